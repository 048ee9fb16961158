// mk_w4_kernel.cuh -- the kernel of the products with 4-bit weights (mk_w4.cu says what it computes
// and why so), instantiated for each type of the activations in a file of its own.
#pragma once
#include <algorithm>
#include <atomic>

#include "../../include/fleet_mk.h"
#include "mk_w4.cuh"

namespace mk {
int set_last_error(int code, const char* msg);   // mk_runtime.cu: the message mk_last_error() returns
}

namespace w4 {

constexpr int WARPS = 16, THREADS = WARPS * 32;
constexpr int SMEM_LIMIT = 227 * 1024;
constexpr int MAX_EXPERTS = 1024;
constexpr int MAX_DEVICES = 64;
constexpr int MAX_COLS = 16;           // columns of an item
constexpr int SMALL_T = MAX_COLS;      // tokens and slots of the two-launch experts
constexpr int SMALL_SLOTS = 256;

// what a launch computes and where its columns and outputs are
enum Mode {
  LINEAR = 0,        // items: blocks of tb tokens
  GATEUP = 1,        // items: the plan's; columns: an item's slots; out: act [column][ldo]
  DOWN = 2,          // items: the plan's; x: act; out: y [column][ldo] FP32
  GATEUP_SMALL = 3,  // items: the selected experts; columns: the tokens; out: act in the MMA's order
  DOWN_SMALL = 4     // one item; a strip's units run over all selected experts; x: act as above
};

// a warp's step: a unit of RT tiles
template <int RT, int G, bool ZP>
struct Shape {
  static constexpr int GROUPS = UNIT_K / G;          // per unit
  static constexpr int SCALES = RT * GROUPS * 32, ZEROS = ZP ? RT * GROUPS * 16 : 0;
  static constexpr int STAGE = RT * TILE_UNIT_BYTES + SCALES + ZEROS;   // without activations
};

// n / d for 0 <= n < 2^31 by one multiplication: with k = 31 + ceil(log2 d), m = ceil(2^k / d) is off by
// less than d / 2^k of itself, so n m / 2^k is off by less than 1 / d
struct Div {
  uint32_t m;
  int shift, d;
};
inline Div div_by(int d) {
  int c = 0;
  while ((1ll << c) < d) ++c;
  return {(uint32_t)(((1ull << (31 + c)) + d - 1) / d), c - 1, d};
}
__device__ __forceinline__ int operator/(int n, const Div& d) {
  return d.d == 1 ? n : (int)(__umulhi((uint32_t)n, d.m) >> d.shift);
}

struct Args {
  const uint8_t* codes;
  const uint8_t* scales;
  const uint8_t* zeros;     // or null: 8
  Div strips;               // of RT tiles, per weight
  Div units, nv;            // units of K; 16-byte pieces of a staged row (16 units)
  int rows, k, experts;
  int mode, depth;          // depth: stages of a warp's ring, 2, 4 or 8
  int device;
  int n_items;              // LINEAR
  const int* items_n;       // GATEUP, DOWN: the plan
  const int4* items;        // {expert, first column, columns, 0}
  const int* col_token;     // GATEUP: the token of a column
  const int* ids;           // *_SMALL: [t, s]
  const float* weights;     // DOWN_SMALL: [t, s]
  int t, s, tb;             // tokens; slots per token; tokens per item of a LINEAR
  Div s_div;
  int cols;                 // most columns of an item
  const uint16_t* x;
  int64_t ldx;
  int x_vec;                // x rows may be read 16 bytes at a time
  const uint16_t* residual;
  int64_t ldr;
  void* out;
  int64_t ldo;
  int out_f32;
};

// the selected experts of a small batch, in the order of their first slots
struct SmallPlan {
  int first[MAX_EXPERTS];               // an expert's first slot, then its place in the list
  int id[SMALL_SLOTS];                  // the slots
  float weight[SMALL_SLOTS];
  int expert[SMALL_SLOTS];
  uint32_t tokens[SMALL_SLOTS];         // the tokens that selected it, one bit each
  int warp_n[WARPS];
  int n;
};

// ends with every warp past a barrier
__device__ __forceinline__ void plan_small(const Args& a, SmallPlan& p) {
  const int n = a.t * a.s, i = threadIdx.x, lane = i & 31, warp = i >> 5;
  if (n > 32 || warp == 0) {
    const int e = i < n ? a.ids[i] : -1;
    const float w = a.weights && i < n ? a.weights[i] : 0.0f;
    const bool valid = (unsigned)e < (unsigned)a.experts;
    if (i < n) {
      p.id[i] = e;
      p.weight[i] = w;
    }
    if (n <= 32) {   // one warp: the lanes with the same expert, the lowest of them leads
      const uint32_t same = __match_any_sync(~0u, valid ? e : -1);
      const bool leads = valid && (same & ((1u << lane) - 1)) == 0;
      const uint32_t ballot = __ballot_sync(~0u, leads);
      if (leads) {
        const int at = __popc(ballot & ((1u << lane) - 1));
        uint32_t tokens = 0;
        for (uint32_t left = same; left; left &= left - 1) tokens |= 1u << ((__ffs(left) - 1) / a.s_div);
        p.expert[at] = e;
        p.tokens[at] = tokens;
      }
      if (lane == 0) p.n = __popc(ballot);
    } else {
      for (int k = i; k < a.experts; k += THREADS) p.first[k] = SMALL_SLOTS;
      if (i < SMALL_SLOTS) p.tokens[i] = 0;
      __syncthreads();
      if (valid) atomicMin(&p.first[e], i);
      __syncthreads();
      const bool leads = valid && p.first[e] == i;
      const uint32_t ballot = __ballot_sync(~0u, leads);
      if (lane == 0) p.warp_n[warp] = __popc(ballot);
      __syncthreads();
      int at = __popc(ballot & ((1u << lane) - 1));
      for (int w = 0; w < warp; ++w) at += p.warp_n[w];
      if (leads) {
        p.expert[at] = e;
        p.first[e] = at;
      }
      if (i == THREADS - 1) p.n = at + leads;
      __syncthreads();
      if (valid) atomicOr(&p.tokens[p.first[e]], 1u << (i / a.s_div));
    }
  }
  __syncthreads();
}

// the item's activations in the MMA's order: [K / 32][columns][4] 16-byte vectors
__device__ __forceinline__ void stage_x(const Args& a, uint4* xs, int start, int count) {
  const int nv = a.nv.d;
  const uint32_t xs_s = (uint32_t)__cvta_generic_to_shared(xs);
  for (int i = threadIdx.x; i < count * nv; i += THREADS) {
    const int col = i / a.nv, v = i - col * nv;
    const int row = a.mode == GATEUP ? a.col_token[start + col] : start + col;
    const uint16_t* src = a.x + (int64_t)row * a.ldx + 8 * v;
    const int at = ((v >> 2) * count + col) * 4 + (v & 3);
    if (a.x_vec && 8 * v + 8 <= a.k) {
      cp16(xs_s + at * 16, src);
    } else {
      uint32_t h[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) h[j] = 8 * v + j < a.k ? (uint32_t)src[j] : 0u;
      xs[at] = make_uint4(h[0] | h[1] << 16, h[2] | h[3] << 16, h[4] | h[5] << 16, h[6] | h[7] << 16);
    }
  }
}

// at most n copies of this thread's newest stay in flight
__device__ __forceinline__ void wait_older(int n) {
  if (n <= 2) {
    if (n == 2) cp_wait<2>();
    else cp_wait<1>();
  } else if (n <= 4) {
    if (n == 4) cp_wait<4>();
    else cp_wait<3>();
  } else {
    if (n == 8) cp_wait<8>();
    else cp_wait<7>();
  }
}

// XR: the activations travel through the ring; SMALL2: DOWN_SMALL
template <class D, int RT, int NT, int G, bool ZP, bool XR, bool SMALL2>
struct Kernel {
  using S = Shape<RT, G, ZP>;
  const Args& a;
  Masks m;
  int warp, lane, g, t;
  uint32_t ring_s;
  int stage;                     // bytes of a stage
  uint4* xs;
  float* slots;                  // [WARPS][RT NT 4][32]: the parts of strips that an earlier warp began
  float* cw;                     // SMALL2: [experts][16] the tokens' weights
  const SmallPlan* plan;
  int U;                         // units of a strip's sums (SMALL2: over all selected experts)
  // the copy cursor: the next unit to copy, the last one's end, the run of consecutive bytes it is in
  int cp, cp_end, run;
  const uint8_t *code = nullptr, *meta = nullptr, *xsrc = nullptr;
  int x_k;                       // XR LINEAR: the unit's first value
  bool scale_lane, zero_lane;
  int item_start, item_count;    // the columns (XR: of every item)
  uint32_t slot;

  __device__ __forceinline__ Kernel(const Args& args) : a(args) {}

  __device__ __forceinline__ int by_u(int p) const { return SMALL2 ? p / U : p / a.units; }
  __device__ __forceinline__ void locate() {
    const int strip_flat = by_u(cp), q = cp - strip_flat * U;
    int item, strip, u, expert;
    if (SMALL2) {
      item = q / a.units;
      u = q - item * a.units.d;
      strip = strip_flat;
      expert = plan->expert[item];
    } else {
      item = strip_flat / a.strips;
      strip = strip_flat - item * a.strips.d;
      u = q;
      expert = a.mode == LINEAR ? 0 : a.mode == GATEUP_SMALL ? plan->expert[item] : a.items[item].x;
    }
    // consecutive: to the strip's (SMALL2: the expert's) last unit; with RT 2 to the weight's
    run = RT == 2 && !SMALL2 && !XR ? (item + 1) * a.strips.d * U - cp : a.units.d - u;
    const int half = RT == 2 ? 0 : strip & 1, pair = RT == 2 ? strip : strip >> 1;
    const int pairs = RT == 2 ? a.strips.d : a.strips.d >> 1;
    const int64_t first = (int64_t)((expert * pairs + pair) * a.units.d + u) * 2 + half;      // in tiles' units
    code = a.codes + first * TILE_UNIT_BYTES + lane * 16;
    if (scale_lane) meta = a.scales + first * (S::GROUPS * 32) + lane * 16;
    else if (zero_lane) meta = a.zeros + first * (S::GROUPS * 16) + (lane - S::SCALES / 16) * 16;
    if (XR) {
      if (SMALL2) xsrc = reinterpret_cast<const uint8_t*>(a.x) + ((int64_t)(item * a.units.d + u) * item_count * 16 + lane) * 16;
      else xsrc = reinterpret_cast<const uint8_t*>(a.x + (int64_t)(item_start + (lane >> 4)) * a.ldx + u * UNIT_K + (lane & 15) * 8);
      x_k = u * UNIT_K + (lane & 15) * 8;
    }
  }
  __device__ __forceinline__ void copy_x(uint32_t dst, bool on) {
    if (SMALL2) {   // already in the MMA's order
      for (int i = lane; i < item_count * 16; i += 32) cp16_if(on, dst + i * 16, xsrc + (i - lane) * 16);
    } else {        // lane: a 16-byte piece of a column's 256 bytes; two columns a step
      const int left = min(max(2 * (a.k - x_k), 0), 16), piece = lane & 15;
      for (int col = lane >> 4; col < item_count; col += 2) {
        const uint32_t to = dst + (((piece >> 2) * item_count + col) * 4 + (piece & 3)) * 16;
        if (on) cp16_part(to, left > 0 ? xsrc + (int64_t)(col - (lane >> 4)) * a.ldx * 2 : reinterpret_cast<const uint8_t*>(a.x), left);
      }
    }
  }
  template <bool WITH_X>
  __device__ __forceinline__ void issue(uint32_t dst) {
    const bool on = cp < cp_end;
#pragma unroll
    for (int i = 0; i < RT * 2; ++i) cp16_if(on, dst + i * 512 + lane * 16, code + i * 512);
    cp16_if(on && (scale_lane || zero_lane), dst + RT * TILE_UNIT_BYTES + lane * 16, meta);
    if (XR && WITH_X) copy_x(dst + S::STAGE, on);
    cp_commit();
    ++cp;
    code += 2 * TILE_UNIT_BYTES;
    meta += 2 * S::GROUPS * (scale_lane ? 32 : 16);
    if (XR) {
      xsrc += SMALL2 ? item_count * 256 : UNIT_K * 2;
      x_k += UNIT_K;
    }
    if (--run == 0 && cp < cp_end) locate();
  }

  // where warp w's units of a phase begin
  static __device__ __forceinline__ int part_of(int p0, int n, int w) {
    return p0 + (n / WARPS) * w + n % WARPS * w / WARPS;
  }
  // GATEUP_SMALL: act [expert of the plan][unit][32-value part][token][4][8]
  __device__ __forceinline__ uint16_t& act_at(int item, int col, int j) {
    const int64_t part = ((int64_t)item * a.ldo + (j >> 7)) * 4 + (j >> 5 & 3);
    return static_cast<uint16_t*>(a.out)[((part * item_count + col) * 4 + (j >> 3 & 3)) * 8 + (j & 7)];
  }

  // a barrier that warps meet at from two places
  __device__ __forceinline__ void all_warps() { asm volatile("barrier.sync 1, %0;" ::"n"(THREADS) : "memory"); }

  // one finished strip
  __device__ __forceinline__ void finish(int strip_flat, const float (&tot)[RT][NT][4]) {
    const int item = SMALL2 ? 0 : strip_flat / a.strips, strip = strip_flat - item * a.strips.d;
    if (!SMALL2 && a.mode == GATEUP_SMALL && strip == a.strips.d - 1) {   // act's padding to whole units is zero
      const int j0 = a.rows / 2, pad = (int)a.ldo * UNIT_K - j0;
      for (int i = lane; i < pad * item_count; i += 32) act_at(item, i / pad, j0 + i % pad) = 0;
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int ci = 0; ci < 2; ++ci) {
        const int col = n * 8 + 2 * t + ci;
        if (col >= item_count) continue;
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          const float lo = tot[r][n][ci], hi = tot[r][n][2 + ci];     // rows g, g + 8 of the tile
          const int tile = strip * RT + r;
          if (!SMALL2 && (a.mode == GATEUP || a.mode == GATEUP_SMALL)) {   // a gate row and its up row
            const int j = tile * 8 + g;
            if (j >= a.rows / 2) continue;
            // rounded to the activations' type: the down projection's tensor-core operand
            uint16_t v = D::round(__fdiv_rn(lo, 1.0f + expf(-lo)) * hi);
            if (a.mode == GATEUP) {
              static_cast<uint16_t*>(a.out)[(int64_t)(item_start + col) * a.ldo + j] = v;
            } else {
              if (!(plan->tokens[item] >> col & 1)) v = 0;
              act_at(item, col, j) = v;
            }
          } else {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int row = tile * 16 + g + 8 * h;
              if (row >= a.rows) continue;
              float v = h ? hi : lo;
              const int64_t at = item_start + col;
              if (a.residual) v += D::one_to_f32(a.residual[at * a.ldr + row]);
              if (a.out_f32) static_cast<float*>(a.out)[at * a.ldo + row] = v;
              else static_cast<uint16_t*>(a.out)[at * a.ldo + row] = D::round(v);
            }
          }
        }
      }
  }

  // the units [p, p_end) of the phase that begins at unit p0 and has n units; at most 8 NT columns
  __device__ __forceinline__ void units(int p, const int p_end, const int p0, const int n) {
    constexpr int WORDS = RT * NT * 4;
    float tot[RT][NT][4];
    // a lane past the columns reads the last one's activations: its sums are not used
    uint32_t xl[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i)
      xl[i] = (XR ? ring_s + S::STAGE : (uint32_t)__cvta_generic_to_shared(xs)) + (min(i * 8 + g, item_count - 1) * 4 + t) * 16;
    const uint32_t x_h = item_count * 64, x_u = item_count * 256;
    bool met = false;                     // this warp has been at the barrier
    int strip_flat = 0;
    while (p < p_end) {
      strip_flat = by_u(p);
      const int q0 = p - strip_flat * U, q1 = min(U, q0 + p_end - p);
#pragma unroll
      for (int i = 0; i < WORDS; ++i) (&tot[0][0][0])[i] = 0.0f;
      uint32_t x_at = XR ? 0 : q0 * x_u;
      float2 w2[NT];
      int to_expert = 0, expert = 0;        // SMALL2: units to the next expert, its place in the plan
      if (SMALL2) {
        expert = q0 / a.units;
        to_expert = (expert + 1) * a.units.d - q0;
#pragma unroll
        for (int i = 0; i < NT; ++i) w2[i] = *reinterpret_cast<const float2*>(cw + expert * MAX_COLS + i * 8 + 2 * t);
      }
      for (int q = q0; q < q1; ++q) {
        wait_older(a.depth - 1);
        __syncwarp();
        const uint32_t st = ring_s + slot;
        uint4 w[RT][2], xr[XR ? 4 : 1][NT];
        uint32_t sc[RT][S::GROUPS], z0[RT][S::GROUPS], z1[RT][S::GROUPS];
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          w[r][0] = lds128(st + lane * 16 + r * TILE_UNIT_BYTES);
          w[r][1] = lds128(st + lane * 16 + r * TILE_UNIT_BYTES + 512);
#pragma unroll
          for (int i = 0; i < S::GROUPS; ++i) {
            sc[r][i] = lds32(st + g * 4 + RT * TILE_UNIT_BYTES + (r * S::GROUPS + i) * 32);
            if (ZP) {
              const uint32_t z = lds16(st + g * 2 + RT * TILE_UNIT_BYTES + S::SCALES + (r * S::GROUPS + i) * 16);
              z0[r][i] = (z & 0xFFu) * 0x00010001u | D::MAGIC;
              z1[r][i] = (z >> 8) * 0x00010001u | D::MAGIC;
            } else {
              z0[r][i] = z1[r][i] = D::MAGIC + 0x00080008u;
            }
          }
        }
        if (XR) {
#pragma unroll
          for (int h = 0; h < 4; ++h)
#pragma unroll
            for (int i = 0; i < NT; ++i) xr[h][i] = lds128(xl[i] + slot + h * x_h);
        }
        __syncwarp();            // every lane has read the stage
        issue<true>(ring_s + slot);
        slot += stage;
        if (slot == (uint32_t)(a.depth * stage)) slot = 0;
        float acc[RT][NT][4];
#pragma unroll
        for (int h = 0; h < 4; ++h) {
          uint4 xb[NT];
#pragma unroll
          for (int i = 0; i < NT; ++i) xb[i] = XR ? xr[XR ? h : 0][i] : lds128(xl[i] + x_at + h * x_h);
          const int i = h * 32 / G;
#pragma unroll
          for (int r = 0; r < RT; ++r) {
            const uint4& v = w[r][h >> 1];
            if (h * 32 % G == 0) half_chunk<D, NT, true>(m, h & 1 ? v.z : v.x, h & 1 ? v.w : v.y, z0[r][i], z1[r][i], xb, acc[r]);
            else half_chunk<D, NT, false>(m, h & 1 ? v.z : v.x, h & 1 ? v.w : v.y, z0[r][i], z1[r][i], xb, acc[r]);
            if ((h + 1) * 32 % G == 0) fold<D, NT, SMALL2>(sc[r][i], w2, acc[r], tot[r]);
          }
        }
        if (!XR) x_at += x_u;
        if (SMALL2 && --to_expert == 0 && q + 1 < q1) {
          to_expert = a.units.d;
          ++expert;
#pragma unroll
          for (int i = 0; i < NT; ++i) w2[i] = *reinterpret_cast<const float2*>(cw + expert * MAX_COLS + i * 8 + 2 * t);
        }
      }
      p += q1 - q0;
      if (q0 > 0) {                       // an earlier warp began it
#pragma unroll
        for (int i = 0; i < WORDS; ++i) slots[(warp * WORDS + i) * 32 + lane] = (&tot[0][0][0])[i];
        continue;
      }
      if (q1 < U) {                       // the warp's last one: the next warps have the rest
        all_warps();
        met = true;
        for (int v = warp + 1; v < WARPS; ++v) {
          const int from = part_of(p0, n, v), to = part_of(p0, n, v + 1);
          if (from >= (strip_flat + 1) * U) break;
          if (from < to) {
#pragma unroll
            for (int i = 0; i < WORDS; ++i) (&tot[0][0][0])[i] += slots[(v * WORDS + i) * 32 + lane];
          }
        }
      }
      finish(strip_flat, tot);
    }
    if (!met) all_warps();
  }

  __device__ __forceinline__ void run_all(uint8_t* smem, SmallPlan& sp) {
    warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    m = masks<D>();
    constexpr int NS = S::SCALES / 16, NZ = S::ZEROS / 16;
    static_assert(NS + NZ <= 32, "one copy a lane");
    scale_lane = lane < NS;
    zero_lane = ZP && lane >= NS && lane < NS + NZ;
    stage = S::STAGE + (XR ? a.cols * UNIT_K * 2 : 0);
    ring_s = (uint32_t)__cvta_generic_to_shared(smem + warp * (a.depth * stage));
    uint8_t* after = smem + WARPS * (a.depth * stage);
    slots = reinterpret_cast<float*>(after);
    after += WARPS * RT * NT * 4 * 32 * 4;
    xs = reinterpret_cast<uint4*>(after);
    cw = reinterpret_cast<float*>(after);
    plan = &sp;
    int n_items = 1;
    item_start = 0;
    item_count = a.cols;
    U = a.units.d;
    if (SMALL2 || a.mode == GATEUP_SMALL) {
      plan_small(a, sp);
      n_items = sp.n;
      item_count = a.t;
      if (SMALL2) {
        U = sp.n * a.units.d;
        n_items = 1;
        for (int i = threadIdx.x; i < sp.n * MAX_COLS; i += THREADS) {
          const int e = sp.expert[i / MAX_COLS], tok = i % MAX_COLS;
          float w = 0.0f;
          if (tok < a.t)
            for (int k = 0; k < a.s; ++k)
              if (sp.id[tok * a.s + k] == e) w += sp.weight[tok * a.s + k];
          cw[i] = w;
        }
        __syncthreads();
      }
    } else {
      n_items = a.mode == LINEAR ? a.n_items : *a.items_n;
    }
    // the CTA's strips: the first total % grid CTAs have one more
    const int total = n_items * a.strips.d, each = total / (int)gridDim.x, more = total - each * (int)gridDim.x;
    const int lo = each * (int)blockIdx.x + min((int)blockIdx.x, more), hi = lo + each + ((int)blockIdx.x < more);
    if (SMALL2 && U == 0) {   // no slot selects an expert
      for (int strip = lo + warp; strip < hi; strip += WARPS) {
        float zero[RT][NT][4] = {};
        finish(strip, zero);
      }
      return;
    }
    bool staged = false;
    for (int from = lo; from < hi;) {
      // a phase: the strips of one item, or all of them if its columns are the same for all
      int to = hi;
      if (!SMALL2 && a.mode != GATEUP_SMALL) {
        const int item = from / a.strips;
        to = min(hi, (item + 1) * a.strips.d);
        if (a.mode == LINEAR) {
          item_start = item * a.tb;
          item_count = min(a.tb, a.t - item_start);
        } else {
          item_start = a.items[item].y;
          item_count = a.items[item].z;
        }
      }
      const int p0 = from * U, n = (to - from) * U;
      const int p = part_of(p0, n, warp), p_end = part_of(p0, n, warp + 1);
      cp = p;
      cp_end = p_end;
      run = 0;
      slot = 0;
      if (p < p_end) locate();
      if (staged) __syncthreads();   // every warp is done with the last phase's activations and parts
      if (!XR) {
        stage_x(a, xs, item_start, item_count);
        cp_commit();
      }
      for (int s = 0; s < a.depth; ++s) issue<true>(ring_s + s * stage);
      if (!XR) {
        wait_older(a.depth);
        __syncthreads();
      }
      staged = true;
      units(p, p_end, p0, n);
      from = to;
    }
    cp_wait<0>();
  }
};

template <class D, int RT, int NT, int G, bool ZP, bool XR, bool SMALL2>
__global__ void __launch_bounds__(THREADS, 1) w4_kernel(const Args a) {
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ SmallPlan plan;
  Kernel<D, RT, NT, G, ZP, XR, SMALL2> k(a);
  k.run_all(smem, plan);
}

// bytes beside rings and activations: the parts and the small plan (static)
constexpr int parts_bytes(int rt, int cols) { return WARPS * rt * (cols <= 8 ? 1 : 2) * 4 * 32 * 4; }
constexpr int STATIC_BYTES = (sizeof(SmallPlan) + 1023) / 1024 * 1024;
// a ring of two stages of two tiles, for the group size and zero points that take most
constexpr int LEAST_RING = WARPS * 2 * Shape<2, 32, true>::STAGE;

// whether the activations of `cols` columns can be staged beside the least ring
inline bool fits(int units, int cols) {
  return LEAST_RING + parts_bytes(2, cols) + STATIC_BYTES + (int64_t)cols * units * UNIT_K * 2 <= SMEM_LIMIT;
}

// beside a ring that carries the activations: the weights of a small batch's slots
constexpr int CW_BYTES = SMALL_SLOTS * MAX_COLS * 4;
inline bool two_tiles_fit_ring(int cols) {
  return WARPS * 2 * (Shape<2, 32, true>::STAGE + cols * UNIT_K * 2) + parts_bytes(2, cols) + CW_BYTES + STATIC_BYTES <= SMEM_LIMIT;
}

template <class D, int RT, int NT, int G, bool ZP, bool XR, bool SMALL2>
static int launch(Args a, int grid, cudaStream_t s) {
  using S = Shape<RT, G, ZP>;
  const int stage = S::STAGE + (XR ? a.cols * UNIT_K * 2 : 0);
  const int64_t rest = parts_bytes(RT, a.cols) + (SMALL2 ? CW_BYTES : XR ? 0 : (int64_t)a.cols * a.units.d * UNIT_K * 2);
  a.depth = 8;
  while (a.depth > 2 && (int64_t)WARPS * a.depth * stage + rest + STATIC_BYTES > SMEM_LIMIT) a.depth /= 2;
  const auto kernel = w4_kernel<D, RT, NT, G, ZP, XR, SMALL2>;
  static std::atomic<bool> ready[MAX_DEVICES];   // the kernel may use that much shared memory on the device
  cudaError_t e = cudaSuccess;
  if (!ready[a.device].load(std::memory_order_acquire)) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_LIMIT - STATIC_BYTES);
    if (e == cudaSuccess) ready[a.device].store(true, std::memory_order_release);
  }
  if (e == cudaSuccess) {
    kernel<<<grid, THREADS, (size_t)(WARPS * a.depth * stage + rest), s>>>(a);
    e = cudaGetLastError();
  }
  return e == cudaSuccess ? MK_OK : mk::set_last_error(MK_ECUDA, cudaGetErrorString(e));
}

template <class D, int RT, int NT, int G, bool ZP>
static int launch_nt(const Args& a, bool through_ring, int grid, cudaStream_t s) {
  if (a.mode == DOWN_SMALL) return launch<D, RT, NT, G, ZP, true, true>(a, grid, s);
  return through_ring ? launch<D, RT, NT, G, ZP, true, false>(a, grid, s) : launch<D, RT, NT, G, ZP, false, false>(a, grid, s);
}

template <class D, int RT, int G, bool ZP>
static int launch_x(const Args& a, bool xr, int grid, cudaStream_t s) {
  return a.cols <= 8 ? launch_nt<D, RT, 1, G, ZP>(a, xr, grid, s) : launch_nt<D, RT, 2, G, ZP>(a, xr, grid, s);
}

template <class D, int RT>
static int launch_group(const Args& a, int group, bool xr, int grid, cudaStream_t s) {
  if (group == 32) return a.zeros ? launch_x<D, RT, 32, true>(a, xr, grid, s) : launch_x<D, RT, 32, false>(a, xr, grid, s);
  if (group == 64) return a.zeros ? launch_x<D, RT, 64, true>(a, xr, grid, s) : launch_x<D, RT, 64, false>(a, xr, grid, s);
  return a.zeros ? launch_x<D, RT, 128, true>(a, xr, grid, s) : launch_x<D, RT, 128, false>(a, xr, grid, s);
}

// mk_w4_bf16.cu, mk_w4_fp16.cu: `two` tiles a warp or one, the activations through the ring or staged
int launch_bf16(const Args& a, int group, bool two, bool through_ring, int grid, cudaStream_t s);
int launch_fp16(const Args& a, int group, bool two, bool through_ring, int grid, cudaStream_t s);

}  // namespace w4

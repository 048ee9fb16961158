// mk_w4_kernel.cuh -- the kernel of the products with 4-bit weights (mk_w4.cu says what it computes
// and why so), instantiated for each type of the activations in a file of its own.
#pragma once
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "../../include/fleet_mk.h"
#include "mk_w4.cuh"

namespace mk {
int set_last_error(int code, const char* msg);   // mk_runtime.cu: the message mk_last_error() returns
}

namespace w4 {

constexpr int MAX_WARPS = 24;
constexpr int SMEM_LIMIT = 227 * 1024;
constexpr int MAX_EXPERTS = 1024;
constexpr int MAX_DEVICES = 64;
constexpr int MAX_COLS = 16;           // columns of an item (of a LINEAR: 32)
// of an expert's item (64 tokens of 66 experts: 101 us; 12: 111, 16: 109; with the intermediate in one value)
constexpr int GROUPED_COLS = 8;
// most tokens and slots of the two-launch experts (12 tokens: 80 us, grouped 68; with the intermediate in one value)
constexpr int SMALL_T = 8;
constexpr int SMALL_SLOTS = 256;

// what a launch computes and where its columns and outputs are
enum Mode {
  LINEAR = 0,        // items: blocks of tb tokens
  GATEUP = 1,        // items: the plan's; columns: an item's slots; out: act [column][2 planes][ldo / 2]
  DOWN = 2,          // items: the plan's; x: act; out: y [column][ldo] FP32
  GATEUP_SMALL = 3,  // items: the selected experts; columns: the tokens; out: act in the MMA's order
  DOWN_SMALL = 4     // one item; a strip's units run over all selected experts; x: act as above
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
  int mode;
  int device;
  int follows;              // launched behind another launch of the same call
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
  int pairs;                // 16-bit out and residual rows start at 4-byte boundaries
};

// The launches of one call overlap: each lets the next one start while it runs (the next's blocks take
// SMs as this one's leave them) and waits for its predecessor's results before it reads them. What an
// earlier launch of the call writes changes during the life of the kernel that reads it, so no kernel that
// waits takes it through const __restrict__ (loads that may be non-coherent, or moved before the wait).
__device__ __forceinline__ void wait_predecessor() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void start_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// the selected experts of a small batch, in the order of their first slots
struct SmallPlan {
  int first[MAX_EXPERTS];               // an expert's first slot, then its place in the list
  int id[SMALL_SLOTS];                  // the slots
  float weight[SMALL_SLOTS];
  int expert[SMALL_SLOTS];
  uint32_t tokens[SMALL_SLOTS];         // the tokens that selected it, one bit each
  int warp_n[MAX_WARPS];
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
      for (int k = i; k < a.experts; k += blockDim.x) p.first[k] = SMALL_SLOTS;
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
      if (i == (int)blockDim.x - 1) p.n = at + leads;
      __syncthreads();
      if (valid) atomicOr(&p.tokens[p.first[e]], 1u << (i / a.s_div));
    }
  }
  __syncthreads();
}

// the item's activations in the MMA's order: [K / 32][planes][columns][4] 16-byte vectors
template <int PLANES>
__device__ __forceinline__ void stage_x(const Args& a, uint4* xs, int start, int count) {
  const int nv = a.nv.d;
  const uint32_t xs_s = (uint32_t)__cvta_generic_to_shared(xs);
  for (int i = threadIdx.x; i < PLANES * count * nv; i += blockDim.x) {
    const int pc = i / a.nv, v = i - pc * nv;
    const int plane = PLANES > 1 && pc >= count, col = pc - plane * count;
    const int row = a.mode == GATEUP ? a.col_token[start + col] : start + col;
    const uint16_t* src = a.x + (int64_t)row * a.ldx + (plane ? a.ldx / 2 : 0) + 8 * v;
    const int at = ((v >> 2) * PLANES * count + pc) * 4 + (v & 3);
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

// RT, NT: tiles of 16 rows and 8 columns a warp computes at a time. XR: the activations are loaded with
// each unit instead of staged. SMALL2: DOWN_SMALL. WIDE: an activation is the sum of two BF16 planes (DOWN,
// DOWN_SMALL), whatever the type of the scales and outputs.
template <class D, int RT, int NT, int G, bool ZP, bool XR, bool SMALL2, bool WIDE>
struct Kernel {
  using M = std::conditional_t<WIDE, Bf16, D>;    // the MMAs' type
  static constexpr int PLANES = WIDE ? 2 : 1;
  // Warps and the units each has in flight. 8 columns: 24 warps of 80 registers, one unit each, its halves
  // reloaded as they are used (the 1-token head 25.6 us; 16 warps two units ahead 28.3). More columns, or
  // too few rows for two tiles a warp: 16 warps of 128 registers. Both planes with each unit (32 registers): 16
  // warps, one unit each (experts of 1 / 8 tokens 21.1 / 58.3 us; 24 warps, which spill, 22.5 / 61.1; 20 warps 22.5 /
  // 59.3; 16 warps two units ahead 22.5 / 62.9)
  static constexpr bool BOTH = XR && WIDE, NARROW = NT == 1 && (RT == 2 || XR) && !BOTH;
  static constexpr int WARPS = NARROW ? 24 : 16, THREADS = WARPS * 32;
  static constexpr int AHEAD = NARROW || BOTH ? 1 : RT == 2 || NT > 1 ? 2 : 3;
  static constexpr int GROUPS = UNIT_K / G, ZWORDS = GROUPS / 2 > 0 ? GROUPS / 2 : 1;
  // a unit of RT tiles in registers
  struct Unit {
    uint4 w[RT][2];
    uint32_t sc[RT][GROUPS];
    uint32_t z[RT][ZP ? ZWORDS : 1];
    uint4 x[XR ? 4 : 1][PLANES][XR ? NT : 1];
  };

  const Args& a;
  uint32_t magic;
  int warp, lane, g, t;
  uint4* xs;
  float* slots;                  // [WARPS][RT NT 4][32]: the parts of strips that an earlier warp began
  float* cw;                     // SMALL2: [experts][SMALL_T] the tokens' weights
  const SmallPlan* plan;
  int U;                         // units of a strip's sums (SMALL2: over all selected experts)
  // the load cursor: the next unit to load, the last one's end, the run of consecutive bytes it is in
  int cp, cp_end, run;
  const uint8_t *code, *scale, *zero;
  const uint16_t* x_at[XR ? NT : 1];
  int x_k;                       // XR LINEAR: the lane's first value of the unit
  int item_start, item_count;    // the columns (XR: of every item)

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
    scale = a.scales + first * (GROUPS * 32) + g * (GROUPS * 4);
    if (ZP) zero = a.zeros + first * (GROUPS * 16) + g * (GROUPS * 2);
    if (XR) {
      x_k = u * UNIT_K + t * 8;
#pragma unroll
      for (int i = 0; i < NT; ++i) {   // a lane past the columns takes the last one's: its sums are not used
        const int col = min(i * 8 + g, item_count - 1);
        x_at[i] = SMALL2 ? a.x + (((int64_t)(item * a.units.d + u) * 4 * PLANES * item_count + col) * 4 + t) * 8
                         : a.x + (int64_t)(item_start + col) * a.ldx + x_k;
      }
    }
  }
  // the first half of the next unit's codes
  __device__ __forceinline__ void load_half(Unit& n) {
    if (cp >= cp_end) return;
#pragma unroll
    for (int r = 0; r < RT; ++r) n.w[r][0] = ldg128(code + r * TILE_UNIT_BYTES);
  }
  // the next unit's codes, scales and zero points; rest: without that half
  __device__ __forceinline__ void load_weights(Unit& n, bool rest) {
    if (cp >= cp_end) return;
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      if (!rest) n.w[r][0] = ldg128(code + r * TILE_UNIT_BYTES);
      n.w[r][1] = ldg128(code + r * TILE_UNIT_BYTES + 512);
      ldg_words<GROUPS>(scale + r * (GROUPS * 32), n.sc[r]);
      if (ZP) {
        if (GROUPS == 1) n.z[r][0] = ldg16(zero + r * 16);
        else ldg_words<ZP ? ZWORDS : 1>(zero + r * (GROUPS * 16), n.z[r]);
      }
    }
  }
  // its activations, and the cursor on to the unit after it
  __device__ __forceinline__ void load_rest(Unit& n) {
    if (cp >= cp_end) return;
    if (XR) {
#pragma unroll
      for (int h = 0; h < 4; ++h)
#pragma unroll
        for (int p = 0; p < PLANES; ++p)
#pragma unroll
          for (int i = 0; i < NT; ++i) {
            if (SMALL2) n.x[h][p][i] = ldg128_x(x_at[i] + (h * PLANES + p) * item_count * 32);
            else if (x_k + 32 * h < a.k) n.x[h][p][i] = ldg128_x(x_at[i] + 32 * h + (p ? a.ldx / 2 : 0));
            else n.x[h][p][i] = make_uint4(0, 0, 0, 0);
          }
#pragma unroll
      for (int i = 0; i < NT; ++i) x_at[i] += SMALL2 ? PLANES * item_count * 128 : UNIT_K;
      x_k += UNIT_K;
    }
    code += 2 * TILE_UNIT_BYTES;
    scale += 2 * GROUPS * 32;
    if (ZP) zero += 2 * GROUPS * 16;
    ++cp;
    if (--run == 0 && cp < cp_end) locate();
  }
  // where warp w's units of a phase begin
  static __device__ __forceinline__ int part_of(int p0, int n, int w) {
    return p0 + (n / WARPS) * w + n % WARPS * w / WARPS;
  }
  // GATEUP_SMALL: act [expert of the plan][unit][32-value part][2 planes][token][4][8]
  __device__ __forceinline__ uint16_t& act_at(int item, int plane, int col, int j) {
    uint16_t* act = static_cast<uint16_t*>(a.out);
    if (a.mode == GATEUP) return act[(int64_t)(item_start + col) * a.ldo + (plane ? a.ldo / 2 : 0) + j];
    const int64_t part = ((int64_t)item * a.ldo + (j >> 7)) * 4 + (j >> 5 & 3);
    return act[(((part * 2 + plane) * item_count + col) * 4 + (j >> 3 & 3)) * 8 + (j & 7)];
  }

  // a barrier that warps meet at from two places
  __device__ __forceinline__ void all_warps() { asm volatile("barrier.sync 1, %0;" ::"n"(THREADS) : "memory"); }

  // A finished strip. 16-bit outputs go through a transposition, so that a lane holds two rows (which are
  // neighbours in memory) of one column: lane 4 g + t rows 2 t, 2 t + 1 of column 8 n + g.
  __device__ __forceinline__ void finish(int strip_flat, const float (&tot)[RT][NT][4]) {
    const int item = SMALL2 ? 0 : strip_flat / a.strips, strip = strip_flat - item * a.strips.d;
    if (!SMALL2 && (a.mode == GATEUP || a.mode == GATEUP_SMALL)) finish_act(item, strip, tot);
    else if (a.pairs) finish_pairs(strip, tot);
    else finish_single(strip, tot);
  }
  // Gate and up rows: a tile's rows g and g + 8. silu(g) u is kept as two BF16 values, hi + lo: the down
  // projection's tensor-core operands, in FP32's range (an FP16 one would end at 65504) and off by at most 2^-16 of
  // itself, so that the results are those of an FP32 activation but for their own rounding.
  __device__ __forceinline__ void finish_act(int item, int strip, const float (&tot)[RT][NT][4]) {
    const int I = a.rows / 2;
    if (strip == a.strips.d - 1) {   // act's padding is zero (to whole units, or to the row's end)
      const int pad = (a.mode == GATEUP ? (int)a.ldo / 2 : (int)a.ldo * UNIT_K) - I;
      for (int i = lane; i < 2 * pad * item_count; i += 32) {
        const int pc = i / pad;
        act_at(item, pc & 1, pc >> 1, I + i % pad) = 0;
      }
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        uint32_t hi[2], lo[2];
#pragma unroll
        for (int ci = 0; ci < 2; ++ci) {
          const float gt = tot[r][n][ci], up = tot[r][n][2 + ci];
          split_bf16(__fdiv_rn(gt, 1.0f + expf(-gt)) * up, hi[ci], lo[ci]);
        }
        const uint32_t planes[2] = {transpose8(hi[0] | hi[1] << 16), transpose8(lo[0] | lo[1] << 16)};
        const int col = n * 8 + g, j = (strip * RT + r) * 8 + 2 * t;
        if (col < item_count && j < I) {
          const bool selected = a.mode == GATEUP || plan->tokens[item] >> col & 1;
#pragma unroll
          for (int p = 0; p < 2; ++p) {
            const uint32_t two = selected ? planes[p] : 0u;
            if (j + 1 < I) *reinterpret_cast<uint32_t*>(&act_at(item, p, col, j)) = two;
            else act_at(item, p, col, j) = (uint16_t)two;
          }
        }
      }
  }
  __device__ __forceinline__ void finish_pairs(int strip, const float (&tot)[RT][NT][4]) {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      if (n * 8 >= item_count) break;
      const int64_t col = item_start + n * 8 + g;
      const bool live = n * 8 + g < item_count;
#pragma unroll
      for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int row = (strip * RT + r) * 16 + 8 * h + 2 * t;
          float lo = tot[r][n][2 * h], hi = tot[r][n][2 * h + 1];
          if (a.residual) {
            const uint16_t* p = a.residual + col * a.ldr + row;
            uint32_t two = 0;
            if (live && row + 1 < a.rows) two = *reinterpret_cast<const uint32_t*>(p);
            else if (live && row < a.rows) two = *p;
            const float2 f = D::to_f32(transpose8(two));
            lo += f.x;
            hi += f.y;
          }
          const uint32_t two = transpose8(D::round2(lo, hi));
          uint16_t* o = static_cast<uint16_t*>(a.out) + col * a.ldo + row;
          if (live && row + 1 < a.rows) *reinterpret_cast<uint32_t*>(o) = two;
          else if (live && row < a.rows) *o = (uint16_t)two;
        }
    }
  }
  // FP32 outputs and rows that do not start at 4-byte boundaries
  __device__ __forceinline__ void finish_single(int strip, const float (&tot)[RT][NT][4]) {
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int ci = 0; ci < 2; ++ci) {
        if (n * 8 + 2 * t + ci >= item_count) continue;
        const int64_t col = item_start + n * 8 + 2 * t + ci;
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int row = (strip * RT + r) * 16 + g + 8 * h;
            if (row >= a.rows) continue;
            float v = tot[r][n][2 * h + ci];
            if (a.residual) v += D::one_to_f32(a.residual[col * a.ldr + row]);
            if (a.out_f32) static_cast<float*>(a.out)[col * a.ldo + row] = v;
            else static_cast<uint16_t*>(a.out)[col * a.ldo + row] = D::round(v);
          }
      }
  }

  // tot += the unit's products; staged activations at shared address xl + x_off, x_p to the next plane
  __device__ __forceinline__ void multiply(Unit& n, const uint32_t (&xl)[NT], uint32_t x_off, uint32_t x_p,
                                           const float2 (&w2)[NT], const bool (&part)[NT][2], float (&tot)[RT][NT][4]) {
    float acc[RT][NT][4];
#pragma unroll
    for (int h = 0; h < 4; ++h) {
      uint4 xb[PLANES][NT];
#pragma unroll
      for (int p = 0; p < PLANES; ++p)
#pragma unroll
        for (int i = 0; i < NT; ++i) xb[p][i] = XR ? n.x[XR ? h : 0][p][XR ? i : 0] : lds128(xl[i] + x_off + (h * PLANES + p) * x_p);
      const int i = h * 32 / G;
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        uint32_t z0 = M::MAGIC + 0x00080008u, z1 = z0;
        if (ZP) {   // rows g and g + 8 of group i: two bytes
          const uint32_t z = n.z[r][i / 2] >> (i % 2 * 16);
          z0 = (z & 0xFFu) * 0x00010001u | M::MAGIC;
          z1 = (z >> 8 & 0xFFu) * 0x00010001u | M::MAGIC;
        }
        const uint4& v = n.w[r][h >> 1];
        if (h * 32 % G == 0) half_chunk<M, NT, PLANES, true>(magic, h & 1 ? v.z : v.x, h & 1 ? v.w : v.y, z0, z1, xb, acc[r]);
        else half_chunk<M, NT, PLANES, false>(magic, h & 1 ? v.z : v.x, h & 1 ? v.w : v.y, z0, z1, xb, acc[r]);
        if ((h + 1) * 32 % G == 0) fold<D, NT, SMALL2>(n.sc[r][i], w2, part, acc[r], tot[r]);
      }
      if (AHEAD == 1 && h == 1) load_half(n);
    }
  }

  // the units [p, p_end) of the phase that begins at unit p0 and has n units; at most 8 NT columns.
  // un holds the first AHEAD of them.
  __device__ __forceinline__ void units(Unit (&un)[AHEAD], int p, const int p_end, const int p0, const int n) {
    constexpr int WORDS = RT * NT * 4;
    float tot[RT][NT][4];
    // a lane past the columns reads the last one's activations: its sums are not used
    uint32_t xl[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i)
      xl[i] = XR ? 0 : (uint32_t)__cvta_generic_to_shared(xs) + (min(i * 8 + g, item_count - 1) * 4 + t) * 16;
    const uint32_t x_p = item_count * 64, x_u = 4 * PLANES * x_p;
    bool met = false;                     // this warp has been at the barrier
    int next = 0;                         // the place in un of the next unit
    while (p < p_end) {
      const int strip_flat = by_u(p);
      const int q0 = p - strip_flat * U, q1 = min(U, q0 + p_end - p);
#pragma unroll
      for (int i = 0; i < WORDS; ++i) (&tot[0][0][0])[i] = 0.0f;
      uint32_t x_off = q0 * x_u;
      float2 w2[NT];
      bool part[NT][2];
      int to_expert = 0, expert = 0;      // SMALL2: units to the next expert, its place in the plan
      auto weigh = [&]() {
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          w2[i] = *reinterpret_cast<const float2*>(cw + expert * SMALL_T + i * 8 + 2 * t);
          const uint32_t tokens = plan->tokens[expert] >> (i * 8 + 2 * t);
          part[i][0] = tokens & 1;
          part[i][1] = tokens & 2;
        }
      };
      if (SMALL2) {
        expert = q0 / a.units;
        to_expert = (expert + 1) * a.units.d - q0;
        weigh();
      }
      int left = q1 - q0;
      while (left > 0) {
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
          if (next == i && left > 0) {
            multiply(un[i], xl, x_off, x_p, w2, part, tot);
            load_weights(un[i], AHEAD == 1);
            load_rest(un[i]);
            next = i + 1 == AHEAD ? 0 : i + 1;
            --left;
            x_off += x_u;
            if (SMALL2 && --to_expert == 0 && left > 0) {
              to_expert = a.units.d;
              ++expert;
              weigh();
            }
          }
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
    magic = magic_register<M>();
    uint8_t* after = smem;
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
        for (int i = threadIdx.x; i < sp.n * SMALL_T; i += THREADS) {
          const int e = sp.expert[i / SMALL_T], tok = i % SMALL_T;
          float w = 0.0f;
          if (tok < a.t)
            for (int k = 0; k < a.s; ++k)
              if (sp.id[tok * a.s + k] == e) w += sp.weight[tok * a.s + k];
          cw[i] = w;
        }
        __syncthreads();
      }
    } else {
      if (a.follows) wait_predecessor();
      n_items = a.mode == LINEAR ? a.n_items : *a.items_n;
    }
    // the CTA's strips: the first total % grid CTAs have one more
    const int total = n_items * a.strips.d, each = total / (int)gridDim.x, more = total - each * (int)gridDim.x;
    const int lo = each * (int)blockIdx.x + min((int)blockIdx.x, more), hi = lo + each + ((int)blockIdx.x < more);
    start_dependents();
    if (SMALL2 && U == 0) {   // no slot selects an expert
      for (int strip = lo + warp; strip < hi; strip += WARPS) {
        const float zero[RT][NT][4] = {};
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
      if (p < p_end) locate();
      if (staged) __syncthreads();   // every warp is done with the last phase's activations and parts
      Unit un[AHEAD];
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        load_weights(un[i], false);
        if (SMALL2 && i == 0 && a.follows) wait_predecessor();   // its activations: the plan and the weights are not
        load_rest(un[i]);
      }
      if (!XR) stage_x<PLANES>(a, xs, item_start, item_count);
      if (!XR) {
        cp_wait_all();
        __syncthreads();
      }
      staged = true;
      units(un, p, p_end, p0, n);
      from = to;
    }
  }
};

template <class D, int RT, int NT, int G, bool ZP, bool XR, bool SMALL2, bool WIDE>
__global__ void __launch_bounds__(Kernel<D, RT, NT, G, ZP, XR, SMALL2, WIDE>::THREADS, 1) w4_kernel(const Args a) {
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ SmallPlan plan;
  Kernel<D, RT, NT, G, ZP, XR, SMALL2, WIDE> k(a);
  k.run_all(smem, plan);
}

// shared memory: the parts of strips, a small batch's weights, the plan (static), the activations
constexpr int PARTS_BYTES = 32 * 1024;     // at most: 16 warps x 4 x 4 (or 24 x 2 x 4) words of 128 bytes
constexpr int CW_BYTES = SMALL_SLOTS * SMALL_T * 4;
constexpr int STATIC_BYTES = (sizeof(SmallPlan) + 1023) / 1024 * 1024;

// whether the activations of `cols` columns can be staged
inline bool fits(int units, int cols) {
  return PARTS_BYTES + STATIC_BYTES + (int64_t)cols * units * UNIT_K * 2 <= SMEM_LIMIT;
}

template <typename... P>
cudaError_t launch_behind(void (*kernel)(P...), dim3 grid, int threads, int smem, cudaStream_t s, bool follows, P... args) {
  cudaLaunchConfig_t c{};
  cudaLaunchAttribute overlap[1];
  c.gridDim = grid;
  c.blockDim = dim3((unsigned)threads);
  c.dynamicSmemBytes = (size_t)smem;
  c.stream = s;
  overlap[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  overlap[0].val.programmaticStreamSerializationAllowed = 1;
  c.attrs = overlap;
  c.numAttrs = follows ? 1 : 0;
  return cudaLaunchKernelEx(&c, kernel, args...);
}

template <class D, int RT, int NT, int G, bool ZP, bool XR, bool SMALL2, bool WIDE>
static int launch(const Args& a, int grid, cudaStream_t s) {
  using K = Kernel<D, RT, NT, G, ZP, XR, SMALL2, WIDE>;
  constexpr int parts = K::WARPS * RT * NT * 4 * 32 * 4;
  static_assert(parts <= PARTS_BYTES, "the parts of strips");
  const int smem = parts + (SMALL2 ? CW_BYTES : XR ? 0 : K::PLANES * a.cols * a.units.d * UNIT_K * 2);
  const auto kernel = w4_kernel<D, RT, NT, G, ZP, XR, SMALL2, WIDE>;
  static std::atomic<bool> ready[MAX_DEVICES];   // the kernel may use that much shared memory on the device
  cudaError_t e = cudaSuccess;
  if (!ready[a.device].load(std::memory_order_acquire)) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_LIMIT - STATIC_BYTES);
    if (e == cudaSuccess) ready[a.device].store(true, std::memory_order_release);
  }
  if (e == cudaSuccess) e = launch_behind(kernel, dim3((unsigned)grid), K::THREADS, smem, s, a.follows, a);
  return e == cudaSuccess ? MK_OK : mk::set_last_error(MK_ECUDA, cudaGetErrorString(e));
}

// two: two tiles a warp; xr: the activations come with the units (of more than 8 columns, or in two planes: one
// tile a warp, for its registers)
template <class D, int G, bool ZP>
static int launch_form(const Args& a, bool two, bool xr, int grid, cudaStream_t s) {
  if (a.mode == DOWN_SMALL) return launch<D, 1, 1, G, ZP, true, true, true>(a, grid, s);
  if (a.mode == DOWN) {
    if (xr) return launch<D, 1, 1, G, ZP, true, false, true>(a, grid, s);
    return two ? launch<D, 2, 1, G, ZP, false, false, true>(a, grid, s) : launch<D, 1, 1, G, ZP, false, false, true>(a, grid, s);
  }
  if (a.cols <= 8) {
    if (xr) return two ? launch<D, 2, 1, G, ZP, true, false, false>(a, grid, s) : launch<D, 1, 1, G, ZP, true, false, false>(a, grid, s);
    return two ? launch<D, 2, 1, G, ZP, false, false, false>(a, grid, s) : launch<D, 1, 1, G, ZP, false, false, false>(a, grid, s);
  }
  if (xr) return launch<D, 1, 2, G, ZP, true, false, false>(a, grid, s);
  if (a.cols > MAX_COLS) return launch<D, 1, 4, G, ZP, false, false, false>(a, grid, s);
  return two ? launch<D, 2, 2, G, ZP, false, false, false>(a, grid, s) : launch<D, 1, 2, G, ZP, false, false, false>(a, grid, s);
}

template <class D>
static int launch_type(const Args& a, int group, bool two, bool xr, int grid, cudaStream_t s) {
  if (group == 32) return a.zeros ? launch_form<D, 32, true>(a, two, xr, grid, s) : launch_form<D, 32, false>(a, two, xr, grid, s);
  if (group == 64) return a.zeros ? launch_form<D, 64, true>(a, two, xr, grid, s) : launch_form<D, 64, false>(a, two, xr, grid, s);
  return a.zeros ? launch_form<D, 128, true>(a, two, xr, grid, s) : launch_form<D, 128, false>(a, two, xr, grid, s);
}

// mk_w4_bf16.cu, mk_w4_fp16.cu
int launch_bf16(const Args& a, int group, bool two, bool xr, int grid, cudaStream_t s);
int launch_fp16(const Args& a, int group, bool two, bool xr, int grid, cudaStream_t s);

}  // namespace w4

// mk_w4.cu -- products with 4-bit weights for a batch of tokens: mk_w4_linear (one weight) and
// mk_w4_experts (a layer's routed experts: gate/up, SwiGLU, down projection, weighted sum).
// The format and the laid-out order are in mk_w4.cuh.
//
// Formulas. linear: out[t] = x[t] W^T (+ residual[t]). experts: out[t] = (residual[t] +) the sum over
// the token's slots s of w[t, s] W2[e] a(t, e), a = silu(g) u, (g, u) = W13[e] x[t], e = ids[t, s]; a
// slot whose id is outside [0, experts) is empty.
//
// What bounds them. A token costs 2 operations per weight and a weight half a byte, so a batch of T
// tokens does 4 T operations a byte: the stream of codes is the bound for a decode batch, then the
// instructions that turn codes into tensor-core operands (11 per 8 codes), not the tensor cores
// (2 cycles an m16n8k16 per SM against 5.5 cycles for its 128 bytes at 6.5 TB/s). mma.sync takes a
// tile of 16 rows by 8 tokens without padding the batch to a tcgen05 tile's 64 or 128 rows.
//
// The work is a row of sums (a strip: RT tiles of 16 rows, for up to 16 columns) times its units of
// 128 values of K. Each CTA (one per SM, 16 warps) takes an equal range of strips, and each warp an
// equal, contiguous range of the CTA's units, wherever strips begin and end in it: the warps finish
// together whatever the sizes, and nothing is synchronised between them until the end of the range,
// where the warp that began a strip adds the parts of the warps after it, in warp order (the result
// does not depend on timing). A warp streams its units, which lie one after the other in memory,
// through its own ring of cp.async stages. The activations are either staged once in shared memory
// (many strips per CTA use them) or travel with the codes through the rings (few strips per CTA, or
// rows too long for shared memory).
//
// The experts of a small batch (at most 16 tokens) take two launches: gate/up with the tokens as the
// columns of every expert, then the down projection as one long dot product over the selected
// experts' activations, each expert's part scaled by the tokens' weights for it. A larger batch is
// grouped by expert first (plan_kernel), each expert's slots being its columns, and the slots' outputs
// are added afterwards in slot order (combine_kernel).
#include <algorithm>
#include <mutex>

#include "../../include/fleet_mk.h"
#include "mk_w4.cuh"

namespace mk {
int set_last_error(int code, const char* msg);   // mk_runtime.cu: the message mk_last_error() returns
}

using namespace w4;

namespace {

constexpr int WARPS = 16, THREADS = WARPS * 32;
constexpr int SMEM_LIMIT = 227 * 1024;
constexpr int MAX_EXPERTS = 1024;
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

struct Args {
  const uint8_t* codes;
  const uint8_t* scales;
  const uint8_t* zeros;     // or null: 8
  int strips;               // of RT tiles, per weight
  int units, rows, k, experts;
  int mode, depth;          // depth: stages of a warp's ring, 2, 4 or 8
  int n_items;              // LINEAR
  const int* items_n;       // GATEUP, DOWN: the plan
  const int4* items;        // {expert, first column, columns, 0}
  const int* col_token;     // GATEUP: the token of a column
  const int* ids;           // *_SMALL: [t, s]
  const float* weights;     // DOWN_SMALL: [t, s]
  int t, s, tb;             // tokens; slots per token; tokens per item of a LINEAR
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
  int expert[SMALL_SLOTS];
  uint32_t tokens[SMALL_SLOTS];         // the tokens that selected it, one bit each
  int warp_n[WARPS];
  int n;
};

__device__ __forceinline__ void plan_small(const Args& a, SmallPlan& p) {
  const int n = a.t * a.s, i = threadIdx.x, lane = i & 31, warp = i >> 5;
  const int e = i < n ? a.ids[i] : -1;
  const bool valid = (unsigned)e < (unsigned)a.experts;
  for (int k = i; k < a.experts; k += THREADS) p.first[k] = SMALL_SLOTS;
  for (int k = i; k < SMALL_SLOTS; k += THREADS) p.tokens[k] = 0;
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
  if (valid) atomicOr(&p.tokens[p.first[e]], 1u << (i / a.s));
}

// the item's activations in the MMA's order: [K / 32][columns][4] 16-byte vectors
__device__ __forceinline__ void stage_x(const Args& a, uint4* xs, int start, int count) {
  const int nv = a.units * 16;
  const uint32_t xs_s = (uint32_t)__cvta_generic_to_shared(xs);
  for (int i = threadIdx.x; i < count * nv; i += THREADS) {
    const int col = i / nv, v = i - col * nv;
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

// XR: the activations travel through the ring; SMALL2: DOWN_SMALL
template <class D, int RT, int G, bool ZP, bool XR, bool SMALL2>
struct Kernel {
  using S = Shape<RT, G, ZP>;
  const Args& a;
  Masks m;
  int warp, lane, g, t;
  uint8_t* ring;
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

  __device__ __forceinline__ void locate() {
    const int strip_flat = cp / U, q = cp - strip_flat * U;
    int item, strip, u, expert;
    if (SMALL2) {
      item = q / a.units;
      u = q - item * a.units;
      strip = strip_flat;
      expert = plan->expert[item];
    } else {
      item = strip_flat / a.strips;
      strip = strip_flat - item * a.strips;
      u = q;
      expert = a.mode == LINEAR ? 0 : a.mode == GATEUP_SMALL ? plan->expert[item] : a.items[item].x;
    }
    // consecutive: to the strip's (SMALL2: the expert's) last unit; with RT 2 to the weight's
    run = RT == 2 && !SMALL2 && !XR ? (item + 1) * a.strips * U - cp : a.units - u;
    const int half = RT == 2 ? 0 : strip & 1, pair = RT == 2 ? strip : strip >> 1;
    const int pairs = RT == 2 ? a.strips : a.strips >> 1;
    const int64_t first = (((int64_t)expert * pairs + pair) * a.units + u) * 2 + half;      // in tiles' units
    code = a.codes + first * TILE_UNIT_BYTES + lane * 16;
    if (scale_lane) meta = a.scales + first * (S::GROUPS * 32) + lane * 16;
    else if (zero_lane) meta = a.zeros + first * (S::GROUPS * 16) + (lane - S::SCALES / 16) * 16;
    if (XR) {
      if (SMALL2) xsrc = reinterpret_cast<const uint8_t*>(a.x) + ((int64_t)(item * a.units + u) * item_count * 16 + lane) * 16;
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

  // GATEUP_SMALL: act [expert of the plan][unit][32-value part][token][4][8]
  __device__ __forceinline__ uint16_t& act_at(int item, int col, int j) {
    const int64_t part = ((int64_t)item * a.ldo + (j >> 7)) * 4 + (j >> 5 & 3);
    return static_cast<uint16_t*>(a.out)[((part * item_count + col) * 4 + (j >> 3 & 3)) * 8 + (j & 7)];
  }

  // one finished strip
  template <int NT>
  __device__ __forceinline__ void finish(int strip_flat, const float (&tot)[RT][NT][4]) {
    const int item = SMALL2 ? 0 : strip_flat / a.strips, strip = strip_flat - item * a.strips;
    if (!SMALL2 && a.mode == GATEUP_SMALL && strip == a.strips - 1) {   // act's padding to whole units is zero
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
  template <int NT>
  __device__ __forceinline__ void units(int p, const int p_end, const int p0, const int n) {
    constexpr int WORDS = RT * NT * 4;
    float tot[RT][NT][4];
    // a lane past the columns reads the last one's activations: its sums are not used
    const uint4* xl[NT];
    const uint4* xbase = XR ? reinterpret_cast<const uint4*>(ring + S::STAGE) : xs;
#pragma unroll
    for (int i = 0; i < NT; ++i) xl[i] = xbase + min(i * 8 + g, item_count - 1) * 4 + t;
    const int x_h = item_count * 4, x_u = item_count * 16;
    bool tail = false;
    int strip_flat = 0;
    while (p < p_end) {
      strip_flat = p / U;
      const int q0 = p - strip_flat * U, q1 = min(U, q0 + p_end - p);
#pragma unroll
      for (int i = 0; i < WORDS; ++i) (&tot[0][0][0])[i] = 0.0f;
      int x_at = XR ? 0 : q0 * x_u;
      float2 w2[NT];
      int to_expert = 0, expert = 0;        // SMALL2: units to the next expert, its place in the plan
      if (SMALL2) {
        expert = q0 / a.units;
        to_expert = (expert + 1) * a.units - q0;
#pragma unroll
        for (int i = 0; i < NT; ++i) w2[i] = *reinterpret_cast<const float2*>(cw + expert * MAX_COLS + i * 8 + 2 * t);
      }
      for (int q = q0; q < q1; ++q) {
        if (a.depth == 2) cp_wait<1>();
        else if (a.depth == 4) cp_wait<3>();
        else cp_wait<7>();
        __syncwarp();
        const uint8_t* st = ring + slot;
        uint4 w[RT][2], xr[XR ? 4 : 1][NT];
        uint32_t sc[RT][S::GROUPS], z0[RT][S::GROUPS], z1[RT][S::GROUPS];
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          w[r][0] = *reinterpret_cast<const uint4*>(st + r * TILE_UNIT_BYTES + lane * 16);
          w[r][1] = *reinterpret_cast<const uint4*>(st + r * TILE_UNIT_BYTES + 512 + lane * 16);
#pragma unroll
          for (int i = 0; i < S::GROUPS; ++i) {
            sc[r][i] = *reinterpret_cast<const uint32_t*>(st + RT * TILE_UNIT_BYTES + (r * S::GROUPS + i) * 32 + g * 4);
            if (ZP) {
              const uint32_t z =
                  *reinterpret_cast<const uint16_t*>(st + RT * TILE_UNIT_BYTES + S::SCALES + (r * S::GROUPS + i) * 16 + g * 2);
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
            for (int i = 0; i < NT; ++i) xr[h][i] = xl[i][(slot >> 4) + h * x_h];
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
          for (int i = 0; i < NT; ++i) xb[i] = XR ? xr[XR ? h : 0][i] : xl[i][x_at + h * x_h];
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
          to_expert = a.units;
          ++expert;
#pragma unroll
          for (int i = 0; i < NT; ++i) w2[i] = *reinterpret_cast<const float2*>(cw + expert * MAX_COLS + i * 8 + 2 * t);
        }
      }
      p += q1 - q0;
      if (q0 > 0) {                       // an earlier warp began it
#pragma unroll
        for (int i = 0; i < WORDS; ++i) slots[(warp * WORDS + i) * 32 + lane] = (&tot[0][0][0])[i];
      } else if (q1 == U) {
        finish<NT>(strip_flat, tot);
      } else {
        tail = true;                      // the warp's last one: the next warps have the rest
      }
    }
    __syncthreads();
    if (tail) {
      for (int v = warp + 1; v < WARPS; ++v) {
        const int from = p0 + (int)((int64_t)n * v / WARPS), to = p0 + (int)((int64_t)n * (v + 1) / WARPS);
        if (from >= (strip_flat + 1) * U) break;
        if (from < to) {
#pragma unroll
          for (int i = 0; i < WORDS; ++i) (&tot[0][0][0])[i] += slots[(v * WORDS + i) * 32 + lane];
        }
      }
      finish<NT>(strip_flat, tot);
    }
  }

  __device__ __forceinline__ void run_all(uint8_t* smem, SmallPlan& sp) {
    warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    m = masks<D>();
    constexpr int NS = S::SCALES / 16, NZ = S::ZEROS / 16;
    static_assert(NS + NZ <= 32, "one copy a lane");
    scale_lane = lane < NS;
    zero_lane = ZP && lane >= NS && lane < NS + NZ;
    const int nt = a.cols <= 8 ? 1 : 2;
    stage = S::STAGE + (XR ? a.cols * UNIT_K * 2 : 0);
    ring = smem + warp * (a.depth * stage);
    ring_s = (uint32_t)__cvta_generic_to_shared(ring);
    uint8_t* after = smem + WARPS * (a.depth * stage);
    slots = reinterpret_cast<float*>(after);
    after += WARPS * RT * nt * 4 * 32 * 4;
    xs = reinterpret_cast<uint4*>(after);
    cw = reinterpret_cast<float*>(after);
    plan = &sp;
    int n_items = 1;
    item_start = 0;
    item_count = a.cols;
    U = a.units;
    if (SMALL2 || a.mode == GATEUP_SMALL) {
      plan_small(a, sp);
      __syncthreads();
      n_items = sp.n;
      item_count = a.t;
      if (SMALL2) {
        U = sp.n * a.units;
        n_items = 1;
        for (int i = threadIdx.x; i < sp.n * MAX_COLS; i += THREADS) {
          const int e = sp.expert[i / MAX_COLS], tok = i % MAX_COLS;
          float w = 0.0f;
          if (tok < a.t)
            for (int k = 0; k < a.s; ++k)
              if (a.ids[tok * a.s + k] == e) w += a.weights[tok * a.s + k];
          cw[i] = w;
        }
        __syncthreads();
      }
    } else {
      n_items = a.mode == LINEAR ? a.n_items : *a.items_n;
    }
    const int64_t total = (int64_t)n_items * a.strips;   // below 2^31
    const int lo = (int)(total * blockIdx.x / gridDim.x), hi = (int)(total * (blockIdx.x + 1) / gridDim.x);
    if (SMALL2 && U == 0) {   // no slot selects an expert
      for (int strip = lo + warp; strip < hi; strip += WARPS) {
        float zero[RT][2][4] = {};
        finish<2>(strip, zero);
      }
      return;
    }
    bool staged = false;
    for (int from = lo; from < hi;) {
      // a phase: the strips of one item, or all of them if its columns are the same for all
      int to = hi;
      if (!SMALL2 && a.mode != GATEUP_SMALL) {
        const int item = from / a.strips;
        to = min(hi, (item + 1) * a.strips);
        if (a.mode == LINEAR) {
          item_start = item * a.tb;
          item_count = min(a.tb, a.t - item_start);
        } else {
          item_start = a.items[item].y;
          item_count = a.items[item].z;
        }
      }
      const int p0 = from * U, n = (to - from) * U;
      const int p = p0 + (int)((int64_t)n * warp / WARPS), p_end = p0 + (int)((int64_t)n * (warp + 1) / WARPS);
      cp = p;
      cp_end = p_end;
      run = 0;
      slot = 0;
      if (p < p_end) locate();
      if (staged) __syncthreads();   // every warp is done with the last phase's activations and parts
      for (int s = 0; s < a.depth; ++s) issue<true>(ring_s + s * stage);
      if (!XR) {
        stage_x(a, xs, item_start, item_count);
        cp_commit();
        cp_wait<0>();
        __syncthreads();
      }
      staged = true;
      if (item_count <= 8) units<1>(p, p_end, p0, n);
      else units<2>(p, p_end, p0, n);
      from = to;
    }
    cp_wait<0>();
  }
};

template <class D, int RT, int G, bool ZP, bool XR, bool SMALL2>
__global__ void __launch_bounds__(THREADS, 1) w4_kernel(const Args a) {
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ SmallPlan plan;
  Kernel<D, RT, G, ZP, XR, SMALL2> k(a);
  k.run_all(smem, plan);
}

// The slots grouped by expert: columns (slots in expert order), col_token, slot_col (a slot's
// column, -1 if empty), and the items of at most tb columns of one expert. One CTA. A slot's place
// among its expert's columns depends on the order of the counting and changes no result: a column's
// sums do not depend on its place.
__global__ void __launch_bounds__(1024) plan_kernel(const int* __restrict__ ids, int t, int s, int experts, int tb,
                                                    int4* items, int* items_n, int* col_token, int* slot_col) {
  __shared__ int cnt[MAX_EXPERTS], first[MAX_EXPERTS];
  const int n = t * s;
  for (int e = threadIdx.x; e < MAX_EXPERTS; e += blockDim.x) cnt[e] = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += blockDim.x) {
    const int e = ids[i];
    if ((unsigned)e < (unsigned)experts) atomicAdd(&cnt[e], 1);
  }
  __syncthreads();
  if (threadIdx.x < 32) {
    int cols = 0, its = 0;
    for (int e0 = 0; e0 < experts; e0 += 32) {
      const int e = e0 + threadIdx.x, c = e < experts ? cnt[e] : 0, b = (c + tb - 1) / tb;
      int ci = c, bi = b;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(~0u, ci, o), v = __shfl_up_sync(~0u, bi, o);
        if ((int)threadIdx.x >= o) { ci += u; bi += v; }
      }
      const int col0 = cols + ci - c, it0 = its + bi - b;
      if (e < experts) first[e] = col0;
      for (int k = 0; k < b; ++k) items[it0 + k] = make_int4(e, col0 + k * tb, min(tb, c - k * tb), 0);
      cols += __shfl_sync(~0u, ci, 31);
      its += __shfl_sync(~0u, bi, 31);
    }
    if (threadIdx.x == 0) *items_n = its;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += blockDim.x) {
    const int e = ids[i];
    int col = -1;
    if ((unsigned)e < (unsigned)experts) {
      col = atomicAdd(&first[e], 1);
      col_token[col] = i / s;
    }
    slot_col[i] = col;
  }
}

// out[t] = (residual[t] +) sum over slots, in slot order, of w[t, s] y[column of the slot]
template <class D>
__global__ void __launch_bounds__(256) combine_kernel(const float* __restrict__ y, const int* __restrict__ slot_col,
                                                      const float* __restrict__ weights, int s, int h,
                                                      const uint16_t* residual, int64_t ldr, uint16_t* out, int64_t ldo) {
  const int tok = blockIdx.y, j = blockIdx.x * 256 + threadIdx.x;
  if (j >= h) return;
  float v = residual ? D::one_to_f32(residual[(int64_t)tok * ldr + j]) : 0.0f;
  for (int k = 0; k < s; ++k) {
    const int col = slot_col[tok * s + k];
    if (col >= 0) v = fmaf(weights[tok * s + k], y[(int64_t)col * h + j], v);
  }
  out[(int64_t)tok * ldo + j] = D::round(v);
}

int fail(int code, const char* msg) { return mk::set_last_error(code, msg); }

const char* bad_weight(const MkW4* w) {
  if (!w || !w->codes || !w->scales) return "null 4-bit weight";
  if (w->n < 1 || w->k < 1 || w->experts < 1) return "a 4-bit weight has at least one row, value and expert";
  if (w->group != 32 && w->group != 64 && w->group != 128) return "the group size is 32, 64 or 128";
  if (w->dtype != MK_W4_BF16 && w->dtype != MK_W4_FP16) return "the activations are BF16 or FP16";
  if (((uintptr_t)w->codes & 15) || ((uintptr_t)w->scales & 15) || ((uintptr_t)w->zeros & 15))
    return "laid-out codes, scales and zeros start at 16-byte boundaries";
  return nullptr;
}

int units_of(const MkW4* w) { return (w->k + UNIT_K - 1) / UNIT_K; }

void fill(Args& a, const MkW4* w) {
  a.codes = static_cast<const uint8_t*>(w->codes);
  a.scales = static_cast<const uint8_t*>(w->scales);
  a.zeros = static_cast<const uint8_t*>(w->zeros);
  a.units = units_of(w);
  a.rows = w->n;
  a.k = w->k;
  a.experts = w->experts;
}

struct Device {
  int sms = 0;
};
constexpr int MAX_DEVICES = 64;
std::mutex g_mu;
Device g_dev[MAX_DEVICES];

int device_sms(int* sms) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= MAX_DEVICES)
    return fail(MK_ECUDA, "cudaGetDevice failed or device ordinal out of range");
  std::lock_guard<std::mutex> lock(g_mu);
  if (!g_dev[dev].sms) {
    int v = 0;
    if (cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return fail(MK_ECUDA, "device attribute");
    g_dev[dev].sms = v;
  }
  *sms = g_dev[dev].sms;
  return MK_OK;
}

// bytes beside rings and activations: the parts and the small plan (static)
constexpr int parts_bytes(int rt, int cols) { return WARPS * rt * (cols <= 8 ? 1 : 2) * 4 * 32 * 4; }
constexpr int STATIC_BYTES = (sizeof(SmallPlan) + 1023) / 1024 * 1024;
// a ring of two stages of two tiles, for the group size and zero points that take most
constexpr int LEAST_RING = WARPS * 2 * Shape<2, 32, true>::STAGE;

// whether the activations of `cols` columns can be staged beside the least ring
bool fits(int units, int cols) {
  return LEAST_RING + parts_bytes(2, cols) + STATIC_BYTES + (int64_t)cols * units * UNIT_K * 2 <= SMEM_LIMIT;
}

// beside a ring that carries the activations: the weights of a small batch's slots
constexpr int CW_BYTES = SMALL_SLOTS * MAX_COLS * 4;
bool two_tiles_fit_ring(int cols) {
  return WARPS * 2 * (Shape<2, 32, true>::STAGE + cols * UNIT_K * 2) + parts_bytes(2, cols) + CW_BYTES + STATIC_BYTES <= SMEM_LIMIT;
}

template <class D, int RT, int G, bool ZP, bool XR, bool SMALL2>
int launch(Args a, int grid, cudaStream_t s) {
  using S = Shape<RT, G, ZP>;
  const int stage = S::STAGE + (XR ? a.cols * UNIT_K * 2 : 0);
  const int64_t rest = parts_bytes(RT, a.cols) + (SMALL2 ? CW_BYTES : XR ? 0 : (int64_t)a.cols * a.units * UNIT_K * 2);
  a.depth = 8;
  while (a.depth > 2 && (int64_t)WARPS * a.depth * stage + rest + STATIC_BYTES > SMEM_LIMIT) a.depth /= 2;
  const auto kernel = w4_kernel<D, RT, G, ZP, XR, SMALL2>;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_LIMIT - STATIC_BYTES);
  if (e == cudaSuccess) {
    kernel<<<grid, THREADS, (size_t)(WARPS * a.depth * stage + rest), s>>>(a);
    e = cudaGetLastError();
  }
  return e == cudaSuccess ? MK_OK : fail(MK_ECUDA, cudaGetErrorString(e));
}

template <class D, int RT, int G, bool ZP>
int launch_x(const Args& a, bool through_ring, int grid, cudaStream_t s) {
  if (a.mode == DOWN_SMALL) return launch<D, RT, G, ZP, true, true>(a, grid, s);
  return through_ring ? launch<D, RT, G, ZP, true, false>(a, grid, s) : launch<D, RT, G, ZP, false, false>(a, grid, s);
}

template <class D, int RT>
int launch_group(const Args& a, int group, bool xr, int grid, cudaStream_t s) {
  if (group == 32) return a.zeros ? launch_x<D, RT, 32, true>(a, xr, grid, s) : launch_x<D, RT, 32, false>(a, xr, grid, s);
  if (group == 64) return a.zeros ? launch_x<D, RT, 64, true>(a, xr, grid, s) : launch_x<D, RT, 64, false>(a, xr, grid, s);
  return a.zeros ? launch_x<D, RT, 128, true>(a, xr, grid, s) : launch_x<D, RT, 128, false>(a, xr, grid, s);
}

// about `items` items over the SMs; known: exactly that many
int launch_weight(Args& a, const MkW4* w, int64_t items, bool known, bool through_ring, int sms, cudaStream_t s) {
  const int strips = (w->n + STRIP_ROWS - 1) / STRIP_ROWS;
  // enough strips for every CTA: two tiles a warp share the activations
  const bool two = items * strips >= 2 * sms && !(through_ring && !two_tiles_fit_ring(a.cols));
  a.strips = two ? strips : 2 * strips;
  const int grid = (int)(known ? std::min<int64_t>(sms, items * a.strips) : sms);
  if (w->dtype == MK_W4_BF16)
    return two ? launch_group<Bf16, 2>(a, w->group, through_ring, grid, s) : launch_group<Bf16, 1>(a, w->group, through_ring, grid, s);
  return two ? launch_group<Fp16, 2>(a, w->group, through_ring, grid, s) : launch_group<Fp16, 1>(a, w->group, through_ring, grid, s);
}

bool aligned16(const void* p, int64_t ld) { return ((uintptr_t)p & 15) == 0 && ld % 8 == 0; }

struct Plan {   // the workspace of mk_w4_experts, in bytes from its start
  int64_t items, items_n, col_token, slot_col, act, y, bytes;
  int cols, ldact;
  bool small;
};

const char* plan_experts(const MkW4* w13, const MkW4* w2, int64_t t, int64_t s, Plan* p) {
  if (const char* m = bad_weight(w13)) return m;
  if (const char* m = bad_weight(w2)) return m;
  if (w13->dtype != w2->dtype || w13->experts != w2->experts || w13->n % 2 || w13->n / 2 != w2->k || w13->k != w2->n)
    return "W13 [E, 2 I, H] and W2 [E, H, I] do not belong together";
  if (w13->experts > MAX_EXPERTS) return "at most 1024 experts";
  if (t < 0 || s < 0 || t * s >= (1 << 24)) return "slots (tokens x slots per token) are from 0 to 2^24 - 1";
  p->small = t <= SMALL_T && t * s <= SMALL_SLOTS && fits(units_of(w13), (int)std::max<int64_t>(t, 1));
  p->cols = (int)std::min<int64_t>(std::max<int64_t>(t, 1), MAX_COLS);
  while (p->cols > 1 && !(fits(units_of(w13), p->cols) && (p->small || fits(units_of(w2), p->cols)))) --p->cols;
  if (!fits(units_of(w13), p->cols) || (!p->small && !fits(units_of(w2), p->cols))) return "rows are too long for the shared memory";
  const int64_t n = std::max<int64_t>(t * s, 1), items = w13->experts + n / p->cols + 1;
  const int64_t most = std::max((std::max(w13->n, w2->n) / 16 + 2) * std::max<int64_t>(units_of(w13), units_of(w2)), (int64_t)1);
  if (items * most > INT32_MAX / 2) return "too many slots times rows";
  int64_t at = 0;
  auto take = [&](int64_t bytes) { const int64_t r = at; at += (bytes + 255) / 256 * 256; return r; };
  if (p->small) {
    p->act = take(2 * n * t * units_of(w2) * UNIT_K);
  } else {
    p->ldact = (w2->k + 7) / 8 * 8;
    p->items_n = take(4);
    p->items = take(16 * items);
    p->col_token = take(4 * n);
    p->slot_col = take(4 * n);
    p->act = take(2 * n * p->ldact);
    p->y = take(4 * n * w2->n);
  }
  p->bytes = std::max<int64_t>(at, 256);
  return nullptr;
}

}  // namespace

extern "C" int mk_w4_linear(const MkW4* w, const void* x, int64_t ldx, int32_t t, const void* residual, int64_t ldr,
                            void* out, int64_t ldo, int32_t out_f32, void* stream) {
  if (const char* m = bad_weight(w)) return fail(MK_EINVAL, m);
  if (w->experts != 1) return fail(MK_EINVAL, "mk_w4_linear takes one weight");
  if (t < 0) return fail(MK_EINVAL, "a negative number of tokens");
  if (t == 0) return MK_OK;
  if (!x || !out) return fail(MK_EINVAL, "null pointer");
  if (((uintptr_t)x & 1) || ((uintptr_t)residual & 1) || ((uintptr_t)out & (out_f32 ? 3 : 1)))
    return fail(MK_EINVAL, "misaligned x, residual or out");
  int sms = 0;
  if (int rc = device_sms(&sms)) return rc;
  Args a{};
  fill(a, w);
  a.mode = LINEAR;
  a.t = t;
  a.x = static_cast<const uint16_t*>(x);
  a.ldx = ldx;
  a.x_vec = aligned16(x, ldx);
  // even blocks of at most 16 tokens
  const int blocks = (t + MAX_COLS - 1) / MAX_COLS;
  a.tb = (t + blocks - 1) / blocks;
  const bool through_ring = a.x_vec && !fits(a.units, a.tb);
  if (!through_ring)
    while (a.tb > 1 && !fits(a.units, a.tb)) --a.tb;
  if (!through_ring && !fits(a.units, a.tb)) return fail(MK_EINVAL, "rows that are not 16-byte aligned are too long for the shared memory");
  a.n_items = (t + a.tb - 1) / a.tb;
  a.cols = a.tb;
  a.residual = static_cast<const uint16_t*>(residual);
  a.ldr = ldr;
  a.out = out;
  a.ldo = ldo;
  a.out_f32 = out_f32;
  if ((int64_t)a.n_items * (w->n / 16 + 2) * a.units > INT32_MAX / 2) return fail(MK_EINVAL, "too many tokens times weights");
  return launch_weight(a, w, a.n_items, true, through_ring, sms, static_cast<cudaStream_t>(stream));
}

extern "C" int mk_w4_experts_workspace(const MkW4* w13, const MkW4* w2, int32_t t, int32_t slots, int64_t* bytes) {
  Plan p{};
  if (const char* m = plan_experts(w13, w2, t, slots, &p)) return fail(MK_EINVAL, m);
  if (!bytes) return fail(MK_EINVAL, "null pointer");
  *bytes = p.bytes;
  return MK_OK;
}

extern "C" int mk_w4_experts(const MkW4* w13, const MkW4* w2, const void* x, int64_t ldx, const int32_t* ids,
                             const float* weights, int32_t t, int32_t slots, const void* residual, int64_t ldr, void* out,
                             int64_t ldo, void* workspace, int64_t workspace_bytes, void* stream) {
  Plan p{};
  if (const char* m = plan_experts(w13, w2, t, slots, &p)) return fail(MK_EINVAL, m);
  if (t == 0) return MK_OK;
  if (!x || !out || (slots && (!ids || !weights))) return fail(MK_EINVAL, "null pointer");
  if (((uintptr_t)x & 1) || ((uintptr_t)residual & 1) || ((uintptr_t)out & 1)) return fail(MK_EINVAL, "misaligned x, residual or out");
  if (!workspace || workspace_bytes < p.bytes || ((uintptr_t)workspace & 255))
    return fail(MK_EINVAL, "the workspace is missing, too small (mk_w4_experts_workspace) or not at a 256-byte boundary");
  if (t > 65535) return fail(MK_EINVAL, "at most 65535 tokens a call");
  int sms = 0;
  if (int rc = device_sms(&sms)) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  const int64_t items_about = std::min<int64_t>((int64_t)t * slots, w13->experts);
  Args a{}, b{};
  fill(a, w13);
  fill(b, w2);
  a.t = b.t = t;
  a.s = b.s = slots;
  a.ids = b.ids = ids;
  a.cols = b.cols = p.cols;
  a.x = static_cast<const uint16_t*>(x);
  a.ldx = ldx;
  a.x_vec = aligned16(x, ldx);
  a.out = ws + p.act;
  b.x = reinterpret_cast<const uint16_t*>(ws + p.act);
  b.x_vec = 1;
  if (p.small) {
    a.mode = GATEUP_SMALL;
    a.ldo = b.units;
    if (slots)
      if (int rc = launch_weight(a, w13, items_about, false, false, sms, st)) return rc;
    b.mode = DOWN_SMALL;
    b.weights = weights;
    b.residual = static_cast<const uint16_t*>(residual);
    b.ldr = ldr;
    b.out = out;
    b.ldo = ldo;
    return launch_weight(b, w2, 1, true, true, sms, st);
  }
  int4* items = reinterpret_cast<int4*>(ws + p.items);
  int* items_n = reinterpret_cast<int*>(ws + p.items_n);
  int* col_token = reinterpret_cast<int*>(ws + p.col_token);
  int* slot_col = reinterpret_cast<int*>(ws + p.slot_col);
  plan_kernel<<<1, 1024, 0, st>>>(ids, t, slots, w13->experts, p.cols, items, items_n, col_token, slot_col);
  a.mode = GATEUP;
  a.items = b.items = items;
  a.items_n = b.items_n = items_n;
  a.col_token = col_token;
  a.ldo = b.ldx = p.ldact;
  if (int rc = launch_weight(a, w13, items_about, false, false, sms, st)) return rc;
  b.mode = DOWN;
  b.out = ws + p.y;
  b.ldo = w2->n;
  b.out_f32 = 1;
  if (int rc = launch_weight(b, w2, items_about, false, false, sms, st)) return rc;
  const dim3 grid((unsigned)((w2->n + 255) / 256), (unsigned)t);
  const float* y = reinterpret_cast<const float*>(ws + p.y);
  if (w2->dtype == MK_W4_BF16)
    combine_kernel<Bf16><<<grid, 256, 0, st>>>(y, slot_col, weights, slots, w2->n, static_cast<const uint16_t*>(residual), ldr,
                                               static_cast<uint16_t*>(out), ldo);
  else
    combine_kernel<Fp16><<<grid, 256, 0, st>>>(y, slot_col, weights, slots, w2->n, static_cast<const uint16_t*>(residual), ldr,
                                               static_cast<uint16_t*>(out), ldo);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? MK_OK : fail(MK_ECUDA, cudaGetErrorString(e));
}

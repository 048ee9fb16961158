// mk_w4.cu -- products with 4-bit weights for a batch of tokens: mk_w4_linear (one weight) and
// mk_w4_experts (a layer's routed experts: gate/up, SwiGLU, down projection, weighted sum).
// The format and the laid-out order are in mk_w4.cuh.
//
// Formulas. linear: out[t] = x[t] W^T (+ residual[t]). experts: out[t] = (residual[t] +) the sum over
// the token's slots s in slot order of w[t, s] W2[e] a(t, s), a = silu(g) u, (g, u) = W13[e] x[t],
// e = ids[t, s]; a slot whose id is outside [0, experts) is empty.
//
// What bounds them. A token costs 2 operations per weight and a weight half a byte, so a batch of T
// tokens does 4 T operations a byte: below about T = 40 the stream of codes is the bound, not the
// tensor cores (2 cycles an m16n8k16 per SM against 5.5 cycles for its 128 bytes at 6.5 TB/s), and
// mma.sync takes a tile of 16 rows by 8 tokens without padding a decode batch to the 64 or 128 rows
// of a tcgen05 tile.
//
// One kernel, three modes. The work is a list of items (a block of at most 8 NT columns that share a
// weight: the linear's token blocks; an expert and up to 8 NT of the slots routed to it) times the
// weight's tiles; each CTA (one per SM, 16 warps) takes an equal contiguous range of that product. A
// team of kw warps owns a tile and splits its units; each warp streams its units through its own
// cp.async ring (DEPTH - 1 units of 128 values in flight, across tile and item boundaries), so no barrier stands
// between the copies and the MMAs. The item's activations are staged in shared memory in the MMA's
// order. A tile's partial sums meet in shared memory and are added in warp order: the result does
// not depend on timing.
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
enum Mode { LINEAR = 0, GATEUP = 1, DOWN = 2 };

// a warp's step: a unit of RT tiles
template <int RT, int G, bool ZP>
struct Shape {
  static constexpr int GROUPS = UNIT_K / G;          // per unit
  static constexpr int SCALES = RT * GROUPS * 32, ZEROS = ZP ? RT * GROUPS * 16 : 0;
  static constexpr int STAGE = RT * TILE_UNIT_BYTES + SCALES + ZEROS;
  static constexpr int RED_STRIDE = RT * 16 + 4;     // floats per column of the partial sums (4: no bank conflicts)
  static constexpr int RED = WARPS * 8 * RED_STRIDE * 4;
};

struct Args {
  const uint8_t* codes;
  const uint8_t* scales;
  const uint8_t* zeros;     // or null: 8
  int tiles;                // steps of RT tiles down the rows
  int units, rows, k;
  int depth;                // stages of a warp's ring: 2, 4 or 8
  int mode;
  int n_items;              // LINEAR: known on the host; else *items_n
  const int* items_n;
  const int4* items;        // {expert, first column, columns, 0}
  const int* col_token;     // GATEUP: the token of a column
  int t, tb;                // LINEAR: tokens, tokens per item
  int kw;                   // warps per team
  int ks;                   // CTAs (of one cluster) that split K
  const uint16_t* x;
  int64_t ldx;
  int x_vec;                // x rows may be read 16 bytes at a time
  const uint16_t* residual; // LINEAR
  int64_t ldr;
  void* out;                // LINEAR: 16-bit or FP32; GATEUP: act, 16-bit; DOWN: FP32
  int64_t ldo;
  int out_f32;
};

// the warps of one team (named barriers 1..8; a team of one warp needs none)
__device__ __forceinline__ void team_sync(int team, int kw) {
  if (kw == 1) __syncwarp();
  else asm volatile("bar.sync %0, %1;" ::"r"(1 + team), "r"(kw * 32) : "memory");
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// the float at the same shared-memory place in the cluster's CTA `rank`
__device__ __forceinline__ float peer_float(const float* p, int rank) {
  const uint32_t at = (uint32_t)__cvta_generic_to_shared(p);
  uint32_t there;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(at), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(there) : "memory");
  return v;
}

// the item's activations [8 v0, 8 v1) in the MMA's order: [(v - v0) / 4][columns][4] 16-byte vectors
__device__ __forceinline__ void stage_x(const Args& a, uint4* xs, int start, int count, int v0, int v1) {
  const int nv = v1 - v0;
  const uint32_t xs_s = (uint32_t)__cvta_generic_to_shared(xs);
  for (int i = threadIdx.x; i < count * nv; i += THREADS) {
    const int col = i / nv, r = i - col * nv, v = v0 + r;
    const int row = a.mode == GATEUP ? a.col_token[start + col] : start + col;
    const uint16_t* src = a.x + (int64_t)row * a.ldx + 8 * v;
    const int at = ((r >> 2) * count + col) * 4 + (r & 3);
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

// One warp's copies: its units of its team's tiles, in order, across the items of the CTA's range.
template <int RT, int G, bool ZP>
struct Copies {
  using S = Shape<RT, G, ZP>;
  int f = 0, end = 0, left = 0;            // the flat tile, the segment's end, the tile's units to come
  int tile0 = 0;                           // from a flat tile to the tile of the item's weight
  const uint8_t *code = nullptr, *meta = nullptr;
  bool scale_lane, zero_lane;              // lanes 0.. carry the scales' 16-byte pieces, then the zero points'
  uint32_t meta_at;
  int meta_step;

  __device__ __forceinline__ void init(int lane) {
    constexpr int NS = S::SCALES / 16, NZ = S::ZEROS / 16;
    static_assert(NS + NZ <= 32, "one copy a lane");
    scale_lane = lane < NS;
    zero_lane = ZP && lane >= NS && lane < NS + NZ;
    meta_at = RT * TILE_UNIT_BYTES + lane * 16;
  }
  // tile f in units of RT tiles: with RT 1 the two tiles of a strip lie side by side in each unit
  __device__ __forceinline__ void at_tile(const Args& a, int first_unit, int n_units, int lane) {
    const int64_t w = f + tile0;
    const int64_t strip = RT == 2 ? w : w >> 1;
    const int half = RT == 2 ? 0 : (int)(w & 1);
    const int64_t u = (strip * a.units + first_unit) * 2 + half;         // in tiles' units
    code = a.codes + u * TILE_UNIT_BYTES + lane * 16;
    if (scale_lane) meta = a.scales + u * (S::GROUPS * 32) + lane * 16;
    else if (zero_lane) meta = a.zeros + u * (S::GROUPS * 16) + (lane - S::SCALES / 16) * 16;
    left = n_units;
  }
  __device__ __forceinline__ void at_segment(const Args& a, int from, int hi, int team) {
    const int item = from / a.tiles;
    end = min(hi, (item + 1) * a.tiles);
    f = from + team;
    tile0 = ((a.mode == LINEAR ? 0 : a.items[item].x) - item) * a.tiles;
  }
  __device__ __forceinline__ void skip_empty(const Args& a, int hi, int team, int first_unit, int n_units, int lane) {
    while (f >= end && end < hi) at_segment(a, end, hi, team);
    if (f < end) at_tile(a, first_unit, n_units, lane);
  }
};

template <class D, int RT, int G, bool ZP>
struct Kernel {
  using S = Shape<RT, G, ZP>;
  const Args& a;
  Masks m;
  int warp, lane, g, t;
  int kw, teams, team, part;
  int ks, rank, u0, n_units, hi;
  uint8_t* ring;
  uint32_t ring_s;
  float* red;
  uint4* xs;
  Copies<RT, G, ZP> c;
  uint32_t slot = 0;

  __device__ __forceinline__ Kernel(const Args& args) : a(args) {}

  __device__ __forceinline__ void issue(uint32_t dst) {
    const bool on = c.left > 0;
#pragma unroll
    for (int i = 0; i < RT * 2; ++i) cp16_if(on, dst + i * 512 + lane * 16, c.code + i * 512);
    cp16_if(on && (c.scale_lane || c.zero_lane), dst + c.meta_at, c.meta);
    cp_commit();
    c.code += kw * (2 * TILE_UNIT_BYTES);
    c.meta += c.meta_step;
    if (--c.left == 0) {
      c.f += teams;
      c.skip_empty(a, hi, team, u0 + part, n_units, lane);
    }
  }

  // the tiles [seg, seg_end) of one item's columns [start, start + count), count <= 8 NT
  template <int NT>
  __device__ __forceinline__ void segment(int seg, int seg_end, int item, int start, int count) {
    // a lane past the columns reads the last one's activations: its sums are not used
    const uint4* xl[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) xl[n] = xs + (part * 4 * count + min(n * 8 + g, count - 1)) * 4 + t;
    const int x_h = count * 4, x_u = kw * count * 16;
    for (int first = seg; first < seg_end; first += teams) {
      const int f = first + team;
      const bool live = f < seg_end;
      if (!live && ks == 1) break;
      float tot[RT][NT][4];
#pragma unroll
      for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) tot[r][n][i] = 0.0f;
      int x_at = 0;
      for (int u = live ? n_units : 0; u > 0; --u) {
        if (a.depth == 2) cp_wait<1>();
        else if (a.depth == 4) cp_wait<3>();
        else cp_wait<7>();
        __syncwarp();
        const uint8_t* st = ring + slot;
        uint4 w[RT][2];
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
        __syncwarp();            // every lane has read the stage
        issue(ring_s + slot);
        slot = slot == (a.depth - 1) * S::STAGE ? 0 : slot + S::STAGE;
        float acc[RT][NT][4];
#pragma unroll
        for (int h = 0; h < 4; ++h) {
          uint4 xb[NT];
#pragma unroll
          for (int n = 0; n < NT; ++n) xb[n] = xl[n][x_at + h * x_h];
          const int i = h * 32 / G;
#pragma unroll
          for (int r = 0; r < RT; ++r) {
            const uint4& v = w[r][h >> 1];
            if (h * 32 % G == 0) half_chunk<D, NT, true>(m, h & 1 ? v.z : v.x, h & 1 ? v.w : v.y, z0[r][i], z1[r][i], xb, acc[r]);
            else half_chunk<D, NT, false>(m, h & 1 ? v.z : v.x, h & 1 ? v.w : v.y, z0[r][i], z1[r][i], xb, acc[r]);
            if ((h + 1) * 32 % G == 0) fold<D, NT>(sc[r][i], acc[r], tot[r]);
          }
        }
        x_at += x_u;
      }
      // the team's partial sums, [column][row], eight columns at a time, added in warp order
      constexpr int RED_WARP = 8 * S::RED_STRIDE, ROWS = RT * 16;
      float* mine = red + warp * RED_WARP;
      float* theirs = red + team * kw * RED_WARP;
      const int row0 = (f - item * a.tiles) * ROWS, me = part * 32 + lane;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const int cols = min(count - n * 8, 8);
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
          for (int i = 0; i < 4; ++i) mine[(2 * t + (i & 1)) * S::RED_STRIDE + r * 16 + g + (i >> 1) * 8] = tot[r][n][i];
        team_sync(team, kw);
        if (a.mode == GATEUP) {   // a tile's rows 0..7 are gate rows, 8..15 their up rows
          for (int i = me; i < cols * (ROWS / 2); i += kw * 32) {
            const int col = i / (ROWS / 2), q = i % (ROWS / 2), r = (q >> 3) * 16 + (q & 7), j = row0 / 2 + q;
            float gt = 0.0f, up = 0.0f;
            for (int v = 0; v < kw; ++v) {
              gt += theirs[v * RED_WARP + col * S::RED_STRIDE + r];
              up += theirs[v * RED_WARP + col * S::RED_STRIDE + r + 8];
            }
            // rounded to the activations' type: the down projection's tensor-core operand
            if (j < a.rows / 2)
              static_cast<uint16_t*>(a.out)[(int64_t)(start + n * 8 + col) * a.ldo + j] =
                  D::round(__fdiv_rn(gt, 1.0f + expf(-gt)) * up);
          }
        } else {
          auto store = [&](int col, int r, float v) {
            const int64_t row = start + n * 8 + col, o = row * a.ldo + row0 + r;
            if (row0 + r >= a.rows) return;
            if (a.residual) v += D::one_to_f32(a.residual[row * a.ldr + row0 + r]);
            if (a.out_f32) static_cast<float*>(a.out)[o] = v;
            else static_cast<uint16_t*>(a.out)[o] = D::round(v);
          };
          for (int i = me; i < cols * ROWS; i += kw * 32) {
            const int col = i / ROWS, r = i % ROWS;
            float v = 0.0f;
            for (int w = 0; w < kw; ++w) v += theirs[w * RED_WARP + col * S::RED_STRIDE + r];
            if (ks > 1) theirs[col * S::RED_STRIDE + r] = v;   // this thread's own place: the CTA's sum for the cluster
            else store(col, r, v);
          }
          if (ks > 1) {   // K is split over the cluster: each CTA adds and stores the columns col % ks == rank
            cluster_sync();
            for (int i = me; i < cols * ROWS; i += kw * 32) {
              const int col = i / ROWS, r = i % ROWS;
              if (col % ks != rank || !live) continue;
              float v = 0.0f;
              for (int p = 0; p < ks; ++p) v += peer_float(theirs + col * S::RED_STRIDE + r, p);
              store(col, r, v);
            }
            cluster_sync();
          }
        }
        team_sync(team, kw);   // the sums are read before the next ones are written
        if (cols < 8) break;
      }
    }
  }

  __device__ __forceinline__ void run(uint8_t* smem) {
    warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    m = masks<D>();
    ring = smem + warp * (a.depth * S::STAGE);
    ring_s = (uint32_t)__cvta_generic_to_shared(ring);
    red = reinterpret_cast<float*>(smem + WARPS * a.depth * S::STAGE);
    xs = reinterpret_cast<uint4*>(smem + WARPS * a.depth * S::STAGE + S::RED);
    const int n_items = a.mode == LINEAR ? a.n_items : *a.items_n;
    const int64_t total = (int64_t)n_items * a.tiles;   // below 2^31
    ks = a.ks;
    rank = blockIdx.x % ks;
    const int group = blockIdx.x / ks, n_groups = gridDim.x / ks;
    const int lo = (int)(total * group / n_groups);
    hi = (int)(total * (group + 1) / n_groups);
    kw = a.kw, teams = WARPS / kw, team = warp / kw, part = warp - team * kw;
    u0 = a.units * rank / ks;
    const int u1 = a.units * (rank + 1) / ks;
    n_units = max(0, (u1 - u0 - part + kw - 1) / kw);   // this warp's units of a tile
    c.init(lane);
    c.meta_step = kw * 2 * S::GROUPS * (c.scale_lane ? 32 : 16);
    if (lo < hi && n_units > 0) {
      c.at_segment(a, lo, hi, team);
      c.skip_empty(a, hi, team, u0 + part, n_units, lane);
    }
    for (int s = 0; s < a.depth; ++s) issue(ring_s + s * S::STAGE);
    for (int seg = lo; seg < hi;) {
      const int item = seg / a.tiles;
      const int seg_end = min(hi, (item + 1) * a.tiles);
      int start, count;
      if (a.mode == LINEAR) {
        start = item * a.tb;
        count = min(a.tb, a.t - start);
      } else {
        const int4 it = a.items[item];
        start = it.y;
        count = it.z;
      }
      __syncthreads();   // every warp is done with the last item's activations
      stage_x(a, xs, start, count, u0 * 16, u1 * 16);
      cp_commit();
      cp_wait<0>();
      __syncthreads();
      if (count <= 8) segment<1>(seg, seg_end, item, start, count);
      else if (count <= 16) segment<2>(seg, seg_end, item, start, count);
      else segment<4>(seg, seg_end, item, start, count);
      seg = seg_end;
    }
    cp_wait<0>();
  }
};

template <class D, int RT, int G, bool ZP>
__global__ void __launch_bounds__(THREADS, 1) w4_kernel(const Args a) {
  extern __shared__ __align__(16) uint8_t smem[];
  Kernel<D, RT, G, ZP> k(a);
  k.run(smem);
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

void fill(Args& a, const MkW4* w) {
  a.codes = static_cast<const uint8_t*>(w->codes);
  a.scales = static_cast<const uint8_t*>(w->scales);
  a.zeros = static_cast<const uint8_t*>(w->zeros);
  a.units = (w->k + UNIT_K - 1) / UNIT_K;
  a.ks = 1;
  a.rows = w->n;
  a.k = w->k;
}

// shared memory beside the activations for the group size and zero points that take most, at a depth
// that keeps 4 KB a warp in flight (twice what the HBM's rate times its latency asks for)
constexpr int FIXED = WARPS * 2 * Shape<2, 32, true>::STAGE + Shape<2, 32, true>::RED;

// columns (at most `want`, at most 32) whose activations of `units` units fit
int columns_that_fit(int units, int want) { return std::min({(SMEM_LIMIT - FIXED) / (units * UNIT_K * 2), 32, want}); }

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

template <class D, int RT, int G, bool ZP>
int launch(Args a, int grid, cudaStream_t s) {
  using S = Shape<RT, G, ZP>;
  const int xbytes = a.tb * ((a.units + a.ks - 1) / a.ks) * UNIT_K * 2;
  a.depth = RT == 2 ? 2 : 4;
  if (WARPS * a.depth * 2 * S::STAGE + S::RED + xbytes <= SMEM_LIMIT) a.depth *= 2;
  cudaLaunchConfig_t c{};
  cudaLaunchAttribute cluster[1];
  c.gridDim = dim3((unsigned)grid);
  c.blockDim = dim3(THREADS);
  c.dynamicSmemBytes = (size_t)WARPS * a.depth * S::STAGE + S::RED + xbytes;
  c.stream = s;
  cluster[0].id = cudaLaunchAttributeClusterDimension;
  cluster[0].val.clusterDim = {(unsigned)a.ks, 1, 1};
  c.attrs = cluster;
  c.numAttrs = a.ks > 1 ? 1 : 0;
  cudaError_t e = cudaFuncSetAttribute(w4_kernel<D, RT, G, ZP>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_LIMIT);
  if (e == cudaSuccess) e = cudaLaunchKernelEx(&c, w4_kernel<D, RT, G, ZP>, a);
  return e == cudaSuccess ? MK_OK : fail(MK_ECUDA, cudaGetErrorString(e));
}

template <class D, int RT>
int launch_group(const Args& a, int group, int grid, cudaStream_t s) {
  if (group == 32) return a.zeros ? launch<D, RT, 32, true>(a, grid, s) : launch<D, RT, 32, false>(a, grid, s);
  if (group == 64) return a.zeros ? launch<D, RT, 64, true>(a, grid, s) : launch<D, RT, 64, false>(a, grid, s);
  return a.zeros ? launch<D, RT, 128, true>(a, grid, s) : launch<D, RT, 128, false>(a, grid, s);
}

// warps per tile: few tiles are split over many warps, many are left to few
int team_warps(int64_t tiles, int units, int grid) {
  int kw = 16;
  while (kw > 1 && (kw > units || tiles > (int64_t)grid * (WARPS / kw) * 8)) kw /= 2;
  return kw;
}

// `items` (about) items over the CTAs, in groups of ks; a.tiles and a.kw are set here
int launch_weight(Args& a, const MkW4* w, int64_t items, int ctas, cudaStream_t s) {
  const int strips = (w->n + STRIP_ROWS - 1) / STRIP_ROWS;
  const int64_t max_groups = ctas / a.ks;
  const bool two = items * strips >= max_groups * 2;   // enough strips for every CTA: two tiles a warp share the activations
  a.tiles = two ? strips : 2 * strips;
  const int groups = (int)(a.mode == LINEAR ? std::min<int64_t>(max_groups, items * a.tiles) : max_groups);
  a.kw = team_warps(items * a.tiles, a.units / a.ks, groups);
  const int grid = groups * a.ks;
  if (w->dtype == MK_W4_BF16)
    return two ? launch_group<Bf16, 2>(a, w->group, grid, s) : launch_group<Bf16, 1>(a, w->group, grid, s);
  return two ? launch_group<Fp16, 2>(a, w->group, grid, s) : launch_group<Fp16, 1>(a, w->group, grid, s);
}

bool aligned16(const void* p, int64_t ld) { return ((uintptr_t)p & 15) == 0 && ld % 8 == 0; }

struct Plan {   // the workspace of mk_w4_experts, in bytes from its start
  int64_t items, items_n, col_token, slot_col, act, y, bytes;
  int tb1, tb2, ldact;
};

const char* plan_experts(const MkW4* w13, const MkW4* w2, int64_t t, int64_t s, Plan* p) {
  if (const char* m = bad_weight(w13)) return m;
  if (const char* m = bad_weight(w2)) return m;
  if (w13->dtype != w2->dtype || w13->experts != w2->experts || w13->n % 2 || w13->n / 2 != w2->k || w13->k != w2->n)
    return "W13 [E, 2 I, H] and W2 [E, H, I] do not belong together";
  if (w13->experts > MAX_EXPERTS) return "at most 1024 experts";
  const int64_t tiles = std::max(w13->n, w2->n) / 16 + 2;
  if (w13->experts * tiles > INT32_MAX / 2) return "too many experts times rows";
  if (t < 0 || s < 0 || t * s >= (1 << 24)) return "slots (tokens x slots per token) are from 0 to 2^24 - 1";
  const int want = t >= 32 ? 32 : (int)std::max<int64_t>(t, 1);
  p->tb1 = columns_that_fit((w13->k + UNIT_K - 1) / UNIT_K, want);
  p->tb2 = columns_that_fit((w2->k + UNIT_K - 1) / UNIT_K, want);
  if (p->tb1 < 1 || p->tb2 < 1) return "rows are too long for the shared memory";
  p->tb1 = p->tb2 = std::min(p->tb1, p->tb2);
  p->ldact = (w2->k + 7) / 8 * 8;
  const int64_t n = std::max<int64_t>(t * s, 1);
  if ((w13->experts + n / p->tb1 + 1) * tiles > INT32_MAX - 4096) return "too many slots times rows";
  int64_t at = 0;
  auto take = [&](int64_t bytes) { const int64_t r = at; at += (bytes + 255) / 256 * 256; return r; };
  p->items_n = take(4);
  p->items = take(16 * (w13->experts + n / p->tb1 + 1));
  p->col_token = take(4 * n);
  p->slot_col = take(4 * n);
  p->act = take(2 * n * p->ldact);
  p->y = take(4 * n * w2->n);
  p->bytes = at;
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
  a.t = t;
  // split K over a cluster while the tokens' activations do not fit one CTA's shared memory
  const int want = std::min(t, 32);
  for (a.ks = 1; a.ks < 8 && columns_that_fit((a.units + a.ks - 1) / a.ks, want) < want; a.ks *= 2) {}
  a.tb = columns_that_fit((a.units + a.ks - 1) / a.ks, want);
  if (a.tb < 1) return fail(MK_EINVAL, "rows are too long for the shared memory");
  a.n_items = (t + a.tb - 1) / a.tb;
  a.x = static_cast<const uint16_t*>(x);
  a.ldx = ldx;
  a.x_vec = aligned16(x, ldx);
  a.residual = static_cast<const uint16_t*>(residual);
  a.ldr = ldr;
  a.out = out;
  a.ldo = ldo;
  a.out_f32 = out_f32;
  if ((int64_t)a.n_items * (w->n / 16 + 2) > INT32_MAX - 4096) return fail(MK_EINVAL, "too many tokens times rows");
  return launch_weight(a, w, a.n_items, sms, static_cast<cudaStream_t>(stream));
}

extern "C" int mk_w4_experts_workspace(const MkW4* w13, const MkW4* w2, int32_t t, int32_t slots, int64_t* bytes) {
  Plan p;
  if (const char* m = plan_experts(w13, w2, t, slots, &p)) return fail(MK_EINVAL, m);
  if (!bytes) return fail(MK_EINVAL, "null pointer");
  *bytes = p.bytes;
  return MK_OK;
}

extern "C" int mk_w4_experts(const MkW4* w13, const MkW4* w2, const void* x, int64_t ldx, const int32_t* ids,
                             const float* weights, int32_t t, int32_t slots, const void* residual, int64_t ldr, void* out,
                             int64_t ldo, void* workspace, int64_t workspace_bytes, void* stream) {
  Plan p;
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
  int4* items = reinterpret_cast<int4*>(ws + p.items);
  int* items_n = reinterpret_cast<int*>(ws + p.items_n);
  int* col_token = reinterpret_cast<int*>(ws + p.col_token);
  int* slot_col = reinterpret_cast<int*>(ws + p.slot_col);
  plan_kernel<<<1, 1024, 0, st>>>(ids, t, slots, w13->experts, p.tb1, items, items_n, col_token, slot_col);
  const int64_t items_about = std::min<int64_t>((int64_t)t * slots, w13->experts);
  Args a{};
  fill(a, w13);
  a.items = items;
  a.items_n = items_n;
  a.col_token = col_token;
  a.tb = p.tb1;
  a.x = static_cast<const uint16_t*>(x);
  a.ldx = ldx;
  a.x_vec = aligned16(x, ldx);
  a.out = ws + p.act;
  a.ldo = p.ldact;
  a.mode = GATEUP;
  if (int rc = launch_weight(a, w13, items_about, sms, st)) return rc;
  Args b{};
  fill(b, w2);
  b.items = items;
  b.items_n = items_n;
  b.tb = p.tb1;
  b.x = reinterpret_cast<const uint16_t*>(ws + p.act);
  b.ldx = p.ldact;
  b.x_vec = 1;
  b.out = ws + p.y;
  b.ldo = w2->n;
  b.out_f32 = 1;
  b.mode = DOWN;
  if (int rc = launch_weight(b, w2, items_about, sms, st)) return rc;
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

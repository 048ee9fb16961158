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
// team of kw warps owns a tile and splits its chunks; each warp streams its chunks through its own
// cp.async ring (DEPTH - 1 chunks in flight, across tile and item boundaries), so no barrier stands
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
constexpr int STAGE_BYTES = CHUNK_BYTES + 64 + 32;   // codes, up to two groups' scales, their zero points
constexpr int RED_STRIDE = 20;                       // floats per column of a tile's partial sums (16 + 4: no conflicts)
constexpr int SMEM_LIMIT = 227 * 1024;
constexpr int MAX_EXPERTS = 1024;
enum Mode { LINEAR = 0, GATEUP = 1, DOWN = 2 };

template <int NT>
struct Shape {
  static constexpr int DEPTH = NT <= 2 ? 8 : 4;
  static constexpr int RING = WARPS * DEPTH * STAGE_BYTES;
  static constexpr int RED = WARPS * NT * 8 * RED_STRIDE * 4;
  static constexpr int FIXED = RING + RED;
};

struct Args {
  const uint8_t* codes;
  const uint8_t* scales;
  const uint8_t* zeros;     // or null: 8
  int tiles, chunks, groups, gshift, rows, k;
  int n_items;              // LINEAR: known on the host; else *items_n
  const int* items_n;
  const int4* items;        // {expert, first column, columns, 0}
  const int* col_token;     // GATEUP: the token of a column
  int t, tb;                // LINEAR: tokens, tokens per item
  int kw;                   // warps per team
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

// the item's activations in the MMA's order: [K / 32][columns][4] 16-byte vectors
template <int MODE>
__device__ __forceinline__ void stage_x(const Args& a, uint4* xs, int start, int count) {
  const int nv = a.chunks * 8;
  for (int i = threadIdx.x; i < count * nv; i += THREADS) {
    const int col = i / nv, v = i - col * nv;
    const int row = MODE == GATEUP ? a.col_token[start + col] : start + col;
    const uint16_t* src = a.x + (int64_t)row * a.ldx + 8 * v;
    uint4 d;
    if (a.x_vec && 8 * v + 8 <= a.k) {
      d = *reinterpret_cast<const uint4*>(src);
    } else {
      uint32_t h[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) h[j] = 8 * v + j < a.k ? (uint32_t)src[j] : 0u;
      d = make_uint4(h[0] | h[1] << 16, h[2] | h[3] << 16, h[4] | h[5] << 16, h[6] | h[7] << 16);
    }
    xs[((v >> 2) * count + col) * 4 + (v & 3)] = d;
  }
}

template <class D, int NT, bool HALF, int MODE>
__global__ void __launch_bounds__(THREADS, 1) w4_kernel(const Args a) {
  constexpr int DEPTH = Shape<NT>::DEPTH;
  extern __shared__ __align__(16) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  uint8_t* ring = smem + warp * (DEPTH * STAGE_BYTES);
  float* red = reinterpret_cast<float*>(smem + Shape<NT>::RING);
  uint4* xs = reinterpret_cast<uint4*>(smem + Shape<NT>::FIXED);
  const uint32_t ring_s = (uint32_t)__cvta_generic_to_shared(ring);

  const int n_items = MODE == LINEAR ? a.n_items : *a.items_n;
  const int64_t total = (int64_t)n_items * a.tiles;
  const int64_t lo = total * blockIdx.x / gridDim.x, hi = total * (blockIdx.x + 1) / gridDim.x;
  const int kw = a.kw, teams = WARPS / kw, team = warp / kw, part = warp - team * kw;

  // the copy cursor: the team's tiles of each segment (the part of the range within one item)
  int64_t c_f, c_end;
  int c_chunk = part;
  const uint8_t *c_codes = nullptr, *c_scales = nullptr, *c_zeros = nullptr;
  auto at_segment = [&](int64_t from) {
    const int item = (int)(from / a.tiles);
    c_end = min(hi, (int64_t)(item + 1) * a.tiles);
    c_f = from + team;
    const int64_t e = MODE == LINEAR ? 0 : a.items[item].x;
    // base so that tile f - item * tiles is at f
    const int64_t tile0 = (e - item) * a.tiles;
    c_codes = a.codes + tile0 * a.chunks * CHUNK_BYTES;
    c_scales = a.scales + tile0 * a.groups * 32;
    c_zeros = a.zeros ? a.zeros + tile0 * a.groups * 16 : nullptr;
  };
  bool more = lo < hi && part < a.chunks;
  if (more) {
    at_segment(lo);
    while (c_f >= c_end && c_end < hi) at_segment(c_end);
    more = c_f < c_end;
  }
  auto issue = [&](int slot) {
    if (more) {
      const uint32_t dst = ring_s + slot * STAGE_BYTES;
      cp16(dst + lane * 16, c_codes + (c_f * a.chunks + c_chunk) * CHUNK_BYTES + lane * 16);
      const int64_t grp = c_f * a.groups + ((c_chunk * CHUNK_K) >> a.gshift);
      if (lane < (HALF ? 16 : 8))
        cp4(dst + CHUNK_BYTES + lane * 4, c_scales + grp * 32 + lane * 4);
      else if (a.zeros && lane >= 16 && lane < (HALF ? 24 : 20))
        cp4(dst + CHUNK_BYTES + 64 + (lane - 16) * 4, c_zeros + grp * 16 + (lane - 16) * 4);
      c_chunk += kw;
      if (c_chunk >= a.chunks) {
        c_chunk = part;
        c_f += teams;
        while (c_f >= c_end && c_end < hi) at_segment(c_end);
        more = c_f < c_end;
      }
    }
    cp_commit();
  };
#pragma unroll
  for (int s = 0; s < DEPTH - 1; ++s) issue(s);

  int slot = 0;
  for (int64_t seg = lo; seg < hi;) {
    const int item = (int)(seg / a.tiles);
    const int64_t seg_end = min(hi, (int64_t)(item + 1) * a.tiles);
    int start, count;
    if (MODE == LINEAR) {
      start = item * a.tb;
      count = min(a.tb, a.t - start);
    } else {
      const int4 it = a.items[item];
      start = it.y;
      count = it.z;
    }
    __syncthreads();   // every warp is done with the last item's activations
    stage_x<MODE>(a, xs, start, count);
    __syncthreads();
    for (int64_t f = seg + team; f < seg_end; f += teams) {
      float tot[NT][4], acc[NT][4];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) tot[n][i] = acc[n][i] = 0.0f;
      for (int c = part; c < a.chunks; c += kw) {
        cp_wait<DEPTH - 2>();
        __syncwarp();
        const uint8_t* st = ring + slot * STAGE_BYTES;
        const uint4 w = *reinterpret_cast<const uint4*>(st + lane * 16);
        uint32_t sc[HALF ? 2 : 1], z0[HALF ? 2 : 1], z1[HALF ? 2 : 1];
#pragma unroll
        for (int h = 0; h < (HALF ? 2 : 1); ++h) {
          sc[h] = *reinterpret_cast<const uint32_t*>(st + CHUNK_BYTES + h * 32 + g * 4);
          const uint32_t z = a.zeros ? *reinterpret_cast<const uint16_t*>(st + CHUNK_BYTES + 64 + h * 16 + g * 2) : 0x0808u;
          z0[h] = (z & 0xFFu) * 0x00010001u | D::MAGIC;
          z1[h] = (z >> 8) * 0x00010001u | D::MAGIC;
        }
        issue(slot == 0 ? DEPTH - 1 : slot - 1);
        slot = slot == DEPTH - 1 ? 0 : slot + 1;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint4 xb[NT];
#pragma unroll
          for (int n = 0; n < NT; ++n)
            xb[n] = n * 8 + g < count ? xs[((2 * c + h) * count + n * 8 + g) * 4 + t] : make_uint4(0, 0, 0, 0);
          half_chunk<D, NT>(h ? w.z : w.x, h ? w.w : w.y, z0[HALF ? h : 0], z1[HALF ? h : 0], xb, acc);
          if (HALF || h == 1) fold<D, NT>(sc[HALF ? h : 0], acc, tot);
        }
      }
      // the team's partial sums, [column][row], added in warp order
      float* mine = red + warp * (NT * 8 * RED_STRIDE);
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) mine[(n * 8 + 2 * t + (i & 1)) * RED_STRIDE + g + (i >> 1) * 8] = tot[n][i];
      team_sync(team, kw);
      const float* theirs = red + team * kw * (NT * 8 * RED_STRIDE);
      const int row0 = (int)(f - (int64_t)item * a.tiles) * TILE_ROWS, me = part * 32 + lane;
      if (MODE == GATEUP) {   // tile rows 0..7 are gate rows, 8..15 their up rows
        for (int i = me; i < count * 8; i += kw * 32) {
          const int col = i >> 3, r = i & 7, j = row0 / 2 + r;
          float gt = 0.0f, up = 0.0f;
          for (int w = 0; w < kw; ++w) {
            gt += theirs[w * (NT * 8 * RED_STRIDE) + col * RED_STRIDE + r];
            up += theirs[w * (NT * 8 * RED_STRIDE) + col * RED_STRIDE + r + 8];
          }
          // rounded to the activations' type: the down projection's tensor-core operand
          if (j < a.rows / 2)
            static_cast<uint16_t*>(a.out)[(int64_t)(start + col) * a.ldo + j] =
                D::round(__fdiv_rn(gt, 1.0f + expf(-gt)) * up);
        }
      } else {
        for (int i = me; i < count * 16; i += kw * 32) {
          const int col = i >> 4, r = i & 15, n = row0 + r;
          if (n >= a.rows) continue;
          float v = 0.0f;
          for (int w = 0; w < kw; ++w) v += theirs[w * (NT * 8 * RED_STRIDE) + col * RED_STRIDE + r];
          const int64_t o = (int64_t)(start + col) * a.ldo + n;
          if (MODE == LINEAR && a.residual) v += D::one_to_f32(a.residual[(int64_t)(start + col) * a.ldr + n]);
          if (MODE == DOWN || a.out_f32) static_cast<float*>(a.out)[o] = v;
          else static_cast<uint16_t*>(a.out)[o] = D::round(v);
        }
      }
      team_sync(team, kw);   // the sums are read before the next tile's are written
    }
    seg = seg_end;
  }
  cp_wait<0>();
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

int gshift_of(int group) { return group == 32 ? 5 : group == 64 ? 6 : group == 128 ? 7 : -1; }

const char* bad_weight(const MkW4* w) {
  if (!w || !w->codes || !w->scales) return "null 4-bit weight";
  if (w->n < 1 || w->k < 1 || w->experts < 1) return "a 4-bit weight has at least one row, value and expert";
  if (gshift_of(w->group) < 0) return "the group size is 32, 64 or 128";
  if (w->dtype != MK_W4_BF16 && w->dtype != MK_W4_FP16) return "the activations are BF16 or FP16";
  if (((uintptr_t)w->codes & 15) || ((uintptr_t)w->scales & 3) || ((uintptr_t)w->zeros & 3))
    return "laid-out codes start at a 16-byte boundary, scales and zeros at a 4-byte one";
  return nullptr;
}

void fill(Args& a, const MkW4* w) {
  a.codes = static_cast<const uint8_t*>(w->codes);
  a.scales = static_cast<const uint8_t*>(w->scales);
  a.zeros = static_cast<const uint8_t*>(w->zeros);
  a.tiles = (w->n + TILE_ROWS - 1) / TILE_ROWS;
  a.chunks = (w->k + CHUNK_K - 1) / CHUNK_K;
  a.gshift = gshift_of(w->group);
  a.groups = (a.chunks * CHUNK_K + w->group - 1) >> a.gshift;
  a.rows = w->n;
  a.k = w->k;
}

// columns of K values that fit beside the ring (at most 32): 128 bytes per column and chunk
int columns_that_fit(int chunks, int want) {
  const int per = chunks * CHUNK_K * 2;
  for (int nt = want <= 8 ? 1 : want <= 16 ? 2 : 4;; nt /= 2) {
    const int fixed = nt == 1 ? Shape<1>::FIXED : nt == 2 ? Shape<2>::FIXED : Shape<4>::FIXED;
    const int fit = std::min({(SMEM_LIMIT - fixed) / per, nt * 8, want});
    if (fit > nt * 4 || nt == 1) return fit;
  }
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

template <class D, int NT, bool HALF, int MODE>
int launch(const Args& a, int grid, cudaStream_t s) {
  const int smem = Shape<NT>::FIXED + a.tb * a.chunks * CHUNK_K * 2;
  cudaError_t e = cudaFuncSetAttribute(w4_kernel<D, NT, HALF, MODE>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_LIMIT);
  if (e == cudaSuccess) {
    w4_kernel<D, NT, HALF, MODE><<<grid, THREADS, smem, s>>>(a);
    e = cudaGetLastError();
  }
  return e == cudaSuccess ? MK_OK : fail(MK_ECUDA, cudaGetErrorString(e));
}

template <int MODE>
int launch_mode(const Args& a, int dtype, int grid, cudaStream_t s) {
  const int nt = a.tb <= 8 ? 1 : a.tb <= 16 ? 2 : 4;
  const bool half = a.gshift == 5;
#define W4_CASE(D, NT, HALF) return launch<D, NT, HALF, MODE>(a, grid, s)
#define W4_NT(D, HALF)                     \
  if (nt == 1) W4_CASE(D, 1, HALF);        \
  else if (nt == 2) W4_CASE(D, 2, HALF);   \
  else W4_CASE(D, 4, HALF)
  if (dtype == MK_W4_BF16) {
    if (half) { W4_NT(Bf16, true); } else { W4_NT(Bf16, false); }
  } else {
    if (half) { W4_NT(Fp16, true); } else { W4_NT(Fp16, false); }
  }
#undef W4_NT
#undef W4_CASE
}

// warps per tile: few tiles are split over many warps, many are left to few
int team_warps(int64_t tiles, int chunks, int grid) {
  int kw = 16;
  while (kw > 1 && (kw > chunks || tiles > (int64_t)grid * (WARPS / kw) * 4)) kw /= 2;
  return kw;
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
  if (t < 0 || s < 0 || t * s >= (1 << 24)) return "slots (tokens x slots per token) are from 0 to 2^24 - 1";
  const int want = t >= 32 ? 32 : (int)std::max<int64_t>(t, 1);
  p->tb1 = columns_that_fit((w13->k + CHUNK_K - 1) / CHUNK_K, want);
  p->tb2 = columns_that_fit((w2->k + CHUNK_K - 1) / CHUNK_K, want);
  if (p->tb1 < 1 || p->tb2 < 1) return "rows are too long for the shared memory";
  p->tb1 = p->tb2 = std::min(p->tb1, p->tb2);
  p->ldact = (w2->k + 7) / 8 * 8;
  const int64_t n = std::max<int64_t>(t * s, 1);
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
  a.tb = columns_that_fit(a.chunks, std::min(t, 32));
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
  const int64_t total = (int64_t)a.n_items * a.tiles;
  const int grid = (int)std::min<int64_t>(sms, total);
  a.kw = team_warps(total, a.chunks, grid);
  return launch_mode<LINEAR>(a, w->dtype, grid, static_cast<cudaStream_t>(stream));
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
  a.kw = team_warps(items_about * a.tiles, a.chunks, sms);
  if (int rc = launch_mode<GATEUP>(a, w13->dtype, sms, st)) return rc;
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
  b.kw = team_warps(items_about * b.tiles, b.chunks, sms);
  if (int rc = launch_mode<DOWN>(b, w2->dtype, sms, st)) return rc;
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

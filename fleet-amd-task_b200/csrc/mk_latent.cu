// mk_latent.cu -- the latent cache in 8 bits written and read back: mk_latent_append, mk_latent_read. The format
// is in mk_latent.cuh, the attention over it in mk_latent_attend.cu.
//
// append: a block takes one page that some sequence's new tokens are in, so the page's scales have one writer. It
// finds the largest finite |x| of the new tokens' latents and rotary keys, sets the scales (anew if the page's
// first token is among them, else they only grow), rounds the page's earlier codes to a scale that grew, and
// writes the new codes: one rounding to E4M3, x / scale being exact. What is not finite becomes NaN and
// does not count for the scale; |x| beyond 448 2^32 saturates.
//
// All of a page's new values are loaded at once and kept in registers (16 bytes a load, 18 loads a thread at most), so they
// are read once, and their loads do not wait for one another. 8192 tokens of 576 values (14 MB): 7.2 us on B200, 64 of as many
// sequences 2.3, most of it the chain lengths, table, scales, codes.
//
// read: code x scale of each row, rounded once (exact in BF16): a warp resolves the places of the block's 16 rows (of 32 rows:
// 12.5 us for 16384 tokens where 16 took 10.3), then each thread widens 8 codes at a time, so that a warp's stores lie side by
// side: 9.2 us for 16384 tokens (28 MB).
#include "mk_latent.cuh"

namespace latent {
namespace {

constexpr int THREADS = 512, READERS = 256, READ_ROWS = 16;

// 8 values of a row, to 16-byte aligned memory or one by one
template <typename T>
__device__ __forceinline__ void store8(T* p, bool wide, const float (&v)[8]) {
  union { uint4 u; T t[8]; } r;
#pragma unroll
  for (int i = 0; i < 8; ++i) r.t[i] = from_f32<T>(v[i]);
  if (wide) {
    *reinterpret_cast<uint4*>(p) = r.u;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = r.t[i];
  }
}

__device__ __forceinline__ float finite_abs(float v) {
  const float a = fabsf(v);
  return a < __int_as_float(0x7F800000) ? a : 0.0f;
}

// the smallest power of two, from 2^-32 to 2^32, with amax <= 448 of it (448 = 1.75 x 2^8)
__device__ __forceinline__ float scale_of(float amax) {
  const uint32_t u = __float_as_uint(amax);
  int e = (int)(u >> 23) - 127 - 8 + ((u & 0x7FFFFFu) > 0x600000u ? 1 : 0);
  e = min(max(e, -32), 32);
  return __uint_as_float((uint32_t)(e + 127) << 23);
}

struct Write {
  Cache k;
  Batch b;
  const void *x[2];       // latents, rotary keys
  int64_t ld[2];
  int wide[2];
  Div by_c, by_r;         // eights of a token's latents, of its rotary keys
};

// the pages that a sequence's new tokens are in: [first, first + count)
__device__ __forceinline__ int pages_of(const Cache& k, const Batch& b, const Seq& q, int& first) {
  const int lo = max(q.len - q.n, 0), hi = min(q.len, b.capacity);
  first = lo >> k.shift;
  return hi > lo ? ((hi - 1) >> k.shift) - first + 1 : 0;
}

template <typename T> struct Pair;
template <> struct Pair<__nv_bfloat16> { using type = __nv_bfloat162; };
template <> struct Pair<__half> { using type = __half2; };

// LOADS: eights of values that a thread holds, enough for a page's
template <typename T, int LOADS>
__global__ void __launch_bounds__(THREADS) append_kernel(const Write a) {
  __shared__ uint32_t most[2][THREADS / 32];
  const Cache& k = a.k;
  start_dependents();
  wait_predecessor();
  int s = blockIdx.x, first;
  int nth = 0;
  if (a.b.starts)
    locate<THREADS>(a.b.n, [&](int i) { int f; return pages_of(k, a.b, sequence(a.b, i), f); },
                    [](int) { return (int)blockIdx.x; }, s, nth);
  if (s >= a.b.n) return;
  const Seq q = sequence(a.b, s);
  if (nth >= pages_of(k, a.b, q, first)) return;
  const int j = first + nth, p = a.b.table[s * a.b.ldt + j];
  // the page's new tokens [lo, hi), offsets in the page; its first new token is row `row`
  const int begin = max(q.len - q.n, 0), lo = max(begin - (j << k.shift), 0);
  const int hi = min(min(q.len, a.b.capacity) - (j << k.shift), k.page), m = hi - lo;
  const int row = q.row + ((j << k.shift) + lo) - (q.len - q.n);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // an item is 8 values: all tokens' latents, then their rotary keys
  const int c_eights = k.d_c / 8, r_eights = k.d_r / 8, latents = m * c_eights, items = latents + m * r_eights;
  const auto part_of = [&](int i) { return i >= latents; };
  const auto place_of = [&](int i, int& token, int& at) {
    const int part = part_of(i), e = part ? i - latents : i;
    token = part ? e / a.by_r : e / a.by_c;
    at = (e - token * (part ? r_eights : c_eights)) * 8;
  };
  using T2 = typename Pair<T>::type;
  union Eight { uint4 u; T t[8]; T2 pair[4]; } v[LOADS];
#pragma unroll
  for (int l = 0; l < LOADS; ++l) {
    const int i = threadIdx.x + l * THREADS;
    v[l].u = make_uint4(0, 0, 0, 0);
    if (i < items) {
      int token, at;
      place_of(i, token, at);
      const int part = part_of(i);
      const T* x = static_cast<const T*>(a.x[part]) + (row + token) * a.ld[part] + at;
      if (a.wide[part]) {
        v[l].u = *reinterpret_cast<const uint4*>(x);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[l].t[e] = x[e];
      }
    }
  }
  if (p < 0 || p >= k.pages) return;
  float2 old = make_float2(0.0f, 0.0f);
  if (lo > 0) old = *reinterpret_cast<const float2*>(k.scales + 2 * (int64_t)p);
  // the largest |x| as bits, whose order that of numbers above 0 is, NaN's above infinity's; only where something is not finite
  // the finite values' apart
  const auto largest = [&](bool finite, uint32_t (&out)[2]) {
    uint32_t top[2] = {0, 0};
#pragma unroll
    for (int l = 0; l < LOADS; ++l) {
      if (threadIdx.x + l * THREADS >= items) break;
      uint32_t big;
      if (finite) {
        float m = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) m = fmaxf(m, finite_abs(to_f32(v[l].t[e])));
        big = __float_as_uint(m);
      } else {
        const auto m = __hmax2_nan(__hmax2_nan(__habs2(v[l].pair[0]), __habs2(v[l].pair[1])), __hmax2_nan(__habs2(v[l].pair[2]), __habs2(v[l].pair[3])));
        big = __float_as_uint(to_f32(__hmax_nan(m.x, m.y)));
      }
      const int part = part_of(threadIdx.x + l * THREADS);
      top[0] = part ? top[0] : max(top[0], big);
      top[1] = part ? max(top[1], big) : top[1];
    }
#pragma unroll
    for (int part = 0; part < 2; ++part) {
      top[part] = __reduce_max_sync(0xFFFFFFFFu, top[part]);
      if (lane == 0) most[part][warp] = top[part];
    }
    __syncthreads();            // (and every thread has the old scales)
#pragma unroll
    for (int part = 0; part < 2; ++part) {
      out[part] = 0;
#pragma unroll
      for (int w = 0; w < THREADS / 32; ++w) out[part] = max(out[part], most[part][w]);
    }
  };
  constexpr uint32_t INF = 0x7F800000u;
  uint32_t top[2];
  largest(false, top);
  const bool odd = top[0] >= INF || top[1] >= INF;
  if (odd) {
    __syncthreads();
    largest(true, top);
  }
  float scale[2], inv[2];
#pragma unroll
  for (int part = 0; part < 2; ++part) {
    const float was = part ? old.y : old.x;
    scale[part] = scale_of(__uint_as_float(top[part]));
    if (lo > 0) scale[part] = fmaxf(scale[part], was);
    inv[part] = 1.0f / scale[part];
    const int ld = part ? LD_R : k.ld_c, eights = part ? r_eights : c_eights;
    uint8_t* codes = (part ? k.r : k.c) + ((int64_t)p << k.shift) * ld;
    if (lo > 0 && scale[part] != was) {
      const float ratio = was / scale[part];
      for (int i = threadIdx.x; i < lo * eights; i += THREADS) {
        const int token = i / eights;
        uint16_t* at = reinterpret_cast<uint16_t*>(codes + token * ld + (i - token * eights) * 8);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 f = decode2(at[e]);
          at[e] = encode2(f.x * ratio, f.y * ratio);
        }
      }
    }
  }
  if (threadIdx.x == 0) *reinterpret_cast<float2*>(k.scales + 2 * (int64_t)p) = make_float2(scale[0], scale[1]);
  const float nan = __int_as_float(0x7FC00000);
#pragma unroll
  for (int l = 0; l < LOADS; ++l) {
    const int i = threadIdx.x + l * THREADS;
    if (i >= items) break;
    int token, at;
    place_of(i, token, at);
    const int part = part_of(i);
    const float by = part ? inv[1] : inv[0];
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      x[e] = to_f32(v[l].t[e]);
      x[e] = odd && !isfinite(x[e]) ? nan : x[e] * by;
    }
    uint8_t* codes = part ? k.r + (((int64_t)p << k.shift) + lo + token) * LD_R : k.c + (((int64_t)p << k.shift) + lo + token) * k.ld_c;
    *reinterpret_cast<uint2*>(codes + at) = make_uint2(encode2(x[0], x[1]) | (uint32_t)encode2(x[2], x[3]) << 16,
                                                       encode2(x[4], x[5]) | (uint32_t)encode2(x[6], x[7]) << 16);
  }
}

struct Read {
  Cache k;
  Batch b;
  void* out[2];
  int64_t ld[2];
  int wide[2], fill;      // fill: rows of no sequence become zeros
  Div by_each;            // the items of a row
};

template <typename T>
__global__ void __launch_bounds__(READERS) read_kernel(const Read a) {
  __shared__ int64_t token_of[READ_ROWS];               // a row's token in the cache, -1: in none, -2: the row is left alone
  __shared__ int page_of[READ_ROWS];
  __shared__ int begun;
  const Cache& k = a.k;
  start_dependents();
  wait_predecessor();
  const int first = blockIdx.x * READ_ROWS, rows = min(READ_ROWS, a.b.rows - first);
  const bool few = a.b.n <= 32;
  if (a.b.starts && !few) {     // the sequences that start at or before the block's first row: all threads count them
    if (threadIdx.x == 0) begun = 0;
    __syncthreads();
    int mine = 0;
    for (int i = threadIdx.x; i < a.b.n; i += READERS) mine += a.b.starts[i] <= first;
    mine = __reduce_add_sync(0xFFFFFFFFu, mine);
    if (threadIdx.x % 32 == 0 && mine > 0) atomicAdd(&begun, mine);
    __syncthreads();
  }
  if (threadIdx.x < 32) {       // a lane for each row
    const int lane = threadIdx.x, row = first + lane;
    int s = row;
    Seq q{0, 0, 0};
    if (a.b.starts && few) {    // a lane for each sequence too: the last that starts at or before the row, by halves
      const int start = lane < a.b.n ? a.b.starts[lane] : INT32_MAX;
      const Seq held = lane < a.b.n ? sequence(a.b, lane) : q;
      s = -1;
#pragma unroll
      for (int step = 32; step >= 1; step /= 2) {
        const int next = s + step, there = __shfl_sync(0xFFFFFFFFu, start, min(next, 31));
        if (next < a.b.n && there <= row) s = next;
      }
      q.row = __shfl_sync(0xFFFFFFFFu, held.row, max(s, 0));
      q.n = __shfl_sync(0xFFFFFFFFu, held.n, max(s, 0));
      q.len = __shfl_sync(0xFFFFFFFFu, held.len, max(s, 0));
    } else {
      if (a.b.starts)
        for (s = begun - 1; s + 1 < a.b.n && a.b.starts[s + 1] <= row;) ++s;
      if (lane < rows && s >= 0 && s < a.b.n) q = sequence(a.b, s);
    }
    int64_t token = a.fill ? -1 : -2;
    int p = -1;
    if (lane < rows && s >= 0 && s < a.b.n && row >= q.row && row < q.row + q.n) {
      const int pos = q.len - q.n + (row - q.row);
      token = -1;
      if (pos >= 0 && pos < a.b.capacity) {
        p = a.b.table[s * a.b.ldt + (pos >> k.shift)];
        if (p >= 0 && p < k.pages) token = ((int64_t)p << k.shift) + (pos & (k.page - 1));
      }
    }
    if (lane < rows) {
      token_of[lane] = token;
      page_of[lane] = p;
    }
  }
  __syncthreads();
  // an item is 8 codes, so that a warp's stores lie side by side; all of a thread's are loaded before the first is stored
  constexpr int ITEMS = (READ_ROWS * (MAX_DC + LD_R) / 8 + READERS - 1) / READERS;
  const int each = a.by_each.d, c_items = k.d_c / 8;
  uint2 codes[ITEMS];
  float scales[ITEMS];
#pragma unroll
  for (int l = 0; l < ITEMS; ++l) {
    const int i = threadIdx.x + l * READERS, r = i / a.by_each, item = i - r * each, part = item >= c_items, at = (part ? item - c_items : item) * 8;
    codes[l] = make_uint2(0, 0);
    scales[l] = 0.0f;
    if (r < rows && token_of[r] >= 0) {
      codes[l] = *reinterpret_cast<const uint2*>(part ? k.r + token_of[r] * LD_R + at : k.c + token_of[r] * k.ld_c + at);
      scales[l] = k.scales[2 * (int64_t)page_of[r] + part];
    }
  }
#pragma unroll
  for (int l = 0; l < ITEMS; ++l) {
    const int i = threadIdx.x + l * READERS, r = i / a.by_each, item = i - r * each, part = item >= c_items, at = (part ? item - c_items : item) * 8;
    if (r >= rows || token_of[r] == -2) continue;
    const uint32_t u[2] = {codes[l].x, codes[l].y};
    float v[8];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 f = decode2((uint16_t)(u[e / 2] >> (e % 2 * 16)));
      v[2 * e] = f.x * scales[l];
      v[2 * e + 1] = f.y * scales[l];
    }
    store8(static_cast<T*>(a.out[part]) + (first + r) * a.ld[part] + at, a.wide[part], v);
  }
}

int wide(const void* p, int64_t ld) { return (uintptr_t)p % 16 == 0 && ld % 8 == 0; }

}  // namespace
}  // namespace latent

using namespace latent;

extern "C" int mk_latent_append(const MkLatent* l, const MkLatentBatch* b, const void* c, int64_t ldc, const void* r, int64_t ldr,
                                int32_t rows, int32_t dtype, void* stream) {
  Write a{};
  if (const int e = check(l, b, rows, dtype, a.k, a.b)) return e;
  if (rows == 0 || b->n == 0) return MK_OK;
  if (!c || !r) return fail(MK_EINVAL, "null pointer");
  if (((uintptr_t)c | (uintptr_t)r) & 1) return fail(MK_EINVAL, "misaligned values");
  a.x[0] = c;
  a.x[1] = r;
  a.ld[0] = ldc;
  a.ld[1] = ldr;
  a.wide[0] = wide(c, ldc);
  a.wide[1] = wide(r, ldr);
  a.by_c = div_by(l->d_c / 8);
  a.by_r = div_by(l->d_r / 8);
  // a sequence's rows are in at most rows / page + 2 pages, and in no more pages than rows
  const int64_t most = b->starts ? rows / l->page + 2 * (int64_t)b->n : rows;
  const unsigned grid = (unsigned)(most < rows ? most : rows);
  // a page's eights of values over the threads (without starts a page gets one token)
  const int64_t held = !b->starts ? 1 : l->page < rows ? l->page : rows, eights = held * ((l->d_c + l->d_r) / 8);
  const auto s = static_cast<cudaStream_t>(stream);
  const auto launch = [&](auto kernel) { return launch_early(kernel, dim3(grid), THREADS, 0, s, a); };
  cudaError_t e;
  if (eights <= THREADS) e = dtype == MK_BF16 ? launch(append_kernel<__nv_bfloat16, 1>) : launch(append_kernel<__half, 1>);
  else if (eights <= 9 * THREADS) e = dtype == MK_BF16 ? launch(append_kernel<__nv_bfloat16, 9>) : launch(append_kernel<__half, 9>);
  else e = dtype == MK_BF16 ? launch(append_kernel<__nv_bfloat16, 18>) : launch(append_kernel<__half, 18>);
  return e == cudaSuccess ? MK_OK : fail(MK_ECUDA, cudaGetErrorString(e));
}

extern "C" int mk_latent_read(const MkLatent* l, const MkLatentBatch* b, void* c, int64_t ldc, void* r, int64_t ldr, int32_t rows,
                              int32_t dtype, int32_t fill, void* stream) {
  Read a{};
  if (const int e = check(l, b, rows, dtype, a.k, a.b)) return e;
  if (rows == 0 || (b->n == 0 && !fill)) return MK_OK;
  if (!c || !r) return fail(MK_EINVAL, "null pointer");
  if (((uintptr_t)c | (uintptr_t)r) & 1) return fail(MK_EINVAL, "misaligned values");
  a.out[0] = c;
  a.out[1] = r;
  a.ld[0] = ldc;
  a.ld[1] = ldr;
  a.wide[0] = wide(c, ldc);
  a.wide[1] = wide(r, ldr);
  a.fill = fill != 0;
  a.by_each = div_by((l->d_c + l->d_r) / 8);
  const unsigned grid = ((unsigned)rows + READ_ROWS - 1) / READ_ROWS;
  const cudaError_t e = launch_early(dtype == MK_BF16 ? read_kernel<__nv_bfloat16> : read_kernel<__half>, dim3(grid), READERS, 0,
                                     static_cast<cudaStream_t>(stream), a);
  return e == cudaSuccess ? MK_OK : fail(MK_ECUDA, cudaGetErrorString(e));
}

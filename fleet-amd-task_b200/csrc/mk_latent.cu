// mk_latent.cu -- the latent cache in 8 bits written and read back: mk_latent_append, mk_latent_read. The format
// is in mk_latent.cuh, the attention over it in mk_latent_attend.cu.
//
// append: a block takes one page that some sequence's new tokens are in, so the page's scales have one writer. It
// finds the largest finite |x| of the new tokens' latents and rotary keys, sets the scales (anew if the page's
// first token is among them, else they only grow), rounds the page's earlier codes to a scale that grew, and
// writes the new codes: one rounding to E4M3, x / scale being exact. What is not finite becomes NaN and
// does not count for the scale; |x| beyond 448 2^32 saturates.
//
// read: code x scale of each row, rounded once (exact in BF16).
#include "mk_latent.cuh"

namespace latent {
namespace {

constexpr int THREADS = 256;

// 8 values of a row, from 16-byte aligned memory or one by one
template <typename T>
__device__ __forceinline__ void load8(const T* p, bool wide, float (&v)[8]) {
  union { uint4 u; T t[8]; } r;
  if (wide) {
    r.u = *reinterpret_cast<const uint4*>(p);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) r.t[i] = p[i];
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = to_f32(r.t[i]);
}

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
};

// the pages that a sequence's new tokens are in: [first, first + count)
__device__ __forceinline__ int pages_of(const Cache& k, const Batch& b, const Seq& q, int& first) {
  const int lo = max(q.len - q.n, 0), hi = min(q.len, b.capacity);
  first = lo >> k.shift;
  return hi > lo ? ((hi - 1) >> k.shift) - first + 1 : 0;
}

template <typename T>
__global__ void __launch_bounds__(THREADS) append_kernel(const Write a) {
  __shared__ float most[2][THREADS / 32];
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
  const int j = first + nth;
  const int p = a.b.table[s * a.b.ldt + j];
  if (p < 0 || p >= k.pages) return;
  // the page's new tokens [lo, hi), offsets in the page; its first new token is row `row`
  const int begin = max(q.len - q.n, 0), lo = max(begin - (j << k.shift), 0);
  const int hi = min(min(q.len, a.b.capacity) - (j << k.shift), k.page), m = hi - lo;
  const int row = q.row + ((j << k.shift) + lo) - (q.len - q.n);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
  for (int part = 0; part < 2; ++part) {
    const int chunks = (part ? k.d_r : k.d_c) / 8;
    const T* x = static_cast<const T*>(a.x[part]) + row * a.ld[part];
    float amax = 0.0f;
    for (int i = threadIdx.x; i < m * chunks; i += THREADS) {
      float v[8];
      load8(x + (i / chunks) * a.ld[part] + i % chunks * 8, a.wide[part], v);
#pragma unroll
      for (int e = 0; e < 8; ++e) amax = fmaxf(amax, finite_abs(v[e]));
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, o));
    if (lane == 0) most[part][warp] = amax;
  }
  const float old[2] = {k.scales[2 * (int64_t)p], k.scales[2 * (int64_t)p + 1]};
  __syncthreads();
#pragma unroll
  for (int part = 0; part < 2; ++part) {
    float amax = 0.0f;
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) amax = fmaxf(amax, most[part][w]);
    float scale = scale_of(amax);
    if (lo > 0) scale = fmaxf(scale, old[part]);
    const int d = part ? k.d_r : k.d_c, ld = part ? LD_R : k.ld_c, chunks = d / 8;
    uint8_t* codes = (part ? k.r : k.c) + ((int64_t)p << k.shift) * ld;
    if (lo > 0 && scale != old[part]) {
      const float ratio = old[part] / scale;
      for (int i = threadIdx.x; i < lo * chunks; i += THREADS) {
        uint16_t* at = reinterpret_cast<uint16_t*>(codes + (i / chunks) * ld + i % chunks * 8);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 v = decode2(at[e]);
          at[e] = encode2(v.x * ratio, v.y * ratio);
        }
      }
    }
    const T* x = static_cast<const T*>(a.x[part]) + row * a.ld[part];
    const float inv = 1.0f / scale, nan = __int_as_float(0x7FC00000);
    for (int i = threadIdx.x; i < m * chunks; i += THREADS) {
      float v[8];
      load8(x + (i / chunks) * a.ld[part] + i % chunks * 8, a.wide[part], v);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = isfinite(v[e]) ? v[e] * inv : nan;
      uint2 w;
      w.x = encode2(v[0], v[1]) | (uint32_t)encode2(v[2], v[3]) << 16;
      w.y = encode2(v[4], v[5]) | (uint32_t)encode2(v[6], v[7]) << 16;
      *reinterpret_cast<uint2*>(codes + (lo + i / chunks) * ld + i % chunks * 8) = w;
    }
    if (threadIdx.x == 0) k.scales[2 * (int64_t)p + part] = scale;
  }
}

struct Read {
  Cache k;
  Batch b;
  void* out[2];
  int64_t ld[2];
  int wide[2], fill;      // fill: rows of no sequence become zeros
};

template <typename T>
__global__ void __launch_bounds__(THREADS) read_kernel(const Read a) {
  const Cache& k = a.k;
  start_dependents();
  wait_predecessor();
  const int row = blockIdx.x * (THREADS / 32) + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (row >= a.b.rows) return;
  int s = row;
  if (a.b.starts) {             // the last sequence that starts at or before the row
    int lo = 0, hi = a.b.n;
    while (lo < hi) {
      const int mid = (lo + hi) / 2;
      if (a.b.starts[mid] <= row) lo = mid + 1;
      else hi = mid;
    }
    s = lo - 1;
  }
  int p = -1, off = 0;
  bool mine = false;
  if (s >= 0 && s < a.b.n) {
    const Seq q = sequence(a.b, s);
    mine = row >= q.row && row < q.row + q.n;
    const int pos = q.len - q.n + (row - q.row);
    if (mine && pos >= 0 && pos < a.b.capacity) {
      p = a.b.table[s * a.b.ldt + (pos >> k.shift)];
      off = pos & (k.page - 1);
    }
  }
  if (!mine && !a.fill) return;
  const bool live = p >= 0 && p < k.pages;
#pragma unroll
  for (int part = 0; part < 2; ++part) {
    const int d = part ? k.d_r : k.d_c, ld = part ? LD_R : k.ld_c;
    const uint8_t* codes = (part ? k.r : k.c) + (((int64_t)p << k.shift) + off) * ld;
    const float scale = live ? k.scales[2 * (int64_t)p + part] : 0.0f;
    T* out = static_cast<T*>(a.out[part]) + row * a.ld[part];
    for (int i = lane * 8; i < d; i += 256) {
      float v[8] = {};
      if (live) {
        const uint2 w = *reinterpret_cast<const uint2*>(codes + i);
        const uint32_t u[2] = {w.x, w.y};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 f = decode2((uint16_t)(u[e / 2] >> (e % 2 * 16)));
          v[2 * e] = f.x * scale;
          v[2 * e + 1] = f.y * scale;
        }
      }
      store8(out + i, a.wide[part], v);
    }
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
  // a sequence's rows are in at most rows / page + 2 pages, and in no more pages than rows
  const int64_t most = b->starts ? rows / l->page + 2 * (int64_t)b->n : rows;
  const unsigned grid = (unsigned)(most < rows ? most : rows);
  const cudaError_t e = launch_early(dtype == MK_BF16 ? append_kernel<__nv_bfloat16> : append_kernel<__half>, grid, THREADS, 0,
                                     static_cast<cudaStream_t>(stream), a);
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
  const unsigned grid = ((unsigned)rows + THREADS / 32 - 1) / (THREADS / 32);
  const cudaError_t e = launch_early(dtype == MK_BF16 ? read_kernel<__nv_bfloat16> : read_kernel<__half>, grid, THREADS, 0,
                                     static_cast<cudaStream_t>(stream), a);
  return e == cudaSuccess ? MK_OK : fail(MK_ECUDA, cudaGetErrorString(e));
}

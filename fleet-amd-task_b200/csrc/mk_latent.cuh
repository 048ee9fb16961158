// mk_latent.cuh -- the latent cache in 8 bits: format, and what its kernels share.
//
// A cache is `pages` pages of `page` tokens (16, 32, 64 or 128). A token is d_c latent values (key and value of every
// head) and d_r rotary key values (of every head's key), E4M3 codes in rows of ld_c = d_c rounded up to 128 and
// ld_r = 64 bytes; the bytes behind a row's values are zero and stay so. scales [pages, 2] FP32: a page's
// latents and rotary keys stand for code x scale.
//
// Scales are powers of two, the smallest 2^e with |x| <= 448 2^e for what the page holds, e from -32 to 32: E4M3
// keeps the same relative precision at any scale, so nothing is lost by it, codes x scale are exact in
// BF16, and where a page's scale grows its earlier codes are only shifted (exact down to E4M3's subnormals).
//
// A batch is a table of pages, the sequences' lengths (this step's tokens included) and, if not one row each,
// the starts of their rows. What these arrays hold is not known on the host, so kernels take nothing of it on trust: a
// length below 0 counts as 0, rows are cut to the call's, and a token past the table's width or in a page outside the cache
// is none: it is not written, reads as zeros and is seen by nobody. (The rows' tokens go by the length as given, so of a length
// past the table the last rows have none.) starts ascend; where they do not, sequences share rows and pages, so that results
// are undefined, but no address leaves the call's tensors, and sums over the sequences saturate (plus), so that a call
// does no more than one of its sizes may.
#ifndef MK_LATENT_CUH
#define MK_LATENT_CUH

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "../../include/fleet_mk.h"

namespace mk {
int set_last_error(int code, const char* msg);   // mk_runtime.cu: the message mk_last_error() returns
}

namespace latent {

constexpr int MAX_DC = 512, LD_R = 64, MAX_PAGE = 128;

struct Cache {
  uint8_t *c, *r;
  float* scales;
  int pages, page, shift, d_c, d_r, ld_c;      // page = 1 << shift
};

struct Batch {
  const int32_t *table, *lens, *starts;
  int64_t ldt;
  int n, capacity;                             // capacity: tokens that a table's row can name
  int rows;                                    // the call's rows
};

// One sequence: its rows [row, row + n) of the call are its tokens [len - n, len), len as the caller has it.
struct Seq {
  int row, n, len;
};

__host__ __device__ __forceinline__ Seq sequence(const Batch& b, int s) {
  Seq q;
  q.len = max(b.lens[s], 0);
  if (!b.starts) {
    q.row = s;
    q.n = s < b.rows ? 1 : 0;
  } else {
    q.row = min(max(b.starts[s], 0), b.rows);
    q.n = max(min(max(b.starts[s + 1], 0), b.rows) - q.row, 0);        // (both in [0, rows]: their difference has 32 bits)
  }
  return q;
}

__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

__device__ __forceinline__ float2 decode2(uint16_t codes) {
  return __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(codes, __NV_E4M3)));
}
__device__ __forceinline__ uint16_t encode2(float a, float b) {      // NaN stays NaN, finite values saturate
  return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
}

// The sum of two numbers that are not negative, 2^31 - 1 at most: rows of starts that go down count again and again, and
// their parts may pass that.
__host__ __device__ __forceinline__ int plus(int a, int b) {
  const uint32_t sum = (uint32_t)a + (uint32_t)b;
  return sum < 0x7FFFFFFFu ? (int)sum : 0x7FFFFFFF;
}

// The item (of n with count(i) parts each, at most 2^31 - 1 in all) that holds part which(all parts) of them, and the
// part's place in it; every thread of the block calls it, once. item is n if there is no such part.
template <int THREADS, typename Count, typename Which>
__device__ __forceinline__ void locate(int n, Count count, Which which, int& item, int& place) {
  __shared__ int warps[THREADS / 32], found[2];
  if (n <= 32) {                // every warp by itself, an item a lane
    const int i = threadIdx.x & 31, mine = i < n ? count(i) : 0;
    int upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xFFFFFFFFu, upto, o);
      if (i >= o) upto = plus(upto, v);
    }
    const int at = which(__shfl_sync(0xFFFFFFFFu, upto, 31));
    const uint32_t holds = __ballot_sync(0xFFFFFFFFu, at >= upto - mine && at < upto);
    const int lane = holds ? __ffs(holds) - 1 : 0;
    item = holds ? lane : n;
    place = at - __shfl_sync(0xFFFFFFFFu, upto - mine, lane);
    return;
  }
  const int per = (n + THREADS - 1) / THREADS, lo = min((int)threadIdx.x * per, n), hi = min(lo + per, n);
  int mine = 0;
  for (int i = lo; i < hi; ++i) mine = plus(mine, count(i));
  int upto = mine;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xFFFFFFFFu, upto, o);
    if (lane >= o) upto = plus(upto, v);
  }
  if (threadIdx.x == 0) found[0] = n;
  if (lane == 31) warps[warp] = upto;
  __syncthreads();
  int total = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) {
    if (w < warp) upto = plus(upto, warps[w]);
    total = plus(total, warps[w]);
  }
  const int at = which(total);
  if (at >= upto - mine && at < upto) {
    int left = at - (upto - mine), i = lo;
    for (int c; i < hi - 1 && left >= (c = count(i)); ++i) left -= c;
    found[0] = i;
    found[1] = left;
  }
  __syncthreads();
  item = found[0];
  place = found[1];
}

// Every kernel here is launched so that it may start before its predecessor on the stream has ended, and reads and writes
// nothing before wait_predecessor(); start_dependents() lets its successor do the same.
__device__ __forceinline__ void wait_predecessor() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void start_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
template <typename... P, typename... A>
cudaError_t launch_early(void (*kernel)(P...), dim3 grid, int threads, size_t smem, cudaStream_t s, A... args) {
  cudaLaunchAttribute early[1];
  early[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t c{};
  c.gridDim = grid;
  c.blockDim = dim3(threads);
  c.dynamicSmemBytes = smem;
  c.stream = s;
  c.attrs = early;
  c.numAttrs = 1;
  return cudaLaunchKernelEx(&c, kernel, args...);
}

// Division by a number that the host knows: x / d = (mulhi(x, mul) + x) >> shift for 0 <= x < 2^31.
struct Div {
  uint32_t mul;
  int shift, d;
};
__device__ __forceinline__ int operator/(int x, const Div& d) { return (int)((__umulhi((uint32_t)x, d.mul) + (uint32_t)x) >> d.shift); }
inline Div div_by(int d) {
  Div v{0, 0, d};
  while ((1ll << v.shift) < d) ++v.shift;
  v.mul = (uint32_t)(((1ull << 32) * ((1ull << v.shift) - d)) / d + 1);
  return v;
}

// Places of the attention's work are 1 << coarse units, so many that all groups' together pass 2^31 - 1 for no lengths: a
// call has at most rows x heads / 16 groups and one more for each sequence, of `capacity` tokens in units of 64 and `fixed`
// places more. -1: too many groups for any.
inline int coarse_of(int64_t rows, int64_t heads, int64_t n, int64_t capacity, int fixed) {
  const int64_t groups = rows * heads / 16 + n, units = capacity / 64 + 1;
  for (int coarse = 0; coarse < 31; ++coarse)
    if (groups * ((units >> coarse) + 1 + fixed) <= INT32_MAX) return coarse;
  return -1;
}

inline int fail(int code, const char* msg) { return mk::set_last_error(code, msg); }

// The host's checks of what every call is handed; MK_OK and the kernels' structs, or the error.
inline int check(const MkLatent* l, const MkLatentBatch* b, int32_t rows, int32_t dtype, Cache& cache, Batch& batch) {
  if (!l || !b) return fail(MK_EINVAL, "null cache or batch");
  if (l->page != 16 && l->page != 32 && l->page != 64 && l->page != 128) return fail(MK_EINVAL, "a page holds 16, 32, 64 or 128 tokens");
  if (l->d_c < 8 || l->d_c > MAX_DC || l->d_c % 8 || l->d_r < 8 || l->d_r > LD_R || l->d_r % 8)
    return fail(MK_EINVAL, "d_c is from 8 to 512, d_r from 8 to 64, both multiples of 8");
  if (l->pages < 1 || (int64_t)l->pages * l->page > INT32_MAX) return fail(MK_EINVAL, "a cache holds from 1 page to 2^31 - 1 tokens");
  if (b->n < 0 || b->pages < 1 || (int64_t)b->pages * l->page > 1 << 30 || b->ldt < 0)
    return fail(MK_EINVAL, "a batch has 0 or more sequences of 1 page to 2^30 tokens each");
  if (rows < 0 || (!b->starts && rows != b->n)) return fail(MK_EINVAL, "without starts a batch has one row for each sequence");
  if (dtype != MK_BF16 && dtype != MK_FP16) return fail(MK_EINVAL, "values are BF16 or FP16");
  if (!l->c || !l->r || !l->scales || (b->n && (!b->table || !b->lens))) return fail(MK_EINVAL, "null pointer");
  if (((uintptr_t)l->c | (uintptr_t)l->r) % 128 || (uintptr_t)l->scales % 8 ||
      ((uintptr_t)b->table | (uintptr_t)b->lens | (uintptr_t)b->starts) % 4)
    return fail(MK_EINVAL, "misaligned codes (128 bytes), scales (8), table, lens or starts (4)");
  cache = {static_cast<uint8_t*>(l->c), static_cast<uint8_t*>(l->r), l->scales, l->pages, l->page,
           l->page == 16 ? 4 : l->page == 32 ? 5 : l->page == 64 ? 6 : 7, l->d_c, l->d_r, (l->d_c + 127) / 128 * 128};
  batch = {b->table, b->lens, b->starts, b->ldt, b->n, b->pages * l->page, rows};
  return MK_OK;
}

}  // namespace latent
#endif

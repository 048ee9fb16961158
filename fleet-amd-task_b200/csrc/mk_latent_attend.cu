// mk_latent_attend.cu -- attention over the latent cache in 8 bits: mk_latent_attend. The format is in mk_latent.cuh.
//
// Formulas. Row i of the n of a sequence is its token P = len - n + i; for each head h, with q = (qc, qr),
//   s_j = scale (qc . c_j + qr . r_j), j = 0 .. P;  out = sum_j softmax(s)_j c_j;  lse = log sum_j exp(s_j).
// A row that sees no token (an empty sequence, P < 0, pages outside the cache) gives zeros and lse -inf.
//
// A block takes one (row, head), a warp every fourth token.
#include "mk_latent.cuh"

namespace latent {
namespace {

constexpr int WARPS = 4, PER = MAX_DC / 32;

struct Attend {
  Cache k;
  Batch b;
  const void* q;
  void* out;
  float* lse;
  int64_t qt, qh, ot, oh;
  int heads;
  float scale;
};

template <typename T>
__global__ void __launch_bounds__(WARPS * 32) attend_kernel(const Attend a) {
  __shared__ float part[WARPS][MAX_DC], stat[WARPS][2];
  const Cache& k = a.k;
  const int row = blockIdx.x, h = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int s = row;
  if (a.b.starts) {
    int lo = 0, hi = a.b.n;
    while (lo < hi) {
      const int mid = (lo + hi) / 2;
      if (a.b.starts[mid] <= row) lo = mid + 1;
      else hi = mid;
    }
    s = lo - 1;
  }
  if (s < 0 || s >= a.b.n) return;
  const Seq seq = sequence(a.b, s);
  if (row < seq.row || row >= seq.row + seq.n) return;
  const int sees = min(seq.len - seq.n + (row - seq.row) + 1, a.b.capacity);
  const T* q = static_cast<const T*>(a.q) + row * a.qt + h * a.qh;
  float qc[PER], qr[2], o[PER] = {}, m = -INFINITY, l = 0.0f;
#pragma unroll
  for (int i = 0; i < PER; ++i) qc[i] = lane + 32 * i < k.d_c ? to_f32(q[lane + 32 * i]) : 0.0f;
#pragma unroll
  for (int i = 0; i < 2; ++i) qr[i] = lane + 32 * i < k.d_r ? to_f32(q[k.d_c + lane + 32 * i]) : 0.0f;
  for (int j = warp; j < sees; j += WARPS) {
    const int p = a.b.table[s * a.b.ldt + (j >> k.shift)];
    if (p < 0 || p >= k.pages) continue;
    const int64_t at = ((int64_t)p << k.shift) + (j & (k.page - 1));
    const float sc = k.scales[2 * (int64_t)p], sr = k.scales[2 * (int64_t)p + 1];
    float c[PER], dot = 0.0f;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      c[i] = lane + 32 * i < k.d_c ? decode2(k.c[at * k.ld_c + lane + 32 * i]).x * sc : 0.0f;
      dot += qc[i] * c[i];
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (lane + 32 * i < k.d_r) dot += qr[i] * decode2(k.r[at * LD_R + lane + 32 * i]).x * sr;
#pragma unroll
    for (int e = 16; e > 0; e >>= 1) dot += __shfl_xor_sync(0xFFFFFFFFu, dot, e);
    const float v = dot * a.scale, to = fmaxf(m, isnan(v) ? 0.0f : v);   // (a NaN is the weights', not the largest score's)
    const float was = m == -INFINITY ? 0.0f : expf(m - to), is = expf(v - to);
    m = to;
    l = l * was + is;
#pragma unroll
    for (int i = 0; i < PER; ++i) o[i] = o[i] * was + is * c[i];
  }
#pragma unroll
  for (int i = 0; i < PER; ++i) part[warp][lane + 32 * i] = o[i];
  if (lane == 0) {
    stat[warp][0] = m;
    stat[warp][1] = l;
  }
  __syncthreads();
  float top = -INFINITY, total = 0.0f, w[WARPS];
  for (int i = 0; i < WARPS; ++i) top = fmaxf(top, stat[i][0]);
  for (int i = 0; i < WARPS; ++i) {
    w[i] = stat[i][0] == -INFINITY ? 0.0f : expf(stat[i][0] - top);
    total += w[i] * stat[i][1];
  }
  T* out = static_cast<T*>(a.out) + row * a.ot + h * a.oh;
  for (int c = threadIdx.x; c < k.d_c; c += WARPS * 32) {
    float v = 0.0f;
    for (int i = 0; i < WARPS; ++i) v += w[i] * part[i][c];
    out[c] = from_f32<T>(top == -INFINITY ? 0.0f : v / total);
  }
  if (a.lse && threadIdx.x == 0) a.lse[(int64_t)row * a.heads + h] = top == -INFINITY ? top : top + logf(total);
}

}  // namespace
}  // namespace latent

using namespace latent;

extern "C" int mk_latent_attend_workspace(const MkLatent* l, int32_t n, int32_t rows, int32_t heads, int64_t* bytes) {
  if (!l || !bytes || n < 0 || rows < 0 || heads < 1) return fail(MK_EINVAL, "null pointer or a negative size");
  *bytes = 0;
  return MK_OK;
}

extern "C" int mk_latent_attend(const MkLatent* l, const MkLatentBatch* b, const void* q, int64_t qt, int64_t qh, int32_t rows,
                                int32_t heads, int32_t dtype, float scale, void* out, int64_t ot, int64_t oh, float* lse,
                                void* workspace, int64_t workspace_bytes, void* stream) {
  Attend a{};
  if (const int e = check(l, b, rows, dtype, a.k, a.b)) return e;
  if (heads < 1 || heads > 1024) return fail(MK_EINVAL, "heads are from 1 to 1024");
  if (rows == 0 || b->n == 0) return MK_OK;
  if (!q || !out) return fail(MK_EINVAL, "null pointer");
  if (((uintptr_t)q | (uintptr_t)out) & 1 || (uintptr_t)lse & 3) return fail(MK_EINVAL, "misaligned q, out or lse");
  a.q = q;
  a.out = out;
  a.lse = lse;
  a.qt = qt;
  a.qh = qh;
  a.ot = ot;
  a.oh = oh;
  a.heads = heads;
  a.scale = scale;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)rows, (unsigned)heads);
  cfg.blockDim = dim3(WARPS * 32);
  cfg.stream = static_cast<cudaStream_t>(stream);
  const cudaError_t e = dtype == MK_BF16 ? cudaLaunchKernelEx(&cfg, attend_kernel<__nv_bfloat16>, a)
                                          : cudaLaunchKernelEx(&cfg, attend_kernel<__half>, a);
  return e == cudaSuccess ? MK_OK : fail(MK_ECUDA, cudaGetErrorString(e));
}

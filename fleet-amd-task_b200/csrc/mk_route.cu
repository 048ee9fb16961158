// mk_route.cu -- routing of a batch of tokens to experts: mk_route.
//
// Formulas, per token with logits l[0..E): scores s = softmax(l) or 1 / (1 + exp(-l)); the order is by
// c = s + bias, without a bias by s (a softmax's numerators exp(l - max), which the division would
// only round together). With n_group > 1 the experts form equal consecutive groups; a group's score
// is its largest c or the sum of its two largest; the topk_group best groups stay. ids are the topk
// largest c among them in descending order, ties to the lowest index (of groups too); weights are
// s[ids], divided by their sum if asked (0 if the sum is 0), times the scaling. n_forced experts
// E, E + 1, ... with weight 1 follow each token's topk. A logit of -inf scores 0; a NaN counts as
// -inf, +inf logits of a softmax share its probability.
//
// One warp per token: lane l holds experts l V .. l V + V - 1 (V = ceil(E / 32) rounded to a built
// width) in registers, so one pass reads the logits and everything else is shuffles: topk rounds of
// one redux over order-preserving integer keys and one ballot for the lowest lane that has it.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "../../include/fleet_mk.h"

namespace mk {
int set_last_error(int code, const char* msg);   // mk_runtime.cu: the message mk_last_error() returns
}

namespace {

constexpr int WARPS = 8, MAX_E = 512, MAX_TOPK = 32, MAX_GROUPS = 32;
constexpr uint32_t FULL = 0xFFFFFFFFu;

struct Args {
  const void* logits;
  int64_t ld;
  const float* bias;
  int32_t* ids;
  float* weights;
  int t, e, topk, n_group, topk_group, gsize, forced;
  uint32_t gmul;        // ceil(2^20 / gsize): e / gsize = e * gmul >> 20 for e < 512
  float scaling;
  int sigmoid, top2, renorm;
};

__device__ __forceinline__ float ninf() { return -__int_as_float(0x7F800000); }
// unsigned order of the key = order of the float; every float's key is above 0
__device__ __forceinline__ uint32_t key_of(float v) {
  const uint32_t u = __float_as_uint(v);
  return (u >> 31) ? ~u : u | 0x80000000u;
}

template <typename L>
__device__ __forceinline__ float load(const L* p);
template <>
__device__ __forceinline__ float load<float>(const float* p) { return *p; }
template <>
__device__ __forceinline__ float load<__nv_bfloat16>(const __nv_bfloat16* p) { return __bfloat162float(*p); }

template <typename L, int V>
__global__ void __launch_bounds__(WARPS * 32) route_kernel(const Args a) {
  __shared__ float cs[WARPS][V * 32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t tok = (int64_t)blockIdx.x * WARPS + warp;
  if (tok >= a.t) return;
  const L* row = static_cast<const L*>(a.logits) + tok * a.ld;
  float s[V], c[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int e = lane * V + i;
    s[i] = e < a.e ? load<L>(row + e) : ninf();
    if (isnan(s[i])) s[i] = ninf();
  }
  float sum = 1.0f;   // what a score is divided by
  if (a.sigmoid) {
#pragma unroll
    for (int i = 0; i < V; ++i) s[i] = __fdiv_rn(1.0f, __fadd_rn(1.0f, expf(-s[i])));
  } else {
    float m = ninf();
#pragma unroll
    for (int i = 0; i < V; ++i) m = fmaxf(m, s[i]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(FULL, m, o));
    sum = 0.0f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      s[i] = m == ninf() ? 0.0f : s[i] == m ? 1.0f : expf(s[i] - m);
      sum += s[i];
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(FULL, sum, o);
    if (sum == 0.0f) sum = 1.0f;
  }
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int e = lane * V + i;
    c[i] = s[i];
    if (a.bias && e < a.e) c[i] = __fadd_rn(a.sigmoid ? s[i] : __fdiv_rn(s[i], sum), a.bias[e]);
    if (isnan(c[i])) c[i] = ninf();
  }
  uint32_t kept = FULL;
  if (a.n_group > 1) {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (lane * V + i < a.e) cs[warp][lane * V + i] = c[i];
    __syncwarp();
    float score = ninf();
    if (lane < a.n_group) {
      float m1 = ninf(), m2 = ninf();
      for (int i = 0; i < a.gsize; ++i) {
        const float v = cs[warp][lane * a.gsize + i];
        m2 = fmaxf(m2, fminf(m1, v));
        m1 = fmaxf(m1, v);
      }
      score = a.top2 && a.gsize > 1 ? __fadd_rn(m1, m2) : m1;
      if (isnan(score)) score = ninf();
    }
    int better = 0;
    for (int j = 0; j < a.n_group; ++j) {
      const float o = __shfl_sync(FULL, score, j);
      better += o > score || (o == score && j < lane);
    }
    kept = __ballot_sync(FULL, lane < a.n_group && better < a.topk_group);
  }
  uint32_t key[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const uint32_t e = lane * V + i, grp = e * a.gmul >> 20;
    key[i] = e < (uint32_t)a.e && (kept >> (grp & 31) & 1) ? key_of(c[i]) : 0u;
  }
  int my_id = 0;
  float my_s = 0.0f;
  for (int k = 0; k < a.topk; ++k) {
    uint32_t best = 0;
#pragma unroll
    for (int i = 0; i < V; ++i) best = max(best, key[i]);
    const uint32_t top = __reduce_max_sync(FULL, best);
    const int who = __ffs(__ballot_sync(FULL, best == top)) - 1;
    int at = 0;
    float sc = 0.0f;
    bool done = false;
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (!done && key[i] == top) {
        at = i;
        sc = s[i];
        done = true;
        if (lane == who) key[i] = 0;
      }
    const int id = __shfl_sync(FULL, lane * V + at, who);
    const float w = __shfl_sync(FULL, sc, who);
    if (lane == k) { my_id = id; my_s = w; }
  }
  const bool mine = lane < a.topk;
  float w = mine && !a.sigmoid ? __fdiv_rn(my_s, sum) : my_s;
  if (a.renorm) {
    float all = mine ? w : 0.0f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(FULL, all, o);
    w = all == 0.0f ? 0.0f : __fdiv_rn(w, all);
  }
  const int64_t o = tok * (a.topk + a.forced);
  if (mine) {
    a.ids[o + lane] = my_id;
    a.weights[o + lane] = w * a.scaling;
  }
  if (lane < a.forced) {
    a.ids[o + a.topk + lane] = a.e + lane;
    a.weights[o + a.topk + lane] = 1.0f;
  }
}

int fail(int code, const char* msg) { return mk::set_last_error(code, msg); }

template <typename L>
cudaError_t launch(const Args& a, cudaStream_t s) {
  const unsigned grid = (unsigned)((a.t + WARPS - 1) / WARPS);
  const int v = (a.e + 31) / 32;
  if (v <= 1) route_kernel<L, 1><<<grid, WARPS * 32, 0, s>>>(a);
  else if (v <= 2) route_kernel<L, 2><<<grid, WARPS * 32, 0, s>>>(a);
  else if (v <= 4) route_kernel<L, 4><<<grid, WARPS * 32, 0, s>>>(a);
  else if (v <= 5) route_kernel<L, 5><<<grid, WARPS * 32, 0, s>>>(a);
  else if (v <= 8) route_kernel<L, 8><<<grid, WARPS * 32, 0, s>>>(a);
  else route_kernel<L, 16><<<grid, WARPS * 32, 0, s>>>(a);
  return cudaGetLastError();
}

}  // namespace

extern "C" int mk_route(const MkRoute* r, const void* logits, int64_t ld, int32_t t, const float* bias, int32_t* ids,
                        float* weights, void* stream) {
  if (!r) return fail(MK_EINVAL, "null routing parameters");
  if (r->experts < 1 || r->experts > MAX_E) return fail(MK_EINVAL, "experts are from 1 to 512");
  if (r->topk < 1 || r->topk > MAX_TOPK || r->topk > r->experts) return fail(MK_EINVAL, "topk is from 1 to 32 and at most the experts");
  if (r->n_group < 1 || r->n_group > MAX_GROUPS || r->experts % r->n_group)
    return fail(MK_EINVAL, "n_group is from 1 to 32 and divides the experts");
  if (r->topk_group < 1 || r->topk_group > r->n_group || r->topk > r->topk_group * (r->experts / r->n_group))
    return fail(MK_EINVAL, "topk_group is from 1 to n_group and its groups hold at least topk experts");
  if (r->n_forced < 0 || r->n_forced > MAX_TOPK) return fail(MK_EINVAL, "n_forced is from 0 to 32");
  if (r->score != MK_ROUTE_SOFTMAX && r->score != MK_ROUTE_SIGMOID) return fail(MK_EINVAL, "score is softmax or sigmoid");
  if (r->logits_dtype != MK_ROUTE_FP32 && r->logits_dtype != MK_ROUTE_BF16) return fail(MK_EINVAL, "logits are FP32 or BF16");
  if (t < 0) return fail(MK_EINVAL, "a negative number of tokens");
  if (t == 0) return MK_OK;
  if (!logits || !ids || !weights) return fail(MK_EINVAL, "null pointer");
  const uintptr_t need = r->logits_dtype == MK_ROUTE_FP32 ? 3 : 1;
  if (((uintptr_t)logits & need) || ((uintptr_t)bias & 3) || ((uintptr_t)ids & 3) || ((uintptr_t)weights & 3))
    return fail(MK_EINVAL, "misaligned logits, bias, ids or weights");
  Args a{};
  a.logits = logits;
  a.ld = ld;
  a.bias = bias;
  a.ids = ids;
  a.weights = weights;
  a.t = t;
  a.e = r->experts;
  a.topk = r->topk;
  a.n_group = r->n_group;
  a.topk_group = r->topk_group;
  a.gsize = r->experts / r->n_group;
  a.gmul = ((1u << 20) + a.gsize - 1) / a.gsize;
  a.forced = r->n_forced;
  a.scaling = r->scaling;
  a.sigmoid = r->score == MK_ROUTE_SIGMOID;
  a.top2 = r->group_top2 != 0;
  a.renorm = r->renormalize != 0;
  const cudaError_t e = r->logits_dtype == MK_ROUTE_FP32 ? launch<float>(a, static_cast<cudaStream_t>(stream))
                                                          : launch<__nv_bfloat16>(a, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? MK_OK : fail(MK_ECUDA, cudaGetErrorString(e));
}

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
// One warp per token: lane l holds experts l V .. l V + V - 1 in registers, V the smallest built width
// with 32 V >= E, so one pass reads the logits (16 bytes a lane at a time where they are aligned)
// and the rest is registers and shuffles. The selection ranks few candidates instead of sorting: no
// expert below the topk-th best of the 32 lanes' best ones can be among the topk, so the experts at
// or above that (about 1.5 topk for scores spread over the lanes) go to shared memory, one to a lane,
// and a lane counts how many are better than its own. More than 32 of them (long ties, more topk than
// lanes with experts) are taken one by one instead.
//
// 16384 tokens of 256 experts (sigmoid, bias, 8 groups by their two best, topk 8, renormalised) read 17 MB,
// 2.6 us at the copy rate, and take 15.9 us: bound by issue (82 % of the issue slots, 830 instructions a
// token, about 160 of them the exact exponentials and reciprocals). topk rounds over all experts
// took 38 us. Two tokens a warp (16 lanes of 16 experts) took 18.2. One token: 2.3 us, a launch.
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
  int lanes;            // log2 of the lanes that hold a group, or -1 (a lane's experts are of several)
  int vec, bias_vec;    // rows, the bias may be read a lane's share at a time
  float scaling;
  int sigmoid, top2, renorm;
};

__device__ __forceinline__ float ninf() { return -__int_as_float(0x7F800000); }
// unsigned order of the key = order of the float; every float's key is above 0
__device__ __forceinline__ uint32_t key_of(float v) {
  const uint32_t u = __float_as_uint(v);
  return u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float logistic(float x) { return __frcp_rn(__fadd_rn(1.0f, expf(-x))); }

// V values from p, aligned to the largest power of two (at most 16 bytes) that divides their size
template <typename L, int V>
__device__ __forceinline__ void load_lane(const L* p, float (&s)[V]) {
  constexpr int BYTES = V * sizeof(L), STEP = BYTES % 16 == 0 ? 16 : BYTES % 8 == 0 ? 8 : BYTES % 4 == 0 ? 4 : 2;
  L v[V];
#pragma unroll
  for (int i = 0; i < BYTES / STEP; ++i) {
    const char* src = reinterpret_cast<const char*>(p) + i * STEP;
    char* dst = reinterpret_cast<char*>(v) + i * STEP;
    if (STEP == 16) *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(src);
    else if (STEP == 8) *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(src);
    else if (STEP == 4) *reinterpret_cast<uint32_t*>(dst) = *reinterpret_cast<const uint32_t*>(src);
    else *reinterpret_cast<uint16_t*>(dst) = *reinterpret_cast<const uint16_t*>(src);
  }
#pragma unroll
  for (int i = 0; i < V; ++i) s[i] = to_f32(v[i]);
}

template <typename L, int V>
__global__ void __launch_bounds__(WARPS * 32) route_kernel(const Args a) {
  __shared__ __align__(16) uint64_t shared[WARPS][V * 32 > 64 ? V * 16 : 32];   // scores of the groups, or candidates
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t tok = (int64_t)blockIdx.x * WARPS + warp;
  if (tok >= a.t) return;
  const L* row = static_cast<const L*>(a.logits) + tok * a.ld;
  const int past = lane * V + V - a.e;     // above 0: this lane's last `past` places hold no expert
  float c[V];           // logits, then the selection's values
  if (a.vec) {
    if (lane * V < a.e) {
      load_lane<L, V>(row + lane * V, c);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) c[i] = ninf();
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) c[i] = lane * V + i < a.e ? to_f32(row[lane * V + i]) : ninf();
  }
#pragma unroll
  for (int i = 0; i < V; ++i) c[i] = fmaxf(c[i], ninf());   // a NaN is the other argument's loss
  float sum = 1.0f, m = 0.0f;   // of a softmax
  if (a.sigmoid) {
#pragma unroll
    for (int i = 0; i < V; ++i) c[i] = logistic(c[i]);
  } else {
    m = ninf();
#pragma unroll
    for (int i = 0; i < V; ++i) m = fmaxf(m, c[i]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(FULL, m, o));
    sum = 0.0f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      c[i] = m == ninf() ? 0.0f : c[i] == m ? 1.0f : expf(c[i] - m);
      sum += c[i];
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(FULL, sum, o);
    if (sum == 0.0f) sum = 1.0f;
  }
  if (a.bias) {
    float b[V];
    if (a.bias_vec && past <= 0) {
      load_lane<float, V>(a.bias + lane * V, b);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) b[i] = lane * V + i < a.e ? a.bias[lane * V + i] : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < V; ++i) c[i] = fmaxf(__fadd_rn(a.sigmoid ? c[i] : __fdiv_rn(c[i], sum), b[i]), ninf());
  }
  uint32_t key[V];
#pragma unroll
  for (int i = 0; i < V; ++i) key[i] = key_of(c[i]);
  if (past > 0) {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (i >= V - past) {
        key[i] = 0;
        c[i] = ninf();
      }
  }
  if (a.n_group > 1) {
    const bool top2 = a.top2 && a.gsize > 1;
    float score = ninf();
    int mine, stride;     // this lane's group; the lane of group j is j * stride
    if (a.lanes >= 0) {
      float m1 = ninf(), m2 = ninf();
#pragma unroll
      for (int i = 0; i < V; ++i) {
        m2 = fmaxf(m2, fminf(m1, c[i]));
        m1 = fmaxf(m1, c[i]);
      }
      for (int o = 1; o < 1 << a.lanes; o <<= 1) {
        const float o1 = __shfl_xor_sync(FULL, m1, o), o2 = __shfl_xor_sync(FULL, m2, o);
        m2 = fmaxf(fminf(m1, o1), fmaxf(m2, o2));
        m1 = fmaxf(m1, o1);
      }
      score = top2 ? __fadd_rn(m1, m2) : m1;
      mine = lane >> a.lanes;
      stride = 1 << a.lanes;
    } else {
      float* cs = reinterpret_cast<float*>(shared[warp]);
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (lane * V + i < a.e) cs[lane * V + i] = c[i];
      __syncwarp();
      if (lane < a.n_group) {
        float m1 = ninf(), m2 = ninf();
        for (int i = 0; i < a.gsize; ++i) {
          const float v = cs[lane * a.gsize + i];
          m2 = fmaxf(m2, fminf(m1, v));
          m1 = fmaxf(m1, v);
        }
        score = top2 ? __fadd_rn(m1, m2) : m1;
      }
      __syncwarp();
      mine = lane;
      stride = 1;
    }
    if (isnan(score)) score = ninf();
    int better = 0;
    for (int j = 0; j < a.n_group; ++j) {
      const float o = __shfl_sync(FULL, score, j * stride);
      better += o > score || (o == score && j < mine);
    }
    const bool keep = mine < a.n_group && better < a.topk_group;
    const uint32_t kept = __ballot_sync(FULL, keep);   // by lane, or by group
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (a.lanes >= 0 ? !keep : !(kept >> (((lane * V + i) * a.gmul >> 20) & 31) & 1)) key[i] = 0;
  }
  // the topk-th best of the lanes' best (equal ones leave together: fewer than topk may stay above it)
  uint32_t best = 0;
#pragma unroll
  for (int i = 0; i < V; ++i) best = max(best, key[i]);
  uint32_t least = 0;
#pragma unroll 2
  for (int k = 0; k < a.topk; ++k) {
    least = __reduce_max_sync(FULL, best);
    best = best == least ? 0 : best;
  }
  least = max(least, 1u);
  int count = 0;
#pragma unroll
  for (int i = 0; i < V; ++i) count += key[i] >= least;
  int upto = count;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(FULL, upto, o);
    if (lane >= o) upto += v;
  }
  const int total = __shfl_sync(FULL, upto, 31);
  int id = 0;
  if (total <= 32) {
    uint64_t* cand = shared[warp];    // (key, the higher the lower the expert)
    int at = upto - count;
    cand[lane] = 0;                   // below every candidate
    __syncwarp();
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (key[i] >= least) cand[at++] = (uint64_t)key[i] << 32 | (uint32_t)~(lane * V + i);
    __syncwarp();
    const uint64_t mine = lane < total ? cand[lane] : 0;
    int rank = 0;
    for (int j = 0; j < total; j += 4) {
      const ulonglong2 u = *reinterpret_cast<const ulonglong2*>(cand + j), v = *reinterpret_cast<const ulonglong2*>(cand + j + 2);
      rank += (u.x > mine) + (u.y > mine) + (v.x > mine) + (v.y > mine);
    }
    __syncwarp();
    int* ranked = reinterpret_cast<int*>(cand);
    if (lane < total && rank < a.topk) ranked[rank] = ~(uint32_t)mine;
    __syncwarp();
    if (lane < a.topk) id = ranked[lane];
  } else {
    for (int k = 0; k < a.topk; ++k) {
      uint32_t most = 0;
#pragma unroll
      for (int i = 0; i < V; ++i) most = max(most, key[i]);
      const uint32_t top = __reduce_max_sync(FULL, most);
      const int who = __ffs(__ballot_sync(FULL, most == top)) - 1;
      int at = 0;
#pragma unroll
      for (int i = V - 1; i >= 0; --i)
        if (key[i] == top) at = i;
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (lane == who && i == at) key[i] = 0;
      const int winner = __shfl_sync(FULL, lane * V + at, who);
      if (lane == k) id = winner;
    }
  }
  const bool mine = lane < a.topk;
  float w = 0.0f;
  if (mine) {           // the score again, from its logit
    const float x = fmaxf(to_f32(row[id]), ninf());
    if (a.sigmoid) w = logistic(x);
    else w = __fdiv_rn(m == ninf() ? 0.0f : x == m ? 1.0f : expf(x - m), sum);
  }
  if (a.renorm) {
    float all = w;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(FULL, all, o);
    w = all == 0.0f ? 0.0f : __fdiv_rn(w, all);
  }
  const int64_t o = tok * (a.topk + a.forced);
  if (mine) {
    a.ids[o + lane] = id;
    a.weights[o + lane] = w * a.scaling;
  }
  if (lane < a.forced) {
    a.ids[o + a.topk + lane] = a.e + lane;
    a.weights[o + a.topk + lane] = 1.0f;
  }
}

int fail(int code, const char* msg) { return mk::set_last_error(code, msg); }

template <typename L, int V>
cudaError_t launch_width(Args a, cudaStream_t s) {
  // a lane's share as vectors: its size's largest power of two up to 16 divides the rows' starts, and no
  // lane's share crosses the row's end
  constexpr int BYTES = V * sizeof(L), STEP = BYTES % 16 == 0 ? 16 : BYTES % 8 == 0 ? 8 : BYTES % 4 == 0 ? 4 : 2;
  a.vec = a.e % V == 0 && (uintptr_t)a.logits % STEP == 0 && a.ld * (int64_t)sizeof(L) % STEP == 0;
  constexpr int BSTEP = V % 4 == 0 ? 16 : V % 2 == 0 ? 8 : 4;
  a.bias_vec = (uintptr_t)a.bias % BSTEP == 0;
  a.lanes = -1;
  if (a.gsize % V == 0)
    for (int l = 0; l <= 5; ++l)
      if (a.gsize / V == 1 << l) a.lanes = l;
  // (the launch's own result: the last error may be another call's)
  cudaLaunchConfig_t c{};
  c.gridDim = dim3(((unsigned)a.t + WARPS - 1) / WARPS);
  c.blockDim = dim3(WARPS * 32);
  c.stream = s;
  return cudaLaunchKernelEx(&c, route_kernel<L, V>, a);
}

template <typename L>
cudaError_t launch(const Args& a, cudaStream_t s) {
  const int v = (a.e + 31) / 32;
  return v <= 1 ? launch_width<L, 1>(a, s) : v <= 2 ? launch_width<L, 2>(a, s) : v <= 3 ? launch_width<L, 3>(a, s)
       : v <= 4 ? launch_width<L, 4>(a, s) : v <= 5 ? launch_width<L, 5>(a, s) : v <= 6 ? launch_width<L, 6>(a, s)
       : v <= 8 ? launch_width<L, 8>(a, s) : v <= 12 ? launch_width<L, 12>(a, s) : launch_width<L, 16>(a, s);
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

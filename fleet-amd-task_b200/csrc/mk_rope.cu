// mk_rope.cu -- rotary positions of a batch of tokens: mk_rope.
//
// Formulas. Of each head's `width` values the `dim` from `start` on are pairs (a_i, b_i), i < dim / 2; at
// position p pair i turns by t_i = p inv_freq[i]:  a' = m (a cos t - b sin t), b' = m (b cos t + a sin t),
// m the scale of a stretched context. Pairs are (i, i + dim / 2) (half), (2 i, 2 i + 1) (interleaved), or
// read from (2 i, 2 i + 1) and written to (i, i + dim / 2) (pairs to half). The other values are copied where
// the output is another tensor. A token at a negative position is left out: its output stays as it was.
//
// An angle of a far position needs more than 32 bits (position 2^20 times an inv_freq of 1 leaves 4 bits
// of an FP32 angle's fraction), so turns are counted in 64: p (inv_freq / 2 pi) less its nearest whole
// number, then sincospif in FP32: within 2^-23 of a turn for positions up to 2^31 and frequencies up to 1 (the product's two
// roundings and that of 1 / 2 pi, each 2^-53 of up to 2^28.4 turns), within 2^-25 for positions up to 2^28.
//
// A block takes some tokens, or some heads of one. Each thread loads VEC pairs of a head and COPIES times VEC values that are
// copied, 16 bytes at a time where all rows allow it; then the block computes its tokens' sines and cosines while the
// loads are on their way, then all is turned and stored. Nothing of the block is stored before all of it is loaded,
// so the output may be the input even where the layout changes.
//
// 8192 tokens of 16 heads of 192 values, the last 64 turned: 101 MB, a floor of 15.4 us; 17.5 us on the device.
#include "mk_latent.cuh"

namespace {

constexpr int MAX_DIM = 512, TABLE = 1024, COPIES = 4, SMS = 148;     // TABLE: pairs whose turns a block holds
// threads of a block: a head's pairs at least; for the wide form 128 (8192 tokens: 17.5 us, 256 threads 19.0, 512 20.7)
__host__ __device__ constexpr int threads_of(int vec) { return vec == 8 ? 128 : MAX_DIM / 2; }

using latent::Div;
using latent::fail;
using latent::operator/;
using latent::to_f32;

struct Args {
  const double* inv_freq;
  const void *x, *positions;
  void* out;
  int64_t xt, xh, ot, oh;       // strides of tokens and heads, in values
  int t, heads, start, dim, layout, pos64;
  int tokens, group, rest;      // of a block: tokens and heads; the vectors of a head that are copied by the loop at the end
  Div by_turned, by_copied, by_group;   // of a head: vectors of pairs, copied vectors; the heads
  float scale;
};

__device__ __forceinline__ void two(__nv_bfloat16* d, float a, float b) { *reinterpret_cast<__nv_bfloat162*>(d) = __floats2bfloat162_rn(a, b); }
__device__ __forceinline__ void two(__half* d, float a, float b) { *reinterpret_cast<__half2*>(d) = __floats2half2_rn(a, b); }

template <typename T, int VEC>
struct Vec { alignas(VEC * sizeof(T)) T v[VEC]; };

template <typename T, int VEC>
__global__ void __launch_bounds__(threads_of(VEC)) rope_kernel(const Args a) {
  constexpr int THREADS = threads_of(VEC);
  __shared__ float2 turn[TABLE];        // (cos, sin) times the scale
  __shared__ bool live[TABLE];
  using V = Vec<T, VEC>;
  latent::start_dependents();
  latent::wait_predecessor();
  const int pairs = a.dim / 2, turned = a.by_turned.d, copied = a.by_copied.d;
  const int64_t first = (int64_t)blockIdx.x * a.tokens;
  const int h0 = blockIdx.y * a.group, heads = min(a.group, a.heads - h0), tokens = (int)min((int64_t)a.tokens, a.t - first);
  const int rows = tokens * heads;      // (several tokens only where a block takes all heads)
  const bool split = a.layout != MK_ROPE_HALF, join = a.layout == MK_ROPE_INTERLEAVED;
  const T* x = static_cast<const T*>(a.x) + first * a.xt + h0 * a.xh;
  T* out = static_cast<T*>(a.out) + first * a.ot + h0 * a.oh;
  // this thread's vectors of pairs: place i of row r
  const int r = (int)threadIdx.x / a.by_turned, i = threadIdx.x - r * turned, tok = r / a.by_group, h = r - tok * a.group;
  const bool turns = r < rows;
  V u, w;
  if (turns) {
    const T* p = x + tok * a.xt + h * a.xh + a.start;
    u = *reinterpret_cast<const V*>(p + (split ? 2 * i : i) * VEC);
    w = *reinterpret_cast<const V*>(p + (split ? 2 * i + 1 : i + turned) * VEC);
  }
  // the values before and behind the turned ones are copied: place c of row cr
  const auto copy_of = [&](int k, int& cr, int& c) {
    const int n = threadIdx.x + k * THREADS;
    cr = n / a.by_copied;
    c = (n - cr * copied) * VEC;
    c += c < a.start ? 0 : a.dim;
    return cr < rows;
  };
  V moved[COPIES];
  if (copied > 0) {
#pragma unroll
    for (int k = 0; k < COPIES; ++k) {
      int cr, c;
      if (copy_of(k, cr, c)) {
        const int t = cr / a.by_group;
        moved[k] = *reinterpret_cast<const V*>(x + t * a.xt + (cr - t * a.group) * a.xh + c);
      }
    }
  }
  for (int n = threadIdx.x; n < tokens * pairs; n += THREADS) {
    const int t = n / pairs, pair = n - t * pairs;
    const int64_t position = a.pos64 ? static_cast<const int64_t*>(a.positions)[first + t] : (int64_t)static_cast<const int32_t*>(a.positions)[first + t];
    const double turns = (double)position * (a.inv_freq[pair] * 0.15915494309189533577);
    float s, c;
    sincospif(2.0f * (float)(turns - rint(turns)), &s, &c);
    turn[n] = make_float2(c * a.scale, s * a.scale);
    if (pair == 0) live[t] = position >= 0;
  }
  __syncthreads();
  if (turns && live[tok]) {
    const float2* cs = turn + tok * pairs + i * VEC;
    V lo, hi;
    float ra[VEC], rb[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      // split: pair j of the 2 VEC neighbours u, w
      const float va = to_f32(split ? (2 * j < VEC ? u.v[2 * j % VEC] : w.v[2 * j % VEC]) : u.v[j]);
      const float vb = to_f32(split ? (2 * j + 1 < VEC ? u.v[(2 * j + 1) % VEC] : w.v[(2 * j + 1) % VEC]) : w.v[j]);
      ra[j] = va * cs[j].x - vb * cs[j].y;
      rb[j] = vb * cs[j].x + va * cs[j].y;
    }
    if constexpr (VEC == 1) {
      lo.v[0] = latent::from_f32<T>(ra[0]);
      hi.v[0] = latent::from_f32<T>(rb[0]);
    } else {                    // two values a conversion
#pragma unroll
      for (int j = 0; j < VEC / 2; ++j) {
        two(lo.v + 2 * j, join ? ra[j] : ra[2 * j], join ? rb[j] : ra[2 * j + 1]);
        two(hi.v + 2 * j, join ? ra[j + VEC / 2] : rb[2 * j], join ? rb[j + VEC / 2] : rb[2 * j + 1]);
      }
    }
    T* p = out + tok * a.ot + h * a.oh + a.start;
    *reinterpret_cast<V*>(p + (join ? 2 * i : i) * VEC) = lo;
    *reinterpret_cast<V*>(p + (join ? 2 * i + 1 : i + turned) * VEC) = hi;
  }
  if (copied > 0) {
#pragma unroll
    for (int k = 0; k < COPIES; ++k) {
      int cr, c;
      if (copy_of(k, cr, c)) {
        const int t = cr / a.by_group;
        if (live[t]) *reinterpret_cast<V*>(out + t * a.ot + (cr - t * a.group) * a.oh + c) = moved[k];
      }
    }
  }
  // heads too wide for the threads' registers
  for (int64_t n = threadIdx.x; n < (int64_t)rows * a.rest; n += THREADS) {
    const int cr = (int)(n / a.rest), t = cr / a.by_group, hh = cr - t * a.group;
    int c = (int)(n - (int64_t)cr * a.rest) * VEC;
    c += c < a.start ? 0 : a.dim;
    if (live[t]) *reinterpret_cast<V*>(out + t * a.ot + hh * a.oh + c) = *reinterpret_cast<const V*>(x + t * a.xt + hh * a.xh + c);
  }
}

template <typename T>
cudaError_t launch(Args a, int width, cudaStream_t s) {
  const bool wide = ((uintptr_t)a.x | (uintptr_t)a.out) % 16 == 0 && (a.xt | a.xh | a.ot | a.oh) % 8 == 0 &&
                    a.dim % 16 == 0 && a.start % 8 == 0 && width % 8 == 0;
  const int vec = wide ? 8 : 1, THREADS = threads_of(vec), turned = a.dim / 2 / vec, rest = a.x != a.out ? (width - a.dim) / vec : 0;
  const int copied = rest <= THREADS * COPIES ? rest : 0;
  int most = THREADS / turned;                  // heads that a block's threads hold
  if (copied > 0 && THREADS * COPIES / copied < most) most = THREADS * COPIES / copied;
  a.rest = rest - copied;
  a.group = most < a.heads ? most : a.heads;
  // whole tokens where they fit, but a block for each of the SMs first
  const int fit = most / a.heads, held = TABLE / (a.dim / 2), spread = (a.t - 1) / (2 * SMS) + 1;
  a.tokens = fit < 1 ? 1 : fit < held ? fit : held;
  a.tokens = a.tokens < spread ? a.tokens : spread;
  a.by_turned = latent::div_by(turned);
  a.by_copied = copied > 0 ? latent::div_by(copied) : Div{0, 0, 0};
  a.by_group = latent::div_by(a.group);
  const dim3 grid((unsigned)((a.t + (int64_t)a.tokens - 1) / a.tokens), (unsigned)((a.heads + a.group - 1) / a.group));
  return latent::launch_early(wide ? rope_kernel<T, 8> : rope_kernel<T, 1>, grid, THREADS, 0, s, a);
}

}  // namespace

extern "C" int mk_rope(const MkRope* r, const void* positions, int32_t t, const void* x, int64_t xt, int64_t xh, int32_t heads,
                       int32_t width, int32_t start, void* out, int64_t ot, int64_t oh, void* stream) {
  if (!r) return fail(MK_EINVAL, "null rotary parameters");
  if (r->dim < 2 || r->dim > MAX_DIM || r->dim % 2) return fail(MK_EINVAL, "dim is even and from 2 to 512");
  if (r->layout < MK_ROPE_HALF || r->layout > MK_ROPE_PAIRS_TO_HALF)
    return fail(MK_EINVAL, "layout is half, interleaved or pairs to half");
  if (r->dtype != MK_BF16 && r->dtype != MK_FP16) return fail(MK_EINVAL, "values are BF16 or FP16");
  if (t < 0 || heads < 0 || width < 0 || start < 0 || (int64_t)start + r->dim > width)
    return fail(MK_EINVAL, "the rotary part lies within a head, and no size is negative");
  if ((int64_t)heads * width > INT32_MAX || heads > 65535) return fail(MK_EINVAL, "a token has at most 65535 heads of together fewer than 2^31 values");
  if (t == 0 || heads == 0) return MK_OK;
  if (!r->inv_freq || !positions || !x || !out) return fail(MK_EINVAL, "null pointer");
  if (((uintptr_t)r->inv_freq & 7) || ((uintptr_t)positions & (r->pos64 ? 7 : 3)) || (((uintptr_t)x | (uintptr_t)out) & 1))
    return fail(MK_EINVAL, "misaligned inv_freq, positions, x or out");
  Args a{};
  a.inv_freq = r->inv_freq;
  a.x = x;
  a.positions = positions;
  a.out = out;
  a.xt = xt;
  a.xh = xh;
  a.ot = ot;
  a.oh = oh;
  a.t = t;
  a.heads = heads;
  a.start = start;
  a.dim = r->dim;
  a.layout = r->layout;
  a.pos64 = r->pos64 != 0;
  a.scale = r->scale;
  const cudaError_t e = r->dtype == MK_BF16 ? launch<__nv_bfloat16>(a, width, static_cast<cudaStream_t>(stream))
                                             : launch<__half>(a, width, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? MK_OK : fail(MK_ECUDA, cudaGetErrorString(e));
}

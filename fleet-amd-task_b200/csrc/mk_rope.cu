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
// number, then sincospif in FP32: within 2^-25 of a turn for positions up to 2^31.
//
// A block takes some tokens: their dim / 2 sines and cosines go to shared memory once for all heads, then
// each thread takes VEC pairs of a head at a time: 16-byte loads and stores where all rows allow them,
// single values otherwise. A head's pairs are in one warp, loaded before any is stored, so the output may
// be the input even where the layout changes.
#include "mk_latent.cuh"

namespace {

constexpr int THREADS = 256, MAX_DIM = 512, TABLE = 512;   // TABLE: pairs whose turns a block holds

struct Args {
  const double* inv_freq;
  const void *x, *positions;
  void* out;
  int64_t xt, xh, ot, oh;       // strides of tokens and heads, in values
  int t, heads, width, start, dim, layout, tokens, pos64, copy;
  float scale;
};

using latent::to_f32;
__device__ __forceinline__ void from_f32(__nv_bfloat16& d, float v) { d = __float2bfloat16_rn(v); }
__device__ __forceinline__ void from_f32(__half& d, float v) { d = __float2half_rn(v); }

template <typename T, int VEC>
struct Vec { alignas(VEC * sizeof(T)) T v[VEC]; };

template <typename T, int VEC>
__global__ void __launch_bounds__(THREADS) rope_kernel(const Args a) {
  __shared__ float2 turn[TABLE];        // (cos, sin) times the scale
  using V = Vec<T, VEC>;
  latent::start_dependents();
  latent::wait_predecessor();
  const int pairs = a.dim / 2, units = pairs / VEC;
  const int64_t first = (int64_t)blockIdx.x * a.tokens;
  const int count = (int)min((int64_t)a.tokens, a.t - first);
  auto position = [&](int i) {
    return a.pos64 ? static_cast<const int64_t*>(a.positions)[first + i] : (int64_t)static_cast<const int32_t*>(a.positions)[first + i];
  };
  for (int i = threadIdx.x; i < count * pairs; i += THREADS) {
    const double turns = (double)position(i / pairs) * (a.inv_freq[i % pairs] * 0.15915494309189533577);
    float s, c;
    sincospif(2.0f * (float)(turns - rint(turns)), &s, &c);
    turn[i] = make_float2(c * a.scale, s * a.scale);
  }
  __syncthreads();
  // a head's units on consecutive lanes of one warp: `lanes` (a power of two) of them, ROUNDS units a lane
  constexpr int ROUNDS = MAX_DIM / 2 / VEC / 32;
  int lanes = 1;
  while (lanes < units && lanes < 32) lanes *= 2;
  const int lane = threadIdx.x % lanes, per = THREADS / lanes;
  const bool split = a.layout != MK_ROPE_HALF, join = a.layout == MK_ROPE_INTERLEAVED;
  const int rows = count * a.heads;
  for (int r0 = 0; r0 < rows; r0 += per) {
    const int r = r0 + threadIdx.x / lanes, tok = r / a.heads;
    const bool live = r < rows && position(tok) >= 0;
    const T* x = static_cast<const T*>(a.x) + (first + tok) * a.xt + (int64_t)(r - tok * a.heads) * a.xh + a.start;
    T* out = static_cast<T*>(a.out) + (first + tok) * a.ot + (int64_t)(r - tok * a.heads) * a.oh + a.start;
    V u[ROUNDS], w[ROUNDS];
#pragma unroll
    for (int k = 0; k < ROUNDS; ++k) {
      const int i = (lane + k * lanes) * VEC;
      if (live && i < pairs) {
        u[k] = *reinterpret_cast<const V*>(x + (split ? 2 * i : i));
        w[k] = *reinterpret_cast<const V*>(x + (split ? 2 * i + VEC : i + pairs));
      }
    }
    __syncwarp();
#pragma unroll
    for (int k = 0; k < ROUNDS; ++k) {
      const int i = (lane + k * lanes) * VEC;
      if (live && i < pairs) {
        V lo, hi;
        T* p = u[k].v;
        T* q = w[k].v;
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float2 cs = turn[tok * pairs + i + j];
          // split: pair j of the 2 VEC neighbours u, w
          const float va = to_f32(split ? (2 * j < VEC ? p[2 * j % VEC] : q[2 * j % VEC]) : p[j]);
          const float vb = to_f32(split ? (2 * j + 1 < VEC ? p[(2 * j + 1) % VEC] : q[(2 * j + 1) % VEC]) : q[j]);
          const float ra = va * cs.x - vb * cs.y, rb = vb * cs.x + va * cs.y;
          if (join) {
            from_f32(2 * j < VEC ? lo.v[2 * j % VEC] : hi.v[2 * j % VEC], ra);
            from_f32(2 * j + 1 < VEC ? lo.v[(2 * j + 1) % VEC] : hi.v[(2 * j + 1) % VEC], rb);
          } else {
            from_f32(lo.v[j], ra);
            from_f32(hi.v[j], rb);
          }
        }
        *reinterpret_cast<V*>(out + (join ? 2 * i : i)) = lo;
        *reinterpret_cast<V*>(out + (join ? 2 * i + VEC : i + pairs)) = hi;
      }
    }
  }
  if (a.copy) {
    const int before = a.start / VEC, rest = (a.width - a.dim) / VEC;
    for (int64_t i = threadIdx.x; i < (int64_t)rows * rest; i += THREADS) {
      const int r = (int)(i / rest), c = (int)(i - (int64_t)r * rest), tok = r / a.heads, h = r - tok * a.heads;
      const int at = c < before ? c * VEC : c * VEC + a.dim;
      if (position(tok) >= 0)
        *reinterpret_cast<V*>(static_cast<T*>(a.out) + (first + tok) * a.ot + h * a.oh + at) =
            *reinterpret_cast<const V*>(static_cast<const T*>(a.x) + (first + tok) * a.xt + h * a.xh + at);
    }
  }
}

using latent::fail;

template <typename T>
cudaError_t launch(Args a, cudaStream_t s) {
  const bool wide = ((uintptr_t)a.x | (uintptr_t)a.out) % 16 == 0 && (a.xt | a.xh | a.ot | a.oh) % 8 == 0 &&
                    a.dim % 16 == 0 && a.start % 8 == 0 && a.width % 8 == 0;
  a.tokens = 1;
  const unsigned grid = (unsigned)((a.t + (int64_t)a.tokens - 1) / a.tokens);
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
  if ((int64_t)heads * width > INT32_MAX) return fail(MK_EINVAL, "a token's heads hold fewer than 2^31 values");
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
  a.width = width;
  a.start = start;
  a.dim = r->dim;
  a.layout = r->layout;
  a.pos64 = r->pos64 != 0;
  a.copy = x != out && width > r->dim;
  a.scale = r->scale;
  const cudaError_t e = r->dtype == MK_BF16 ? launch<__nv_bfloat16>(a, static_cast<cudaStream_t>(stream))
                                             : launch<__half>(a, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? MK_OK : fail(MK_ECUDA, cudaGetErrorString(e));
}

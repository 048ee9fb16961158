// mk_latent_attend.cu -- attention over the latent cache in 8 bits: mk_latent_attend. The format is in mk_latent.cuh.
//
// Formulas. Row i of the n of a sequence is its token P = len - n + i; for each head h, with q = (qc, qr),
//   s_j = scale (qc . c_j + qr . r_j), j = 0 .. P;  out = sum_j softmax(s)_j c_j;  lse = log sum_j exp(s_j).
// A row that sees no token (an empty sequence, P < 0, pages outside the cache) gives zeros and lse -inf.
//
// Why E4M3 operands, and how nothing is lost by them. A token is 576 bytes and 16 heads do 35 thousand operations on
// it: HBM brings an SM a tile of 128 tokens in 1.7 us, which leaves no time to widen its codes to 16 bits (147 KB
// of shared memory written and read back). So the codes go to tcgen05.mma (kind::f8f6f4) as they arrive by TMA, twice:
// as the keys of S = K q^T (128 tokens x N, K-major) and, the same bytes, as the values of O = C^T P (128 latent
// values x N, MN-major). What is not in 8 bits is split into pieces that are, each a column of its own, for the tensor core's
// time goes by the 128 rows of the tile (32 + N / 4 clocks a product of 128 x N x 32, measured alone, in any layout):
//   q    = scale_q (q1 + q2 / 16 (+ q3 / 256)) in E4M3: each piece takes 4 bits and the remainder's sign one more, so
//          two hold a BF16 value but for what is below 2^-14 of an x of up to 448 (the row's largest has 224 or more: 2^-21.8 of
//          it), three an FP16 value but for what is below 2^-18 (2^-25.8);
//   p    = x 2^-7, for BF16 x rounded to FP16 = x1 + x2 / 8 + x3 / 64 in E5M2: within 2^-11 (3, 4 and 4 bits are all of
//          FP16's 11), or 2^-30 of the row's largest where that is more: an eighth to a quarter of half a step of a BF16 output. An FP16
//          output's half step is 2^-11 itself, so there x = ... + x4 / 512 has what the rounding to FP16 took away: within
//          2^-15 + 2^-18, or 2^-33 of the row's largest (64 sequences of up to 8192 tokens
//          41.9 us, with three pieces 41.0; 512 tokens behind 3584 189 and 182). The sum of the weights takes x unrounded.
// A page's scales (keys: sc latent, sr rotary) multiply the scores' two accumulators in FP32. As the values' scale, sc
// goes into the exponent: t = s + log2 sc, p = 2^(t - ref), so the pieces are relative to the largest p |c|, and the sum
// of the weights takes p / sc. ref is a tile's maximum of t, taken anew (with O rescaled in tensor memory) only where some t
// is more than 8 above it.
//
// What bounds it, on B200 (64 sequences of 8192 and of 16384 tokens, their difference): in the middle of a run a tile of 16
// rows takes 1.73 us from HBM, 6.3 of the measured 6.5 TB/s, and 1.29 where all sequences name the same 64 pages, which L2
// holds: the chain of load, scores, softmax and sums over two stages. FP16, whose products have a third to
// a half more columns: 1.83 and 1.61. With 256 latent values the chain counts from HBM too: 1.32 (4.6 TB/s) and 1.13. 64 sequences of up
// to 8192 tokens (153 MB, 23.5 us at HBM's rate) take 42 us, of which 5.5 are the start (the batch's lengths, a table's
// page, the first tile and the queries, one after the other), 1.2 a run's end, 5 merge_kernel. A single sequence of 32768
// tokens takes 14 us, most of it those.
//
// The work is units of 64 tokens of a group of R rows (a row is a token's head) of a sequence; each block (one per SM)
// takes an equal run of all units, whatever the lengths, as tiles of two. A group within one run is finished there, one
// that several runs share leaves partial sums, which merge_kernel joins. Warps 0 to 7 are the softmax: a warp holds 32 of a
// tile's 128 tokens (the lanes of tensor memory that it may read) for half of the rows. Warp 9 issues the scores' products and
// warp 10 the sums', warps 8 and 11 the loads (every other page each: a copy takes 80 clocks to issue); each only ever waits
// for what comes next.
#include <cuda.h>

#include <atomic>
#include <cfloat>

#include "mk_device.cuh"
#include "mk_latent.cuh"

namespace latent {
namespace {

using mk::mbar_arrive;
using mk::mbar_init;
using mk::smem_u32;

constexpr int MAX_CTAS = 148, TILE = 128, UNIT = 64, THREADS = 384, SOFTMAX = 256, LOADERS = 2;
constexpr int SUB = TILE * 128, STAGE = 4 * SUB + TILE * LD_R;      // a tile: up to 4 x [128 tokens][128 B], then [128][64 B]
// A wait's default limit, and that of a block's end for its own copies and products in flight, which no caller shortens.
constexpr uint64_t TIMEOUT_NS = 2000000000ull;
constexpr float X_SCALE = 7.0f, RAISE = 8.0f;                       // x = 2^7 at ref, 2^15 at most

struct Bf16 {
  using half_type = __nv_bfloat16;
  using pair_type = __nv_bfloat162;
  static constexpr int pieces = 2, weights = 3;
};
struct Fp16 {
  using half_type = __half;
  using pair_type = __half2;
  static constexpr int pieces = 3, weights = 4;
};

template <typename T, int R_>
struct Config {
  static constexpr int R = R_, H = R_ / 2, PIECES = T::pieces, W = T::weights;
  static constexpr int NS = R * PIECES, NO = R * W;
  static constexpr int BUFS = 4 * NS + 4 * NO <= 512 ? 2 : 1;       // buffers of scores in tensor memory
  static constexpr int O_COL = BUFS * 2 * NS;
  static constexpr int QC = 2 * STAGE, QR = QC + 4 * NS * 128, PB = QR + NS * 64, SMEM = PB + 2 * NO * 128;
  static_assert(O_COL + 4 * NO <= 512 && SMEM + 1024 + 2048 <= 232448, "tensor memory, shared memory");
};

struct Args {
  Cache k;
  Batch b;
  const void* q;
  void* out;
  float* lse;
  int64_t qt, qh, ot, oh;
  int heads, subs, box, wide;   // subs: 128-byte columns of a latent; box: rows of a TMA box; wide: 16-byte loads of q
  int coarse;                   // a place is 1 << coarse units (more than one only where places would pass 2^31)
  Div by_heads, by_subs, by_blocks;
  float scale;
  int4* meta;                   // [blocks]: of a group that begins in the run before and goes on in this one, the runs that
                                // hold some of it (or 0), its first row, its rows
  float2* stat;                 // [R][2][MAX_CTAS]: ref, sum of the group's middle or end, of its beginning (side by side for the join)
  float* part;                  // [2 blocks][R][128 subs]
  int32_t* error;               // (or null) where a block whose wait ran out leaves its code
  uint64_t limit;               // of a wait, in ns
};

// ---- a block's share of the units ----------------------------------------------------------
// Runs are cut by cost, in places: a group costs its units and FIXED more (its queries, its first tile's maximum, its
// outputs; fitted: a unit 0.8 us, a group 4; 5 units cost 300 sequences of up to 4096 tokens 1 us of 89).
constexpr int FIXED = 4;
template <int R>
__device__ __forceinline__ int groups_of(const Args& a, const Seq& q) { return (q.n * a.heads + R - 1) / R; }
__device__ __forceinline__ int units_of(const Args& a, const Seq& q) { return max(1, (min(q.len, a.b.capacity) + UNIT - 1) / UNIT); }
__device__ __forceinline__ int places_of(const Args& a, int units) { return ((units - 1) >> a.coarse) + 1 + FIXED; }
__device__ __forceinline__ int begin_of(int total, int block, const Div& blocks) {
  const int each = total / blocks, more = total - each * blocks.d;
  return each * block + min(block, more);
}
// the block whose run holds place `at` < total
__device__ __forceinline__ int holder_of(int total, int at, int blocks) {
  const int each = (uint32_t)total / (uint32_t)blocks, more = total - each * blocks, wide = more * (each + 1);
  return at < wide ? (uint32_t)at / (uint32_t)(each + 1) : more + (uint32_t)(at - wide) / (uint32_t)max(each, 1);
}

struct Work {
  int b, g, at, left;           // the sequence, its group, the place in the group's cost, what is left of the run
};
struct Segment {
  Seq q;
  int s;                        // the sequence
  int r0, rows;                 // rows [r0, r0 + rows) of the sequence's n x heads
  int u0, u1, units;            // units [u0, u1) of the group's
  int end;                      // past the last token of this segment
  int tiles;
};

template <int R>
__device__ __forceinline__ bool next(const Args& a, Work& w, Segment& s) {
  while (w.left > 0 && w.b < a.b.n) {
    s.q = sequence(a.b, w.b);
    if (w.g >= groups_of<R>(a, s.q)) {
      ++w.b;
      w.g = 0;
      continue;
    }
    s.s = w.b;
    s.units = units_of(a, s.q);
    const int places = places_of(a, s.units), to = min(places, w.at + w.left);
    s.u0 = max(w.at - FIXED, 0) << a.coarse;
    s.u1 = min(max(to - FIXED, 0) << a.coarse, s.units);
    s.r0 = w.g * R;
    s.rows = min(R, s.q.n * a.heads - s.r0);
    w.left -= to - w.at;
    w.at = to;
    if (to == places) {
      ++w.g;
      w.at = 0;
    }
    if (s.u1 <= s.u0) continue;
    // past the tokens that its last row sees
    s.end = min(min(s.u1 * UNIT, a.b.capacity), s.q.len - s.q.n + (s.r0 + s.rows - 1) / a.by_heads + 1);
    s.tiles = max(0, (s.end - s.u0 * UNIT + TILE - 1) / TILE);
    return true;
  }
  return false;
}

// ---- tcgen05 -------------------------------------------------------------------------------
__device__ __forceinline__ uint64_t descriptor(uint32_t addr, uint32_t lead, uint32_t stride, uint64_t swizzle) {
  return (uint64_t)((addr >> 4) & 0x3FFF) | (uint64_t)(lead >> 4) << 16 | (uint64_t)(stride >> 4) << 32 | 1ull << 46 | swizzle << 61;
}
constexpr uint64_t SWIZZLE_NONE = 0, SWIZZLE_128 = 2, SWIZZLE_64 = 4;
// FP32 accumulators; types 0 E4M3, 1 E5M2; transposed: MN-major
__host__ __device__ constexpr uint32_t instruction(uint32_t b_type, bool transposed, uint32_t n) {
  return 1u << 4 | 0u << 7 | b_type << 10 | (transposed ? 3u << 15 : 0u) | (n >> 3) << 17 | (uint32_t)(TILE >> 4) << 24;
}
__device__ __forceinline__ uint32_t elect_one() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xFFFFFFFF;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
  return r;
}
// The whole warp calls these with the same operands and its elected lane issues: operands that the compiler has to make
// uniform out of one lane's branch cost 80 to 130 clocks a product, more than the product (32 + N / 4).
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t add, uint32_t elected) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %4, 0;\n\tsetp.ne.u32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(add), "r"(elected)
      : "memory");
}
__device__ __forceinline__ void commit(uint64_t* bar, uint32_t elected) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.u32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar)), "r"(elected)
      : "memory");
}
__device__ __forceinline__ void expect_bytes(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
// a box of a tensor map, brought by the elected lane (`issues`)
__device__ __forceinline__ void copy(uint32_t to, const CUtensorMap* map, int x, int y, uint32_t bar, uint32_t issues) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.u32 q, %5, 0;\n\t"
      "@q cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];\n\t}" ::"r"(to), "l"(map),
      "r"(x), "r"(y), "r"(bar), "r"(issues)
      : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// 8 or 16 columns of this warp's 32 lanes
__device__ __forceinline__ void tmem_load(uint32_t addr, float (&v)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7])
               : "r"(addr));
}
__device__ __forceinline__ void tmem_load(uint32_t addr, float (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]), "=f"(v[9]),
        "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15])
      : "r"(addr));
}
__device__ __forceinline__ void tmem_store(uint32_t addr, const float (&v)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(addr), "f"(v[0]), "f"(v[1]),
               "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7])
               : "memory");
}
__device__ __forceinline__ void tmem_store(uint32_t addr, const float (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(addr),
      "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]), "f"(v[8]), "f"(v[9]), "f"(v[10]),
      "f"(v[11]), "f"(v[12]), "f"(v[13]), "f"(v[14]), "f"(v[15])
      : "memory");
}
// (the loaded values may be used from here on)
template <int N, int M>
__device__ __forceinline__ void tmem_wait_load(float (&v)[N][M]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int i = 0; i < M; ++i) asm volatile("" : "+f"(v[n][i]));
}
__device__ __forceinline__ void tmem_wait_store() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Whether a barrier's phase is over. (mbarrier.try_wait may sleep, and woke up 700 to 2000 clocks late: 66 us for the 64
// sequences of up to 8192 tokens that took 55 without it.)
__device__ __forceinline__ bool come(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity & 1)
      : "memory");
  return ok != 0;
}
// A warp's wait of at most `limit` ns: false where it ran out.
__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, uint64_t limit) {
  bool ok = come(bar, parity);
  if (!ok) {
    const uint64_t begin = mk::globaltimer();
#pragma unroll 1
    do ok = come(bar, parity);
    while (!ok && mk::globaltimer() - begin <= limit);
  }
  return __all_sync(~0u, ok);
}

__device__ __forceinline__ void softmax_sync() { asm volatile("bar.sync 1, 256;" ::: "memory"); }
__device__ __forceinline__ bool softmax_any(bool v) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbarrier.cta.red.or.pred q, 1, 256, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"((uint32_t)v)
      : "memory");
  return r != 0;
}
__device__ __forceinline__ float exp2_fast(float v) {      // within 2^-22; below 2^-126: 0
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
// Of 32 lanes' v[N], lane l gets the whole of v[l % N].
template <int N, typename Op>
__device__ __forceinline__ float across(float (&v)[N], Op op) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int n = N / 2; n >= 1; n /= 2)
#pragma unroll
    for (int i = 0; i < n; ++i) {
      const bool up = lane & n;
      const float keep = up ? v[i + n] : v[i], give = up ? v[i] : v[i + n];
      v[i] = op(keep, __shfl_xor_sync(~0u, give, n));
    }
#pragma unroll
  for (int o = N; o < 32; o *= 2) v[0] = op(v[0], __shfl_xor_sync(~0u, v[0], o));
  return v[0];
}

__device__ __forceinline__ float lse_of(float ref, float sum) {
  return sum == 0.0f ? -INFINITY : (ref - X_SCALE + log2f(sum)) * 0.693147181f;
}

template <int R>
struct Shared {
  uint64_t full[2], empty[2], scored[2], taken[2], weighed[2], summed[2], asked, drained[2];
  uint32_t tmem;
  // A softmax thread's wait ran out: what the block has left to write becomes NaN, and it reports it. (Written by those threads alone,
  // with a barrier before each reading: they all leave a segment, or none does.)
  volatile int lost;
  volatile int late;            // a wait for the block's own copies or products ran out: reported
  float4 gran[2][TILE / 16];    // of each 16 tokens: sc, sr, log2 sc, 1 / sc (0: no such page)
  // of this segment and the next:
  float qc[2][R], qr[2][R];     // the rows' factors of the two accumulators, log2 e included
  int sees[2][R];               // the tokens that they see
  int64_t at[2][R];             // their outputs
  float red[4][R];              // of each 32 tokens
  float ref[R], inv[R];
};

// The W pieces of N weights x as bytes of E5M2, the upper byte of an FP16 value: x1 + x2 / 8 + x3 / 64 of x rounded to FP16
// or, with what that rounding took away, ... + x4 / 512 of x.
template <int W, int N>
__device__ __forceinline__ void pieces_of(const float (&x)[N], uint32_t (&p)[W][N / 4]) {
#pragma unroll
  for (int i = 0; i < N / 4; ++i) {
    uint32_t w[W][2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const float x0 = x[4 * i + 2 * k], x1 = x[4 * i + 2 * k + 1];
      __half2 v = __floats2half2_rn(x0, x1), rest;
      if constexpr (W == 4) {
        const float2 f = __half22float2(v);
        rest = __floats2half2_rn((x0 - f.x) * 64.0f, (x1 - f.y) * 64.0f);
      }
#pragma unroll
      for (int n = 0; n < W; ++n) {
        uint32_t u;
        memcpy(&u, &v, 4);
        u += 0x00800080u;       // to nearest: magnitudes stay below 2^15.8, so nothing carries over
        w[n][k] = u;
        if (n + 1 < W) {
          u &= 0xFF00FF00u;
          __half2 h;
          memcpy(&h, &u, 4);
          v = __hmul2(__hsub2(v, h), __float2half2_rn(8.0f));
          if constexpr (W == 4)
            if (n == 1) v = __hadd2(v, rest);
        }
      }
    }
#pragma unroll
    for (int n = 0; n < W; ++n) p[n][i] = __byte_perm(w[n][0], w[n][1], 0x7531);
  }
}

// Eight values from any address.
__device__ __noinline__ uint4 load_apart(const uint16_t* p) {
  return make_uint4(p[0] | (uint32_t)p[1] << 16, p[2] | (uint32_t)p[3] << 16, p[4] | (uint32_t)p[5] << 16, p[6] | (uint32_t)p[7] << 16);
}
__device__ __forceinline__ float2 unpack(__nv_bfloat162 v) { return __bfloat1622float2(v); }
__device__ __forceinline__ float2 unpack(__half2 v) { return __half22float2(v); }

// A segment's queries: each row's scales, and its values' pieces in the order that the products read (K-major, swizzled as
// TMA does it), zeros behind its values and in absent rows. x = q / scale_q has at most 448 and is exact in FP16 down to
// 2^-24. A row with an infinity or a NaN gets a NaN for its factor, which makes all its scores and outputs NaN.
template <typename T, int R>
__device__ __forceinline__ void ask(const Args& a, const Segment& s, uint8_t* smem, Shared<R>& sh, int set) {
  using C = Config<T, R>;
  using E2 = typename T::pair_type;
  constexpr int PER = SOFTMAX / R, EACH = 16 / PER;     // threads of a row, their eights of 128 latent values
  constexpr int N = 4 * EACH + 1;                       // a thread's eights: latents, and one of the rotary part
  const int row = threadIdx.x / PER, sub = threadIdx.x % PER, n = a.subs * EACH;
  const bool live = row < s.rows;
  const int f = s.r0 + (live ? row : 0), tok = f / a.by_heads;
  const uint16_t* q = static_cast<const uint16_t*>(a.q) + (s.q.row + tok) * a.qt + (f - tok * a.heads) * a.qh;
  union Eight { uint4 u; E2 e[4]; } v[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int at = i + 1 < N ? (sub + i * PER) * 8 : sub * 8;
    const bool there = live && (i + 1 < N ? at < a.k.d_c : sub < LD_R / 8 && at < a.k.d_r);
    const uint16_t* p = q + (i + 1 < N ? at : a.k.d_c + at);
    v[i].u = make_uint4(0, 0, 0, 0);
    if (a.wide) {
      if (there) v[i].u = *reinterpret_cast<const uint4*>(p);
    } else {
      if (there) v[i].u = load_apart(p);
    }
  }
  E2 most[2];
  memset(most, 0, sizeof(most));
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const E2 m = __hmax2_nan(__hmax2_nan(__habs2(v[i].e[0]), __habs2(v[i].e[1])), __hmax2_nan(__habs2(v[i].e[2]), __habs2(v[i].e[3])));
    most[i + 1 == N] = __hmax2_nan(most[i + 1 == N], m);
  }
  float inv[2];
#pragma unroll
  for (int part = 0; part < 2; ++part) {
    // (bits of values that are not negative have their order, a NaN's are above an infinity's)
    uint32_t u = __float_as_uint(unpack(most[part]).x);
    u = max(u, __float_as_uint(unpack(most[part]).y));
#pragma unroll
    for (int o = PER / 2; o > 0; o >>= 1) u = max(u, __shfl_xor_sync(~0u, u, o));
    // the smallest power of two with the largest <= 448 of it
    const int e2 = max((int)(u >> 23) - 127 - 8 + ((u & 0x7FFFFFu) > 0x600000u ? 1 : 0), -120);
    inv[part] = __uint_as_float((uint32_t)(127 - e2) << 23);
    if (sub == 0)
      (part ? sh.qr : sh.qc)[set][row] = u < 0x7F800000u ? __uint_as_float((uint32_t)(e2 + 127) << 23) * (a.scale * 1.44269504f) : __int_as_float(0x7FC00000);
  }
  // an eight's pieces to `to` and on, R rows of `width` bytes apart (R is a multiple of 16, so the swizzle is the same)
  const auto split = [](const Eight& v, float by, uint8_t* to, int width) {
    __half2 x[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 y = unpack(v.e[e]);
      x[e] = __floats2half2_rn(y.x * by, y.y * by);
    }
#pragma unroll
    for (int n = 0; n < C::PIECES; ++n) {
      uint32_t w[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        w[e] = __nv_cvt_halfraw2_to_fp8x2(x[e], __NV_SATFINITE, __NV_E4M3);
        if (n + 1 < C::PIECES) x[e] = __hmul2(__hsub2(x[e], __half2(__nv_cvt_fp8x2_to_halfraw2((uint16_t)w[e], __NV_E4M3))), __float2half2_rn(16.0f));
      }
      *reinterpret_cast<uint2*>(to + n * R * width) = make_uint2(w[0] | w[1] << 16, w[2] | w[3] << 16);
    }
  };
  // (16-byte cells, swizzled by the row)
  const auto cell = [](int eight, int by) { return (eight & 1) * 8 + ((eight >> 1 ^ by) << 4); };
#pragma unroll
  for (int i = 0; i + 1 < N; ++i) {
    if (i >= n) break;
    split(v[i], inv[0], smem + C::QC + i / EACH * (C::NS * 128) + row * 128 + cell(sub + i % EACH * PER, row & 7), 128);
  }
  if (sub < LD_R / 8) split(v[N - 1], inv[1], smem + C::QR + row * 64 + cell(sub, row >> 1 & 3), 64);
}

// ---- the attention -------------------------------------------------------------------------
template <typename T, int R>
__global__ void __launch_bounds__(THREADS, 1) attend_kernel(const __grid_constant__ Args a, const __grid_constant__ CUtensorMap map_c,
                                                             const __grid_constant__ CUtensorMap map_r) {
  using C = Config<T, R>;
  using E = typename T::half_type;
  extern __shared__ uint8_t raw[];
  __shared__ Shared<R> sh;
  uint8_t* smem = raw + ((1024 - (smem_u32(raw) & 1023)) & 1023);
  const uint32_t base = smem_u32(smem);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Cache& k = a.k;

  if (warp == 8) {
    if (lane < 2) {
      mbar_init(&sh.full[lane], LOADERS);
      mbar_init(&sh.empty[lane], 1);
      mbar_init(&sh.drained[lane], 1);
      mbar_init(&sh.scored[lane], 1);
      mbar_init(&sh.taken[lane], SOFTMAX / 32);
      mbar_init(&sh.weighed[lane], SOFTMAX / 32);
      mbar_init(&sh.summed[lane], 1);
    }
    if (lane == 0) {
      mbar_init(&sh.asked, SOFTMAX / 32);
      sh.lost = sh.late = 0;
      asm volatile("prefetch.tensormap [%0];" ::"l"(&map_c) : "memory");
      asm volatile("prefetch.tensormap [%0];" ::"l"(&map_r) : "memory");
    }
    mk::fence_barrier_init();
  }
  start_dependents();
  wait_predecessor();
  // (not before: a predecessor on this SM may still have to allocate tensor memory of its own)
  if (warp == 9) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&sh.tmem)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    fence_before();
  }
  // this block's run of the units, and its first segment: once for all roles (each by itself the first time: 11.4 us for one
  // sequence of 1027 tokens on the device, 11.3 so)
  Work work{};
  Segment s;
  int place, total = 0, lo = 0;
  {
    const auto count = [&](int i) {
      const Seq q = sequence(a.b, i);
      return groups_of<R>(a, q) * places_of(a, units_of(a, q));
    };
    const auto which = [&](int all) {
      total = all;
      return lo = begin_of(all, blockIdx.x, a.by_blocks);
    };
    locate<THREADS>(a.b.n, count, which, work.b, place);
    work.left = begin_of(total, blockIdx.x + 1, a.by_blocks) - lo;
    if (work.b < a.b.n) {
      const int places = places_of(a, units_of(a, sequence(a.b, work.b)));
      work.at = place;
      if (place >= places) {
        work.g = (uint32_t)place / (uint32_t)places;
        work.at = place - work.g * places;
      }
    }
  }
  const Work start = work;
  bool more = next<R>(a, work, s);
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = sh.tmem;
  int it = 0;                   // tiles so far

  if (warp == 8 || warp == 11) {
    // ---- loads: a tile's pages, and the scales of their tokens
    bool ok = true;
    // this loader's boxes: every other one (a box's first 16 tokens name its page)
    const int each = a.box / 16, loader = warp == 11;
    const uint32_t elected = elect_one();
    for (; ok && more; more = next<R>(a, work, s)) {
      for (int t = 0; t < s.tiles; ++t, ++it) {
        const int st = it & 1, pos0 = s.u0 * UNIT + t * TILE, pos = pos0 + 16 * lane;
        int page = -1;
        const bool mine = lane < TILE / 16 && lane / each % LOADERS == loader;
        if (mine && pos < s.end) {
          page = a.b.table[s.s * a.b.ldt + (pos >> k.shift)];
          if (page >= k.pages) page = -1;
        }
        const int rows = __popc(__ballot_sync(~0u, page >= 0 && lane % each == 0)) * a.box;
        const int y = (page << k.shift) + (pos & (k.page - 1));
        if (it >= 2 && !(ok = wait(&sh.empty[st], (it - 2) >> 1, a.limit))) break;
        const uint32_t to = base + st * STAGE, full = smem_u32(&sh.full[st]);
        if (lane == 0) expect_bytes(full, rows * (a.subs * 128 + LD_R));
        __syncwarp();
#pragma unroll 1
        for (int from = loader * each; from < TILE / 16; from += LOADERS * each) {
          const int at = __shfl_sync(~0u, y, from), named = __shfl_sync(~0u, page, from);
          const uint32_t issues = elected != 0 && named >= 0;
          copy(to + 4 * SUB + from * 16 * LD_R, &map_r, 0, at, full, issues);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (j >= a.subs) break;
            copy(to + j * SUB + from * 16 * 128, &map_c, j * 128, at, full, issues);
          }
        }
        if (mine) {
          float4 g = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
          if (page >= 0) {
            const float2 scale = *reinterpret_cast<const float2*>(k.scales + 2 * (int64_t)page);
            const float v = fmaxf(scale.x, 5.42101086e-20f);    // 2^-64: a page that was never written has scale 0
            g = make_float4(scale.x, scale.y, log2f(v), 1.0f / v);
          }
          sh.gran[st][lane] = g;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.full[st]);
      }
    }
    for (int i = max(it - 2, 0); i < it; ++i)                                      // no copy outlives the block
      if (!wait(&sh.full[i & 1], i >> 1, TIMEOUT_NS)) sh.late = 1;
  } else if (warp == 9) {
    // ---- scores
    constexpr uint32_t ASK = instruction(0, false, C::NS);
    const uint32_t elected = elect_one();
    const uint64_t latents = descriptor(base, 16, 1024, SWIZZLE_128), rotary = descriptor(base + 4 * SUB, 16, 512, SWIZZLE_64);
    const uint64_t q_c = descriptor(base + C::QC, 16, 1024, SWIZZLE_128), q_r = descriptor(base + C::QR, 16, 512, SWIZZLE_64);
    bool ok = true;
    int segments = 0;
    for (; ok && more; more = next<R>(a, work, s)) {
      if (s.tiles == 0) continue;
      ok = wait(&sh.asked, segments++, a.limit);
      for (int t = 0; t < s.tiles && ok; ++t, ++it) {
        const int st = it & 1, buf = it % C::BUFS;
        ok = (it < C::BUFS || wait(&sh.taken[buf], it / C::BUFS - 1, a.limit)) && wait(&sh.full[st], it >> 1, a.limit);
        if (!ok) break;
        fence_after();
        const uint32_t d = tmem + buf * 2 * C::NS;
        const uint64_t c = latents + (st * STAGE >> 4), r = rotary + (st * STAGE >> 4);
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) mma(d + C::NS, r + (kk * 32 >> 4), q_r + (kk * 32 >> 4), ASK, kk > 0, elected);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (j >= a.subs) break;
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            mma(d, c + ((j * SUB + kk * 32) >> 4), q_c + ((j * C::NS * 128 + kk * 32) >> 4), ASK, j > 0 || kk > 0, elected);
        }
        commit(&sh.scored[buf], elected);
      }
    }
    commit(&sh.drained[0], elected);
    if (!wait(&sh.drained[0], 0, TIMEOUT_NS)) sh.late = 1;
  } else if (warp == 10) {
    // ---- sums (a tile's weights come after its scores, so its stage is free once they are used)
    constexpr uint32_t SUM = instruction(1, true, C::NO);
    const uint32_t elected = elect_one();
    const uint64_t latents = descriptor(base, SUB, 1024, SWIZZLE_128), weights = descriptor(base + C::PB, 128, 2048, SWIZZLE_NONE);
    bool ok = true;
    if (lane == 0) {
      int4 m = make_int4(0, 0, 0, 0);
      if (start.b < a.b.n) {
        const Seq q = sequence(a.b, start.b);
        // the group's first unit is at place `first`: this run is the second that holds some of it, or not
        const int first = lo - start.at + FIXED, last = lo - start.at + places_of(a, units_of(a, q)) - 1;
        m = make_int4(0, q.row * a.heads + start.g * R, min(R, q.n * a.heads - start.g * R), 0);
        if (start.at > FIXED && blockIdx.x > 0 && begin_of(total, blockIdx.x - 1, a.by_blocks) <= first)
          m.x = min(holder_of(total, last, gridDim.x), (int)gridDim.x - 1) - (int)blockIdx.x + 2;
      }
      a.meta[blockIdx.x] = m;
    }
    __syncwarp();
    for (; ok && more; more = next<R>(a, work, s)) {
      for (int t = 0; t < s.tiles; ++t, ++it) {
        const int st = it & 1, n = s.end - (s.u0 * UNIT + t * TILE);       // tokens that count
        if (!(ok = wait(&sh.weighed[st], it >> 1, a.limit))) break;
        fence_after();
        const uint64_t v = latents + (st * STAGE >> 4), w = weights + (st * C::NO * 128 >> 4);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (j >= a.subs) break;
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            mma(tmem + C::O_COL + j * C::NO, v + ((j * SUB + kk * 4096) >> 4), w + (kk * 512 >> 4), SUM, kk > 0 || t > 0, elected && kk * 32 < n);
        }
        commit(&sh.empty[st], elected);
        commit(&sh.summed[st], elected);
      }
    }
    commit(&sh.drained[1], elected);
    if (!wait(&sh.drained[1], 0, TIMEOUT_NS)) sh.late = 1;
  } else {
    // ---- softmax: this thread's token of each tile for half of the rows, and its latent value of each 128
    constexpr int H = C::H, AHEAD = R == 16 ? 4 : 1;      // (32 rows' registers allow one column of the outputs at a time)
    const int tid = threadIdx.x, tok = tid % TILE, half = warp / 4;
    const uint32_t lanes = tmem + ((uint32_t)(warp % 4) * 32 << 16) + half * H;
    bool dead = false;
    const auto prepare = [&](const Segment& s, int set) {
      softmax_sync();           // what was in this set has been read
      if (tid < R) {
        const int f = s.r0 + tid, row = f / a.by_heads;
        sh.sees[set][tid] = tid < s.rows ? min(max(s.q.len - s.q.n + 1 + row, 0), a.b.capacity) : INT32_MAX;
        sh.at[set][tid] = (s.q.row + row) * a.ot + (f - row * a.heads) * a.oh;
      }
      if (s.tiles > 0 && !dead) {
        ask<T, R>(a, s, smem, sh, set);
        mk::fence_proxy_async_smem();
      }
      softmax_sync();
      if (s.tiles > 0 && !dead && lane == 0) mbar_arrive(&sh.asked);
    };
    float ref[H], l[H];
    Segment ahead;
    if (more) prepare(s, 0);
    for (int set = 0; more; set ^= 1) {
      const int first_sees = min(max(s.q.len - s.q.n + 1 + s.r0 / a.by_heads, 0), a.b.capacity);
      float qc[H], qr[H];
#pragma unroll
      for (int h = 0; h < H; ++h) {
        ref[h] = -FLT_MAX;
        l[h] = 0.0f;
        qc[h] = sh.qc[set][half * H + h];
        qr[h] = sh.qr[set][half * H + h];
      }
      for (int t = 0; t < s.tiles && !dead; ++t, ++it) {
        const int st = it & 1, buf = it % C::BUFS, pos0 = s.u0 * UNIT + t * TILE, pos = pos0 + tok;
        bool ok = wait(&sh.full[st], it >> 1, a.limit);
        const float4 g = sh.gran[st][tok >> 4];
        ok = wait(&sh.scored[buf], it / C::BUFS, a.limit) && ok;
        fence_after();
        const bool none = pos >= s.end || g.w == 0.0f;
        float v[H];
        {
          float sc[2 * C::PIECES][H];
#pragma unroll
          for (int p = 0; p < 2 * C::PIECES; ++p) tmem_load(lanes + buf * 2 * C::NS + p * R, sc[p]);
          tmem_wait_load(sc);
#pragma unroll
          for (int h = 0; h < H; ++h) {
            float x = sc[1][h], y = sc[C::PIECES + 1][h];
            if (C::PIECES == 3) {
              x = fmaf(sc[2][h], 0.0625f, x);
              y = fmaf(sc[C::PIECES + 2 * (C::PIECES == 3)][h], 0.0625f, y);
            }
            x = fmaf(x, 0.0625f, sc[0][h]) * g.x;
            y = fmaf(y, 0.0625f, sc[C::PIECES][h]) * g.y;
            v[h] = fmaf(x, qc[h], fmaf(y, qr[h], g.z));
          }
        }
        fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.taken[buf]);
        if (none) {
#pragma unroll
          for (int h = 0; h < H; ++h) v[h] = -INFINITY;
        } else if (pos >= first_sees) {
#pragma unroll
          for (int h = 0; h < H; ++h)
            if (pos >= sh.sees[set][half * H + h]) v[h] = -INFINITY;
        }
        bool rises = false;
#pragma unroll
        for (int h = 0; h < H; ++h) rises |= v[h] > ref[h] + RAISE;
        if (!ok) sh.lost = 1;
        if (softmax_any(rises || !ok)) {
          if (sh.lost) {
            dead = true;
            break;
          }
          float m[H], f[H];
#pragma unroll
          for (int h = 0; h < H; ++h) m[h] = v[h];
          // (a NaN is no largest value)
          sh.red[warp % 4][half * H + lane % H] = across<H>(m, [](float x, float y) { return fmaxf(x, y); });
          softmax_sync();
#pragma unroll
          for (int h = 0; h < H; ++h) {
            const int row = half * H + h;
            const float top = fmaxf(ref[h], fmaxf(fmaxf(sh.red[0][row], sh.red[1][row]), fmaxf(sh.red[2][row], sh.red[3][row])));
            f[h] = exp2_fast(ref[h] - top);
            l[h] *= f[h];
            ref[h] = top;
          }
          if (t > 0) {
            if (!wait(&sh.summed[st ^ 1], (it - 1) >> 1, a.limit)) sh.lost = 1;
            fence_after();
            for (int j = 0; j < a.subs; ++j) {
              float o[C::W][H];
#pragma unroll
              for (int p = 0; p < C::W; ++p) tmem_load(lanes + C::O_COL + j * C::NO + p * R, o[p]);
              tmem_wait_load(o);
#pragma unroll
              for (int p = 0; p < C::W; ++p) {
#pragma unroll
                for (int h = 0; h < H; ++h) o[p][h] *= f[h];
                tmem_store(lanes + C::O_COL + j * C::NO + p * R, o[p]);
              }
            }
            tmem_wait_store();
          }
        }
        {
          // (this stage's tile before has been summed, so its weights' place is free too)
          float x[H];
          uint32_t p[C::W][H / 4];
#pragma unroll
          for (int h = 0; h < H; ++h) {
            x[h] = exp2_fast(v[h] - (ref[h] - X_SCALE));
            l[h] = fmaf(x[h], g.w, l[h]);
          }
          pieces_of(x, p);
          // rows of the operand in 16s: [W R / 16][128 tokens][16]
          uint8_t* w = smem + C::PB + st * C::NO * 128 + tok * 16;
#pragma unroll
          for (int i = 0; i < C::W; ++i) {
            if constexpr (H == 8) *reinterpret_cast<uint2*>(w + i * 2048 + half * 8) = make_uint2(p[i][0], p[i][1]);
            else *reinterpret_cast<uint4*>(w + (i * 2 + half) * 2048) = make_uint4(p[i][0], p[i][1], p[i][2], p[i][3]);
          }
        }
        // 0 x NaN is NaN: what no row sees becomes zero, a NaN that only later rows see (their scores are NaN) too
        if ((none && tok < ((s.end - pos0 + 31) & ~31)) || (!none && pos >= first_sees)) {
          for (int j = half; j < a.subs; j += 2) {
            // (the lanes' rows begin in one bank: each begins at a cell of its own)
            uint8_t* const from = smem + st * STAGE + j * SUB + tok * 128;
            const auto cell = [&](int i) { return reinterpret_cast<uint4*>(from + (i ^ (tok & 7)) * 16); };
            if (none) {
#pragma unroll
              for (int i = 0; i < 8; ++i) *cell(i) = make_uint4(0, 0, 0, 0);
            } else {
              const auto clean = [](uint32_t x) { return x & ~((((x & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u) / 128 * 255); };
#pragma unroll 1
              for (int i = 0; i < 8; ++i) {
                const uint4 u = *cell(i);
                *cell(i) = make_uint4(clean(u.x), clean(u.y), clean(u.z), clean(u.w));
              }
            }
          }
        }
        mk::fence_proxy_async_smem();
        fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.weighed[st]);
      }
      // the next segment's queries are prepared while this one's last sum runs
      more = next<R>(a, work, ahead);
      if (more) prepare(ahead, set ^ 1);
      // ---- the segment's end: whole groups are finished, others leave their sums
      if (s.tiles > 0 && !dead && !wait(&sh.summed[(it - 1) & 1], (it - 1) >> 1, a.limit)) sh.lost = 1;
      fence_after();
      sh.red[warp % 4][half * H + lane % H] = across<H>(l, [](float x, float y) { return x + y; });
      if (tok == 0) {
#pragma unroll
        for (int h = 0; h < H; ++h) sh.ref[half * H + h] = ref[h];
      }
      softmax_sync();
      if (sh.lost) dead = true;
      const bool whole = s.u0 == 0 && s.u1 == s.units;
      const int64_t slot = (2 * (int64_t)blockIdx.x + (s.u0 == 0)) * R;
      if (tid < s.rows) {
        const float sum = dead ? __int_as_float(0x7FC00000) : sh.red[0][tid] + sh.red[1][tid] + sh.red[2][tid] + sh.red[3][tid];
        if (!whole) {
          a.stat[(tid * 2 + (s.u0 == 0)) * MAX_CTAS + blockIdx.x] = make_float2(sh.ref[tid], sum);
        } else if (a.lse) {
          a.lse[(int64_t)s.q.row * a.heads + s.r0 + tid] = lse_of(sh.ref[tid], sum);
        }
        sh.inv[tid] = sum == 0.0f ? 0.0f : 1.0f / sum;
      }
      softmax_sync();           // (what was read here may be written again from now on: the next segment may have no tile)
      const int rows = s.rows - half * H;
      E* out[H];
      float inv[H];
#pragma unroll
      for (int h = 0; h < H; ++h) {
        out[h] = static_cast<E*>(a.out) + sh.at[set][half * H + h] + tok;
        inv[h] = sh.inv[half * H + h];
      }
      float* part = a.part + (slot + half * H) * (a.subs * 128) + tok;
#pragma unroll AHEAD
      for (int j = 0; j < 4; ++j) {
        if (j >= a.subs) break;
        float o[C::W][H];
#pragma unroll
        for (int p = 0; p < C::W; ++p)
#pragma unroll
          for (int h = 0; h < H; ++h) o[p][h] = 0.0f;
        if (s.tiles > 0) {
#pragma unroll
          for (int p = 0; p < C::W; ++p) tmem_load(lanes + C::O_COL + j * C::NO + p * R, o[p]);
          tmem_wait_load(o);
        }
#pragma unroll
        for (int p = C::W - 1; p > 0; --p)
#pragma unroll
          for (int h = 0; h < H; ++h) o[p - 1][h] = fmaf(o[p][h], 0.125f, o[p - 1][h]);
        if (!whole) {
#pragma unroll
          for (int h = 0; h < H; ++h)
            if (h < rows) part[h * (a.subs * 128) + j * 128] = o[0][h];
        } else if (j * 128 + tok < k.d_c) {
#pragma unroll
          for (int h = 0; h < H; ++h)
            if (h < rows) out[h][j * 128] = from_f32<E>(o[0][h] * inv[h]);      // (what no token adds to is 0 x 0)
        }
      }
      fence_before();
      s = ahead;
    }
  }
  __syncwarp();
  __syncthreads();
  if (threadIdx.x == 0 && (sh.lost || sh.late) && a.error) *a.error = MK_DERR_WAIT_TIMEOUT;
  if (warp == 9) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
}

// The groups that several blocks' runs share: a job is 128 latent values of one row of one, the partial sums of all its runs
// in their order, by one warp or, where there are fewer jobs than warps, by up to 8 of a block with a share of the runs each.
constexpr int MERGE_WARPS = 8;
template <typename T, int R, int SIDE>          // SIDE: the parts that a warp reads side by side, of 128 / SIDE values each
__device__ __forceinline__ void join(const Args& a, const int4* groups, int n_groups, float (*weights)[MAX_CTAS], float4 (*sums)[32]) {
  using E = typename T::half_type;
  constexpr int LANES = 32 / SIDE;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, ld = a.subs * 128, jobs = n_groups * R * a.subs * SIDE;
  int warps = 1;
  while (warps < MERGE_WARPS && 2 * warps * jobs <= (int)gridDim.x * MERGE_WARPS) warps *= 2;
  const int teams = MERGE_WARPS / warps, team = warp / warps, share = warps * SIDE, part = warp % warps * SIDE + lane / LANES;
#pragma unroll 1
  for (int first = blockIdx.x * teams; first < jobs; first += gridDim.x * teams) {
    const int job = min(first + team, jobs - 1), row = job % R, rest = job / R, group = rest / SIDE / a.by_subs;
    const int4 g = groups[group];
    const int n = first + team < jobs && row < g.z ? g.x : 0, dim = (rest - group * a.subs * SIDE) * (128 / SIDE) + lane % LANES * 4;
    // the first part begins the group (its block's second place), the others continue it
    const float2* stat = a.stat + row * 2 * MAX_CTAS + g.w - 1;
    const float* parts = a.part + ((int64_t)2 * (g.w - 1) * R + row) * ld + dim;
    const auto place = [&](int p) { return (2 * p + (p == 0)) * R; };
    const auto load = [&](int p) { return *reinterpret_cast<const float4*>(parts + place(p) * ld); };
    // several parts at a time, the first on their way before their weights are known (a loop's rest would wait for each)
    constexpr int AT_ONCE = SIDE == 1 ? 4 : 5;
    float4 v[AT_ONCE];
    const auto fetch = [&](int from) {
#pragma unroll
      for (int k = 0; k < AT_ONCE; ++k) {
        v[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (from + k * share < n) v[k] = load(from + k * share);
      }
    };
    fetch(part);
    constexpr int CHUNKS = (MAX_CTAS + 31) / 32;
    float2 st[CHUNKS];
    float ref = -FLT_MAX, l = 0.0f;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      st[c] = make_float2(-FLT_MAX, 0.0f);
      if (c * 32 + lane < n) st[c] = stat[c * 32 + lane + (c * 32 + lane == 0 ? MAX_CTAS : 0)];
    }
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) ref = fmaxf(ref, st[c].x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ref = fmaxf(ref, __shfl_xor_sync(~0u, ref, o));
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c)
      if (c * 32 + lane < n) {
        const float w = exp2_fast(st[c].x - ref);
        weights[warp][c * 32 + lane] = w;
        l = fmaf(w, st[c].y, l);
      }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(~0u, l, o);
    __syncwarp();
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    const auto add = [&](float w, const float4& x) {
      o.x = fmaf(w, x.x, o.x);
      o.y = fmaf(w, x.y, o.y);
      o.z = fmaf(w, x.z, o.z);
      o.w = fmaf(w, x.w, o.w);
    };
    for (int from = part; from < n; from += AT_ONCE * share) {
      float4 now[AT_ONCE];
#pragma unroll
      for (int k = 0; k < AT_ONCE; ++k) now[k] = v[k];
      fetch(from + AT_ONCE * share);
#pragma unroll
      for (int k = 0; k < AT_ONCE; ++k)
        if (from + k * share < n) add(weights[warp][from + k * share], now[k]);
    }
    __syncwarp();
#pragma unroll
    for (int x = LANES; x < 32; x *= 2) {
      o.x += __shfl_xor_sync(~0u, o.x, x);
      o.y += __shfl_xor_sync(~0u, o.y, x);
      o.z += __shfl_xor_sync(~0u, o.z, x);
      o.w += __shfl_xor_sync(~0u, o.w, x);
    }
    if (warps > 1) {
      sums[warp][lane] = o;
      __syncthreads();
      o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      for (int w = 0; w < warps; ++w) add(1.0f, sums[team * warps + w][lane]);
      __syncthreads();
    }
    if (n == 0 || part > 0) continue;
    const int f = g.y + row, tok = f / a.by_heads;
    if (a.lse && dim == 0) a.lse[f] = lse_of(ref, l);
    E* out = static_cast<E*>(a.out) + tok * a.ot + (f - tok * a.heads) * a.oh + dim;
    const float inv = l == 0.0f ? 0.0f : 1.0f / l, x[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (dim + e < a.k.d_c) out[e] = from_f32<E>(x[e] * inv);
  }
}

template <typename T, int R, int SIDE>
__global__ void __launch_bounds__(MERGE_WARPS * 32) merge_kernel(const Args a, int blocks) {
  static_assert(MAX_CTAS <= MERGE_WARPS * 32, "a thread for each block's run");
  __shared__ int4 groups[MAX_CTAS];                     // of each: the runs, the first row, the rows, the second run
  __shared__ int counts[MERGE_WARPS];
  __shared__ float weights[MERGE_WARPS][MAX_CTAS];
  __shared__ float4 sums[MERGE_WARPS][32];
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  start_dependents();
  wait_predecessor();
  int4 g = make_int4(0, 0, 0, 0);
  if (tid < blocks) g = a.meta[tid];
  g.w = tid;
  const uint32_t ballot = __ballot_sync(~0u, g.x > 0);
  if (lane == 0) counts[warp] = __popc(ballot);
  __syncthreads();
  int n_groups = 0, at = 0;
#pragma unroll
  for (int w = 0; w < MERGE_WARPS; ++w) {
    if (w == warp) at = n_groups;
    n_groups += counts[w];
  }
  if (g.x > 0) groups[at + __popc(ballot & ((1u << lane) - 1))] = g;
  __syncthreads();
  join<T, R, SIDE>(a, groups, n_groups, weights, sums);
}

// ---- the host's side -----------------------------------------------------------------------
int tensor_map(CUtensorMap* map, void* base, uint64_t cols, uint64_t rows, uint32_t box, CUtensorMapSwizzle swizzle) {
  using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                              const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static std::atomic<Encode> known{nullptr};
  Encode encode = known.load(std::memory_order_acquire);
  if (!encode) {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult q{};
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q) != cudaSuccess || !fn || q != cudaDriverEntryPointSuccess)
      return fail(MK_ECUDA, "cuTensorMapEncodeTiled is not available from the driver");
    encode = reinterpret_cast<Encode>(fn);
    known.store(encode, std::memory_order_release);
  }
  const cuuint64_t dims[2] = {cols, rows}, strides[1] = {cols};
  const cuuint32_t boxes[2] = {cols < 128 ? (cuuint32_t)cols : 128, box}, ones[2] = {1, 1};
  if (encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, base, dims, strides, boxes, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
    return fail(MK_EINVAL, "the codes make no tensor map");
  return MK_OK;
}

constexpr int MAX_DEVICES = 64;

cudaError_t multiprocessors(int device, int* n) {
  static std::atomic<int> known[MAX_DEVICES];
  *n = known[device].load(std::memory_order_relaxed);
  if (*n) return cudaSuccess;
  const cudaError_t e = cudaDeviceGetAttribute(n, cudaDevAttrMultiProcessorCount, device);
  if (e == cudaSuccess) known[device].store(*n, std::memory_order_relaxed);
  return e;
}

template <typename T, int R>
int launch(const Args& a, const CUtensorMap& c, const CUtensorMap& r, int device, int blocks, bool side, cudaStream_t s) {
  static std::atomic<bool> ready[MAX_DEVICES];   // the kernel may use that much shared memory on the device
  cudaError_t e = cudaSuccess;
  if (!ready[device].load(std::memory_order_acquire)) {
    e = cudaFuncSetAttribute(attend_kernel<T, R>, cudaFuncAttributeMaxDynamicSharedMemorySize, Config<T, R>::SMEM + 1024);
    if (e == cudaSuccess) ready[device].store(true, std::memory_order_release);
  }
  if (e == cudaSuccess) e = launch_early(attend_kernel<T, R>, dim3(blocks), THREADS, Config<T, R>::SMEM + 1024, s, a, c, r);
  if (e == cudaSuccess) e = launch_early(side ? merge_kernel<T, R, 4> : merge_kernel<T, R, 1>, dim3(2 * blocks), MERGE_WARPS * 32, 0, s, a, blocks);
  return e == cudaSuccess ? MK_OK : fail(MK_ECUDA, cudaGetErrorString(e));
}

constexpr int64_t META_BYTES = (MAX_CTAS * sizeof(int4) + 255) / 256 * 256;
// Rows of a group: 32 where sequences have 64 rows or more each and 16 would make 24 tiles a block or more, by the table's width:
// their tokens are brought and multiplied half as often (37 sequences at 4096, 128 heads: 79 us, with 16 rows 110; 512
// tokens of a prompt behind 3584: 137, with 16 178). 16 otherwise, whose scores have two buffers in tensor memory and whose
// runs start sooner (1 sequence at 8192, 128 heads: 16.4 us, with 32 rows 18.5), and with fewer rows a group of 32 is half
// empty (300 sequences of up to 4096, 16 heads: 82 us, with 32 rows 121). The lengths are the device's, so a table that is much wider
// than its sequences takes 32 rows sooner than they would: 8 sequences of up to 8192, 4 drafts each, behind 65536: 28 us, with 16 23.
// (Calls in a row in a captured graph, on the device.)
int rows_of_group(int64_t n, int64_t rows, int64_t heads, int64_t capacity) {
  return rows * heads >= 64 * n && rows * heads / 16 * (capacity / TILE) >= 24 * MAX_CTAS ? 32 : 16;
}
int64_t workspace(int rows, int subs) { return META_BYTES + (int64_t)2 * MAX_CTAS * rows * (2 + subs * 128) * 4; }

}  // namespace
}  // namespace latent

using namespace latent;

extern "C" int mk_latent_attend_workspace(const MkLatent* l, int32_t n, int32_t rows, int32_t heads, int64_t* bytes) {
  if (!l || !bytes || n < 0 || rows < 0 || heads < 1) return fail(MK_EINVAL, "null pointer or a negative size");
  *bytes = workspace(rows_of_group(n, rows, heads, 1 << 30), (l->d_c + 127) / 128);      // the most, whatever the table
  return MK_OK;
}

extern "C" int mk_latent_attend(const MkLatent* l, const MkLatentBatch* b, const void* q, int64_t qt, int64_t qh, int32_t rows,
                                int32_t heads, int32_t dtype, float scale, void* out, int64_t ot, int64_t oh, float* lse,
                                void* workspace, int64_t workspace_bytes, void* stream) {
  return mk_latent_attend_status(l, b, q, qt, qh, rows, heads, dtype, scale, out, ot, oh, lse, workspace, workspace_bytes, nullptr, 0, stream);
}

extern "C" int mk_latent_attend_status(const MkLatent* l, const MkLatentBatch* b, const void* q, int64_t qt, int64_t qh, int32_t rows,
                                       int32_t heads, int32_t dtype, float scale, void* out, int64_t ot, int64_t oh, float* lse,
                                       void* workspace, int64_t workspace_bytes, int32_t* error, int64_t wait_ns, void* stream) {
  Args a{};
  if (const int e = check(l, b, rows, dtype, a.k, a.b)) return e;
  if (heads < 1 || heads > 1024 || (int64_t)rows * heads > 1 << 30) return fail(MK_EINVAL, "heads are from 1 to 1024, rows x heads at most 2^30");
  if (wait_ns < 0 || (uintptr_t)error & 3) return fail(MK_EINVAL, "a negative limit or a misaligned error word");
  if (rows == 0 || b->n == 0) return MK_OK;
  if (!q || !out || !workspace) return fail(MK_EINVAL, "null pointer");
  if (((uintptr_t)q | (uintptr_t)out) & 1 || (uintptr_t)lse & 3 || (uintptr_t)workspace & 255)
    return fail(MK_EINVAL, "misaligned q, out, lse or workspace (256 bytes)");
  a.coarse = coarse_of(rows, heads, b->n, a.b.capacity, FIXED);
  if (a.coarse < 0) return fail(MK_EINVAL, "a call has at most 2^31 / 5 groups of 16 rows of a sequence");
  a.subs = a.k.ld_c / 128;
  const int group = rows_of_group(b->n, rows, heads, a.b.capacity);
  if (workspace_bytes < latent::workspace(group, a.subs)) return fail(MK_EINVAL, "the workspace is too small");
  int device = 0, sms = 0;
  if (cudaGetDevice(&device) != cudaSuccess || device < 0 || device >= MAX_DEVICES ||
      multiprocessors(device, &sms) != cudaSuccess)
    return fail(MK_ECUDA, "cudaGetDevice failed or device ordinal out of range");
  a.q = q;
  a.out = out;
  a.lse = lse;
  a.qt = qt;
  a.qh = qh;
  a.ot = ot;
  a.oh = oh;
  a.heads = heads;
  a.scale = scale;
  a.error = error;
  a.limit = wait_ns ? (uint64_t)wait_ns : TIMEOUT_NS;
  a.box = a.k.page < UNIT ? a.k.page : UNIT;
  a.wide = (uintptr_t)q % 16 == 0 && qt % 8 == 0 && qh % 8 == 0;
  a.by_heads = div_by(heads);
  a.by_subs = div_by(a.subs);
  a.meta = static_cast<int4*>(workspace);
  a.stat = reinterpret_cast<float2*>(static_cast<char*>(workspace) + META_BYTES);
  a.part = reinterpret_cast<float*>(a.stat + (int64_t)2 * MAX_CTAS * group);
  CUtensorMap c, r;
  const uint64_t tokens = (uint64_t)a.k.pages * a.k.page;
  if (const int e = tensor_map(&c, a.k.c, a.k.ld_c, tokens, a.box, CU_TENSOR_MAP_SWIZZLE_128B)) return e;
  if (const int e = tensor_map(&r, a.k.r, LD_R, tokens, a.box, CU_TENSOR_MAP_SWIZZLE_64B)) return e;
  const int blocks = sms < MAX_CTAS ? sms : MAX_CTAS;
  a.by_blocks = div_by(blocks);
  // Few groups that may be shared by all runs, by the table's width: the join takes quarters of the columns, a warp reading 4
  // parts side by side, so that all of a row's are on their way at once (1 sequence at 32768: 13.1 us, without 14.4). Otherwise
  // not: few parts do not pay for it (1 sequence at 1027: 10.4 us, with it 11.0; 8 sequences of 4 drafts 22.9 and 26.3).
  const int64_t shared = (rows * (int64_t)heads + b->n * (int64_t)(group - 1)) / group;
  const bool side = 4 * shared * group * a.subs <= 2 * blocks && a.b.capacity / UNIT + 1 > MAX_CTAS;
  const auto s = static_cast<cudaStream_t>(stream);
  // (FP16's three pieces of a query leave no room for 32 rows in tensor memory)
  if (dtype == MK_FP16) return launch<Fp16, 16>(a, c, r, device, blocks, side, s);
  return group == 32 ? launch<Bf16, 32>(a, c, r, device, blocks, side, s) : launch<Bf16, 16>(a, c, r, device, blocks, side, s);
}

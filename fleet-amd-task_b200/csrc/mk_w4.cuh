// mk_w4.cuh -- the 4-bit weight format and the warp-level pieces of its products (mk_w4.cu).
//
// A weight W [N, K] is 4-bit codes with one scale, and optionally one zero point, per row and group
// of 32, 64 or 128 values along K: W[n, k] = s[n, k / G] (q[n, k] - z[n, k / G]), z = 8 without zero
// points. Products sum exactly that: q - z is an integer of at most 5 bits (exact in BF16 and FP16),
// its product with a 16-bit activation is exact in FP32, a group is summed by the tensor cores in
// FP32 and the group's sum is multiplied by its scale in FP32. Nothing is rounded to 16 bits before
// the result: the experts' intermediate silu(g) u goes to the down projection as the sum of two BF16 values.
//
// The laid-out form (fleet/w4.py lay_out) is the order in which the lanes of a warp want the codes
// for mma.sync m16n8k16 with the weights as the 16-row operand and the tokens as its 8 columns. A
// strip is 32 rows (two tiles of 16), a unit 128 values of K:
//   codes  [experts][strips][units][2 tiles][2 chunks of 64][32 lanes][4 words]: lane 4 g + t, word
//          2 h + j (h, j in 0..1) holds the tile's rows g and g + 8 at the four values
//          k = 64 chunk + 32 h + 8 t + 4 j + (0..3): bits 4i..4i+3 (k even) and 16+4i.. (k odd) are,
//          for i = 0..3, (row g, k 0/1), (row g + 8, k 0/1), (row g, k 2/3), (row g + 8, k 2/3): the
//          four A registers of one MMA, two codes each, a shift and one AND-OR from a 16-bit float
//   scales [experts][strips][units][2 tiles][8][128 / G groups][2]: for g the groups' scales of rows g
//          and g + 8, one load a lane
//   zeros  the same, bytes, or none
// The MMA's k slots are a permutation of the values (lane t of a quad has 8 consecutive ones of each
// 32), the same one for the activations: a sum does not ask for their order, and a lane's share of
// the activations is then one 16-byte load per 32 values. Rows and K are padded to whole strips and
// units with scale 0 and activations 0.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace w4 {

constexpr int STRIP_ROWS = 32, UNIT_K = 128, TILE_UNIT_BYTES = 1024;   // a tile's codes of a unit

struct Bf16 {
  static constexpr uint32_t MAGIC = 0x43004300u;   // 128 + code in the low mantissa bits
  static __device__ __forceinline__ uint32_t sub2(uint32_t a, uint32_t b) {
    const __nv_bfloat162 d = __hsub2(reinterpret_cast<const __nv_bfloat162&>(a), reinterpret_cast<const __nv_bfloat162&>(b));
    return reinterpret_cast<const uint32_t&>(d);
  }
  static __device__ __forceinline__ float2 to_f32(uint32_t v) {
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xFFFF0000u));
  }
  static __device__ __forceinline__ float one_to_f32(uint16_t v) { return __uint_as_float((uint32_t)v << 16); }
  static __device__ __forceinline__ uint16_t round(float v) { return __bfloat16_as_ushort(__float2bfloat16_rn(v)); }
  static __device__ __forceinline__ uint32_t round2(float lo, float hi) { return (uint32_t)round(lo) | (uint32_t)round(hi) << 16; }
  static __device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                             uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
  // d = a b
  static __device__ __forceinline__ void mma0(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                              uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
  }
};

struct Fp16 {
  static constexpr uint32_t MAGIC = 0x64006400u;   // 1024 + code
  static __device__ __forceinline__ uint32_t sub2(uint32_t a, uint32_t b) {
    const __half2 d = __hsub2(reinterpret_cast<const __half2&>(a), reinterpret_cast<const __half2&>(b));
    return reinterpret_cast<const uint32_t&>(d);
  }
  static __device__ __forceinline__ float2 to_f32(uint32_t v) {
    return __half22float2(reinterpret_cast<const __half2&>(v));
  }
  static __device__ __forceinline__ float one_to_f32(uint16_t v) { return __half2float(__ushort_as_half(v)); }
  static __device__ __forceinline__ uint16_t round(float v) { return __half_as_ushort(__float2half_rn(v)); }
  static __device__ __forceinline__ uint32_t round2(float lo, float hi) { return (uint32_t)round(lo) | (uint32_t)round(hi) << 16; }
  static __device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                             uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
  // d = a b
  static __device__ __forceinline__ void mma0(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                              uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
  }
};

// v = hi + lo to 16 significant bits (2^-16 of v at most), in FP32's range: both are BF16. An infinity is
// hi alone, and so is what would round to one.
__device__ __forceinline__ void split_bf16(float v, uint32_t& hi, uint32_t& lo) {
  hi = __bfloat16_as_ushort(__float2bfloat16_rn(v));
  if ((hi & 0x7F80u) == 0x7F80u) hi = __float_as_uint(v) >> 16;
  const float rest = v - __uint_as_float(hi << 16);
  lo = isinf(v) ? 0u : (uint32_t)__bfloat16_as_ushort(__float2bfloat16_rn(rest));
}

// weights are read once: past L1
__device__ __forceinline__ uint4 ldg128(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
// N (1, 2 or 4) words
template <int N>
__device__ __forceinline__ void ldg_words(const void* p, uint32_t (&v)[N]) {
  if (N == 4) {
    const uint4 q = ldg128(p);
    v[0] = q.x, v[N > 1 ? 1 : 0] = q.y, v[N > 2 ? 2 : 0] = q.z, v[N > 3 ? 3 : 0] = q.w;
  } else if (N == 2) {
    asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0,%1}, [%2];" : "=r"(v[0]), "=r"(v[N > 1 ? 1 : 0]) : "l"(p));
  } else {
    asm volatile("ld.global.nc.L1::no_allocate.u32 %0, [%1];" : "=r"(v[0]) : "l"(p));
  }
}
__device__ __forceinline__ uint32_t ldg16(const void* p) {
  uint16_t v;
  asm volatile("ld.global.nc.L1::no_allocate.u16 %0, [%1];" : "=h"(v) : "l"(p));
  return v;
}
// activations that other CTAs of the launch's predecessor wrote
__device__ __forceinline__ uint4 ldg128_x(const void* p) {
  uint4 v;
  asm volatile("ld.global.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
__device__ __forceinline__ uint4 lds128(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at));
  return v;
}
__device__ __forceinline__ void cp16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// an 8 x 8 matrix of 16-bit values, lane 4 g + t holding columns 2 t, 2 t + 1 of row g, transposed
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(v));
  return d;
}

// (w & 0x000F000F) | magic in one instruction: the magic in a register (an instruction takes one
// immediate, and the compiler would otherwise spend two)
__device__ __forceinline__ uint32_t and_or(uint32_t w, uint32_t magic) {
  uint32_t d;
  asm("lop3.b32 %0, %1, 0x000F000F, %2, 0xEA;" : "=r"(d) : "r"(w), "r"(magic));
  return d;
}

template <class D>
__device__ __forceinline__ uint32_t magic_register() {
  uint32_t m;
  asm volatile("mov.b32 %0, %1;" : "=r"(m) : "n"(D::MAGIC));
  return m;
}

// one word's four A registers: codes to 16-bit floats, their zero points taken off (exact)
template <class D>
__device__ __forceinline__ void decode(uint32_t magic, uint32_t w, uint32_t z0, uint32_t z1, uint32_t (&a)[4]) {
  a[0] = D::sub2(and_or(w, magic), z0);
  a[1] = D::sub2(and_or(w >> 4, magic), z1);
  a[2] = D::sub2(and_or(w >> 8, magic), z0);
  a[3] = D::sub2(and_or(w >> 12, magic), z1);
}

// 32 values of K: two words against each column tile's 16 bytes of activations (of every plane: an
// activation is the sum of its planes); FIRST: acc = instead of acc +=
template <class D, int NT, int PLANES, bool FIRST>
__device__ __forceinline__ void half_chunk(uint32_t magic, uint32_t w0, uint32_t w1, uint32_t z0, uint32_t z1,
                                           const uint4 (&xb)[PLANES][NT], float (&acc)[NT][4]) {
  uint32_t a[4];
  decode<D>(magic, w0, z0, z1, a);
#pragma unroll
  for (int p = 0; p < PLANES; ++p)
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      if (FIRST && p == 0) D::mma0(acc[n], a[0], a[1], a[2], a[3], xb[p][n].x, xb[p][n].y);
      else D::mma(acc[n], a[0], a[1], a[2], a[3], xb[p][n].x, xb[p][n].y);
    }
  decode<D>(magic, w1, z0, z1, a);
#pragma unroll
  for (int p = 0; p < PLANES; ++p)
#pragma unroll
    for (int n = 0; n < NT; ++n) D::mma(acc[n], a[0], a[1], a[2], a[3], xb[p][n].z, xb[p][n].w);
}

// tot += scale (rows g, g + 8) * acc (CW: * cw, the columns' weights, of the columns that take part: an
// infinite scale or a NaN is not the others')
template <class D, int NT, bool CW>
__device__ __forceinline__ void fold(uint32_t scale, const float2 (&cw)[NT], const bool (&part)[NT][2], const float (&acc)[NT][4],
                                     float (&tot)[NT][4]) {
  const float2 s = D::to_f32(scale);
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    if (!CW || part[n][0]) {
      tot[n][0] = fmaf(CW ? s.x * cw[n].x : s.x, acc[n][0], tot[n][0]);
      tot[n][2] = fmaf(CW ? s.y * cw[n].x : s.y, acc[n][2], tot[n][2]);
    }
    if (!CW || part[n][1]) {
      tot[n][1] = fmaf(CW ? s.x * cw[n].y : s.x, acc[n][1], tot[n][1]);
      tot[n][3] = fmaf(CW ? s.y * cw[n].y : s.y, acc[n][3], tot[n][3]);
    }
  }
}

}  // namespace w4

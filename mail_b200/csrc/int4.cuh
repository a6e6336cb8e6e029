// 4-bit expert weights: the storage format and its register-level decoding.
//
//   W[n, k] = (q[n, k] - 8) * s[n, k / group],  q in 0..15
//
// Byte b of a weight row holds q[2b] in its low and q[2b + 1] in its high
// nibble; s is in the activations' 16-bit type. A 32-bit word so holds eight
// consecutive k, k0 in its lowest nibble. Masking 0x000f000f at shifts of 0,
// 4, 8 and 12 gives the pairs (k0, k4), (k1, k5), (k2, k6), (k3, k7), each
// nibble in the low mantissa bits of a 16-bit half; setting the exponent of
// 128 (bf16) or 1024 (fp16) there makes it the number 128 + q or 1024 + q,
// exactly, and one packed subtraction leaves q - 8. The activations are paired
// the same way, so the order of k inside a product does not matter.
#pragma once
#include "common.cuh"

namespace moe {
namespace u4 {

__device__ __forceinline__ uint32_t as_u32(__nv_bfloat162 v) { return *reinterpret_cast<uint32_t*>(&v); }
__device__ __forceinline__ uint32_t as_u32(__half2 v) { return *reinterpret_cast<uint32_t*>(&v); }
__device__ __forceinline__ __nv_bfloat162 as_bf162(uint32_t v) { return *reinterpret_cast<__nv_bfloat162*>(&v); }
__device__ __forceinline__ __half2 as_half2(uint32_t v) { return *reinterpret_cast<__half2*>(&v); }

// (v & mask) | bits in one instruction; written in C the two constants cost two.
__device__ __forceinline__ uint32_t and_or(uint32_t v, uint32_t mask, uint32_t bits) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(v), "r"(mask), "r"(bits));
  return r;
}

// The 16-bit activation types.
template <typename T>
struct Act;

template <>
struct Act<__nv_bfloat16> {
  static constexpr int kDtype = MOE_BF16;
  // q - 8 of word w: pairs (k0, k4), (k1, k5), (k2, k6), (k3, k7)
  static __device__ __forceinline__ void decode(uint32_t w, uint32_t (&p)[4]) {
    const __nv_bfloat162 off = as_bf162(0x43084308u);  // 136
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = as_u32(__hsub2(as_bf162(and_or(w >> (4 * i), 0x000f000fu, 0x43004300u)), off));
  }
  static __device__ __forceinline__ uint32_t scale2(uint32_t p, uint32_t s2) {
    return as_u32(__hmul2(as_bf162(p), as_bf162(s2)));
  }
  static __device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
  static __device__ __forceinline__ __nv_bfloat16 from_float(float v) { return __float2bfloat16_rn(v); }
  // d = a b, or d += a b
  static __device__ __forceinline__ void mma_first(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
  }
  static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};

template <>
struct Act<__half> {
  static constexpr int kDtype = MOE_F16;
  static __device__ __forceinline__ void decode(uint32_t w, uint32_t (&p)[4]) {
    // ten mantissa bits also hold a nibble four bits up: 1024 + 16 q, which a
    // packed fma turns into q - 8 (exact: 1024 / 16 + 8 = 72)
    const __half2 off = as_half2(0x64086408u);   // 1032
    const __half2 sixteenth = as_half2(0x2c002c00u), off16 = as_half2(0xd480d480u);  // 1 / 16, -72
    const uint32_t v = w >> 8;
    p[0] = as_u32(__hsub2(as_half2(and_or(w, 0x000f000fu, 0x64006400u)), off));
    p[1] = as_u32(__hfma2(as_half2(and_or(w, 0x00f000f0u, 0x64006400u)), sixteenth, off16));
    p[2] = as_u32(__hsub2(as_half2(and_or(v, 0x000f000fu, 0x64006400u)), off));
    p[3] = as_u32(__hfma2(as_half2(and_or(v, 0x00f000f0u, 0x64006400u)), sixteenth, off16));
  }
  static __device__ __forceinline__ uint32_t scale2(uint32_t p, uint32_t s2) {
    return as_u32(__hmul2(as_half2(p), as_half2(s2)));
  }
  static __device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
  static __device__ __forceinline__ __half from_float(float v) { return __float2half_rn(v); }
  // d = a b, or d += a b
  static __device__ __forceinline__ void mma_first(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
  }
  static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};

// Eight consecutive activations (16 bytes) as the pairs of decode().
__device__ __forceinline__ void pair_up(const uint4& v, uint32_t (&p)[4]) {
  p[0] = __byte_perm(v.x, v.z, 0x5410);
  p[1] = __byte_perm(v.x, v.z, 0x7632);
  p[2] = __byte_perm(v.y, v.w, 0x5410);
  p[3] = __byte_perm(v.y, v.w, 0x7632);
}

// silu(g) * u; for g below about -87, 1 + exp(-g) overflows and the quotient
// is 0, the limit of silu there.
__device__ __forceinline__ float silu_mul(float g, float u) { return __fdividef(g, 1.0f + __expf(-g)) * u; }

inline bool group_ok(int group) { return group == 32 || group == 64 || group == 128; }

}  // namespace u4
}  // namespace moe

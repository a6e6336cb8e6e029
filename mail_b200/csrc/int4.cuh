// 4-bit expert weights: the storage format and its register-level decoding.
//
//   W[n, k] = (q[n, k] - 8) * s[n, k / group],  q in 0..15
//
// Byte b of a weight row holds q[2b] in its low and q[2b + 1] in its high
// nibble; s is in the activations' 16-bit type. A 32-bit word so holds eight
// consecutive k, k0 in its lowest nibble. Masking a nibble in both halves of
// the word at once gives one of the pairs (k0, k4), (k1, k5), (k2, k6),
// (k3, k7). Put into the mantissas of two 16-bit numbers under an exponent
// that makes their step 1 it is the number M + q, exactly.
#pragma once
#include "common.cuh"

namespace moe {
namespace u4 {

__device__ __forceinline__ uint32_t as_u32(__nv_bfloat162 v) { return *reinterpret_cast<uint32_t*>(&v); }
__device__ __forceinline__ uint32_t as_u32(__half2 v) { return *reinterpret_cast<uint32_t*>(&v); }
__device__ __forceinline__ __nv_bfloat162 as_bf162(uint32_t v) { return *reinterpret_cast<__nv_bfloat162*>(&v); }
__device__ __forceinline__ __half2 as_half2(uint32_t v) { return *reinterpret_cast<__half2*>(&v); }

// (v & mask) | bits in one instruction; written in C the two constants cost two.
template <uint32_t MASK>
__device__ __forceinline__ uint32_t and_or(uint32_t v, uint32_t bits) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(v), "n"(MASK), "r"(bits));
  return r;
}

// The exponents that decode() sets, kept in registers: as constants they would
// be moved into one for each use.
struct Exponents {
  uint32_t first, rest;
};
template <uint32_t FIRST, uint32_t REST>
__device__ __forceinline__ Exponents held_exponents() {
  Exponents e;
  asm volatile("mov.b32 %0, %1;" : "=r"(e.first) : "n"(FIRST));
  asm volatile("mov.b32 %0, %1;" : "=r"(e.rest) : "n"(REST));
  return e;
}

// The 16-bit activation types.
template <typename T>
struct Act;

template <>
struct Act<__nv_bfloat16> {
  // (M + q) / kUnit of word w: pairs (k0, k4) with M = 128, from the lowest four
  // mantissa bits as they stand; (k1, k5), (k2, k6), (k3, k7) with M = 16, shifted
  // to the highest four. Left as it is, M costs no instruction for each weight;
  // kOffset, -(M + 8) / kUnit, multiplied by the same activations, takes it out
  // of the sums. The largest M + q of a group of 128 add up to less than 2^13, so
  // in units of 2^13 no group's sum overflows, whatever the activations are; at
  // the other end the unit costs sums 2^-136, an eighth of bf16's smallest step.
  static constexpr float kUnit = 8192.f;
  static __device__ __forceinline__ Exponents exponents() { return held_exponents<0x3c803c80u, 0x3b003b00u>(); }
  static __device__ __forceinline__ void decode(uint32_t w, const Exponents& e, uint32_t (&p)[4]) {
    p[0] = and_or<0x000f000fu>(w, e.first);
    p[1] = and_or<0x00780078u>(w >> 1, e.rest);
    p[2] = and_or<0x00780078u>(w >> 5, e.rest);
    p[3] = and_or<0x00780078u>(w >> 9, e.rest);
  }
  static constexpr uint32_t kOffset[4] = {0xbc88bc88u, 0xbb40bb40u, 0xbb40bb40u, 0xbb40bb40u};  // -136, -24, ..
  static __device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
  static __device__ __forceinline__ __nv_bfloat16 from_float(float v) { return __float2bfloat16_rn(v); }
  // d = a b + c, d = a b, d += a b
  static __device__ __forceinline__ void mma_from(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1,
                                                  const float (&c)[4]) {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
  }
  static __device__ __forceinline__ void mma_first(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    const float zero[4] = {0.f, 0.f, 0.f, 0.f};
    mma_from(d, a, b0, b1, zero);
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
  // M + q: ten mantissa bits take (k1, k5) as it stands, with M = 64; the other
  // pairs shifted to the highest four, with M = 16. (Sums of fp16 activations
  // are far from fp32's limits.)
  static constexpr float kUnit = 1.f;
  static __device__ __forceinline__ Exponents exponents() { return held_exponents<0x54005400u, 0x4c004c00u>(); }
  static __device__ __forceinline__ void decode(uint32_t w, const Exponents& e, uint32_t (&p)[4]) {
    p[0] = and_or<0x03c003c0u>(w << 6, e.rest);
    p[1] = and_or<0x00f000f0u>(w, e.first);
    p[2] = and_or<0x03c003c0u>(w >> 2, e.rest);
    p[3] = and_or<0x03c003c0u>(w >> 6, e.rest);
  }
  static constexpr uint32_t kOffset[4] = {0xce00ce00u, 0xd480d480u, 0xce00ce00u, 0xce00ce00u};  // -24, -72, ..
  static __device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
  static __device__ __forceinline__ __half from_float(float v) { return __float2half_rn(v); }
  // d = a b + c, d = a b, d += a b
  static __device__ __forceinline__ void mma_from(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1,
                                                  const float (&c)[4]) {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
  }
  static __device__ __forceinline__ void mma_first(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    const float zero[4] = {0.f, 0.f, 0.f, 0.f};
    mma_from(d, a, b0, b1, zero);
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

// Decoding of the 8-bit cache format (see q8_cache.cu for the format).
#pragma once
#include <stdint.h>

namespace sdv2 {
namespace q8 {

constexpr int kMinExp = -126;
constexpr int kNotFinite = -128;  // exponent byte of a vector that reads back as NaN

__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// Two bf16 copies of 2^e (-126 <= e <= 127), or of NaN.
__device__ __forceinline__ uint32_t scale_bits(int e, bool not_finite) {
  return not_finite ? 0x7FC07FC0u : static_cast<uint32_t>(e + 127) * 0x00800080u;
}

// Four bytes (sign above a 7-bit magnitude m) as two pairs of bf16 subnormals, +-m * 2^-133: a byte doubled and
// masked with 0x807F has its sign in bf16's sign bit and m in its seven fraction bits.
__device__ __forceinline__ void spread4(uint32_t w, uint32_t& lo, uint32_t& hi) {
  lo = __byte_perm(w, 0u, 0x1100) & 0x807F807Fu;
  hi = __byte_perm(w, 0u, 0x3322) & 0x807F807Fu;
}

// The values +-m * 2^-6 * scale of four bytes; every step is exact while the result is a normal bf16 number.
__device__ __forceinline__ void decode4(uint32_t w, uint32_t scale2, uint32_t& lo, uint32_t& hi) {
  spread4(w, lo, hi);
  lo = mul_bf16x2(mul_bf16x2(lo, 0x7F007F00u), scale2);  // 2^127 first: 2^(e+133) itself can pass bf16's range
  hi = mul_bf16x2(mul_bf16x2(hi, 0x7F007F00u), scale2);
}

}  // namespace q8
}  // namespace sdv2

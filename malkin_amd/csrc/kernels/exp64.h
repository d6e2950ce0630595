// 2^x in 64 bits by a table and a short series, for sums of probabilities.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <cfloat>

namespace mk {
namespace {

typedef uint32_t v2u __attribute__((ext_vector_type(2)));

// NaN counts as -inf, +inf as the largest float.
__device__ __forceinline__ float clean(float z) { return fminf(fmaxf(z, -INFINITY), FLT_MAX); }

// p f + c with c in scalar registers (left to itself the compiler copies the constant into the result first, and a power
// takes twice the instructions).
__device__ __forceinline__ double fma_s(double p, double f, double c) {
  double r;
  asm("v_fma_f64 %0, %1, %2, %3" : "=v"(r) : "v"(p), "v"(f), "s"(c));
  return r;
}

// 2^(d / 64) in two factors, by a table and a short series (Tang, Table-driven implementation of the exponential function,
// 1989): d = 64 n + j + g, |g| <= 1/2; the table has 2^(j / 64), and 2^(g / 64) is the series of
// e^x to x^4 (x = g ln 2 / 64 at most 0.0054: what follows is below 4e-14 of it). d is rounded by adding 1.5 * 2^52,
// whose low word then holds 64 n + j; a table entry's high word is kept less j << 14, so that adding that word << 14 puts
// n into the exponent. |d| < 64000.
constexpr int kTable = 64;
// 2^(j / 64), rounded, less j << 46 (j << 14 of the high word).
__device__ const uint64_t kPowers[kTable] = {
    0x3ff0000000000000, 0x3fefec9a3e778061, 0x3fefd9b0d3158574, 0x3fefc74518759bc8,
    0x3fefb5586cf9890f, 0x3fefa3ec32d3d1a2, 0x3fef9301d0125b51, 0x3fef829aaea92de0,
    0x3fef72b83c7d517b, 0x3fef635beb6fcb75, 0x3fef54873168b9aa, 0x3fef463b88628cd6,
    0x3fef387a6e756238, 0x3fef2b4565e27cdd, 0x3fef1e9df51fdee1, 0x3fef1285a6e4030b,
    0x3fef06fe0a31b715, 0x3feefc08b26416ff, 0x3feef1a7373aa9cb, 0x3feee7db34e59ff7,
    0x3feedea64c123422, 0x3feed60a21f72e2a, 0x3feece086061892d, 0x3feec6a2b5c13cd0,
    0x3feebfdad5362a27, 0x3feeb9b2769d2ca7, 0x3feeb42b569d4f82, 0x3feeaf4736b527da,
    0x3feeab07dd485429, 0x3feea76f15ad2148, 0x3feea47eb03a5585, 0x3feea23882552225,
    0x3feea09e667f3bcd, 0x3fee9fb23c651a2f, 0x3fee9f75e8ec5f74, 0x3fee9feb564267c9,
    0x3feea11473eb0187, 0x3feea2f336cf4e62, 0x3feea589994cce13, 0x3feea8d99b4492ed,
    0x3feeace5422aa0db, 0x3feeb1ae99157736, 0x3feeb737b0cdc5e5, 0x3feebd829fde4e50,
    0x3feec49182a3f090, 0x3feecc667b5de565, 0x3feed503b23e255d, 0x3feede6b5579fdbf,
    0x3feee89f995ad3ad, 0x3feef3a2b84f15fb, 0x3feeff76f2fb5e47, 0x3fef0c1e904bc1d2,
    0x3fef199bdd85529c, 0x3fef27f12e57d14b, 0x3fef3720dcef9069, 0x3fef472d4a07897c,
    0x3fef5818dcfba487, 0x3fef69e603db3285, 0x3fef7c97337b9b5f, 0x3fef902ee78b3ff6,
    0x3fefa4afa2a490da, 0x3fefba1bee615a27, 0x3fefd0765b6e4540, 0x3fefe7c1819e90d8,
};
struct Power {
  double factor, rest;  // their product is the power
};
__device__ __forceinline__ Power pow2(double d, const double* table) {
  constexpr double kRound = 0x1.8p52, k1 = 6.931471805599453094e-1 / 64;
  const double r = d + kRound, g = d - (r - kRound);
  const uint32_t word = (uint32_t)__builtin_bit_cast(uint64_t, r);
  v2u t = __builtin_bit_cast(v2u, table[word & (kTable - 1)]);
  t[1] += word << 14;
  double p = fma_s(g, k1 * k1 * k1 * k1 / 24, k1 * k1 * k1 / 6);
  p = fma_s(p, g, k1 * k1 / 2);
  p = fma_s(p, g, k1);
  return Power{__builtin_bit_cast(double, t), __builtin_fma(p, g, 1.0)};
}
// 2^(x c / 64) of it, x c as above, in one rounding less.
__device__ __forceinline__ Power pow2_of(double x, double c, const double* table) {
  constexpr double kRound = 0x1.8p52, k1 = 6.931471805599453094e-1 / 64;
  const double r = __builtin_fma(x, c, kRound), g = __builtin_fma(x, c, -(r - kRound));
  const uint32_t word = (uint32_t)__builtin_bit_cast(uint64_t, r);
  v2u t = __builtin_bit_cast(v2u, table[word & (kTable - 1)]);
  t[1] += word << 14;
  double p = fma_s(g, k1 * k1 * k1 * k1 / 24, k1 * k1 * k1 / 6);
  p = fma_s(p, g, k1 * k1 / 2);
  p = fma_s(p, g, k1);
  return Power{__builtin_bit_cast(double, t), __builtin_fma(p, g, 1.0)};
}
// The table to LDS, where lanes read entries of their own; a barrier follows before its first use.
__device__ __forceinline__ void load_table(double* table) {
  if (threadIdx.x < kTable) table[threadIdx.x] = __builtin_bit_cast(double, kPowers[threadIdx.x]);
}

}  // namespace
}  // namespace mk

// Weights exp((x - max) / temperature) of a vocabulary in 64 bits: what the verification of drafts and the truncated sampling
// share.
#pragma once
#include "q35_common.h"
#include "q35hip.h"

namespace q35 {

// 2^(z / 32) for z <= 0 to 2e-12 relative: z = 32 n + j + r with |r| <= 1/2, as 2^n 2^(j / 32) 2^(r / 32): a table in LDS (32
// entries of 8 bytes, one pair of banks each: no conflicts) and the Taylor series of e^(r ln 2 / 32) to r^4 (the rest is
// below (ln 2 / 64)^5 / 5! = 1.3e-12; z's own rounding adds 2^-53 |z| / 32). 11 operations of 64 bits where a series over
// |f| <= 1/2 to f^9 takes 14: they come on top of the loads in the passes over the vocabulary (statistics of 32 rows of up to
// 8 drafts: 28.7 us with 14, 26.3 with 11, 19.3 with one).
constexpr int kVTab = 32;
__device__ __forceinline__ double exp2_neg(double z, const double* tab) {
  constexpr double c1 = 0.69314718055994530942 / kVTab, c2 = c1 * c1 / 2.0, c3 = c1 * c2 / 3.0, c4 = c1 * c3 / 4.0;
  z = fmax(z, -1100.0 * kVTab);  // 0 from there on, also for -inf
  const double n = __builtin_rint(z), r = z - n;
  const int k = (int)n;
  const double e = __builtin_fma(__builtin_fma(__builtin_fma(__builtin_fma(c4, r, c3), r, c2), r, c1), r, 1.0);
  return __builtin_ldexp(e * tab[k & (kVTab - 1)], k >> 5);
}
// Threads 0 .. 31 fill the table (a barrier before its use is the caller's): the series of 2^f to f^13, |f| <= 1/2.
__device__ __forceinline__ void exp2_table(double* tab, int tid) {
  if (tid >= kVTab) return;
  constexpr double L = 0.69314718055994530942;
  const bool up = 2 * tid > kVTab;
  const double f = (double)(up ? tid - kVTab : tid) * (L / kVTab);
  double e = 1.0;
#pragma unroll
  for (int k = 13; k > 0; --k) e = __builtin_fma(e * (1.0 / k), f, 1.0);
  tab[tid] = up ? 2.0 * e : e;
}
// exp((x - m) / T) for x <= m (no NaN), inv_t = 32 log2(e) / T: 1 at the maximum, also an infinite one.
__device__ __forceinline__ double v_weight(float x, float m, double inv_t, const double* tab) {
  return x == m ? 1.0 : exp2_neg(((double)x - (double)m) * inv_t, tab);
}
// A NaN counts as -inf.
__device__ __forceinline__ float v_clean(float x) { return fmaxf(x, -INFINITY); }

__device__ __forceinline__ int wave_min_i32(int v) {
#pragma unroll
  for (int o = 32; o; o >>= 1) v = min(v, __shfl_xor(v, o));
  return v;
}

}  // namespace q35

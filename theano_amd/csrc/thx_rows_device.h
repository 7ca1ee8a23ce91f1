// Device-side helpers of the row operators (thx_layernorm.cpp, thx_vocab.cpp).
#pragma once

#include "kernels/thx_common.h"

namespace thx {

// What sums, statistics and probabilities of T data are computed in.
template <class T> struct AccOf { typedef float type; };
template <> struct AccOf<double> { typedef double type; };

// Elements of a 16-byte vector.
template <class T> struct Width { enum { value = 16 / (int)sizeof(T) }; };

// The value of a lane's partner in step STEP (1, 2, 4 ... 32, in this order) of a reduction over 2 * STEP lanes.  Within
// 16 lanes a permutation on the way into the vector unit instead of a round trip through LDS; for steps 4 and 8 it
// mirrors 8 and 16 lanes, which reaches the other half as well, and the lanes of a half hold the same value by then.
template <int STEP>
THX_DEV int partner_bits(int v) {
  if constexpr (STEP == 1) return __builtin_amdgcn_update_dpp(0, v, 0xB1, 0xf, 0xf, true);
  else if constexpr (STEP == 2) return __builtin_amdgcn_update_dpp(0, v, 0x4E, 0xf, 0xf, true);
  else if constexpr (STEP == 4) return __builtin_amdgcn_update_dpp(0, v, 0x141, 0xf, 0xf, true);
  else if constexpr (STEP == 8) return __builtin_amdgcn_update_dpp(0, v, 0x140, 0xf, 0xf, true);
  else return __shfl_xor(v, STEP, 64);
}
template <int STEP>
THX_DEV float partner(float v) { return __int_as_float(partner_bits<STEP>(__float_as_int(v))); }
template <int STEP>
THX_DEV double partner(double v) {
  const long long b = __double_as_longlong(v);
  const unsigned lo = (unsigned)partner_bits<STEP>((int)b), hi = (unsigned)partner_bits<STEP>((int)(b >> 32));
  return __longlong_as_double((long long)(((unsigned long long)hi << 32) | lo));
}

// Sum and maximum over LANES neighbouring lanes, in every one of them.  All lanes of the wave take part.
template <int LANES, class A>
THX_DEV A lanes_sum(A v) {
  if constexpr (LANES >= 2) v += partner<1>(v);
  if constexpr (LANES >= 4) v += partner<2>(v);
  if constexpr (LANES >= 8) v += partner<4>(v);
  if constexpr (LANES >= 16) v += partner<8>(v);
  if constexpr (LANES >= 32) v += partner<16>(v);
  if constexpr (LANES >= 64) v += partner<32>(v);
  return v;
}
THX_DEV float larger(float a, float b) { return __builtin_fmaxf(a, b); }
THX_DEV double larger(double a, double b) { return __builtin_fmax(a, b); }
template <class A>
THX_DEV A wave_largest(A v) {
  v = larger(v, partner<1>(v));
  v = larger(v, partner<2>(v));
  v = larger(v, partner<4>(v));
  v = larger(v, partner<8>(v));
  v = larger(v, partner<16>(v));
  return larger(v, partner<32>(v));
}

// A vector of a large result: past the caches where nothing reads it soon.
template <class T, int V>
THX_DEV void store_out(T* p, const Vec<T, V>& v, bool nt) {
  if (nt) store_vec<T, V, true, true>(p, v);
  else store_vec<T, V, false, true>(p, v);
}

// The compiler forgets what it knows about a vector's values: without this it keeps single-precision copies of a row's
// elements from the first use to the second, which is twice the registers.
template <class T, int V>
THX_DEV void forget(Vec<T, V>& v) {
  thx_u32x4& raw = *(thx_u32x4*)&v;
  asm volatile("" : "+v"(raw));
}

}  // namespace thx

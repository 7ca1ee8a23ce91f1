// Device-side helpers of the row operators (thx_layernorm.cpp, thx_vocab.cpp).
#pragma once

#include "kernels/thx_common.h"

namespace thx {

// What sums, statistics and probabilities of T data are computed in.
template <class T> struct AccOf { typedef float type; };
template <> struct AccOf<double> { typedef double type; };

// Elements of a 16-byte vector.
template <class T> struct Width { enum { value = 16 / (int)sizeof(T) }; };

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

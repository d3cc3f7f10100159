// Shared device code of the log-probability kernels: a row's running softmax
// statistics, and vector accesses at element alignment.
#pragma once

#include "nq_common.hpp"

namespace nq {

// 8 consecutive elements at any element's address, as fp32 (unaligned-access mode:
// still one or two 16-byte loads).
template <typename T> struct Any8;
template <> struct Any8<bf16> { typedef __bf16 type __attribute__((ext_vector_type(8), aligned(2))); };
template <> struct Any8<float> { typedef float type __attribute__((ext_vector_type(8), aligned(4))); };

template <typename T, bool STREAM = false>
__device__ __forceinline__ floatx8 load8_any(const T* p) {
  const auto* q = reinterpret_cast<const typename Any8<T>::type*>(p);
  return __builtin_convertvector(STREAM ? __builtin_nontemporal_load(q) : *q, floatx8);
}
// Written once and not read here again: past the caches.
template <typename T>
__device__ __forceinline__ void store8_stream(T* p, floatx8 v) {
  typedef T V8 __attribute__((ext_vector_type(8)));
  typedef typename Any8<T>::type A8;
  __builtin_nontemporal_store((A8)__builtin_convertvector(v, V8), reinterpret_cast<A8*>(p));
}

// The maximum m of a set of values and l = sum of 2^((x - m) c) over it; (-inf, 0) for
// nothing.  A NaN or +inf among the values makes l NaN; a set of -inf has l 0.
struct RowStat {
  float m, l;
};
__device__ __forceinline__ float finite_max(float m) { return m == -INFINITY ? 0.f : m; }
__device__ __forceinline__ RowStat join(RowStat a, RowStat b, float c) {
  const float m = fmaxf(a.m, b.m), base = finite_max(m);
  return RowStat{m, a.l * fast_exp2((a.m - base) * c) + b.l * fast_exp2((b.m - base) * c)};
}

}  // namespace nq

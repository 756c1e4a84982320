// Scalar pieces of the linear-layer cross entropy of the kernels.
#pragma once
#include "common.cuh"
#include "math.cuh"

namespace kn {

// exp(v - m) for v <= m.  A masked score of -inf contributes 0 also when the whole row is masked
// (m = -inf); NaN stays NaN, so that it reaches the sum although the maximum skips it.
template <typename T> __device__ __forceinline__ T exp_from(T v, T m) {
  return v == -Math<T>::inf() ? (T)0 : Math<T>::exp_fast(v - m);
}

// d loss / d score of class v (0-based) without the factor g: softmax minus one-hot, 0 on a skipped
// instance whatever its scores are.
template <typename T> __device__ __forceinline__ T grad_score(T s, T hi, T lo, int32_t label, int64_t v) {
  const T p = Math<T>::exp_fast((s - hi) - lo);
  return label == 0 ? (T)0 : (label == v + 1 ? p - (T)1 : p);
}

// the factor of all gradients: dy, divided by the number of used instances for a mean
template <typename T> struct GradScale {
  const int32_t* count;        // null: no division
  T dy;
  __device__ __forceinline__ T value() const {
    if (!count) return dy;
    const int32_t c = __ldg(count);
    return c > 0 ? dy / (T)c : (T)0;
  }
};

}  // namespace kn

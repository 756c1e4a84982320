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

// lse as its rounded value and the remainder, and the loss lse - s[label], from an instance's maximum
// and sum, in Float64.  In this order log s survives beside a maximum of the type's lowest value (every
// class masked by it).  A label outside 0..V gives NaN.
template <typename T>
__device__ __forceinline__ T finish_instance(T m, double s, T label_score, int32_t label, int64_t V, T* lse_hi, T* lse_lo) {
  const double ls = ::log(s);
  const T hi = (T)((double)m + ls);
  *lse_hi = hi;
  *lse_lo = isfinite(hi) ? (T)(((double)m - (double)hi) + ls) : (T)0;
  if (label == 0) return (T)0;
  if (label < 0 || label > V) return (T)NAN;
  return (T)(((double)m - (double)label_score) + ls);
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

// the counter of the statistics kernel that follows in the stream
__device__ __forceinline__ void clear_done(uint32_t* done) {
  if (done && threadIdx.x == 0 && blockIdx.x == 0 && blockIdx.y == 0 && blockIdx.z == 0) *done = 0;
}

template <typename T> __device__ __forceinline__ T sum_parts(const T* p, int64_t stride, int parts) {
  T s = p[0];
  for (int k = 1; k < parts; k++) s += p[k * stride];
  return s;
}

}  // namespace kn

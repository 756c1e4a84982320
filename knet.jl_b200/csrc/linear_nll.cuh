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
    const int32_t c = *count;
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

// K scores v, v + STEP, ... of one instance: their parts in order, one part of all of them at a time so
// that the loads overlap, and the bias; -inf past the last class
template <typename T, int K, int STEP>
__device__ __forceinline__ void load_scores(T (&t)[K], const T* x, int64_t v, int64_t V, int64_t stride, int parts, const T* bias) {
#pragma unroll
  for (int k = 0; k < K; k++) t[k] = v + k * STEP < V ? x[v + k * STEP] : -Math<T>::inf();
  for (int p = 1; p < parts; p++) {
#pragma unroll
    for (int k = 0; k < K; k++)
      if (v + k * STEP < V) t[k] += x[p * stride + v + k * STEP];
  }
  if (bias) {
#pragma unroll
    for (int k = 0; k < K; k++)
      if (v + k * STEP < V) t[k] += bias[v + k * STEP];
  }
}

// total and count over the instances in a fixed order, by one CTA
template <typename T, int THREADS>
__device__ __forceinline__ void add_losses(const T* per_instance, const int32_t* labels, int64_t N, T* total, int32_t* count) {
  __shared__ double sd[32];
  __shared__ int sc[32];
  double a = 0.0;
  int c = 0;
  for (int64_t n0 = threadIdx.x; n0 < N; n0 += 8 * THREADS) {      // eight loads in flight
    T v[8];
    int32_t l[8];
#pragma unroll
    for (int k = 0; k < 8; k++) {
      const int64_t n = n0 + (int64_t)k * THREADS;
      l[k] = n < N ? labels[n] : 0;
      v[k] = n < N ? __ldcg(per_instance + n) : (T)0;
    }
#pragma unroll
    for (int k = 0; k < 8; k++)
      if (l[k] != 0) {
        a += (double)v[k];
        c++;
      }
  }
  a = block_reduce(a, [](double x, double y) { return x + y; }, 0.0, sd);
  c = block_reduce(c, [](int x, int y) { return x + y; }, 0, sc);
  if (threadIdx.x == 0) {
    *total = (T)a;
    *count = c;
  }
}
// the same by the last CTA of the grid to get here; `done` counts them
template <typename T, int THREADS>
__device__ __forceinline__ void last_adds_losses(const T* per_instance, const int32_t* labels, int64_t N, T* total,
                                                 int32_t* count, uint32_t* done) {
  __shared__ uint32_t last;
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) last = atomicAdd(done, 1u);
  __syncthreads();
  if (last + 1 != gridDim.x) return;
  __threadfence();
  add_losses<T, THREADS>(per_instance, labels, N, total, count);
}

}  // namespace kn

// The linear-layer cross entropy where the instances times the classes are few: the scores fit a small
// workspace, so a product leaves them there and a second kernel takes softmax statistics or gradients
// from them.  Which product depends on what bounds it:
//   few instances    W is read once at memory speed (row_dot or col_sum, by W's layout); tiles would
//                    waste all but a few of their rows
//   few outputs      64x64 tiles on the FMA pipe (Float64: on the FP64 tensor instruction) with the
//                    summed axis split over CTAs, as there are too few tiles for the SMs
// All of them leave sums as `parts`: [part of the summed axis][instance][column], added in order by
// the kernel that reads them.
#pragma once
#include "linear_nll.cuh"

namespace kn {

template <typename T> struct Strided {
  const T* p;
  int64_t si, sc;      // element (i, c) at p + i*si + c*sc
};

// ---- tiles ---------------------------------------------------------------------------------------
// acc(i, j) = sum_c A(i, c) * B(j, c) over a part of c, for a 64x64 tile of (i, j), c in steps through
// shared memory: four steps of 16 (Float64: 8) are in flight as asynchronous copies of single elements,
// which may go anywhere, so operands have any strides with one of the two equal to 1.  Float64 is bound by the FP64
// unit: loss and gradients of 10007x512, 2048 instances, 84 GFLOP, 3.27 ms (25.7 TFLOP/s; the library's largest product
// on this device reaches 35), Float32 at these sizes by latency (27 us for 1000x512, 512 instances).
constexpr int kTile = 64, kSimtThreads = 256, kSimtStages = 4;
template <typename T> constexpr int kStep = sizeof(T) == 8 ? 8 : 16;

// one element into shared memory, 0 where `in` is false (the address is then not read)
template <typename T> __device__ __forceinline__ void copy_element(T* dst, const T* src, bool in) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src),
               "n"((int)sizeof(T)), "r"(in ? (int)sizeof(T) : 0)
               : "memory");
}

// this thread's elements of one operand's steps: neighbouring threads walk the contiguous axis.  MASK: where
// the summed axis is the instances, x of a skipped one (label 0) is taken as 0, since its dS of 0 times what a
// padded batch holds there may be NaN.
template <typename T, bool MASK> struct TileCopy {
  static constexpr int S = kStep<T>, PER = S * kTile / kSimtThreads;
  const T* p[PER];
  uint32_t at[PER];            // places in a stage
  int c[PER];                  // summed index in a step; past any bound for a row outside
  int64_t advance;
  const int32_t* labels;       // of the summed indices from this part's first on, or null
  int32_t used[PER];           // the next step's
  __device__ __forceinline__ TileCopy(const Strided<T>& a, int64_t i0, int64_t c0, int64_t I, const int32_t* labels_, int64_t left)
      : advance(S * a.sc), labels(labels_ ? labels_ + c0 : nullptr) {
#pragma unroll
    for (int r = 0; r < PER; r++) {
      const int i = a.sc == 1 ? threadIdx.x / S + kSimtThreads / S * r : threadIdx.x % kTile;
      const int k = a.sc == 1 ? threadIdx.x % S : threadIdx.x / kTile + kSimtThreads / kTile * r;
      const bool in = i0 + i < I;
      p[r] = in ? a.p + (i0 + i) * a.si + (c0 + k) * a.sc : a.p;
      at[r] = (uint32_t)(k * (kTile + 4) + i);
      c[r] = in ? k : 1 << 30;
    }
    if constexpr (MASK) look(0, left);
  }
  __device__ __forceinline__ void look(int k, int64_t left) {
#pragma unroll
    for (int r = 0; r < PER; r++) used[r] = !labels || (c[r] < left && labels[(int64_t)k * S + c[r]] != 0);
  }
  // step k into `stage`; `left` summed indices remain from its first on
  __device__ __forceinline__ void start(T* stage, int k, int64_t left) {
#pragma unroll
    for (int r = 0; r < PER; r++) {
      const bool in = c[r] < left && (!MASK || used[r]);
      copy_element(stage + at[r], in ? p[r] + k * advance : p[r], in);
    }
    if constexpr (MASK) look(k + 1, left - S);
  }
};

// D += A * B for 8 x 8 doubles, 4 summed indices, by one warp: lane holds A(lane/4, lane%4),
// B(lane%4, lane/4) and D(lane/4, 2*(lane%4) + {0, 1})
__device__ __forceinline__ void dmma(double (&d)[2], double a, double b) {
  asm("mma.sync.aligned.m8n8k4.row.col.f64.f64.f64.f64 {%0, %1}, {%2}, {%3}, {%0, %1};" : "+d"(d[0]), "+d"(d[1]) : "d"(a), "d"(b));
}

template <typename T> struct TileShared {
  union {
    struct {
      T a[kSimtStages][kStep<T>][kTile + 4], b[kSimtStages][kStep<T>][kTile + 4];
    } in;
    T out[kTile][kTile + 1];
  };
};

template <typename T, bool MASK, typename Epi>
__global__ void __launch_bounds__(kSimtThreads, 3)
simt_product_kernel(Strided<T> a, Strided<T> b, const int32_t* mask_a, const int32_t* mask_b, int64_t I, int64_t J, int64_t C, int64_t c_part,
                    uint32_t* done, Epi epi) {
  chain_begin();
  clear_done(done);
  __shared__ __align__(16) TileShared<T> sh;
  const int ty = threadIdx.x / 16, tx = threadIdx.x % 16;
  const int64_t i0 = (int64_t)blockIdx.y * kTile, j0 = (int64_t)blockIdx.x * kTile;
  const int64_t c_lo = (int64_t)blockIdx.z * c_part, c_hi = min(C, c_lo + c_part);
  T acc[4][4];
#pragma unroll
  for (int u = 0; u < 4; u++)
#pragma unroll
    for (int w = 0; w < 4; w++) acc[u][w] = (T)0;
  // Float64: warp w owns rows 32*(w%2).. and columns 16*(w/2).. as 4 x 2 blocks of 8 x 8
  const int lane = threadIdx.x & 31, wr = (threadIdx.x >> 5 & 1) * 32, wc = (threadIdx.x >> 6) * 16;
  constexpr int S = kStep<T>;
  const int steps = (int)((c_hi - c_lo + S - 1) / S);
  TileCopy<T, MASK> ca(a, i0, c_lo, I, mask_a, c_hi - c_lo), cb(b, j0, c_lo, J, mask_b, c_hi - c_lo);
  auto start = [&](int k) {
    if (k < steps) {
      const int64_t left = c_hi - c_lo - (int64_t)k * S;
      ca.start(&sh.in.a[k % kSimtStages][0][0], k, left);
      cb.start(&sh.in.b[k % kSimtStages][0][0], k, left);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");      // empty past the last step, so that the count stays right
  };
#pragma unroll
  for (int k = 0; k < kSimtStages - 1; k++) start(k);
  for (int k = 0; k < steps; k++) {
    asm volatile("cp.async.wait_group %0;" ::"n"(kSimtStages - 2) : "memory");
    __syncthreads();                                          // step k has landed; step k - 1 has been used by all
    start(k + kSimtStages - 1);
    const int buf = k % kSimtStages;
    if constexpr (sizeof(T) == 8) {
#pragma unroll
      for (int c = 0; c < S; c += 4) {
        double av[4], bv[2];
#pragma unroll
        for (int u = 0; u < 4; u++) av[u] = sh.in.a[buf][c + (lane & 3)][wr + 8 * u + (lane >> 2)];
#pragma unroll
        for (int w = 0; w < 2; w++) bv[w] = sh.in.b[buf][c + (lane & 3)][wc + 8 * w + (lane >> 2)];
#pragma unroll
        for (int u = 0; u < 4; u++) {
          dmma(reinterpret_cast<double(&)[2]>(acc[u][0]), av[u], bv[0]);
          dmma(reinterpret_cast<double(&)[2]>(acc[u][2]), av[u], bv[1]);
        }
      }
    } else {
#pragma unroll
      for (int c = 0; c < S; c++) {
        T av[4], bv[4];
#pragma unroll
        for (int u = 0; u < 4; u++) av[u] = sh.in.a[buf][c][ty * 4 + u];
#pragma unroll
        for (int w = 0; w < 4; w++) bv[w] = sh.in.b[buf][c][tx * 4 + w];
#pragma unroll
        for (int u = 0; u < 4; u++)
#pragma unroll
          for (int w = 0; w < 4; w++) acc[u][w] = Math<T>::fma(av[u], bv[w], acc[u][w]);
      }
    }
  }
  if constexpr (sizeof(T) == 8) {      // from the blocks to 4 x 4 per thread, as the epilogues expect it
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();
#pragma unroll
    for (int u = 0; u < 4; u++)
#pragma unroll
      for (int w = 0; w < 2; w++)
#pragma unroll
        for (int e = 0; e < 2; e++) sh.out[wr + 8 * u + (lane >> 2)][wc + 8 * w + 2 * (lane & 3) + e] = acc[u][2 * w + e];
    __syncthreads();
#pragma unroll
    for (int u = 0; u < 4; u++)
#pragma unroll
      for (int w = 0; w < 4; w++) acc[u][w] = sh.out[ty * 4 + u][tx * 4 + w];
  }
  epi(acc, i0 + ty * 4, j0 + tx * 4, I, J);
}

// the sums of one part of c
template <typename T> struct PartsEpi {
  T* parts;
  __device__ __forceinline__ void operator()(T (&acc)[4][4], int64_t i0, int64_t j0, int64_t I, int64_t J) const {
    T* out = parts + (int64_t)blockIdx.z * I * J;
#pragma unroll
    for (int u = 0; u < 4; u++)
#pragma unroll
      for (int w = 0; w < 4; w++)
        if (i0 + u < I && j0 + w < J) out[(i0 + u) * J + j0 + w] = acc[u][w];
  }
};

// out(i, j) (+)= g * acc
template <typename T> struct StoreEpi {
  T* out;
  int64_t ld;
  int add;
  GradScale<T> g;
  __device__ __forceinline__ void operator()(T (&acc)[4][4], int64_t i0, int64_t j0, int64_t I, int64_t J) const {
    const T f = g.value();
#pragma unroll
    for (int u = 0; u < 4; u++) {
      if (i0 + u >= I) break;
#pragma unroll
      for (int w = 0; w < 4; w++) {
        if (j0 + w >= J) break;
        T* p = out + (i0 + u) * ld + j0 + w;
        const T v = acc[u][w] * f;
        *p = add ? *p + v : v;
      }
    }
  }
};

// ---- few instances ------------------------------------------------------------------------------------
// A matrix of `rows` rows of `cols` contiguous elements, pitch between rows, and NB vectors y.
template <typename T> struct Matrix {
  const T* p;
  int64_t rows, cols, pitch;
};

template <typename T, int VEC> __device__ __forceinline__ Pack<T, VEC> ld_cached(const T* p) {
  return *reinterpret_cast<const Pack<T, VEC>*>(p);
}

// parts[z part][n][row] = sum over a part of the columns of M(row, c) * y(n, c): a warp takes four
// rows, its lanes the columns; the vectors come through L1.  Bound by the one read of M: 50257x1024 Float32,
// one vector 33 us (6.2 TB/s), eight 54 us, where the vectors' loads and 8 FMAs per element show.
template <typename T, int NB, int VEC>
__global__ void __launch_bounds__(256, 2)
row_dot_kernel(Matrix<T> m, const T* y, int64_t ldy, int64_t N, int64_t c_part, uint32_t* done, T* parts) {
  chain_begin();
  clear_done(done);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t r0 = ((int64_t)blockIdx.x * 8 + warp) * 4;
  const int64_t n0 = (int64_t)blockIdx.y * NB;
  const int64_t c_lo = (int64_t)blockIdx.z * c_part, c_hi = min(m.cols, c_lo + c_part);
  if (r0 >= m.rows) return;
  T acc[4][NB];
#pragma unroll
  for (int r = 0; r < 4; r++)
#pragma unroll
    for (int n = 0; n < NB; n++) acc[r][n] = (T)0;
  const T* row[4];
#pragma unroll
  for (int r = 0; r < 4; r++) row[r] = m.p + min(r0 + r, m.rows - 1) * m.pitch;
  const T* yv[NB];
#pragma unroll
  for (int n = 0; n < NB; n++) yv[n] = y + min(n0 + n, N - 1) * ldy;
  constexpr int UN = NB >= 8 ? 1 : 2;              // packs per row in flight
  for (int64_t c = c_lo + lane * VEC; c < c_hi; c += 32 * VEC * UN) {
    Pack<T, VEC> w[UN][4];
#pragma unroll
    for (int u = 0; u < UN; u++)
#pragma unroll
      for (int r = 0; r < 4; r++)
        if (c + u * 32 * VEC < c_hi) w[u][r] = ld_stream<T, VEC>(row[r] + c + u * 32 * VEC);
#pragma unroll
    for (int u = 0; u < UN; u++)
      if (c + u * 32 * VEC < c_hi) {
#pragma unroll
        for (int n = 0; n < NB; n++) {
          const Pack<T, VEC> v = ld_cached<T, VEC>(yv[n] + c + u * 32 * VEC);
#pragma unroll
          for (int r = 0; r < 4; r++)
#pragma unroll
            for (int e = 0; e < VEC; e++) acc[r][n] = Math<T>::fma(w[u][r].v[e], v.v[e], acc[r][n]);
        }
      }
  }
#pragma unroll
  for (int n = 0; n < NB; n++)
#pragma unroll
    for (int r = 0; r < 4; r++) {
      const T s = warp_reduce(acc[r][n], [](T a, T b) { return a + b; });
      if (lane == 0 && r0 + r < m.rows && n0 + n < N) parts[((int64_t)blockIdx.z * N + n0 + n) * m.rows + r0 + r] = s;
    }
}

// the sums of the 8 warps of a CTA in warp 0: two warps at a time hand over to the others, so that two
// slots of shared memory suffice
template <typename T, int NB>
__device__ __forceinline__ void join_warps(T (&acc)[NB][4], T (*red)[NB][128]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int h = 6; h > 0; h -= 2) {                 // warps h, h+1 -> 0, 1
    __syncthreads();
    if (warp == h || warp == h + 1) {
#pragma unroll
      for (int n = 0; n < NB; n++)
#pragma unroll
        for (int e = 0; e < 4; e++) red[warp - h][n][e * 32 + lane] = acc[n][e];
    }
    __syncthreads();
    if (warp < 2) {
#pragma unroll
      for (int n = 0; n < NB; n++)
#pragma unroll
        for (int e = 0; e < 4; e++) acc[n][e] += red[warp][n][e * 32 + lane];
    }
  }
  __syncthreads();
  if (warp == 1) {
#pragma unroll
    for (int n = 0; n < NB; n++)
#pragma unroll
      for (int e = 0; e < 4; e++) red[0][n][e * 32 + lane] = acc[n][e];
  }
  __syncthreads();
  if (warp == 0) {
#pragma unroll
    for (int n = 0; n < NB; n++)
#pragma unroll
      for (int e = 0; e < 4; e++) acc[n][e] += red[0][n][e * 32 + lane];
  }
}

// parts[z part][n][col] = sum over a part of the rows of M(r, col) * y(n, r): a CTA takes 128 columns,
// its 8 warps share the rows; the vectors' entries come transposed through shared memory.  768x50257 Float32, eight
// vectors 51 us, 768x50256 Float64, one vector 70 us (4.4 TB/s): two CTAs of 128 registers, with the loads of a
// batch of rows issued before the batch in front of it is used.
constexpr int kColRows = 128;
template <typename T, int NB, int VEC>
__global__ void __launch_bounds__(256, 2)
col_sum_kernel(Matrix<T> m, const T* y, int64_t ldy, int64_t N, int64_t r_part, uint32_t* done, T* parts) {
  chain_begin();
  clear_done(done);
  constexpr int Q = 4 / VEC;                       // packs per thread: 4 columns
  constexpr int YV = NB < 16 / (int)sizeof(T) ? NB : 16 / (int)sizeof(T);
  __shared__ __align__(16) T ys[kColRows][NB];
  __shared__ __align__(16) T red[2][NB][128];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t j0 = (int64_t)blockIdx.x * 128, n0 = (int64_t)blockIdx.y * NB;
  const int64_t r_lo = (int64_t)blockIdx.z * r_part, r_hi = min(m.rows, r_lo + r_part);
  int64_t col[Q];
  bool in[Q];
#pragma unroll
  for (int q = 0; q < Q; q++) {
    col[q] = j0 + (lane + 32 * q) * VEC;
    in[q] = col[q] < m.cols;                        // cols is a multiple of VEC where VEC > 1
  }
  T acc[NB][4];
#pragma unroll
  for (int n = 0; n < NB; n++)
#pragma unroll
    for (int e = 0; e < 4; e++) acc[n][e] = (T)0;
  for (int64_t rc = r_lo; rc < r_hi; rc += kColRows) {
    __syncthreads();
    for (int k = threadIdx.x; k < kColRows * NB; k += 256) {
      const int n = k / kColRows, r = k % kColRows;
      ys[r][n] = rc + r < r_hi && n0 + n < N ? y[(n0 + n) * ldy + rc + r] : (T)0;
    }
    __syncthreads();
    // rows warp, warp + 8, ... of the 128, UN at a time, the next batch in flight while one is used
    constexpr int UN = (NB >= 8 ? 4 : 8) / (sizeof(T) / 4), BATCHES = kColRows / (8 * UN);
    Pack<T, VEC> w[2][UN][Q];
    // all rows and columns inside: no bounds, one address per row
    const bool full = j0 + 128 <= m.cols && rc + kColRows <= r_hi;
    const T* from = m.p + (rc + warp) * m.pitch + j0 + lane * VEC;
    auto fetch = [&](Pack<T, VEC> (&to)[UN][Q], int batch) {
      if (full) {
#pragma unroll
        for (int u = 0; u < UN; u++, from += 8 * m.pitch)
#pragma unroll
          for (int q = 0; q < Q; q++) to[u][q] = ld_stream<T, VEC>(from + q * 32 * VEC);
        return;
      }
#pragma unroll
      for (int u = 0; u < UN; u++)
#pragma unroll
        for (int q = 0; q < Q; q++) {
          const int64_t r = rc + warp + 8 * (batch * UN + u);
          if (in[q] && r < r_hi) to[u][q] = ld_stream<T, VEC>(m.p + r * m.pitch + col[q]);
          else
#pragma unroll
            for (int e = 0; e < VEC; e++) to[u][q].v[e] = (T)0;
        }
    };
    fetch(w[0], 0);
#pragma unroll
    for (int b = 0; b < BATCHES; b++) {
      if (b + 1 < BATCHES) fetch(w[(b + 1) & 1], b + 1);
#pragma unroll
      for (int u = 0; u < UN; u++) {
#pragma unroll
        for (int k = 0; k < NB; k += YV) {
          const Pack<T, YV> v = *reinterpret_cast<const Pack<T, YV>*>(&ys[warp + 8 * (b * UN + u)][k]);
#pragma unroll
          for (int n = 0; n < YV; n++)
#pragma unroll
            for (int q = 0; q < Q; q++)
#pragma unroll
              for (int e = 0; e < VEC; e++)
                acc[k + n][q * VEC + e] = Math<T>::fma(w[b & 1][u][q].v[e], v.v[n], acc[k + n][q * VEC + e]);
        }
      }
    }
  }
  join_warps<T, NB>(acc, red);
  if (warp == 0) {
#pragma unroll
    for (int n = 0; n < NB; n++)
#pragma unroll
      for (int q = 0; q < Q; q++)
        if (in[q] && n0 + n < N)
#pragma unroll
          for (int e = 0; e < VEC; e++) parts[((int64_t)blockIdx.z * N + n0 + n) * m.cols + col[q] + e] = acc[n][q * VEC + e];
  }
}

// out(r, c) = g * sum_n a(n, r) * b(n, c): few instances, bound by the stores (50257x768 Float32, eight
// instances 58 us).  A CTA takes 64 rows and
// 128 columns, a warp eight rows; a's entries come through shared memory, eight instances at a time.
// Skipped instances (label 0) are passed over: 0 times what a padded batch holds there may be NaN.
template <typename T, int VEC>
__global__ void __launch_bounds__(256)
outer_kernel(const T* a, int64_t lda, const T* b, int64_t ldb, const int32_t* labels, int64_t N,
             int64_t R, int64_t C, T* out, int64_t ld, GradScale<T> g) {
  chain_begin();
  constexpr int Q = 4 / VEC, NB = 8;
  __shared__ __align__(16) T as[NB][64];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t r0 = (int64_t)blockIdx.x * 64, j0 = (int64_t)blockIdx.y * 128;
  T acc[8][4];
#pragma unroll
  for (int r = 0; r < 8; r++)
#pragma unroll
    for (int e = 0; e < 4; e++) acc[r][e] = (T)0;
  for (int64_t n0 = 0; n0 < N; n0 += NB) {
    __syncthreads();
    for (int k = threadIdx.x; k < NB * 64; k += 256) {
      const int n = k >> 6, r = k & 63;
      as[n][r] = n0 + n < N && r0 + r < R ? a[(n0 + n) * lda + r0 + r] : (T)0;
    }
    __syncthreads();
#pragma unroll
    for (int n = 0; n < NB; n++) {
      if (n0 + n >= N) break;
      if (labels[n0 + n] == 0) continue;
      T av[8];
#pragma unroll
      for (int r = 0; r < 8; r++) av[r] = as[n][warp * 8 + r];
#pragma unroll
      for (int q = 0; q < Q; q++) {
        const int64_t c = j0 + (lane + 32 * q) * VEC;
        if (c < C) {
          const Pack<T, VEC> v = ld_cached<T, VEC>(b + (n0 + n) * ldb + c);
#pragma unroll
          for (int r = 0; r < 8; r++)
#pragma unroll
            for (int e = 0; e < VEC; e++) acc[r][q * VEC + e] = Math<T>::fma(av[r], v.v[e], acc[r][q * VEC + e]);
        }
      }
    }
  }
  const T f = g.value();
#pragma unroll
  for (int r = 0; r < 8; r++) {
    const int64_t row = r0 + warp * 8 + r;
    if (row >= R) break;
#pragma unroll
    for (int q = 0; q < Q; q++) {
      const int64_t c = j0 + (lane + 32 * q) * VEC;
      if (c < C) {
        Pack<T, VEC> v;
#pragma unroll
        for (int e = 0; e < VEC; e++) v.v[e] = acc[r][q * VEC + e] * f;
        st_stream<T, VEC>(out + row * ld + c, v);
      }
    }
  }
}

// ---- from the scores ------------------------------------------------------------------------------------
// lse and loss of each instance from the parts of its scores; GROUP threads (a warp or the CTA) per
// instance.  The last CTA to finish adds the losses in a fixed order (`done` counts CTAs; the product
// that ran before set it to 0).
template <typename T, int GROUP>
__global__ void __launch_bounds__(GROUP < 256 ? 256 : GROUP)
lnll_rows_kernel(const T* scores, int parts, const T* bias, const int32_t* labels, int64_t N,
                 int64_t V, T* lse, T* per_instance, T* total, int32_t* count,
                 uint32_t* done) {
  chain_begin();
  constexpr int THREADS = GROUP < 256 ? 256 : GROUP;
  constexpr int KEEP = 8;                      // scores in flight per thread; the first ones stay in registers
  __shared__ T red[32];
  __shared__ double redd[32];
  const int sub = threadIdx.x % GROUP;
  const int64_t n = (int64_t)blockIdx.x * (THREADS / GROUP) + threadIdx.x / GROUP;
  const int64_t stride = N * V;
  if (GROUP == THREADS || n < N) {
    const T* x = scores + n * V;
    T keep[KEEP];
    T m = -Math<T>::inf();
    load_scores<T, KEEP, GROUP>(keep, x, sub, V, stride, parts, bias);
#pragma unroll
    for (int k = 0; k < KEEP; k++) m = fmax(m, keep[k]);
    for (int64_t v0 = sub + (int64_t)KEEP * GROUP; v0 < V; v0 += (int64_t)KEEP * GROUP) {
      T t[KEEP];
      load_scores<T, KEEP, GROUP>(t, x, v0, V, stride, parts, bias);
#pragma unroll
      for (int k = 0; k < KEEP; k++) m = fmax(m, t[k]);
    }
    auto larger = [](T a, T b) { return (T)fmax(a, b); };
    if constexpr (GROUP == 32) m = warp_reduce(m, larger);
    else m = block_reduce(m, larger, (T)-Math<T>::inf(), red);
    double s = 0.0;
#pragma unroll
    for (int k = 0; k < KEEP; k++) s += (double)exp_from(keep[k], m);
    for (int64_t v0 = sub + (int64_t)KEEP * GROUP; v0 < V; v0 += (int64_t)KEEP * GROUP) {
      T t[KEEP];
      load_scores<T, KEEP, GROUP>(t, x, v0, V, stride, parts, bias);
      T e = (T)0;
#pragma unroll
      for (int k = 0; k < KEEP; k++) e += exp_from(t[k], m);
      s += (double)e;
    }
    auto plus = [](double a, double b) { return a + b; };
    if constexpr (GROUP == 32) s = warp_reduce(s, plus);
    else s = block_reduce(s, plus, 0.0, redd);
    if (sub == 0) {
      const int32_t lab = labels[n];
      per_instance[n] = finish_instance(m, s, lab > 0 && lab <= V ? (T)(sum_parts(x + lab - 1, stride, parts) + (bias ? bias[lab - 1] : (T)0)) : (T)0,
                                        lab, V, lse + n, lse + N + n);
      __threadfence();
    }
  }
  last_adds_losses<T, THREADS>(per_instance, labels, N, total, count, done);
}

// The same for many classes: a CTA takes 2048 classes of one instance and leaves their maximum and sum at
// [chunk][instance], as the tiles of the larger forms do.  With `done` (few instances) the last CTA to
// finish joins them, a warp per instance, and adds the losses; else lnll_join_kernel follows.
constexpr int kChunk = 2048;
template <typename T>
__global__ void __launch_bounds__(256)
lnll_chunks_kernel(const T* scores, int parts, const T* bias, const int32_t* labels, int64_t N,
                   int64_t V, uint32_t chunks, T* part_m, T* part_s, T* label_score,
                   T* lse, T* per_instance, T* total, int32_t* count,
                   uint32_t* done) {
  chain_begin();
  __shared__ T red[32];
  __shared__ uint32_t last;
  const int64_t n = blockIdx.x / chunks, chunk = blockIdx.x % chunks, v0 = chunk * kChunk;
  const T* x = scores + n * V;
  T t[kChunk / 256];
  T m = -Math<T>::inf();
  const int64_t lab = (int64_t)labels[n] - 1 - v0;
  load_scores<T, kChunk / 256, 256>(t, x, v0 + threadIdx.x, V, N * V, parts, bias);
#pragma unroll
  for (int k = 0; k < kChunk / 256; k++)
    if (k * 256 + threadIdx.x == lab && v0 + lab < V) label_score[n] = t[k];
#pragma unroll
  for (int k = 0; k < kChunk / 256; k++) m = fmax(m, t[k]);
  m = block_reduce(m, [](T a, T b) { return (T)fmax(a, b); }, (T)-Math<T>::inf(), red);
  T s = (T)0;
#pragma unroll
  for (int k = 0; k < kChunk / 256; k++) s += exp_from(t[k], m);
  s = block_reduce(s, [](T a, T b) { return a + b; }, (T)0, red);
  if (threadIdx.x == 0) {
    part_m[chunk * N + n] = m;
    part_s[chunk * N + n] = s;
  }
  if (!done) return;
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) last = atomicAdd(done, 1u);
  __syncthreads();
  if (last + 1 != gridDim.x) return;
  __threadfence();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int64_t i = warp; i < N; i += 8) {
    T mm = -Math<T>::inf();
    for (uint32_t k = lane; k < chunks; k += 32) mm = fmax(mm, __ldcg(part_m + k * N + i));
    mm = warp_reduce(mm, [](T p, T q) { return (T)fmax(p, q); });
    double sd = 0.0;
    for (uint32_t k = lane; k < chunks; k += 32) {
      const T v = __ldcg(part_s + k * N + i), d = __ldcg(part_m + k * N + i) - mm;
      if (v != (T)0) sd += (double)(v * exp(d));                 // an empty chunk is (-inf, 0)
    }
    sd = warp_reduce(sd, [](double p, double q) { return p + q; });
    if (lane == 0) {
      const int32_t l = labels[i];
      per_instance[i] = finish_instance(mm, sd, l > 0 && l <= V ? __ldcg(label_score + i) : (T)0, l, V, lse + i, lse + N + i);
    }
  }
  __threadfence();
  __syncthreads();
  add_losses<T, 256>(per_instance, labels, N, total, count);
}

// dS (without g) over the first part of the scores; `blocks` CTAs per instance
template <typename T>
__global__ void __launch_bounds__(256)
lnll_grad_kernel(T* scores, int parts, const T* bias, const int32_t* labels,
                 const T* lse, int64_t N, int64_t V, uint32_t blocks) {
  chain_begin();
  const int64_t n = blockIdx.x / blocks;
  const T hi = lse[n], lo = lse[N + n];
  const int32_t lab = labels[n];
  T* x = scores + n * V;
  const int64_t v0 = (int64_t)(blockIdx.x % blocks) * 1024 + threadIdx.x;
  T t[4];
  load_scores<T, 4, 256>(t, x, v0, V, N * V, parts, bias);
#pragma unroll
  for (int k = 0; k < 4; k++)
    if (v0 + k * 256 < V) x[v0 + k * 256] = grad_score(t[k], hi, lo, lab, v0 + k * 256);
}

// out = g * (the parts, added in order), n numbers in rows of J, `ld` apart in `out`
template <typename T>
__global__ void __launch_bounds__(256)
lnll_sum_kernel(const T* parts, int64_t n, int64_t J, int64_t ld, int count, T* out, int add, GradScale<T> g) {
  chain_begin();
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  const T a = sum_parts(parts + i, n, count) * g.value();
  const int64_t to = J == ld ? i : i / J * ld + i % J;
  out[to] = add ? out[to] + a : a;
}

}  // namespace kn

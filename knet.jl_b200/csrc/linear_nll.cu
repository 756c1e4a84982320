// Softmax cross entropy of a linear output layer, scores = W x (+ b), without the score matrix:
//   forward   lse_n = log sum_v exp(s_vn),  loss = sum over used n of lse_n - s_{label_n, n}
//   backward  dS = (exp(s - lse) - onehot) * g,  dx = W' dS,  dW = dS x',  db = sum_n dS
// The forward keeps per instance and tile of the vocabulary the maximum and the sum of
// exponentials; the backward computes the scores again, a piece of the vocabulary at a time, turns
// them into dS in the workspace and multiplies that piece by W and x.  Knet composes the same from
// `W*x .+ b` and nll (src/ops20/loss.jl:37-41), which keeps scores, logsoftmax and their gradients.
//
// An instance's loss is lse - s[label]; the forward hands lse on as an unevaluated sum of two
// numbers (its rounding alone would be a relative error of |lse| * 2^-24 in every p of that
// instance), so that p = exp((s - hi) - lo).
#include <atomic>

#include "linear_nll.cuh"
#include "linear_nll_mma.cuh"
#include "linear_nll_small.cuh"

namespace kn {

// ---- epilogues of the FMA and FP64 tiles -----------------------------------------------------------------
// i = instance, j = class: the tile's maximum and sum of exponentials per instance, and the score at
// the label.  The 16 threads of an instance row are neighbours in a half warp.
template <typename T> struct StatsEpi {
  const T* bias;
  const int32_t* labels;
  T *part_m, *part_s, *label_score;
  int64_t N;
  __device__ __forceinline__ void operator()(T (&acc)[4][4], int64_t i0, int64_t j0, int64_t I, int64_t J) const {
    T bv[4];
#pragma unroll
    for (int w = 0; w < 4; w++) bv[w] = (bias && j0 + w < J) ? bias[j0 + w] : (T)0;
#pragma unroll
    for (int u = 0; u < 4; u++) {
      const int64_t i = i0 + u;
      const int32_t lab = i < I ? labels[i] : 0;
      T m = -Math<T>::inf();
#pragma unroll
      for (int w = 0; w < 4; w++) {
        acc[u][w] = j0 + w < J ? acc[u][w] + bv[w] : -Math<T>::inf();
        m = fmax(m, acc[u][w]);
        if (i < I && j0 + w < J && lab == j0 + w + 1) label_score[i] = acc[u][w];
      }
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) m = fmax(m, __shfl_xor_sync(0xffffffffu, m, o));
      T s = (T)0;
#pragma unroll
      for (int w = 0; w < 4; w++) s += exp_from(acc[u][w], m);
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
      if (i < I && (threadIdx.x & 15) == 0) {
        part_m[(int64_t)blockIdx.x * N + i] = m;
        part_s[(int64_t)blockIdx.x * N + i] = s;
      }
    }
  }
};

// i = instance, j = class of the piece: dS without the factor g
template <typename T> struct GradScoresEpi {
  const T* bias;               // of the piece's first class
  const int32_t* labels;
  const T* lse;                // N rounded values, then N remainders
  T* ds;                       // [n][class of the piece], row pitch ld
  int64_t N, ld, v0;
  __device__ __forceinline__ void operator()(T (&acc)[4][4], int64_t i0, int64_t j0, int64_t I, int64_t J) const {
#pragma unroll
    for (int u = 0; u < 4; u++) {
      const int64_t i = i0 + u;
      if (i >= I) break;
      const int32_t lab = labels[i];
      const T hi = lse[i], lo = lse[N + i];
#pragma unroll
      for (int w = 0; w < 4; w++) {
        if (j0 + w >= J) break;
        const T s = acc[u][w] + (bias ? bias[j0 + w] : (T)0);
        ds[i * ld + j0 + w] = grad_score(s, hi, lo, lab, v0 + j0 + w);
      }
    }
  }
};

// ---- joining the tiles of the vocabulary ---------------------------------------------------------------
// A CTA takes 32 instances; its 32 warps share the tiles of the vocabulary: the maximum first, then the
// sums relative to it, added in Float64 (8 warps took 25 us for 197 tiles of 4096 instances).
template <typename T>
__global__ void __launch_bounds__(1024)
lnll_join_kernel(const T* part_m, const T* part_s, const T* label_score,
                 const int32_t* labels, int64_t N, int64_t V, int64_t tiles, T* lse,
                 T* per_instance, T* total, int32_t* count, uint32_t* done) {
  chain_begin();
  __shared__ T sm[32][32];
  __shared__ double ss[32][32];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int64_t n = (int64_t)blockIdx.x * 32 + lane;
  T m = -Math<T>::inf();
  if (n < N) {
#pragma unroll 8
    for (int64_t t = w; t < tiles; t += 32) m = fmax(m, part_m[t * N + n]);
  }
  sm[w][lane] = m;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 32; k++) m = fmax(m, sm[k][lane]);
  double s = 0.0;
  if (n < N) {
#pragma unroll 8
    for (int64_t t = w; t < tiles; t += 32) {
      const T d = part_m[t * N + n] - m, v = part_s[t * N + n];
      if (v != (T)0) s += (double)(v * exp(d));      // an empty tile is (-inf, 0)
    }
  }
  ss[w][lane] = s;
  __syncthreads();
  if (w == 0 && n < N) {
    s = ss[0][lane];
    for (int k = 1; k < 32; k++) s += ss[k][lane];
    const int32_t lab = labels[n];
    per_instance[n] = finish_instance(m, s, lab > 0 && lab <= V ? label_score[n] : (T)0, lab, V, lse + n, lse + N + n);
  }
  last_adds_losses<T, 1024>(per_instance, labels, N, total, count, done);
}

// an empty batch
template <typename T> __global__ void lnll_none_kernel(T* total, int32_t* count) {
  chain_begin();
  *total = (T)0;
  *count = 0;
}

// db[j] = g * sum_n ds[n][j]: a CTA takes 32 classes, its 32 warps share the instances.  Cut over gridDim.y
// parts of `rows` instances, the plain sums of each go to parts[part][j].
template <typename T>
__global__ void __launch_bounds__(1024)
lnll_bias_kernel(const T* ds, int64_t ld, int64_t N, int64_t J, int64_t rows, T* out, GradScale<T> g) {
  chain_begin();
  __shared__ T part[32][33];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int64_t j = (int64_t)blockIdx.x * 32 + lane;
  const int64_t n0 = (int64_t)blockIdx.y * rows, n1 = min(N, n0 + rows);
  T a = (T)0;
  if (j < J)
#pragma unroll 8
    for (int64_t n = n0 + w; n < n1; n += 32) a += ds[n * ld + j];
  part[w][lane] = a;
  __syncthreads();
  if (w == 0 && j < J) {
    for (int k = 1; k < 32; k++) a += part[k][lane];
    out[blockIdx.y * J + j] = gridDim.y > 1 ? a : a * g.value();
  }
}

template <typename T> __global__ void lnll_zero_kernel(T* p, int64_t n) {
  chain_begin();
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i < n) p[i] = (T)0;
}
template <typename T> void lnll_zero(T* p, int64_t n, cudaStream_t st) {
  if (p && n > 0) launch_chained(lnll_zero_kernel<T>, (unsigned)((n + 255) / 256), 256, 0, st, p, n);
}

// ---- host ---------------------------------------------------------------------------------------------
template <typename T> struct Head {
  const T* w;
  int trans;                   // 0: w is (V,H), 1: (H,V)
  const T* bias;
  const T* x;
  const int32_t* labels;
  int64_t V, H, N;
  Strided<T> weights(int64_t v0) const {      // element (class v0 + i, feature c)
    return trans ? Strided<T>{w + v0 * H, H, 1} : Strided<T>{w + v0, 1, V};
  }
};

constexpr size_t kAlign = 256;
inline size_t up(size_t n) { return (n + kAlign - 1) / kAlign * kAlign; }

constexpr int kPlanSMs = 148;

// ---- plans; the tensor-core form (Float32) --------------------------------------------------------------
inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// The bias gradient's rows of dS are cut where there are many and few classes: one CTA of 32 warps would
// walk them alone.  At most 64 parts of 2048 rows or more, together two CTAs per SM.
inline int64_t bias_parts(int64_t rows, int64_t J) {
  int64_t k = 2 * kPlanSMs / ceil_div(J, 32);
  k = k > rows / 2048 ? rows / 2048 : k;
  return k > 64 ? 64 : k < 1 ? 1 : k;
}
// numbers in the parts of any J classes: more than one part of ceil(J / 32) CTAs are at most two CTAs per SM
constexpr size_t kBiasRoom = 2 * kPlanSMs * 32;

// Which form a call takes.
//   kSmall   up to 2^24 scores and either few instances or little work: the scores go to the workspace
//   kMma     Float32 beyond that
//   kPieces  the rest (Float64 with many scores)
// Few instances: kSmall reads W once per 8 instances, kMma reads it, writes it in two planes and reads those whatever
// their number.  50257x1024, forward / with gradients, us, kSmall and kMma: 8 instances 59 and 133 / 248 and 462,
// 16 instances 103 and 133 / 419 and 465, 17 instances 147 and 134 / 524 and 477, 24 instances 148 and 133 / 562 and
// 470, 32 instances 195 and 132 / 730 and 472.
// Work: FMA tiles and kMma with gradients: 300x256, 400 instances (2^25) 65 and 77 us, 500x512, 512 instances (2^27)
// 92 and 81 us, 1000x512, 512 instances (2^28) 120 and 85 us.
enum Form { kSmall, kMma, kPieces };
constexpr int64_t kFewInstances = 16;
template <typename T> Form form(int64_t V, int64_t H, int64_t N) {
  const bool fits = N * V <= (1 << 24);
  if (fits && N <= kFewInstances) return kSmall;
  if (sizeof(T) == 4 && ((double)V * H * N >= (double)(1 << 26) || !fits)) return kMma;
  return fits && (double)V * H * N < (double)(1ll << 32) ? kSmall : kPieces;
}

// Parts (at most 8, of at least 64 terms) of the sums of `tiles` FP64 tiles that take the SMs the least time:
// an SM gets ceil(tiles * parts / SMs) CTAs, one alone keeps its FP64 unit at about 0.6 of the rate of three, two
// at 0.85, and writing and reading a part weighs as much as 40 terms.  Measured, loss and gradients:
// 4645x1102, 318 instances 662 us with parts only below a round of three CTAs per SM, 605 us so.
inline void even_parts(int64_t tiles, int64_t len, int64_t bytes, int64_t& part, int& parts) {
  int64_t most = (64 << 20) / (bytes + 1), best = 1;
  most = most > 8 ? 8 : most;
  most = most > len / 64 ? len / 64 : most;
  double cost = 0;
  for (int64_t k = 1; k <= most || k == 1; k++) {
    const int64_t n = ceil_div(tiles * k, kPlanSMs);
    const double c = (double)n / k / (n == 1 ? 0.6 : n == 2 ? 0.85 : 1.0) * (1.0 + (k > 1 ? 40.0 * k / len : 0.0));
    if (k == 1 || c < cost) {
      cost = c;
      best = k;
    }
  }
  part = ceil_div(ceil_div(len, best), 64) * 64;
  parts = (int)ceil_div(len, part);
}
// Parts of the summed axes of the three products in kSmall: no more CTAs than three per SM (Float32 tiles:
// all run at once) or eight (few instances: the last round costs little), parts of at least 64 or
// 128 terms, at most 64 parts.  Float64 tiles, which the FP64 unit bounds, by even_parts where there is a
// tile for every second SM.
struct SmallPlan {
  int64_t few, s_part, x_part, w_part;         // few: by vectors, not tiles; lengths of the parts
  int s_parts, x_parts, w_parts;
  int64_t chunks;                              // of 2048 classes, where the statistics go by chunks
  size_t scores, parts, stats, bias, total;
};
template <typename T> SmallPlan small_plan(int64_t V, int64_t H, int64_t N, int trans, int backward) {
  SmallPlan p{};
  p.few = N <= 32;
  auto cut = [&](int64_t ctas, int64_t len, int64_t unit, int64_t bytes, int64_t& part, int& parts) {
    if (sizeof(T) == 8 && unit == 64 && ctas * 2 >= kPlanSMs) return even_parts(ctas, len, bytes, part, parts);
    int64_t k = unit == 64 ? 3 * kPlanSMs / ctas : ceil_div(8 * kPlanSMs, ctas);
    k = k > len / unit ? len / unit : k;
    k = k > 64 ? 64 : k;
    k = k > (64 << 20) / (bytes + 1) ? (64 << 20) / (bytes + 1) : k;
    k = k < 1 ? 1 : k;
    part = ceil_div(ceil_div(len, k), unit) * unit;
    parts = (int)ceil_div(len, part);
  };
  const int64_t sz = sizeof(T), groups = ceil_div(N, 8);
  if (p.few) {
    cut(ceil_div(V, trans ? 32 : 128) * groups, H, 128, N * V * sz, p.s_part, p.s_parts);
    cut(ceil_div(H, trans ? 128 : 32) * groups, V, 128, N * H * sz, p.x_part, p.x_parts);
    p.w_parts = 1;
  } else {
    cut(ceil_div(N, kTile) * ceil_div(V, kTile), H, 64, N * V * sz, p.s_part, p.s_parts);
    cut(ceil_div(N, kTile) * ceil_div(H, kTile), V, 64, N * H * sz, p.x_part, p.x_parts);
    cut(ceil_div(V, kTile) * ceil_div(H, kTile), N, 64, V * H * sz, p.w_part, p.w_parts);
  }
  size_t at = up(4);
  p.scores = at;
  at += up((size_t)p.s_parts * N * V * sz);
  p.parts = at;
  p.stats = at;
  p.chunks = V > 4 * kChunk ? ceil_div(V, kChunk) : 0;
  if (!backward && p.chunks) at += up((size_t)(2 * p.chunks + 1) * N * sz);
  if (backward) {
    const size_t x = p.few || p.x_parts > 1 ? (size_t)p.x_parts * N * H * sz : 0, w = p.w_parts > 1 ? (size_t)p.w_parts * V * H * sz : 0;
    at += up(x > w ? x : w);
    p.bias = at;
    at += up(kBiasRoom * sz);
  }
  p.total = at;
  return p;
}

// Pieces of the vocabulary and parts of the products' sums.  Workspace bounds: 256 MB of split weights in
// the forward; 128 MB of dS, twice as much of its split forms and 192 MB of split weights in the backward.  Within them the backward takes
// the piece with the fewest waves of tiles over its three products (a product's tiles are 128 x 256, a
// pair's two of them, and its time is proportional to the summed length), charging each piece for its
// launches.  Only the smallest piece of each number of pieces is tried: for four million classes that takes the host
// 10 us, every size of a piece 0.7 ms.  Where a
// product has tiles for less than half of the SMs, its sum is cut into parts of at least 128 (a chunk);
// the scores only if all of them fit 64 MB with their parts, dW only if there is one piece.
struct MmaPlan {
  int64_t piece, wld, xld, dld;        // classes per piece; row pitches of split w, x and dS (elements)
  int s_parts, x_parts, w_parts;
  int64_t chunks;                      // of 2048 classes, where the scores are in the workspace (s_parts > 1)
  size_t done, xs, ws, xmag, wmag, label, part_m, part_s, scores, maxima, ds, dx_ds, dw_ds, parts, db, bias, total;
};

inline int64_t cut_sum(int64_t tiles, int64_t len, int64_t bytes) {
  if (tiles * 2 > kPlanSMs) return 1;
  int64_t k = kPlanSMs / tiles;
  k = k > ceil_div(len, 128) ? ceil_div(len, 128) : k;
  k = k > (64 << 20) / (bytes + 1) ? (64 << 20) / (bytes + 1) : k;
  return k < 1 ? 1 : k;
}

inline MmaPlan mma_plan(int64_t V, int64_t H, int64_t N, int trans, int backward) {
  MmaPlan p{};
  const int64_t all = ceil_div(V, kTN), nt = ceil_div(N, kTM), hj = ceil_div(H, kTN), hi = ceil_div(H, kTM);
  p.s_parts = p.x_parts = p.w_parts = 1;
  int64_t most = (int64_t)(256u << 20) / 4 / (ceil_div(H, 64) * 64) / kTN;
  most = most < 1 ? 1 : most;
  p.piece = kTN * ceil_div(all, ceil_div(all, most));      // of the forward
  // the backward's scores are the forward's bit for bit, summed in the same parts, whatever its own pieces
  if (p.piece >= V) p.s_parts = (int)cut_sum(nt * all, H, N * V * 4);
  if (backward) {
    // the largest piece within the bounds, then the smallest piece of each number of pieces
    const int64_t row = ceil_div(H, 64) * 64 * 4 * kTN, most_ds = (128ll << 20) / (kTN * N * 4), most_w = (192ll << 20) / row;
    int64_t m = most_ds < most_w ? most_ds : most_w;
    m = m < 1 ? 1 : m > all ? all : m;
    double best = 0;
    for (bool first = true; m > 0; first = false) {
      const int64_t pieces = ceil_div(all, m);
      if (!first && pieces * 1500.0 >= best) break;
      m = ceil_div(all, pieces);
      int64_t sp = kPlanSMs / (nt * hj);
      sp = sp < 1 ? 1 : sp > 2 * m ? 2 * m : sp > 16 ? 16 : sp;
      const int64_t wt = trans ? 2 * m * hj : hi * m;
      const int64_t wp = m == all ? cut_sum(wt, N, V * H * 4) : 1;
      const double t = (double)ceil_div(nt * m, kPlanSMs) * H + (double)ceil_div(nt * hj * sp, kPlanSMs) * ceil_div(m * kTN, sp) +
                       (double)ceil_div(wt * wp, kPlanSMs) * ceil_div(N, wp) + 1500.0;
      const double cost = t * pieces;
      if (first || cost <= best) {
        best = cost;
        p.piece = m * kTN;
        p.x_parts = (int)sp;
        p.w_parts = (int)wp;
      }
      m--;
    }
  }
  p.chunks = V > 4 * kChunk ? ceil_div(V, kChunk) : 0;
  const int64_t vp = p.piece < V ? p.piece : V;
  // pitches of whole 128-byte lines: a box of 32 summed indices (64 bytes) then never straddles two sectors
  // (dx of 1000 classes, 8192 x 8192, with a pitch of 1000: 479 us)
  p.wld = ceil_div(trans ? H : vp, 64) * 64;
  p.xld = ceil_div(H, 64) * 64;
  p.dld = ceil_div(vp, 64) * 64;
  size_t at = 0;
  auto put = [&](size_t& where, size_t bytes) {
    where = at;
    at += up(bytes);
  };
  put(p.done, 16);
  put(p.xs, (size_t)N * p.xld * 4);
  put(p.ws, (size_t)(trans ? vp : H) * p.wld * 4);
  put(p.xmag, (size_t)N * 4);
  put(p.wmag, (size_t)vp * 4);
  if (p.s_parts > 1) put(p.scores, (size_t)p.s_parts * N * vp * 4);
  if (!backward) {
    put(p.label, (size_t)N * 4);
    put(p.part_m, (size_t)(p.s_parts > 1 ? p.chunks : all) * N * 4);
    put(p.part_s, (size_t)(p.s_parts > 1 ? p.chunks : all) * N * 4);
  } else {
    put(p.maxima, (size_t)(N + vp) * 4);
    put(p.ds, (size_t)N * p.dld * 4);
    put(p.dx_ds, (size_t)N * p.dld * 4);
    put(p.dw_ds, (size_t)N * p.dld * 4);
    const size_t x = p.x_parts > 1 ? (size_t)p.x_parts * N * H * 4 : 0, w = p.w_parts > 1 ? (size_t)p.w_parts * V * H * 4 : 0;
    put(p.parts, x > w ? x : w);
    put(p.db, (size_t)ceil_div(N, kGradRows) * vp * 4);
    put(p.bias, kBiasRoom * 4);
  }
  p.total = at;
  return p;
}

// Float64 with many scores: pieces of equal size with at most 128 MB of dS
struct PiecePlan {
  int64_t piece, x_part, w_part;
  int x_parts, w_parts;
  size_t parts, bias, total;
};
template <typename T> PiecePlan piece_plan(int64_t V, int64_t H, int64_t N) {
  PiecePlan p{};
  int64_t most = (int64_t)((128u << 20) / sizeof(T)) / N / kTile;
  most = most < 1 ? 1 : most;
  const int64_t all = ceil_div(V, kTile);
  p.piece = ceil_div(all, ceil_div(all, most)) * kTile;
  p.piece = p.piece < V ? p.piece : V;
  const int64_t nt = ceil_div(N, kTile), ht = ceil_div(H, kTile), vt = ceil_div(p.piece, kTile), sz = sizeof(T);
  even_parts(nt * ht, p.piece, N * H * sz, p.x_part, p.x_parts);
  even_parts(vt * ht, N, p.piece * H * sz, p.w_part, p.w_parts);
  const size_t x = p.x_parts > 1 ? (size_t)p.x_parts * N * H * sz : 0, w = p.w_parts > 1 ? (size_t)p.w_parts * p.piece * H * sz : 0;
  p.parts = up((size_t)N * p.piece * sz);
  p.bias = p.parts + up(x > w ? x : w);
  p.total = p.bias + up(kBiasRoom * sz);
  return p;
}

template <typename T> size_t workspace(int64_t V, int64_t H, int64_t N, int trans, int backward) {
  const Form f = form<T>(V, H, N);
  if (f == kMma) return mma_plan(V, H, N, trans, backward).total;
  if (f == kSmall) return small_plan<T>(V, H, N, trans, backward).total;
  if (backward) return piece_plan<T>(V, H, N).total;
  const int64_t tiles = (V + kTile - 1) / kTile;
  return up(4) + up((size_t)N * sizeof(T)) + 2 * up((size_t)tiles * N * sizeof(T));
}
template <typename T> size_t workspace_any(int64_t V, int64_t H, int64_t N, int backward) {
  const size_t a = workspace<T>(V, H, N, 0, backward), b = workspace<T>(V, H, N, 1, backward);
  return a > b ? a : b;
}

template <typename T, typename Epi>
void simt_product(Strided<T> a, Strided<T> b, int64_t I, int64_t J, int64_t C, int64_t c_part, uint32_t* done, Epi epi, cudaStream_t st) {
  const dim3 grid((unsigned)ceil_div(J, kTile), (unsigned)ceil_div(I, kTile), (unsigned)ceil_div(C, c_part));
  launch_chained(simt_product_kernel<T, false, Epi>, grid, kSimtThreads, 0, st, a, b, (const int32_t*)nullptr, (const int32_t*)nullptr, I, J, C,
                 c_part, done, epi);
}
// out (I x J, rows `ld` apart) = or += g * (parts, added in order)
template <typename T>
void sum_parts_to(const T* parts, int64_t I, int64_t J, int64_t ld, int count, T* out, int add, GradScale<T> g, cudaStream_t st) {
  launch_chained(lnll_sum_kernel<T>, (unsigned)ceil_div(I * J, 256), 256, 0, st, parts, I * J, J, ld, count, out, add, g);
}
// out (I x J, rows `ld` apart) = or += g * sum_c A(i, c) B(j, c), through `parts` where the sum is cut
template <typename T>
void tile_product_out(Strided<T> a, Strided<T> b, int64_t I, int64_t J, int64_t C, int64_t c_part, int cuts, T* out, int64_t ld, int add,
                      T* parts, GradScale<T> g, cudaStream_t st) {
  if (cuts == 1) {
    simt_product<T>(a, b, I, J, C, C, nullptr, StoreEpi<T>{out, ld, add, g}, st);
  } else {
    simt_product<T>(a, b, I, J, C, c_part, nullptr, PartsEpi<T>{parts}, st);
    sum_parts_to<T>(parts, I, J, ld, cuts, out, add, g, st);
  }
}
// dW's: the sum runs over the instances, of which the labels tell the skipped ones in the operand that is x
template <typename T, typename Epi>
void simt_product_dw(Strided<T> a, Strided<T> b, bool a_is_x, const int32_t* labels, int64_t I, int64_t J, int64_t N, int64_t c_part,
                     const Epi& epi, cudaStream_t st) {
  const dim3 grid((unsigned)ceil_div(J, kTile), (unsigned)ceil_div(I, kTile), (unsigned)ceil_div(N, c_part));
  launch_chained(simt_product_kernel<T, true, Epi>, grid, kSimtThreads, 0, st, a, b, a_is_x ? labels : nullptr, a_is_x ? nullptr : labels, I, J, N,
                 c_part, (uint32_t*)nullptr, epi);
}
template <typename T>
void tile_product_dw(Strided<T> a, Strided<T> b, bool a_is_x, const int32_t* labels, int64_t I, int64_t J, int64_t N, int64_t n_part, int cuts,
                     T* out, int64_t ld, T* parts, GradScale<T> g, cudaStream_t st) {
  if (cuts == 1) {
    simt_product_dw<T>(a, b, a_is_x, labels, I, J, N, N, StoreEpi<T>{out, ld, 0, g}, st);
  } else {
    simt_product_dw<T>(a, b, a_is_x, labels, I, J, N, n_part, PartsEpi<T>{parts}, st);
    sum_parts_to<T>(parts, I, J, ld, cuts, out, 0, g, st);
  }
}

// packs of VEC elements are possible where base addresses and pitches are multiples of 16 bytes
template <typename T> bool aligned16(const T* p, int64_t pitch) {
  return ((uintptr_t)p & 15) == 0 && pitch * (int64_t)sizeof(T) % 16 == 0;
}

// parts of sum_c M(r, c) y(n, c) (by_row) or sum_r M(r, c) y(n, r)
template <typename T, int NB>
void few_product_nb(bool by_row, const Matrix<T>& m, const T* y, int64_t ldy, int64_t N, int64_t part, int parts, uint32_t* done, T* out,
                    cudaStream_t st) {
  constexpr int VEC = 16 / sizeof(T);
  const unsigned groups = (unsigned)ceil_div(N, NB);
  const bool wide = aligned16(m.p, m.pitch) && m.cols % VEC == 0;
  if (by_row) {
    const dim3 grid((unsigned)ceil_div(m.rows, 32), groups, (unsigned)parts);
    if (wide && aligned16(y, ldy)) launch_chained(row_dot_kernel<T, NB, VEC>, grid, 256, 0, st, m, y, ldy, N, part, done, out);
    else launch_chained(row_dot_kernel<T, NB, 1>, grid, 256, 0, st, m, y, ldy, N, part, done, out);
  } else {
    const dim3 grid((unsigned)ceil_div(m.cols, 128), groups, (unsigned)parts);
    if (wide) launch_chained(col_sum_kernel<T, NB, VEC>, grid, 256, 0, st, m, y, ldy, N, part, done, out);
    else launch_chained(col_sum_kernel<T, NB, 1>, grid, 256, 0, st, m, y, ldy, N, part, done, out);
  }
}
template <typename T>
void few_product(bool by_row, const Matrix<T>& m, const T* y, int64_t ldy, int64_t N, int64_t part, int parts, uint32_t* done, T* out,
                 cudaStream_t st) {
  if (N == 1) few_product_nb<T, 1>(by_row, m, y, ldy, N, part, parts, done, out, st);
  else if (N == 2) few_product_nb<T, 2>(by_row, m, y, ldy, N, part, parts, done, out, st);
  else if (N <= 4) few_product_nb<T, 4>(by_row, m, y, ldy, N, part, parts, done, out, st);
  else few_product_nb<T, 8>(by_row, m, y, ldy, N, part, parts, done, out, st);
}

// sizes whose tile counts fit a launch grid (features are rows of a tile grid in dW)
inline bool sizes_ok(int64_t V, int64_t H, int64_t N) {
  const int64_t most = (int64_t)65535 * kTile;
  return V <= 0x7fffffff && H <= most && N <= most && V <= most;
}

int linear_nll_wait_flag_read_clear() { return wait_flag_read_clear(); }

template <typename T> bool odd(const T* p) { return (uintptr_t)p % sizeof(T) != 0; }

template <typename T> int check(const Head<T>& h, const void* ws, size_t have, size_t need) {
  if (h.V <= 0 || h.H <= 0 || h.N < 0 || (h.trans != 0 && h.trans != 1)) return KN_EINVAL;
  if (!sizes_ok(h.V, h.H, h.N)) return KN_ESIZE;
  if (h.N == 0) return KN_OK;
  if (!h.w || !h.x || !h.labels) return KN_EINVAL;
  if (odd(h.w) || odd(h.x) || odd(h.bias) || odd(h.labels)) return KN_EALIGN;
  if (!ws || have < need) return KN_EWORKSPACE;
  if ((uintptr_t)ws % kAlign) return KN_EALIGN;
  return KN_OK;
}

// One operand of a product: `rows` x `cols` in memory (cols contiguous), two planes.
struct Planes {
  const __half* p;
  int64_t rows, cols, ld, plane;
};
// its map in the role of the tile's `tile` rows; mn: those rows are the contiguous axis
inline int operand_map(CUtensorMap* map, const Planes& o, bool mn, int tile) {
  return tensor_map_planes(map, o.p, o.rows, o.cols, o.ld, o.plane, mn ? 64 : kBK, mn ? kBK : tile,
                           mn ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B);
}

// the kernel's shared memory is beyond the default limit: raised once per device
template <int CG, typename Epi> int allow_smem() {
  static std::atomic<uint64_t> done{0};
  int dev = 0;
  if (cudaError_t e = cudaGetDevice(&dev)) return (int)e;
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (done.load(std::memory_order_relaxed) & bit) return 0;
  if (cudaError_t e = cudaFuncSetAttribute(mma_kernel<CG, Epi>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kMmaSmem)) return (int)e;
  done.fetch_or(bit, std::memory_order_relaxed);
  return 0;
}

template <int CG, typename Epi>
int mma_product_cg(const Planes& a, bool a_mn, const Planes& b, bool b_mn, int64_t I, int64_t J, int64_t C, int splits, const Epi& epi,
                   cudaStream_t st) {
  static_assert(sizeof(CUtensorMap) == 128, "kernel parameter");
  CUtensorMap am, bm;
  if (int rc = operand_map(&am, a, a_mn, kTM)) return rc;
  if (int rc = operand_map(&bm, b, b_mn, kTN / CG)) return rc;
  MmaTiles tl;
  tl.i_tiles = (uint32_t)ceil_div(I, kTM * CG);
  tl.j_tiles = (uint32_t)ceil_div(J, kTN);
  tl.blocks = (uint32_t)ceil_div(C, kBK);
  tl.blocks_per_split = (uint32_t)ceil_div(tl.blocks, splits);
  tl.splits = (uint32_t)splits;
  tl.a_mn = a_mn;
  tl.b_mn = b_mn;
  if (int rc = allow_smem<CG, Epi>()) return rc;
  const uint64_t tiles = (uint64_t)tl.i_tiles * tl.j_tiles * tl.splits;
  if (tiles > 0x7fffffff) return KN_ESIZE;
  const uint64_t workers = (uint64_t)sm_count() / CG;
  const unsigned grid = (unsigned)(tiles < workers ? tiles : workers) * CG;
  return (int)launch_chained_cluster(CG, mma_kernel<CG, Epi>, grid, kMmaThreads, kMmaSmem, st, am, bm, tl, epi);
}

// Pairs of CTAs are faster by a thirteenth (see linear_nll_mma.cuh) but need tiles of 256 rows: not where those
// would add more to the rows (forward of 20000x1024: 850 instances in pairs 161 us, alone 150 us).
template <typename Epi>
int mma_product(const Planes& a, bool a_mn, const Planes& b, bool b_mn, int64_t I, int64_t J, int64_t C, int splits, const Epi& epi,
                cudaStream_t st) {
  const int64_t one = ceil_div(I, kTM), two = 2 * ceil_div(I, 2 * kTM);
  if (13 * two <= 14 * one) return mma_product_cg<2>(a, a_mn, b, b_mn, I, J, C, splits, epi, st);
  return mma_product_cg<1>(a, a_mn, b, b_mn, I, J, C, splits, epi, st);
}

// W's classes [v0, v0 + vp) and, with the first piece, x in two planes, each class and each instance with a scale
// of its own
struct SplitState {
  Planes w, x;
  const uint32_t *wmag, *xmag;
};
// W by columns in one kernel (see there) where a CTA's share of the rows is 128 at most: the shares of all CTAs that run
// at once then fit L2 (50257x1024 102 us; 32000x4096 so 258 us, by the two 271 us, but 25357x5169, rows of any
// alignment, 363-569 and 280 us).  A backward that is given the maxima reads W once (66 and 166 us).
constexpr int64_t kSplitRows = 128 * kSplitCtas;
template <int GROUP>
void split_launch(bool rows, const SplitJob& w, const SplitJob& x, bool with_x, bool given, uint32_t* zeros, int64_t nzeros, cudaStream_t st) {
  const int64_t per = 256 / GROUP, bx = with_x ? ceil_div(x.rows, per) : 0;
  if (rows) {
    const int64_t bw = ceil_div(w.rows, per);
    launch_chained(lnll_split_rows_kernel<GROUP>, (unsigned)(bw + bx), 256, 0, st, w, x, (uint32_t)bw, zeros, nzeros);
    return;
  }
  if (w.rows <= kSplitRows && !given) {
    uint32_t ctas = 1;
    while (ctas < kSplitCtas && w.rows >= 64 * (int64_t)ctas) ctas *= 2;
    const int64_t bw = ceil_div(w.cols, kSplitCols) * ctas, padded = ceil_div(bx, ctas) * ctas;
    launch_chained_cluster(ctas, lnll_split_cols_kernel<GROUP>, (unsigned)(bw + padded), 256, 0, st, w, x, (uint32_t)bw, ctas, zeros, nzeros);
    return;
  }
  const uint32_t groups = (uint32_t)ceil_div(w.cols, kSplitCols);
  int64_t share = ceil_div(w.rows, ceil_div(8 * kPlanSMs, groups));      // eight CTAs per SM, 32 rows or more each
  share = share < 32 ? 32 : share;
  const int64_t bw = groups * ceil_div(w.rows, share);
  // ordinary launches: placed under the tail of another kernel, equal shares land unevenly on the SMs (loss and gradients
  // of 25357x5169, 24 instances 1511 us chained, 1456 so, 1427 with the split of dS launched so too)
  if (!given) {
    lnll_zero((float*)w.mag, w.cols, st);
    lnll_colmax_kernel<<<(unsigned)bw, 256, 0, st>>>(w, groups, share);
  }
  lnll_split_wide_kernel<GROUP><<<(unsigned)(bw + bx), 256, 0, st>>>(w, x, (uint32_t)bw, groups, share, zeros, nzeros);
}
// class_max: of W's columns, taken where `given`, else left there if not null
inline SplitState split_operands(const Head<float>& h, const MmaPlan& p, char* ws, int64_t v0, int64_t vp, uint32_t* class_max, bool given,
                                 uint32_t* zeros, int64_t nzeros, cudaStream_t st) {
  SplitJob w, x;
  w.src = h.trans ? h.w + v0 * h.H : h.w + v0;
  w.rows = h.trans ? vp : h.H;
  w.cols = h.trans ? h.H : vp;
  w.pitch = h.trans ? h.H : h.V;
  w.dst = (__half*)(ws + p.ws);
  w.ld = p.wld;
  w.plane = w.rows * p.wld;
  w.labels = nullptr;
  w.mag = class_max && !h.trans ? class_max + v0 : (uint32_t*)(ws + p.wmag);
  given = given && class_max && !h.trans;
  x.src = h.x;
  x.rows = h.N;
  x.cols = x.pitch = h.H;
  x.dst = (__half*)(ws + p.xs);
  x.ld = p.xld;
  x.plane = x.rows * p.xld;
  x.labels = h.labels;
  x.mag = (uint32_t*)(ws + p.xmag);
  auto launch = [&](auto group) { split_launch<decltype(group)::value>(h.trans, w, x, v0 == 0, given, zeros, nzeros, st); };
  // threads per row: 32 features of each stay in registers, of a warp up to twice as many are read again from L1
  // (28212x1352, 120 instances with gradients 423 us by CTAs, 356 by warps)
  if (h.H <= 256) launch(std::integral_constant<int, 8>());
  else if (h.H <= 512) launch(std::integral_constant<int, 16>());
  else if (h.H <= 2048) launch(std::integral_constant<int, 32>());
  else launch(std::integral_constant<int, 256>());
  return SplitState{Planes{w.dst, w.rows, w.cols, w.ld, w.plane}, Planes{x.dst, x.rows, x.cols, x.ld, x.plane}, w.mag, x.mag};
}

// how many parts a sum of C terms really has (each has work, in blocks of 32)
inline int mma_parts(int64_t C, int parts) {
  const int64_t blocks = ceil_div(C, kBK);
  const int64_t k = parts < blocks ? parts : blocks;
  return (int)ceil_div(blocks, ceil_div(blocks, k));
}
// parts of the scores of a piece's classes
inline int mma_scores(const Head<float>& h, const MmaPlan& p, const SplitState& s, int64_t vp, float* scores, uint32_t* done, cudaStream_t st) {
  const MmaStore epi{s.xmag, s.wmag, scores, h.N, vp, vp, h.N * vp, 0, done, GradScale<float>{nullptr, 1.0f}};
  return mma_product(s.x, false, s.w, !h.trans, h.N, vp, h.H, mma_parts(h.H, p.s_parts), epi, st);
}

// lse and loss from the parts of the scores: a warp per instance where there are many, or little to do (forward
// of 1000x16, 4000 instances 30.0 us, with a CTA each 56.7; 500x64, 1000 instances 25.3 and 25.9), a CTA up to
// 8192 classes (4000x64, 200 instances 24.8 us, in chunks 27.6), beyond that chunks of 2048 classes over all SMs
// (50257x1024, one instance 40.4 us, by one CTA 60.0).  The chunks of up to 64 instances are joined by the CTA
// that finishes last (50257x256, one instance 25.3 us, by a launch of its own 27.3; 5000x64, 64 instances 26.4
// and 27.3).
template <typename T>
void statistics(const Head<T>& h, const T* scores, int parts, int64_t chunks, T* stats, T* total, int32_t* count, T* lse,
                T* per_instance, uint32_t* done, cudaStream_t st) {
  if (chunks) {
    T *pm = stats + h.N, *ps = pm + chunks * h.N;
    const bool few = h.N <= 64;
    launch_chained(lnll_chunks_kernel<T>, (unsigned)(chunks * h.N), 256, 0, st, scores, parts, h.bias, h.labels, h.N, h.V, (uint32_t)chunks, pm, ps,
                                                                   stats, lse, per_instance, total, count, few ? done : nullptr);
    if (!few)
      launch_chained(lnll_join_kernel<T>, (unsigned)ceil_div(h.N, 32), 1024, 0, st, pm, ps, stats, h.labels, h.N, h.V, chunks, lse, per_instance, total,
                                                                       count, done);
  } else if (h.V <= 64 || (h.V <= 2048 && h.N >= 1024)) {
    launch_chained(lnll_rows_kernel<T, 32>, (unsigned)ceil_div(h.N, 8), 256, 0, st, scores, parts, h.bias, h.labels, h.N, h.V, lse, per_instance, total,
                                                                       count, done);
  } else {
    launch_chained(lnll_rows_kernel<T, 256>, (unsigned)h.N, 256, 0, st, scores, parts, h.bias, h.labels, h.N, h.V, lse, per_instance, total, count, done);
  }
}

inline int linear_nll_fwd_mma(const Head<float>& h, float* total, int32_t* count, float* lse, float* per_instance, float* class_max, char* ws,
                              cudaStream_t st) {
  const MmaPlan p = mma_plan(h.V, h.H, h.N, h.trans, 0);
  const int64_t all = ceil_div(h.V, kTN);
  uint32_t* done = (uint32_t*)(ws + p.done);
  float *label = (float*)(ws + p.label), *pm = (float*)(ws + p.part_m), *ps = (float*)(ws + p.part_s);
  for (int64_t v0 = 0; v0 < h.V; v0 += p.piece) {
    const int64_t vp = h.V - v0 < p.piece ? h.V - v0 : p.piece;
    const SplitState s = split_operands(h, p, ws, v0, vp, (uint32_t*)class_max, false, nullptr, 0, st);
    if (p.s_parts > 1) {      // one piece
      float* scores = (float*)(ws + p.scores);
      if (int rc = mma_scores(h, p, s, vp, scores, done, st)) return rc;
      statistics<float>(h, scores, mma_parts(h.H, p.s_parts), p.chunks, label, total, count, lse, per_instance, done, st);
      return launch_status();
    }
    const MmaStats epi{s.xmag, s.wmag, h.bias ? h.bias + v0 : nullptr, h.labels, pm, ps, label, done, h.N, vp, v0, v0 / kTN};
    if (int rc = mma_product(s.x, false, s.w, !h.trans, h.N, vp, h.H, 1, epi, st)) return rc;
  }
  launch_chained(lnll_join_kernel<float>, (unsigned)ceil_div(h.N, 32), 1024, 0, st, pm, ps, label, h.labels, h.N, h.V, all, lse, per_instance, total,
                                                                       count, done);
  return launch_status();
}

// db from rows of dS or of its sums over groups of instances
template <typename T>
void bias_gradient(const T* ds, int64_t ld, int64_t rows, int64_t J, T* db, T* parts, GradScale<T> g, cudaStream_t st) {
  const int64_t k = bias_parts(rows, J), part = ceil_div(rows, k);
  const dim3 grid((unsigned)ceil_div(J, 32), (unsigned)ceil_div(rows, part));
  launch_chained(lnll_bias_kernel<T>, grid, 1024, 0, st, ds, ld, rows, J, part, grid.y > 1 ? parts : db, g);
  if (grid.y > 1) sum_parts_to<T>(parts, 1, J, J, (int)grid.y, db, 0, g, st);
}

inline int linear_nll_bwd_mma(const Head<float>& h, const float* lse, const float* class_max, GradScale<float> g, float* dw, float* db, float* dx, char* ws,
                              cudaStream_t st) {
  const MmaPlan p = mma_plan(h.V, h.H, h.N, h.trans, 1);
  float *parts = (float*)(ws + p.parts), *ds = (float*)(ws + p.ds), *dbp = db ? (float*)(ws + p.db) : nullptr;
  uint32_t *rowmax = (uint32_t*)(ws + p.maxima), *colmax = rowmax + h.N;
  for (int64_t v0 = 0; v0 < h.V; v0 += p.piece) {
    const int64_t vp = h.V - v0 < p.piece ? h.V - v0 : p.piece;
    const SplitState s = split_operands(h, p, ws, v0, vp, (uint32_t*)class_max, true, rowmax, h.N + vp, st);
    if (p.s_parts > 1) {
      float* scores = (float*)(ws + p.scores);
      if (int rc = mma_scores(h, p, s, vp, scores, nullptr, st)) return rc;
      const dim3 grid((unsigned)ceil_div(vp, 256), (unsigned)ceil_div(h.N, kGradRows));
      launch_chained(lnll_grad_scores_kernel, grid, 256, 0, st, scores, mma_parts(h.H, p.s_parts), h.bias ? h.bias + v0 : nullptr, h.labels, lse,
                     s.xmag, s.wmag, h.N, vp, v0, ds, p.dld, rowmax, colmax, dbp);
    } else {
      const MmaGradScores e1{s.xmag, s.wmag, h.bias ? h.bias + v0 : nullptr, h.labels, lse, ds, h.N, vp, p.dld, v0, rowmax, colmax, dbp};
      if (int rc = mma_product(s.x, false, s.w, !h.trans, h.N, vp, h.H, 1, e1, st)) return rc;
    }
    if (db) bias_gradient<float>(dbp, vp, ceil_div(h.N, p.s_parts > 1 ? kGradRows : kTM), vp, db + v0, (float*)(ws + p.bias), g, st);
    if (!dx && !dw) continue;
    const int64_t plane = h.N * p.dld;
    const Planes for_dx{(__half*)(ws + p.dx_ds), h.N, vp, p.dld, plane}, for_dw{(__half*)(ws + p.dw_ds), h.N, vp, p.dld, plane};
    // an ordinary launch, as above (10007x515, 333 instances 151 us chained, 145 so)
    lnll_grad_planes_kernel<<<dim3((unsigned)ceil_div(h.N, kPlaneRows), (unsigned)ceil_div(vp, 256)), 256, 0, st>>>(
        ds, p.dld, h.N, vp, s.xmag, s.wmag, rowmax, colmax, dx ? (__half*)for_dx.p : nullptr, dw ? (__half*)for_dw.p : nullptr, plane);
    if (dx) {
      const int k = mma_parts(vp, p.x_parts);
      const MmaStore e2{rowmax, nullptr, k == 1 ? dx : parts, h.N, h.H, h.H, k == 1 ? 0 : h.N * h.H, k == 1 && v0 > 0, nullptr, g};
      if (int rc = mma_product(for_dx, false, s.w, (bool)h.trans, h.N, h.H, vp, k, e2, st)) return rc;
      if (k > 1) sum_parts_to<float>(parts, h.N, h.H, h.H, k, dx, v0 > 0, g, st);
    }
    if (dw) {
      const int k = mma_parts(h.N, p.w_parts);           // more than one only where one piece holds all classes
      const int64_t I = h.trans ? vp : h.H, J = h.trans ? h.H : vp;
      float* out = h.trans ? dw + v0 * h.H : dw + v0;
      const MmaStore e3{h.trans ? colmax : nullptr, h.trans ? nullptr : colmax, k == 1 ? out : parts, I, J, h.trans ? h.H : h.V,
                        k == 1 ? 0 : h.V * h.H, 0, nullptr, g};
      if (int rc = h.trans ? mma_product(for_dw, true, s.x, true, I, J, h.N, k, e3, st) : mma_product(s.x, true, for_dw, true, I, J, h.N, k, e3, st))
        return rc;
      if (k > 1) sum_parts_to<float>(parts, I, J, J, k, dw, 0, g, st);
    }
  }
  return launch_status();
}

// ---- few scores -----------------------------------------------------------------------------------------
template <typename T> Matrix<T> weight_matrix(const Head<T>& h) {
  return h.trans ? Matrix<T>{h.w, h.V, h.H, h.H} : Matrix<T>{h.w, h.H, h.V, h.V};
}
template <typename T> void small_scores(const Head<T>& h, const SmallPlan& p, uint32_t* done, T* scores, cudaStream_t st) {
  if (p.few) few_product<T>(h.trans, weight_matrix(h), h.x, h.H, h.N, p.s_part, p.s_parts, done, scores, st);
  else
    simt_product<T>(Strided<T>{h.x, h.H, 1}, h.weights(0), h.N, h.V, h.H, p.s_part, done, PartsEpi<T>{scores}, st);
}

template <typename T>
int linear_nll_fwd_small(const Head<T>& h, T* total, int32_t* count, T* lse, T* per_instance, char* ws, cudaStream_t st) {
  const SmallPlan p = small_plan<T>(h.V, h.H, h.N, h.trans, 0);
  uint32_t* done = (uint32_t*)ws;
  T* scores = (T*)(ws + p.scores);
  small_scores(h, p, done, scores, st);
  statistics<T>(h, scores, p.s_parts, p.chunks, (T*)(ws + p.stats), total, count, lse, per_instance, done, st);
  return launch_status();
}

template <typename T>
int linear_nll_bwd_small(const Head<T>& h, const T* lse, GradScale<T> g, T* dw, T* db, T* dx, char* ws, cudaStream_t st) {
  const SmallPlan p = small_plan<T>(h.V, h.H, h.N, h.trans, 1);
  T *ds = (T*)(ws + p.scores), *parts = (T*)(ws + p.parts);
  if (!p.few && p.s_parts == 1) {
    simt_product<T>(Strided<T>{h.x, h.H, 1}, h.weights(0), h.N, h.V, h.H, h.H, nullptr,
                    GradScoresEpi<T>{h.bias, h.labels, lse, ds, h.N, h.V, 0}, st);
  } else {
    small_scores(h, p, nullptr, ds, st);
    const int64_t blocks = ceil_div(h.V, 1024);
    launch_chained(lnll_grad_kernel<T>, (unsigned)(blocks * h.N), 256, 0, st, ds, p.s_parts, h.bias, h.labels, lse, h.N, h.V, (uint32_t)blocks);
  }
  if (db) bias_gradient<T>(ds, h.V, h.N, h.V, db, (T*)(ws + p.bias), g, st);
  const Matrix<T> m = weight_matrix(h);
  if (dx) {
    if (p.few) {
      few_product<T>(!h.trans, m, ds, h.V, h.N, p.x_part, p.x_parts, nullptr, parts, st);
      sum_parts_to<T>(parts, h.N, h.H, h.H, p.x_parts, dx, 0, g, st);
    } else {
      const Strided<T> w = h.weights(0);
      tile_product_out<T>(Strided<T>{ds, h.V, 1}, Strided<T>{w.p, w.sc, w.si}, h.N, h.H, h.V, p.x_part, p.x_parts, dx, h.H, 0, parts, g, st);
    }
  }
  if (dw) {
    const int64_t R = m.rows, C = m.cols;
    // rows and columns of W in terms of (dS, x)
    const T *a = h.trans ? ds : h.x, *b = h.trans ? h.x : ds;
    const int64_t lda = h.trans ? h.V : h.H, ldb = h.trans ? h.H : h.V;
    if (p.few) {
      constexpr int VEC = 16 / sizeof(T);
      const dim3 grid((unsigned)ceil_div(R, 64), (unsigned)ceil_div(C, 128));
      if (aligned16(b, ldb) && aligned16(dw, C)) launch_chained(outer_kernel<T, VEC>, grid, 256, 0, st, a, lda, b, ldb, h.labels, h.N, R, C, dw, C, g);
      else launch_chained(outer_kernel<T, 1>, grid, 256, 0, st, a, lda, b, ldb, h.labels, h.N, R, C, dw, C, g);
    } else {
      tile_product_dw<T>(Strided<T>{a, 1, lda}, Strided<T>{b, 1, ldb}, !h.trans, h.labels, R, C, h.N, p.w_part, p.w_parts, dw, C, parts, g, st);
    }
  }
  return launch_status();
}

// ---- many Float64 scores: pieces of the vocabulary on FP64 tiles -------------------------------------------
template <typename T>
int linear_nll_fwd_pieces(const Head<T>& h, T* total, int32_t* count, T* lse, T* per_instance, char* p, cudaStream_t st) {
  const int64_t tiles = ceil_div(h.V, kTile);
  uint32_t* done = (uint32_t*)p;
  T* label_score = (T*)(p += up(4));
  T* part_m = (T*)(p += up((size_t)h.N * sizeof(T)));
  T* part_s = (T*)(p += up((size_t)tiles * h.N * sizeof(T)));
  simt_product<T>(Strided<T>{h.x, h.H, 1}, h.weights(0), h.N, h.V, h.H, h.H, done,
                  StatsEpi<T>{h.bias, h.labels, part_m, part_s, label_score, h.N}, st);
  launch_chained(lnll_join_kernel<T>, (unsigned)ceil_div(h.N, 32), 1024, 0, st, part_m, part_s, label_score, h.labels, h.N, h.V, tiles, lse,
                 per_instance, total, count, done);
  return launch_status();
}

template <typename T>
int linear_nll_bwd_pieces(const Head<T>& h, const T* lse, GradScale<T> g, T* dw, T* db, T* dx, char* ws, cudaStream_t st) {
  const PiecePlan p = piece_plan<T>(h.V, h.H, h.N);
  T *ds = (T*)ws, *parts = (T*)(ws + p.parts);
  for (int64_t v0 = 0; v0 < h.V; v0 += p.piece) {
    const int64_t vp = h.V - v0 < p.piece ? h.V - v0 : p.piece;
    const Strided<T> w = h.weights(v0), d{ds, 1, p.piece}, x{h.x, 1, h.H};
    simt_product<T>(Strided<T>{h.x, h.H, 1}, w, h.N, vp, h.H, h.H, nullptr,
                    GradScoresEpi<T>{h.bias ? h.bias + v0 : nullptr, h.labels, lse, ds, h.N, p.piece, v0}, st);
    if (db) bias_gradient<T>(ds, p.piece, h.N, vp, db + v0, (T*)(ws + p.bias), g, st);
    if (dx)
      tile_product_out<T>(Strided<T>{ds, p.piece, 1}, Strided<T>{w.p, w.sc, w.si}, h.N, h.H, vp, p.x_part, (int)ceil_div(vp, p.x_part), dx, h.H,
                          v0 > 0, parts, g, st);
    if (dw && h.trans) tile_product_dw<T>(d, x, false, h.labels, vp, h.H, h.N, p.w_part, p.w_parts, dw + v0 * h.H, h.H, parts, g, st);
    else if (dw) tile_product_dw<T>(x, d, true, h.labels, h.H, vp, h.N, p.w_part, p.w_parts, dw + v0, h.V, parts, g, st);
  }
  return launch_status();
}

template <typename T>
int linear_nll_fwd(const Head<T>& h, T* total, int32_t* count, T* lse, T* per_instance, T* class_max, void* ws, size_t have, cudaStream_t st) {
  if (!total || !count || (h.N > 0 && (!lse || !per_instance))) return KN_EINVAL;
  if (odd(total) || odd(lse) || odd(per_instance) || odd(class_max) || (uintptr_t)count % 4) return KN_EALIGN;
  const size_t need = h.V > 0 && h.H > 0 && h.N > 0 && sizes_ok(h.V, h.H, h.N) ? workspace<T>(h.V, h.H, h.N, h.trans, 0) : 0;
  if (int rc = check(h, ws, have, need)) return rc;
  if (h.N == 0) {
    launch_chained(lnll_none_kernel<T>, 1, 1, 0, st, total, count);
    return launch_status();
  }
  const Form f = form<T>(h.V, h.H, h.N);
  if constexpr (sizeof(T) == 4) {
    if (f == kMma) return linear_nll_fwd_mma(h, total, count, lse, per_instance, class_max, (char*)ws, st);
  } else if (f == kPieces) {
    return linear_nll_fwd_pieces<T>(h, total, count, lse, per_instance, (char*)ws, st);
  }
  return linear_nll_fwd_small<T>(h, total, count, lse, per_instance, (char*)ws, st);
}

template <typename T>
int linear_nll_bwd(const Head<T>& h, const T* lse, const T* class_max, int average, T dy, const int32_t* count, T* dw, T* db, T* dx, void* ws,
                   size_t have, cudaStream_t st) {
  if (h.N > 0 && (!lse || (average && !count))) return KN_EINVAL;
  if (odd(lse) || odd(class_max) || odd(dw) || odd(db) || odd(dx) || (uintptr_t)count % 4) return KN_EALIGN;
  const size_t need = h.V > 0 && h.H > 0 && h.N > 0 && sizes_ok(h.V, h.H, h.N) ? workspace<T>(h.V, h.H, h.N, h.trans, 1) : 0;
  if (int rc = check(h, ws, have, need)) return rc;
  if (h.N == 0) {
    lnll_zero(dw, h.V * h.H, st);
    lnll_zero(db, h.V, st);
    return launch_status();
  }
  const GradScale<T> g{average ? count : nullptr, dy};
  const Form f = form<T>(h.V, h.H, h.N);
  if constexpr (sizeof(T) == 4) {
    if (f == kMma) return linear_nll_bwd_mma(h, lse, class_max, g, dw, db, dx, (char*)ws, st);
  } else if (f == kPieces) {
    return linear_nll_bwd_pieces<T>(h, lse, g, dw, db, dx, (char*)ws, st);
  }
  return linear_nll_bwd_small<T>(h, lse, g, dw, db, dx, (char*)ws, st);
}

}  // namespace kn

using namespace kn;

#define KN_DEF_LNLL(f_, S, T)                                                                                       \
  KN_EXPORT size_t knet_linear_nll_workspace_##S(int64_t V, int64_t H, int64_t N, int backward) {                   \
    if (V <= 0 || H <= 0 || N <= 0 || !sizes_ok(V, H, N)) return 0;                                                 \
    return workspace_any<T>(V, H, N, backward != 0);                                                                \
  }                                                                                                                 \
  KN_EXPORT int knet_linear_nll_fwd_max_##S(const T* w, int transW, const T* b, const T* x, const int32_t* labels,  \
                                            int64_t V, int64_t H, int64_t N, T* total, int32_t* count, T* lse,      \
                                            T* per_instance, T* class_max, void* workspace,                         \
                                            size_t workspace_bytes, cudaStream_t s) {                               \
    return linear_nll_fwd<T>(Head<T>{w, transW, b, x, labels, V, H, N}, total, count, lse, per_instance, class_max, \
                             workspace, workspace_bytes, s);                                                        \
  }                                                                                                                 \
  KN_EXPORT int knet_linear_nll_bwd_max_##S(const T* w, int transW, const T* b, const T* x, const int32_t* labels,  \
                                            int64_t V, int64_t H, int64_t N, const T* lse, const T* class_max,      \
                                            int average, T dy, const int32_t* count, T* dw, T* db, T* dx,           \
                                            void* workspace, size_t workspace_bytes, cudaStream_t s) {              \
    return linear_nll_bwd<T>(Head<T>{w, transW, b, x, labels, V, H, N}, lse, class_max, average, dy, count, dw, db, \
                             dx, workspace, workspace_bytes, s);                                                    \
  }                                                                                                                 \
  KN_EXPORT int knet_linear_nll_fwd_##S(const T* w, int transW, const T* b, const T* x, const int32_t* labels,      \
                                        int64_t V, int64_t H, int64_t N, T* total, int32_t* count, T* lse,          \
                                        T* per_instance, void* workspace, size_t workspace_bytes, cudaStream_t s) { \
    return knet_linear_nll_fwd_max_##S(w, transW, b, x, labels, V, H, N, total, count, lse, per_instance, nullptr,  \
                                       workspace, workspace_bytes, s);                                              \
  }                                                                                                                 \
  KN_EXPORT int knet_linear_nll_bwd_##S(const T* w, int transW, const T* b, const T* x, const int32_t* labels,      \
                                        int64_t V, int64_t H, int64_t N, const T* lse, int average, T dy,           \
                                        const int32_t* count, T* dw, T* db, T* dx, void* workspace,                 \
                                        size_t workspace_bytes, cudaStream_t s) {                                   \
    return knet_linear_nll_bwd_max_##S(w, transW, b, x, labels, V, H, N, lse, nullptr, average, dy, count, dw, db,  \
                                       dx, workspace, workspace_bytes, s);                                          \
  }
KNET_BOTH_TYPES(KN_DEF_LNLL, lnll)

// Float32 products of the linear-layer cross entropy on the tensor cores.
//
// A row of a Float32 operand (a class of W, an instance of x), scaled by a power of two that brings its largest
// magnitude into [2^14, 2^15), is split into two fp16 terms, hi = fp16(v), lo = fp16(v - hi): together 22 bits,
// and never less than 2^-25 of the scaled value's unit, so entries down to 2^-16 of the row's largest keep a relative
// error of 2^-23.  The row has its own scale, undone in the epilogue, so that a large instance or class costs no
// other one its bits.  dS is kept in Float32 and split twice: for dx = W' dS with a scale per instance, for
// dW = dS x' with one per class, the scales of W's classes and x's instances taken into it, since the sums run over
// those.  (Terms of every magnitude, three in bf16, would make a product of six partial ones.)
// A product takes three of the four partial products (lo*lo is below 2^-22 of it), which are
// exact in Float32; the tensor core adds them.  Its additions truncate: measured on sums of 1024 and 8192
// products, an accumulator that takes n blocks of 32 summed indices comes out low by 0.75 n 2^-23 of its
// value for terms of random signs (n = 4, 8, 16: 3.4e-7, 7.4e-7, 1.5e-6), about twice that for terms of
// one sign.  The accumulator in TMEM therefore takes 256 summed indices, the chunks are added in registers
// with rounding to nearest, and the epilogue multiplies by 1 + 0.75 n 2^-23, which leaves a relative error
// of 5e-7 to 8e-7 in a product and leaves one of terms of one sign up to 9e-7 low.  (Chunks of 128 halve the error;
// 256 give the epilogue 10 us instead of 5 before the tensor core has to wait for it.)
//
// A CTA owns a 128 x 256 tile of the result, or a pair of CTAs (a cluster) one of 256 x 256.  Warp 16 loads
// the operands with TMA into a ring of stages of 32 summed indices (both planes of 128 rows of A and of 256
// rows of B, or the CTA's 128 of them); warp 17, of a pair the first CTA's, issues the products into one of
// two halves of TMEM (256 columns each); warps 0-15 move finished chunks from the other half into registers,
// 64 columns of one row per thread, and run the epilogue while the tensor core works on the next tile.
//
// Alone, a CTA writes 48 KB and reads 72 KB of shared memory per 32 summed indices, 160 bytes per clock at the
// tensor core's full rate where shared memory has 128; in a pair, where each loads half of B, 32 + 48 KB or 107
// bytes.  Scores of 50257 classes x 4096 instances: 818 us alone, 748 us in pairs (1692 TFLOP/s of fp16
// products; the device's own library reaches 1658 on bf16).
#pragma once
#include <cuda_fp16.h>

#include "linear_nll.cuh"
#include "umma.cuh"

namespace kn {

constexpr int kTM = 128, kTN = 256, kBK = 32;
constexpr int kChunkBlocks = 8;                         // 256 summed indices per accumulator
// Registers: 640 threads start with 96 each; the four warps beside the epilogue give up all but 32 and
// the epilogue's 512 threads take 112 (57 344 + 4 096 of 61 440).
constexpr int kEpiWarps = 16, kMmaThreads = (kEpiWarps + 4) * 32;
constexpr uint32_t kStageA = 2 * kTM * kBK * 2;
// a CTA's share of B in a stage, and the stages: 48 KB x 4 alone, 32 KB x 6 in a pair
template <int CG> constexpr uint32_t kStageB = 2 * (kTN / CG) * kBK * 2;
template <int CG> constexpr uint32_t kStageBytes = kStageA + kStageB<CG>;
template <int CG> constexpr uint32_t kStages = CG == 1 ? 4 : 6;
constexpr int kMaxStages = 6;

struct MmaShared {
  uint64_t full[kMaxStages], empty[kMaxStages], acc_full[2], acc_empty[2], drain;
  uint32_t tmem;
  int gave_up;
  float2 stat[2][4][kTM];                               // per tile parity, column quarter and row
  __align__(16) float bias[2][kTN], mag[2][kTN];        // per tile parity
  float colsum[4][kTN];
};
constexpr size_t kMmaSmem = 1024 + (size_t)kStages<1> * kStageBytes<1> + sizeof(MmaShared);
static_assert(kStages<1> * kStageBytes<1> == kStages<2> * kStageBytes<2>, "one size");

// how one launch walks its tiles: rows i fastest, then columns j, then parts of the summed axis
struct MmaTiles {
  uint32_t i_tiles, j_tiles, splits;
  uint32_t blocks, blocks_per_split;                    // of 32 summed indices
  int a_mn, b_mn;                                       // operand stored with its row index contiguous
};

// A wait that gives up (or finds that another role has) makes every role of the CTA leave; the other CTA of
// a pair then runs into its own limits.
template <int CG> __device__ __forceinline__ bool mma_wait(uint64_t* bar, uint32_t parity, int* gave_up) {
  for (uint32_t i = 0; i < kWaitSpins; i++) {
    if (CG == 1 ? mbar_try_wait(bar, parity) : mbar_try_wait_cluster(bar, parity)) return true;
    if (*(volatile int*)gave_up) return false;
    if (i > 256) __nanosleep(128);
  }
  *(volatile int*)gave_up = 1;
  note_wait_timeout();
  return false;
}

// Arithmetic on two neighbours in one instruction.  The epilogues share power and issue slots with the
// tensor core: packed additions in the drain alone took the scores of 50257 classes x 4096 instances from
// 857 to 830 us.
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 r;
  asm("{\n\t.reg .b64 a, b;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tadd.rn.f32x2 a, a, b;\n\tmov.b64 {%0, %1}, a;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 r;
  asm("{\n\t.reg .b64 a, b;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmul.rn.f32x2 a, a, b;\n\tmov.b64 {%0, %1}, a;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("{\n\t.reg .b64 a, b, c;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
      "fma.rn.f32x2 a, a, b, c;\n\tmov.b64 {%0, %1}, a;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return r;
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

// what the epilogue of one tile gets besides the accumulators
struct TileAt {
  int64_t i, j0;               // this thread's row and first of its 64 columns
  uint32_t it, jt, split;      // tile
  uint32_t turn;               // how many tiles this CTA has finished
  int quarter, row;            // which 64 columns, which of the 128 rows
  float gain;                  // makes up for the mean loss of the truncated additions
  MmaShared* sh;
};

// barriers among the 512 epilogue threads; the second tells every one of them whether any says yes
__device__ __forceinline__ void epi_sync() { asm volatile("barrier.cta.sync 1, 512;" ::: "memory"); }
__device__ __forceinline__ bool epi_any(bool yes) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %1, 0;\n\t"
      "barrier.cta.red.or.pred q, 1, 512, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"((uint32_t)yes)
      : "memory");
  return r != 0;
}

template <int CG, typename Epi>
__global__ void __launch_bounds__(kMmaThreads, 1)
mma_kernel(const __grid_constant__ CUtensorMap amap, const __grid_constant__ CUtensorMap bmap, MmaTiles tl, Epi epi) {
  constexpr uint32_t STAGES = kStages<CG>, STAGE = kStageBytes<CG>, BN = kTN / CG;
  extern __shared__ uint8_t raw[];
  uint8_t* stages = reinterpret_cast<uint8_t*>(((uintptr_t)raw + 1023) & ~(uintptr_t)1023);
  MmaShared* sh = reinterpret_cast<MmaShared*>(stages + (size_t)STAGES * STAGE);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = CG == 1 ? 0 : cluster_rank();
  const uint32_t worker = blockIdx.x / CG, workers = gridDim.x / CG;     // a CTA or a pair
  const uint32_t tiles = tl.i_tiles * tl.j_tiles * tl.splits;

  if (threadIdx.x == 0) {
    for (uint32_t s = 0; s < STAGES; s++) {
      mbar_init(&sh->full[s], 1);
      mbar_init(&sh->empty[s], 1);
    }
    for (int b = 0; b < 2; b++) {
      mbar_init(&sh->acc_full[b], 1);
      mbar_init(&sh->acc_empty[b], kEpiWarps * CG);
    }
    mbar_init(&sh->drain, 1);
    sh->gave_up = 0;
    mbar_init_fence();
  }
  __syncwarp();
  if (warp == kEpiWarps + 1) tmem_alloc<CG>(&sh->tmem, 512);
  tcgen05_before_sync();
  if constexpr (CG == 1) __syncthreads();
  else cluster_barrier();
  tcgen05_after_sync();
  const uint32_t tmem = sh->tmem;
  chain_begin();

  if (warp >= kEpiWarps) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 32;");
    if (warp == kEpiWarps) {
      // ---- loads: this CTA's rows of A and its share of B; in a pair all bytes count on the first CTA's barrier
      if (lane == 0) {
        tma_prefetch_map(&amap);
        tma_prefetch_map(&bmap);
        uint32_t n = 0;                                   // stages filled so far
        bool ok = true;
        for (uint32_t t = worker; t < tiles && ok; t += workers) {
          const uint32_t it = t % tl.i_tiles, r = t / tl.i_tiles, jt = r % tl.j_tiles, sp = r / tl.j_tiles;
          const uint32_t k0 = sp * tl.blocks_per_split, k1 = min(k0 + tl.blocks_per_split, tl.blocks);
          const int32_t i0 = (int32_t)((it * CG + rank) * kTM), j0 = (int32_t)(jt * kTN + rank * BN);
          for (uint32_t k = k0; k < k1; k++, n++) {
            const uint32_t s = n % STAGES;
            if (n >= STAGES && !mma_wait<CG>(&sh->empty[s], (n / STAGES - 1) & 1, &sh->gave_up)) {
              ok = false;
              break;
            }
            uint8_t* a = stages + (size_t)s * STAGE;
            uint8_t* b = a + kStageA;
            const int32_t c = (int32_t)(k * kBK);
            if (rank == 0) mbar_arrive_expect_tx(&sh->full[s], STAGE * CG);
            const uint32_t bar = CG == 1 ? 0 : mapa_u32(&sh->full[s], 0);
            auto load = [&](uint8_t* to, const CUtensorMap* map, int32_t x, int32_t y) {
              if constexpr (CG == 1) tma_load_3d(to, map, x, y, 0, &sh->full[s]);
              else tma_load_3d_pair(to, map, x, y, 0, bar);
            };
            if (tl.a_mn) {
              for (int g = 0; g < kTM / 64; g++) load(a + g * 8192, &amap, i0 + g * 64, c);
            } else {
              load(a, &amap, c, i0);
            }
            if (tl.b_mn) {
              for (uint32_t g = 0; g < BN / 64; g++) load(b + g * 8192, &bmap, j0 + (int32_t)g * 64, c);
            } else {
              load(b, &bmap, c, j0);
            }
          }
        }
        // every load issued has landed before this CTA may leave: the first CTA sees it on its barriers (the
        // products that it waits for below have read the second CTA's); after a wait that gave up the second
        // CTA leaves its own loads a millisecond
        if (rank == 0) {
          for (uint32_t m = n > STAGES ? n - STAGES : 0; m < n; m++)
            for (uint32_t i = 0; i < kWaitSpins && !mbar_try_wait(&sh->full[m % STAGES], (m / STAGES) & 1); i++) __nanosleep(64);
        } else if (!ok) {
          for (int i = 0; i < 1000; i++) __nanosleep(1000);
        }
      }
    } else if (warp == kEpiWarps + 1) {
      // ---- products, by the first CTA
      if (lane == 0 && rank == 0) {
        const uint32_t idesc = umma_idesc(kTM * CG, kTN, tl.a_mn, tl.b_mn);
        const uint64_t ad = tl.a_mn ? umma_desc(8192, 1024, 2) : umma_desc(16, 8 * kBK * 2, 4);
        const uint64_t bd = tl.b_mn ? umma_desc(8192, 1024, 2) : umma_desc(16, 8 * kBK * 2, 4);
        // second plane, and 16 summed indices further, in bytes
        const uint32_t alo = tl.a_mn ? 4096 : kTM * kBK * 2, blo = tl.b_mn ? 4096 : BN * kBK * 2;
        const uint32_t ak = tl.a_mn ? 2048 : 32, bk = tl.b_mn ? 2048 : 32;
        uint32_t n = 0, ch = 0;                           // stages and chunks so far
        bool ok = true;
        for (uint32_t t = worker; t < tiles && ok; t += workers) {
          const uint32_t sp = t / (tl.i_tiles * tl.j_tiles);
          const uint32_t k0 = sp * tl.blocks_per_split, k1 = min(k0 + tl.blocks_per_split, tl.blocks);
          for (uint32_t k = k0; k < k1 && ok; ch++) {
            const uint32_t buf = ch & 1, d = tmem + buf * kTN;
            if (ch >= 2 && !mma_wait<CG>(&sh->acc_empty[buf], ((ch >> 1) - 1) & 1, &sh->gave_up)) {
              ok = false;
              break;
            }
            tcgen05_after_sync();
            const uint32_t ke = min(k + kChunkBlocks, k1);
            bool acc = false;
            for (; k < ke; k++, n++) {
              const uint32_t s = n % STAGES;
              if (!mma_wait<CG>(&sh->full[s], (n / STAGES) & 1, &sh->gave_up)) {
                ok = false;
                break;
              }
              tcgen05_after_sync();
              const uint32_t a = smem_u32(stages + (size_t)s * STAGE), b = a + kStageA;
              // the small cross terms first, while the sum is small
#pragma unroll
              for (uint32_t q = 0; q < kBK / 16; q++) {
                umma_f16<CG>(d, umma_at(ad, a + alo + q * ak), umma_at(bd, b + q * bk), idesc, acc);
                umma_f16<CG>(d, umma_at(ad, a + q * ak), umma_at(bd, b + blo + q * bk), idesc, true);
                acc = true;
              }
#pragma unroll
              for (uint32_t q = 0; q < kBK / 16; q++) umma_f16<CG>(d, umma_at(ad, a + q * ak), umma_at(bd, b + q * bk), idesc, true);
              umma_commit<CG>(&sh->empty[s]);
            }
            if (!ok) break;
            umma_commit<CG>(&sh->acc_full[buf]);
          }
        }
        // every product issued is done before TMEM is freed
        umma_commit<CG>(&sh->drain);
        for (uint32_t i = 0; i < kWaitSpins && !mbar_try_wait(&sh->drain, 0); i++) __nanosleep(64);
      }
    }
  } else {
    // ---- accumulators -> registers -> epilogue
    asm volatile("setmaxnreg.inc.sync.aligned.u32 112;");
    const int q = warp & 3, quarter = warp >> 2;
    const uint32_t lane_addr = (uint32_t)(q * 32) << 16;
    uint32_t ch = 0, turn = 0;
    bool ok = true;
    for (uint32_t t = worker; t < tiles && ok; t += workers, turn++) {
      const uint32_t it = t % tl.i_tiles, r = t / tl.i_tiles, jt = r % tl.j_tiles, sp = r / tl.j_tiles;
      const uint32_t k0 = sp * tl.blocks_per_split, k1 = min(k0 + tl.blocks_per_split, tl.blocks);
      epi.stage((int64_t)jt * kTN, sh, turn & 1);        // read after the barrier below
      float2 acc[32];                                   // 64 columns
#pragma unroll
      for (int e = 0; e < 32; e++) acc[e] = both(0.0f);
      for (uint32_t k = k0; k < k1; k += kChunkBlocks, ch++) {
        const uint32_t buf = ch & 1;
        ok = __all_sync(0xffffffffu, mma_wait<CG>(&sh->acc_full[buf], (ch >> 1) & 1, &sh->gave_up));
        if (!ok) break;
        tcgen05_after_sync();
#pragma unroll
        for (int h = 0; h < 4; h++) {
          uint32_t v[16];
          tmem_load16(tmem + lane_addr + buf * kTN + quarter * 64 + h * 16, v);
          tmem_load_wait();
#pragma unroll
          for (int e = 0; e < 16; e += 2) acc[h * 8 + e / 2] = add2(acc[h * 8 + e / 2], make_float2(__uint_as_float(v[e]), __uint_as_float(v[e + 1])));
        }
        tcgen05_before_sync();
        __syncwarp();
        if (lane == 0) {
          if constexpr (CG == 1) mbar_arrive(&sh->acc_empty[buf]);
          else mbar_arrive_remote(mapa_u32(&sh->acc_empty[buf], 0));
        }
      }
      // the epilogue has barriers of its own: all of its warps run it, or none
      if (epi_any(!ok)) break;
      const uint32_t rows = it * CG + rank;              // 128-row tile
      const TileAt at{(int64_t)rows * kTM + q * 32 + lane, (int64_t)jt * kTN + quarter * 64, rows, jt, sp, turn, quarter, q * 32 + lane,
                      1.0f + 0.75f * 0x1p-23f * (float)min((uint32_t)kChunkBlocks, k1 - k0), sh};
      epi(acc, at);
    }
  }
  __syncwarp();
  tcgen05_before_sync();
  if constexpr (CG == 1) __syncthreads();
  else cluster_barrier();
  tcgen05_after_sync();
  if (warp == kEpiWarps + 1) tmem_free<CG>(tmem, 512);
  if constexpr (CG == 2) cluster_barrier();              // neither CTA leaves while the other still frees or signals
}

// ---- scaling ------------------------------------------------------------------------------------------
// An operand's row is multiplied by 2^14 / m, m being the power of two at or below its largest finite magnitude
// (2^-112 at least: data below it stays below 2^14, with terms as fine as before).  Arrays keep that
// magnitude's bits, 0 for a row of zeros.
__device__ __forceinline__ float magnitude(uint32_t max_bits) { return __uint_as_float(max(max_bits & 0x7f800000u, 15u << 23)); }
__device__ __forceinline__ float scale_of(float m) { return __uint_as_float((268u << 23) - __float_as_uint(m)); }
__device__ __forceinline__ float power2(int e) { return __int_as_float((127 + e) << 23); }
__device__ __forceinline__ uint32_t finite_bits(float v) {
  const uint32_t u = __float_as_uint(v) & 0x7fffffffu;
  return u < 0x7f800000u ? u : 0u;
}
// A sum of products of two such operands times 2^-28, the row's m and the column's: acc * a * column * b, in an
// order in which no step leaves the range unless the result does (m is 2^-112 .. 2^127).
struct Unscale {
  float a, b;
};
__device__ __forceinline__ Unscale unscale(float m, float gain) {
  const int e = (int)(__float_as_uint(m) >> 23) - 127, h = e / 2;
  return Unscale{gain * power2(h - 28), power2(e - h)};
}

struct SplitJob {
  const float* src;            // rows x cols, row pitch `pitch`
  int64_t rows, cols, pitch;
  __half* dst;                 // two planes of rows x ld
  int64_t ld, plane;
  const int32_t* labels;       // of the rows, or null: see split_rows
  uint32_t* mag;               // largest finite magnitude per instance or class
};

// v = hi + lo in fp16 for two values; what is not finite goes to hi alone, so that an infinity is not NaN
__device__ __forceinline__ void split_pair(float v0, float v1, uint32_t& hi, uint32_t& lo) {
  const __half2 h = __floats2half2_rn(v0, v1);
  const float2 f = __half22float2(h);
  float r0 = v0 - f.x, r1 = v1 - f.y;
  r0 = r0 == r0 ? r0 : 0.0f;
  r1 = r1 == r1 ? r1 : 0.0f;
  const __half2 l = __floats2half2_rn(r0, r1);
  hi = *reinterpret_cast<const uint32_t*>(&h);
  lo = *reinterpret_cast<const uint32_t*>(&l);
}

// Eight consecutive floats at p, of which `left` are inside the row (0 past its end).  OFF 0..3: p lies OFF floats past a
// multiple of 16 bytes and the aligned 16-byte words around the eight are inside the row; the shift is the same for
// all rows that a thread walks, so it is a constant here.  OFF 4: single loads.  OFF 5: as 0..3 but by the address (rows of a warp that differ in it would else take turns).
__device__ __forceinline__ int offset_of(const float* p) { return (int)(((uintptr_t)p >> 2) & 3); }
template <int OFF> __device__ __forceinline__ void load_at(const float* p, int64_t left, float (&v)[8]) {
  if constexpr (OFF == 5) {
    const int off = offset_of(p);
    const float4* q = reinterpret_cast<const float4*>(p - off);
    const float4 a = q[0], b = q[1], d = off ? q[2] : b;
    const float t[12] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w, d.x, d.y, d.z, d.w};
#pragma unroll
    for (int k = 0; k < 8; k++) v[k] = off == 0 ? t[k] : off == 1 ? t[k + 1] : off == 2 ? t[k + 2] : t[k + 3];
  } else if constexpr (OFF < 4) {
    const float4* q = reinterpret_cast<const float4*>(p - OFF);
    const float4 a = q[0], b = q[1], d = OFF ? q[2] : b;
    const float t[12] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w, d.x, d.y, d.z, d.w};
#pragma unroll
    for (int k = 0; k < 8; k++) v[k] = t[k + OFF];
  } else {
#pragma unroll
    for (int k = 0; k < 8; k++) v[k] = k < left ? p[k] : 0.0f;
  }
}
__device__ __forceinline__ bool words_inside(int off, int64_t c, int64_t cols) { return c - off >= 0 && c - off + (off ? 12 : 8) <= cols; }

// 8 values times their scales in two planes; the pitch is a multiple of 8
__device__ __forceinline__ void store_split(const SplitJob& j, int64_t r, int64_t c, const float (&v)[8]) {
  uint4 hi, lo;
  split_pair(v[0], v[1], hi.x, lo.x);
  split_pair(v[2], v[3], hi.y, lo.y);
  split_pair(v[4], v[5], hi.z, lo.z);
  split_pair(v[6], v[7], hi.w, lo.w);
  *reinterpret_cast<uint4*>(j.dst + r * j.ld + c) = hi;
  *reinterpret_cast<uint4*>(j.dst + j.plane + r * j.ld + c) = lo;
}

// of rows that lie one behind the other
template <int OFF> __device__ __forceinline__ void load_of_row(const float* p, int64_t left, float (&v)[8]) {
  load_at<OFF>(p, left, v);                              // the words around the eight may reach into the rows beside this one
  if (OFF != 4 && left < 8) {
#pragma unroll
    for (int k = 0; k < 8; k++)
      if (k >= left) v[k] = 0.0f;
  }
}
// x, or W whose classes are rows, which lie one behind the other: GROUP threads take a row, read it (up to 32 values per
// thread stay in registers, what is longer comes from L1 the second time) and scale it by its own maximum.  In a
// skipped instance (label 0) whatever has no fp16 value becomes 0: its dS is 0, which times infinity would be NaN in dW.
template <int GROUP, int OFF>
__device__ __forceinline__ void split_row(const SplitJob& j, int64_t r, bool live, uint32_t* red) {
  constexpr int KEEP = 4;
  const int t = threadIdx.x % GROUP;
  const float* row = j.src + r * j.pitch;
  const bool skipped = j.labels && j.labels[r] == 0;
  const bool kept = j.cols <= KEEP * GROUP * 8;
  float v[KEEP][8];
  uint32_t m = 0;
  for (int64_t c0 = t * 8; c0 < j.cols; c0 += KEEP * GROUP * 8) {
#pragma unroll
    for (int k = 0; k < KEEP; k++)
      if (c0 + k * GROUP * 8 < j.cols) load_of_row<OFF>(row + c0 + k * GROUP * 8, j.cols - c0 - k * GROUP * 8, v[k]);
#pragma unroll
    for (int k = 0; k < KEEP; k++)
      if (c0 + k * GROUP * 8 < j.cols) {
#pragma unroll
        for (int e = 0; e < 8; e++) m = max(m, finite_bits(v[k][e]));
      }
  }
  if constexpr (GROUP == 256) {
    m = block_reduce(m, [](uint32_t a, uint32_t b) { return max(a, b); }, 0u, red);
  } else {      // rows of a warp may take different branches of the caller
    const uint32_t mask = GROUP == 32 ? 0xffffffffu : ((1u << GROUP) - 1) << (threadIdx.x & 31 & ~(GROUP - 1));
#pragma unroll
    for (int o = GROUP / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(mask, m, o));
  }
  if (!live) return;
  if (t == 0) j.mag[r] = m;
  const float f = scale_of(magnitude(m));
  for (int64_t c0 = t * 8; c0 < j.cols; c0 += KEEP * GROUP * 8)
#pragma unroll
    for (int k = 0; k < KEEP; k++) {
      const int64_t c = c0 + k * GROUP * 8;
      if (c >= j.cols) break;
      if (!kept) load_of_row<OFF>(row + c, j.cols - c, v[k]);
#pragma unroll
      for (int e = 0; e < 8; e++) {
        v[k][e] *= f;
        if (skipped && !(fabsf(v[k][e]) <= 65504.0f)) v[k][e] = 0.0f;
      }
      store_split(j, r, c, v[k]);
    }
}
template <int GROUP> __device__ __forceinline__ void split_rows(const SplitJob& j, int64_t block, uint32_t* red) {
  if (block * (256 / GROUP) >= j.rows) return;           // the whole CTA
  const int64_t at = block * (256 / GROUP) + threadIdx.x / GROUP;
  const bool live = at < j.rows;
  const int64_t r = live ? at : j.rows - 1;
  // a row's words lie inside the array but at its two ends; one row per CTA where it has barriers
  const bool inside = r * j.pitch >= 3 && (j.rows - 1 - r) * j.pitch >= 12;
  if constexpr (GROUP < 32) return inside ? split_row<GROUP, 5>(j, r, live, red) : split_row<GROUP, 4>(j, r, live, red);
  else switch (inside ? offset_of(j.src + r * j.pitch) : 4) {
      case 0: return split_row<GROUP, 0>(j, r, live, red);
      case 1: return split_row<GROUP, 1>(j, r, live, red);
      case 2: return split_row<GROUP, 2>(j, r, live, red);
      case 3: return split_row<GROUP, 3>(j, r, live, red);
      default: return split_row<GROUP, 4>(j, r, live, red);
    }
}

// maxima of dS's rows and columns, which a kernel that follows takes, begin at 0
__device__ __forceinline__ void clear(uint32_t* zeros, int64_t n) {
  const int64_t blocks = (int64_t)gridDim.x * gridDim.y, b = (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
  for (int64_t i = b * 256 + threadIdx.x; i < n; i += blocks * 256) zeros[i] = 0;
}

// x and W whose classes are rows: the first blocks take W, the others x
template <int GROUP>
__global__ void __launch_bounds__(256, 4)
lnll_split_rows_kernel(SplitJob w, SplitJob x, uint32_t blocks_w, uint32_t* zeros, int64_t nzeros) {
  chain_begin();
  __shared__ uint32_t red[32];
  clear(zeros, nzeros);
  if (blockIdx.x >= blocks_w) split_rows<GROUP>(x, blockIdx.x - blocks_w, red);
  else split_rows<GROUP>(w, blockIdx.x, red);
}

// W whose classes are columns.  A thread takes eight of them and every eighth row (the features), so that its rows
// have one offset in their 16-byte words; a CTA 256 classes.
constexpr int kSplitCols = 256;
template <int UN, int OFF>
__device__ __forceinline__ void col_maxima(const SplitJob& w, int64_t c, int64_t r0, int64_t hi, uint32_t (&m)[8]) {
  for (int64_t r = r0; r < hi; r += 8 * UN) {
    float v[UN][8];
#pragma unroll
    for (int u = 0; u < UN; u++)
      if (r + 8 * u < hi) load_at<OFF>(w.src + (r + 8 * u) * w.pitch + c, w.cols - c, v[u]);
#pragma unroll
    for (int u = 0; u < UN; u++)
      if (r + 8 * u < hi) {
#pragma unroll
        for (int e = 0; e < 8; e++) m[e] = max(m[e], finite_bits(v[u][e]));
      }
  }
}
// from the last row, which the maxima's pass has left in the caches
template <int UN, int OFF>
__device__ __forceinline__ void col_split(const SplitJob& w, int64_t c, int64_t r0, int64_t hi, const float (&f)[8]) {
  for (int64_t r = r0 + (hi - 1 - r0) / 8 * 8; r >= r0; r -= 8 * UN) {
    float v[UN][8];
#pragma unroll
    for (int u = 0; u < UN; u++)
      if (r - 8 * u >= r0) load_at<OFF>(w.src + (r - 8 * u) * w.pitch + c, w.cols - c, v[u]);
#pragma unroll
    for (int u = 0; u < UN; u++)
      if (r - 8 * u >= r0) {
#pragma unroll
        for (int e = 0; e < 8; e++) v[u][e] *= f[e];
        store_split(w, r - 8 * u, c, v[u]);
      }
  }
}
struct ColumnShare {
  int64_t c, r0, hi;           // this thread's first class, first row and the end of the CTA's rows
  bool in;
  int how;                     // offset in a word, 4 at the ends of a row
  __device__ __forceinline__ ColumnShare(const SplitJob& w, int64_t group, int64_t lo, int64_t hi_)
      : c(group * kSplitCols + (threadIdx.x & 31) * 8), r0(lo + (threadIdx.x >> 5)), hi(min(w.rows, hi_)) {
    in = c < w.cols && r0 < hi;
    const int off = in ? offset_of(w.src + r0 * w.pitch + c) : 0;
    how = words_inside(off, c, w.cols) ? off : 4;
  }
  template <int UN> __device__ __forceinline__ void maxima(const SplitJob& w, uint32_t (*part)[kSplitCols]) const {
    uint32_t m[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (in) switch (how) {
        case 0: col_maxima<UN, 0>(w, c, r0, hi, m); break;
        case 1: col_maxima<UN, 1>(w, c, r0, hi, m); break;
        case 2: col_maxima<UN, 2>(w, c, r0, hi, m); break;
        case 3: col_maxima<UN, 3>(w, c, r0, hi, m); break;
        default: col_maxima<UN, 4>(w, c, r0, hi, m);
      }
#pragma unroll
    for (int e = 0; e < 8; e++) part[threadIdx.x >> 5][(threadIdx.x & 31) * 8 + e] = m[e];
  }
  template <int UN> __device__ __forceinline__ void split(const SplitJob& w, const float (&f)[8]) const {
    switch (how) {
      case 0: return col_split<UN, 0>(w, c, r0, hi, f);
      case 1: return col_split<UN, 1>(w, c, r0, hi, f);
      case 2: return col_split<UN, 2>(w, c, r0, hi, f);
      case 3: return col_split<UN, 3>(w, c, r0, hi, f);
      default: return col_split<UN, 4>(w, c, r0, hi, f);
    }
  }
};
__device__ __forceinline__ uint32_t joined(const uint32_t (*part)[kSplitCols]) {      // of column threadIdx.x
  uint32_t a = 0;
#pragma unroll
  for (int k = 0; k < 8; k++) a = max(a, part[k][threadIdx.x]);
  return a;
}

// Few features: a cluster of CTAs takes the 256 classes, each CTA a share of the rows.  The maxima of the shares meet
// through the cluster's shared memory; the second read of a share finds it in L1 and L2.  The clusters of the first
// blocks take W, the other blocks x.
__device__ __forceinline__ uint32_t ld_cluster_u32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
constexpr int kSplitCtas = 8;
template <int GROUP>
__global__ void __launch_bounds__(256, 4)
lnll_split_cols_kernel(SplitJob w, SplitJob x, uint32_t blocks_w, uint32_t ctas, uint32_t* zeros, int64_t nzeros) {
  chain_begin();
  clear(zeros, nzeros);
  __shared__ uint32_t part[8][kSplitCols], mine[kSplitCols], all[kSplitCols];
  if (blockIdx.x >= blocks_w) return split_rows<GROUP>(x, blockIdx.x - blocks_w, mine);
  const uint32_t rank = ctas > 1 ? cluster_rank() : 0;
  const int64_t group = blockIdx.x / ctas, share = (w.rows + ctas - 1) / ctas, col = group * kSplitCols + threadIdx.x;
  const ColumnShare s(w, group, rank * share, (rank + 1) * share);
  s.maxima<2>(w, part);
  __syncthreads();
  uint32_t a = joined(part);
  mine[threadIdx.x] = a;
  if (ctas > 1) {
    cluster_barrier();
    for (uint32_t k = 0; k < ctas; k++) a = max(a, ld_cluster_u32(mapa_u32(&mine[threadIdx.x], k)));
    cluster_barrier();                                   // no CTA leaves while another reads its share
  }
  all[threadIdx.x] = a;
  __syncthreads();
  if (rank == 0 && col < w.cols) w.mag[col] = a;
  if (!s.in) return;
  float f[8];
#pragma unroll
  for (int e = 0; e < 8; e++) f[e] = scale_of(magnitude(all[(threadIdx.x & 31) * 8 + e]));
  s.split<2>(w, f);
}

// Many features, or maxima that are known: the maxima (which begin at 0) by one kernel, the split by another, whose last
// blocks take x.
__global__ void __launch_bounds__(256, 4)
lnll_colmax_kernel(SplitJob w, uint32_t groups, int64_t share) {
  chain_begin();
  __shared__ uint32_t part[8][kSplitCols];
  const uint32_t group = blockIdx.x % groups, turn = blockIdx.x / groups;
  const ColumnShare s(w, group, turn * share, (turn + 1) * share);
  s.maxima<4>(w, part);
  __syncthreads();
  const uint32_t a = joined(part);
  const int64_t col = (int64_t)group * kSplitCols + threadIdx.x;
  if (col < w.cols && a) atomicMax(w.mag + col, a);
}
template <int GROUP>
__global__ void __launch_bounds__(256, 4)
lnll_split_wide_kernel(SplitJob w, SplitJob x, uint32_t blocks_w, uint32_t groups, int64_t share, uint32_t* zeros, int64_t nzeros) {
  chain_begin();
  clear(zeros, nzeros);
  __shared__ uint32_t red[32];
  if (blockIdx.x >= blocks_w) return split_rows<GROUP>(x, blockIdx.x - blocks_w, red);
  const uint32_t group = blockIdx.x % groups, turn = blockIdx.x / groups;
  const ColumnShare s(w, group, turn * share, (turn + 1) * share);
  if (!s.in) return;
  float f[8];
#pragma unroll
  for (int e = 0; e < 8; e++) f[e] = s.c + e < w.cols ? scale_of(magnitude(w.mag[s.c + e])) : 0.0f;
  s.split<2>(w, f);
}

// ---- epilogues -------------------------------------------------------------------------------------------
// A thread holds 64 columns of one row.  The epilogue has to stay below the time of two chunks, about
// 12 000 clocks: the tensor core runs ahead by that much and then waits.
constexpr float kLog2e = 1.4426950408889634f;

// 2^t, t = (s - lse) log2 e rounded: relative error |t| 2^-24 ln 2 and 2^-22 of the instruction, beside what the
// rounding of the scores themselves, |s| 2^-24, does to any exponential of them

__device__ __forceinline__ float exp2_approx(float t) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(t));
  return y;
}

// the bias (0 without one) and the magnitudes (1 without them) of the tile's columns into shared memory
__device__ __forceinline__ void stage_columns(const float* bias, const uint32_t* mag, int64_t j0, int64_t J, MmaShared* sh, int turn) {
  const int col = threadIdx.x & (kTN - 1);
  if (threadIdx.x < kTN) sh->bias[turn][col] = bias && j0 + col < J ? bias[j0 + col] : 0.0f;
  else sh->mag[turn][col] = mag && j0 + col < J ? magnitude(mag[j0 + col]) : 1.0f;
}

// i = instance, j = class: maximum and sum of exponentials of the tile's 256 classes per instance
struct MmaStats {
  const uint32_t *xmag, *wmag;
  const float* bias;
  const int32_t* labels;
  float *part_m, *part_s, *label_score;
  uint32_t* done;              // counter of the joining kernel that follows
  int64_t N, J;                // instances, classes of this launch
  int64_t v0, tile0;           // first class and first tile of this launch
  __device__ __forceinline__ void stage(int64_t j0, MmaShared* sh, int turn) const {
    clear_done(done);
    stage_columns(bias, wmag, j0, J, sh, turn);
  }
  __device__ __forceinline__ void operator()(float2 (&acc)[32], const TileAt& at) const {
    const bool live = at.i < N;
    const Unscale us = unscale(live ? magnitude(xmag[at.i]) : 1.0f, at.gain);
    const int64_t lab = live ? (int64_t)labels[at.i] - 1 - v0 - at.j0 : -1;
    const float4* bs = reinterpret_cast<const float4*>(at.sh->bias[at.turn & 1] + at.quarter * 64);
    const float4* ms = reinterpret_cast<const float4*>(at.sh->mag[at.turn & 1] + at.quarter * 64);
    float m = -CUDART_INF_F;
    const int in = (int)min((int64_t)64, J - at.j0);        // columns that are classes
    const float2 ua = both(us.a), ub = both(us.b);
#pragma unroll
    for (int g = 0; g < 16; g++) {
      const float4 b = bs[g], c = ms[g];
      acc[2 * g] = fma2(mul2(mul2(acc[2 * g], ua), make_float2(c.x, c.y)), ub, make_float2(b.x, b.y));
      acc[2 * g + 1] = fma2(mul2(mul2(acc[2 * g + 1], ua), make_float2(c.z, c.w)), ub, make_float2(b.z, b.w));
    }
    if (in < 64) {
#pragma unroll
      for (int e = 0; e < 32; e++) {
        if (2 * e >= in) acc[e].x = -CUDART_INF_F;
        if (2 * e + 1 >= in) acc[e].y = -CUDART_INF_F;
      }
    }
#pragma unroll
    for (int e = 0; e < 32; e++) m = fmaxf(m, fmaxf(acc[e].x, acc[e].y));
    if (lab >= 0 && lab < 64) {
      float s = 0.0f;
#pragma unroll
      for (int e = 0; e < 32; e++) {
        if (lab == 2 * e) s = acc[e].x;
        if (lab == 2 * e + 1) s = acc[e].y;
      }
      label_score[at.i] = s;
    }
    const float ref = m == -CUDART_INF_F ? 0.0f : m;        // all masked: every term is 0
    const float2 nref = both(-ref), l2e = both(kLog2e);
    float2 s2 = both(0.0f);
#pragma unroll
    for (int e = 0; e < 32; e++) {
      const float2 t = mul2(add2(acc[e], nref), l2e);
      s2 = add2(s2, make_float2(exp2_approx(t.x), exp2_approx(t.y)));
    }
    const float s = s2.x + s2.y;
    float2(&st)[4][kTM] = at.sh->stat[at.turn & 1];
    st[at.quarter][at.row] = make_float2(m, s);
    epi_sync();
    if (at.quarter == 0 && live) {
      float mm = m;
#pragma unroll
      for (int k = 1; k < 4; k++) mm = fmaxf(mm, st[k][at.row].x);
      float ss = 0.0f;
#pragma unroll
      for (int k = 0; k < 4; k++) {
        const float2 o = st[k][at.row];
        if (o.y != 0.0f) ss += o.y * exp2_approx((o.x - mm) * kLog2e);      // an empty quarter is (-inf, 0)
      }
      part_m[(tile0 + at.jt) * N + at.i] = mm;
      part_s[(tile0 + at.jt) * N + at.i] = ss;
    }
  }
};

// Eight lanes that hold one row of eight 16-byte groups each (32 words) exchange them so that lane r
// (of the eight) holds group r of all eight rows: stores then cover 128 contiguous bytes per row
// instead of 16 bytes in each of 32 lines.
__device__ __forceinline__ void transpose8(uint32_t (&w)[32]) {
  const int r = threadIdx.x & 7;
#pragma unroll
  for (int b = 1; b < 8; b <<= 1) {
    const bool up = r & b;
#pragma unroll
    for (int k = 0; k < 8; k++)
      if (!(k & b)) {
#pragma unroll
        for (int c = 0; c < 4; c++) {
          const uint32_t send = up ? w[4 * k + c] : w[4 * (k | b) + c];
          const uint32_t got = __shfl_xor_sync(0xffffffffu, send, b);
          if (up) w[4 * k + c] = got;
          else w[4 * (k | b) + c] = got;
        }
      }
  }
}

// The 32 rows of 32 words of a warp turned: lane c then holds word c of every row.
__device__ __forceinline__ void transpose32(uint32_t (&w)[32]) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int b = 16; b > 0; b >>= 1) {
    const bool up = lane & b;
#pragma unroll
    for (int k = 0; k < 32; k++)
      if (!(k & b)) {
        const uint32_t send = up ? w[k] : w[k | b];
        const uint32_t got = __shfl_xor_sync(0xffffffffu, send, b);
        if (up) w[k] = got;
        else w[k | b] = got;
      }
  }
}

// i = instance, j = class of the piece: dS without g, and what the products that follow need to scale it:
// of each instance the largest |dS| times its class's magnitude (as dS meets W in dx), of each class the largest
// |dS| times its instance's (as it meets x in dW); maxima do not depend on the order of the atomics.  Also dS's sums
// over the tile's instances for the bias gradient.
struct MmaGradScores {
  const uint32_t *xmag, *wmag;
  const float* bias;           // of the piece's first class
  const int32_t* labels;
  const float* lse;            // N rounded values, N remainders
  float* ds;                   // [N][ld], ld a multiple of 64
  int64_t N, J, ld, v0;
  uint32_t *rowmax, *colmax;
  float* db_part;              // [instance tile][J] or null
  __device__ __forceinline__ void stage(int64_t j0, MmaShared* sh, int turn) const { stage_columns(bias, wmag, j0, J, sh, turn); }
  __device__ __forceinline__ void operator()(float2 (&acc)[32], const TileAt& at) const {
    const bool live = at.i < N;
    const float mine = live ? magnitude(xmag[at.i]) : 1.0f;
    const Unscale us = unscale(mine, at.gain);
    const int32_t label = live ? labels[at.i] : 0;            // rows past the last instance act as skipped
    const float hi = live ? lse[at.i] : 0.0f, lo = live ? lse[N + at.i] : 0.0f;
    const float2 ua = both(us.a), ub = both(us.b), nhi = both(-hi), nlo = both(-lo), l2e = both(kLog2e);
    const int64_t hit64 = (int64_t)label - 1 - v0 - at.j0;
    const int hit = hit64 >= 0 && hit64 < 64 ? (int)hit64 : -1;
    const int in = (int)max((int64_t)0, min((int64_t)64, J - at.j0));
    const int lane = threadIdx.x & 31, r8 = lane & 7;
    const int64_t row0 = at.i - lane + (lane & ~7);           // first of the eight rows of this lane's group
    float* out = ds + row0 * ld + at.j0 + 4 * r8;
    uint32_t* top = colmax + at.j0 + 4 * r8;
    const int rows = (int)max((int64_t)0, min((int64_t)8, N - row0));
    float rm = 0.0f;                                          // fmaxf passes over NaN
#pragma unroll
    for (int h = 0; h < 2; h++) {                             // 32 columns at a time, which the registers hold
      const float4* bs = reinterpret_cast<const float4*>(at.sh->bias[at.turn & 1] + at.quarter * 64 + 32 * h);
      const float4* ms = reinterpret_cast<const float4*>(at.sh->mag[at.turn & 1] + at.quarter * 64 + 32 * h);
      const int hit_h = hit - 32 * h, in_h = in - 32 * h;
      uint32_t w[32];
#pragma unroll
      for (int g = 0; g < 8; g++) {
        asm volatile("" ::: "memory");                        // no loads of later columns before this one is done with
        const float4 b4 = bs[g], m4 = ms[g];
#pragma unroll
        for (int k = 0; k < 2; k++) {
          const float2 c = k ? make_float2(m4.z, m4.w) : make_float2(m4.x, m4.y);
          const float2 s = fma2(mul2(mul2(acc[16 * h + 2 * g + k], ua), c), ub, k ? make_float2(b4.z, b4.w) : make_float2(b4.x, b4.y));
          const float2 t = mul2(add2(add2(s, nhi), nlo), l2e);
          float2 d = label == 0 ? both(0.0f) : make_float2(exp2_approx(t.x), exp2_approx(t.y));
          const int e = 4 * g + 2 * k;
          if (hit_h == e) d.x -= 1.0f;
          if (hit_h == e + 1) d.y -= 1.0f;
          if (e >= in_h) d.x = 0.0f;
          if (e + 1 >= in_h) d.y = 0.0f;
          const float2 r = mul2(d, c);
          rm = fmaxf(rm, fmaxf(fabsf(r.x), fabsf(r.y)));
          w[e] = __float_as_uint(d.x);
          w[e + 1] = __float_as_uint(d.y);
        }
      }
      transpose8(w);                                          // now four classes of each of the eight rows
      const int left = in_h - 4 * r8;                         // classes of the four
#pragma unroll
      for (int q = 0; q < 8; q++)
        if (q < rows && left > 0) *reinterpret_cast<uint4*>(out + q * ld + 32 * h) = make_uint4(w[4 * q], w[4 * q + 1], w[4 * q + 2], w[4 * q + 3]);
      if (db_part) {
#pragma unroll
        for (int c = 0; c < 4; c++) {
          float cs = 0.0f;
#pragma unroll
          for (int q = 0; q < 8; q++) cs += __uint_as_float(w[4 * q + c]);
#pragma unroll
          for (int o = 8; o < 32; o <<= 1) cs += __shfl_xor_sync(0xffffffffu, cs, o);
          if (lane < 8) at.sh->colsum[at.row >> 5][at.quarter * 64 + 32 * h + 4 * r8 + c] = cs;
        }
      }
#pragma unroll
      for (int q = 0; q < 8; q++) {
        const float mx = __shfl_sync(0xffffffffu, mine, (lane & ~7) + q);
#pragma unroll
        for (int c = 0; c < 4; c++) w[4 * q + c] = __float_as_uint(fabsf(__uint_as_float(w[4 * q + c]) * mx));
      }
#pragma unroll
      for (int c = 0; c < 4; c++) {
        float cm = 0.0f;
#pragma unroll
        for (int q = 0; q < 8; q++) cm = fmaxf(cm, __uint_as_float(w[4 * q + c]));
#pragma unroll
        for (int o = 8; o < 32; o <<= 1) cm = fmaxf(cm, __shfl_xor_sync(0xffffffffu, cm, o));
        if (lane < 8 && c < left && cm > 0.0f) atomicMax(top + 32 * h + c, __float_as_uint(cm));
      }
    }
    if (live && rm > 0.0f) atomicMax(rowmax + at.i, __float_as_uint(rm));
    if (db_part) {
      epi_sync();
      const int c = threadIdx.x;
      if (c < kTN) {
        const int64_t j = (int64_t)at.jt * kTN + c;
        if (j < J && (int64_t)at.it * kTM < N)                // a pair's second tile may lie past the last instance
          db_part[(int64_t)at.it * J + j] =
              (at.sh->colsum[0][c] + at.sh->colsum[1][c]) + (at.sh->colsum[2][c] + at.sh->colsum[3][c]);
      }
    }
  }
};

// out(i, j) = or += g * acc; with several parts of the summed axis the plain sums go to `out` + part
struct MmaStore {
  const uint32_t *row, *col;   // magnitudes of the result's rows and columns, null where there are none
  float* out;
  int64_t I, J, ld, part;      // part: elements between the parts' results (0: there is one)
  int add;
  uint32_t* done;              // counter of the statistics kernel that follows, or null
  GradScale<float> g;
  __device__ __forceinline__ void stage(int64_t j0, MmaShared* sh, int turn) const {
    clear_done(done);
    stage_columns(nullptr, col, j0, J, sh, turn);
  }
  __device__ __forceinline__ void operator()(float2 (&acc)[32], const TileAt& at) const {
    const Unscale us = unscale(row && at.i < I ? magnitude(row[at.i]) : 1.0f, at.gain);
    const float4* ms = reinterpret_cast<const float4*>(at.sh->mag[at.turn & 1] + at.quarter * 64);
    const float f = part ? 1.0f : g.value();
    const int lane = threadIdx.x & 31, r8 = lane & 7;
    const int64_t row0 = at.i - lane + (lane & ~7);
    float* base = out + at.split * part;
    const bool wide = (ld & 3) == 0 && (J & 3) == 0 && ((uintptr_t)base & 15) == 0;
#pragma unroll
    for (int h = 0; h < 2; h++) {
      uint32_t w[32];
#pragma unroll
      for (int e = 0; e < 16; e++) {
        const float4 m4 = ms[8 * h + e / 2];
        const float2 c = e & 1 ? make_float2(m4.z, m4.w) : make_float2(m4.x, m4.y);
        const float2 v = mul2(mul2(mul2(mul2(acc[16 * h + e], both(us.a)), c), both(us.b)), both(f));
        w[2 * e] = __float_as_uint(v.x);
        w[2 * e + 1] = __float_as_uint(v.y);
      }
      if (wide) {
        transpose8(w);
        const int64_t j = at.j0 + 32 * h + 4 * r8;             // J is a multiple of 4 here
        float* p = base + row0 * ld + j;
#pragma unroll
        for (int q = 0; q < 8; q++)
          if (row0 + q < I && j < J) {
            float4 o = make_float4(__uint_as_float(w[4 * q]), __uint_as_float(w[4 * q + 1]), __uint_as_float(w[4 * q + 2]),
                                   __uint_as_float(w[4 * q + 3]));
            float4* d = reinterpret_cast<float4*>(p + q * ld);
            if (add) {
              const float4 t = *d;
              o = make_float4(t.x + o.x, t.y + o.y, t.z + o.z, t.w + o.w);
            }
            *d = o;
          }
      } else {                                                  // rows start anywhere: a row's 32 columns at a time
        transpose32(w);
        const int64_t i0 = at.i - lane, j = at.j0 + 32 * h + lane;
        float* p = base + i0 * ld + j;
#pragma unroll
        for (int q = 0; q < 32; q++)
          if (i0 + q < I && j < J) {
            float* d = p + q * ld;
            *d = add ? *d + __uint_as_float(w[q]) : __uint_as_float(w[q]);
          }
      }
    }
  }
};

// The same dS, maxima and sums over groups of 8 instances from the parts of the scores of V classes from v0 on
constexpr int kGradRows = 8;
__global__ void __launch_bounds__(256)
lnll_grad_scores_kernel(const float* scores, int parts, const float* bias, const int32_t* labels, const float* lse, const uint32_t* xmag,
                        const uint32_t* wmag, int64_t N, int64_t V, int64_t v0, float* ds, int64_t ld, uint32_t* rowmax, uint32_t* colmax,
                        float* db_part) {
  chain_begin();
  __shared__ float row_top[8][kGradRows];                // one atomic per CTA and row: thousands to one address queue up
  const int64_t v = (int64_t)blockIdx.x * 256 + threadIdx.x, n0 = (int64_t)blockIdx.y * kGradRows;
  const float b = bias && v < V ? bias[v] : 0.0f, mw = v < V ? magnitude(wmag[v]) : 0.0f;
  float t[kGradRows], sum = 0.0f, cm = 0.0f;
#pragma unroll
  for (int k = 0; k < kGradRows; k++) t[k] = v < V && n0 + k < N ? scores[(n0 + k) * V + v] : 0.0f;
  for (int p = 1; p < parts; p++) {
#pragma unroll
    for (int k = 0; k < kGradRows; k++)
      if (v < V && n0 + k < N) t[k] += scores[p * N * V + (n0 + k) * V + v];
  }
#pragma unroll
  for (int k = 0; k < kGradRows; k++) {
    const int64_t n = n0 + k;
    if (n >= N) break;
    const float d = v < V ? grad_score(t[k] + b, lse[n], lse[N + n], labels[n], v0 + v) : 0.0f;
    sum += d;
    if (v < V) ds[n * ld + v] = d;
    cm = fmaxf(cm, fabsf(d * magnitude(xmag[n])));
    const float rm = warp_reduce(fmaxf(0.0f, fabsf(d * mw)), [](float x, float y) { return fmaxf(x, y); });
    if ((threadIdx.x & 31) == 0) row_top[threadIdx.x >> 5][k] = rm;
  }
  __syncthreads();
  if (threadIdx.x < kGradRows && n0 + threadIdx.x < N) {
    float rm = 0.0f;
#pragma unroll
    for (int k = 0; k < 8; k++) rm = fmaxf(rm, row_top[k][threadIdx.x]);
    if (rm > 0.0f) atomicMax(rowmax + n0 + threadIdx.x, __float_as_uint(rm));
  }
  if (v < V && cm > 0.0f) atomicMax(colmax + v, __float_as_uint(cm));
  if (db_part && v < V) db_part[(int64_t)blockIdx.y * V + v] = sum;
}

// dS (rows `ld` apart) as the operands of dx and of dW, two planes each (either may be null): times its class's
// magnitude and scaled by the instance's maximum, times its instance's magnitude and scaled by the class's.  One row
// of dx, or one class of dW, then keeps its terms to 2^-39 of the largest of them, whatever the others hold.  A warp
// takes 256 classes of an instance, a CTA 32 instances; from the last classes, which are still in L2.
constexpr int kPlaneRows = 32;
__global__ void __launch_bounds__(256)
lnll_grad_planes_kernel(const float* ds, int64_t ld, int64_t N, int64_t J, const uint32_t* xmag, const uint32_t* wmag, const uint32_t* rowmax,
                        const uint32_t* colmax, __half* for_dx, __half* for_dw, int64_t plane) {
  chain_begin();
  const int64_t c = (int64_t)(gridDim.y - 1 - blockIdx.y) * 256 + (threadIdx.x & 31) * 8, n0 = (int64_t)blockIdx.x * kPlaneRows + (threadIdx.x >> 5);
  if (c >= J) return;
  float mw[8], sw[8];
#pragma unroll
  for (int k = 0; k < 8; k++) {
    mw[k] = c + k < J ? magnitude(wmag[c + k]) : 0.0f;
    sw[k] = c + k < J ? scale_of(magnitude(colmax[c + k])) : 0.0f;
  }
#pragma unroll
  for (int r = 0; r < kPlaneRows; r += 8) {
    const int64_t n = n0 + r;
    if (n >= N) break;
    const float4 a = *reinterpret_cast<const float4*>(ds + n * ld + c), b = *reinterpret_cast<const float4*>(ds + n * ld + c + 4);
    const float d[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    const float mx = magnitude(xmag[n]), sx = scale_of(magnitude(rowmax[n]));
    uint4 hi, lo;
    uint32_t *h = &hi.x, *l = &lo.x;
    if (for_dx) {
#pragma unroll
      for (int k = 0; k < 8; k += 2)
        split_pair(c + k < J ? d[k] * mw[k] * sx : 0.0f, c + k + 1 < J ? d[k + 1] * mw[k + 1] * sx : 0.0f, h[k / 2], l[k / 2]);
      *reinterpret_cast<uint4*>(for_dx + n * ld + c) = hi;
      *reinterpret_cast<uint4*>(for_dx + plane + n * ld + c) = lo;
    }
    if (for_dw) {
#pragma unroll
      for (int k = 0; k < 8; k += 2)
        split_pair(c + k < J ? d[k] * mx * sw[k] : 0.0f, c + k + 1 < J ? d[k + 1] * mx * sw[k + 1] : 0.0f, h[k / 2], l[k / 2]);
      *reinterpret_cast<uint4*>(for_dw + n * ld + c) = hi;
      *reinterpret_cast<uint4*>(for_dw + plane + n * ld + c) = lo;
    }
  }
}

}  // namespace kn

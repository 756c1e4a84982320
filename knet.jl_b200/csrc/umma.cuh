// Matrix products on the 5th-generation tensor cores: tcgen05 instructions, the descriptors of their
// shared-memory operands, and tiled TMA loads, as inline PTX for sm_100a.
//
// Rules the helpers rely on: one thread issues tcgen05.mma and its commits; TMEM is allocated and
// freed by one whole warp; a warp reads the 32 TMEM lanes of its rank in its group of four; every
// TMA load starts at a multiple of 16 bytes along the contiguous axis; no load is multicast.  (A pair's commit
// signals the barriers of both its CTAs through tcgen05.commit's cluster form, which reads no memory.)
#pragma once
#include <cuda.h>

#include "tma.cuh"

namespace kn {

// ---- TMEM ------------------------------------------------------------------------------------------
// CG is the number of CTAs (1 or a cluster of 2) that work on one product; for a pair one warp of each
// calls these.
template <int CG> __device__ __forceinline__ void tmem_alloc(uint32_t* addr_smem, uint32_t columns) {
  if constexpr (CG == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(addr_smem)), "r"(columns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  } else {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(addr_smem)), "r"(columns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
}
template <int CG> __device__ __forceinline__ void tmem_free(uint32_t addr, uint32_t columns) {
  if constexpr (CG == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(columns) : "memory");
  else asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(columns) : "memory");
}
__device__ __forceinline__ void tcgen05_before_sync() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tcgen05_after_sync() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// 16 columns of this warp's 32 lanes: thread t receives lane t's values
__device__ __forceinline__ void tmem_load16(uint32_t addr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tmem_load_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

// ---- products ---------------------------------------------------------------------------------------
// Instruction descriptor of kind::f16 with fp16 operands and Float32 accumulators: M x N tile; an
// operand is "mn" when its row index (not the summed one) is the contiguous axis in memory.
__host__ __device__ inline uint32_t umma_idesc(uint32_t m, uint32_t n, bool a_mn, bool b_mn) {
  return (1u << 4) | ((uint32_t)a_mn << 15) | ((uint32_t)b_mn << 16) | ((n >> 3) << 17) | ((m >> 4) << 24);
}

// Shared-memory descriptor: start, leading and stride byte offsets in units of 16 bytes, version 1,
// swizzle mode (2: 128 bytes, 4: 64 bytes).
//   summed index contiguous, rows of 64 bytes, 64-byte swizzle: `stride` = 8 rows, `leading` unused;
//   row index contiguous, 64 rows (128 bytes) per line, 128-byte swizzle: `stride` = 8 summed
//   indices (1024 bytes), `leading` = the next 64 rows.
__host__ __device__ inline uint64_t umma_desc(uint32_t leading, uint32_t stride, uint32_t swizzle) {
  return ((uint64_t)((leading >> 4) & 0x3fff) << 16) | ((uint64_t)((stride >> 4) & 0x3fff) << 32) | (1ull << 46) |
         ((uint64_t)swizzle << 61);
}
__device__ __forceinline__ uint64_t umma_at(uint64_t desc, uint32_t smem_addr) {
  return desc | (uint64_t)((smem_addr >> 4) & 0x3fff);
}

// D (TMEM) = A * B (+ D), 16 summed indices.  For a pair the first CTA issues it: each CTA holds its half of
// A's rows and of D, and half of B's rows, at the same shared-memory addresses.
template <int CG> __device__ __forceinline__ void umma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate) {
  if constexpr (CG == 1)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        :
        : "r"(d), "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        :
        : "r"(d), "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate)
        : "memory");
}
// the barrier (of a pair: both CTAs' barriers at that address) gets one arrival when all products issued so
// far by this thread are done
template <int CG> __device__ __forceinline__ void umma_commit(uint64_t* bar) {
  if constexpr (CG == 1)
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
  else
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)),
                 "h"((uint16_t)3)
                 : "memory");
}

// ---- barriers and loads -----------------------------------------------------------------------------
__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// one box of a 3-d tensor into this CTA's shared memory
__device__ __forceinline__ void tma_load_3d(void* dst_smem, const CUtensorMap* map, int32_t x, int32_t y, int32_t z, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(
          smem_u32(dst_smem)),
      "l"((uint64_t)map), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z)
      : "memory");
}
// the same into this CTA's half of a pair; the barrier is the first CTA's (a shared::cluster address)
__device__ __forceinline__ void tma_load_3d_pair(void* dst_smem, const CUtensorMap* map, int32_t x, int32_t y, int32_t z, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(
          smem_u32(dst_smem)),
      "l"((uint64_t)map), "r"(bar), "r"(x), "r"(y), "r"(z)
      : "memory");
}
// one arrival on a barrier of another CTA of the cluster
__device__ __forceinline__ void mbar_arrive_remote(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void tma_prefetch_map(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"((uint64_t)map) : "memory");
}

// ---- host: tensor maps ------------------------------------------------------------------------------
typedef CUresult (*EncodeTiled)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
inline EncodeTiled encode_tiled() {
  static const EncodeTiled f = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult r;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &r) != cudaSuccess ||
        r != cudaDriverEntryPointSuccess)
      p = nullptr;
    cudaGetLastError();
    return reinterpret_cast<EncodeTiled>(p);
  }();
  return f;
}

// A map over two planes (rows x cols, row pitch ld elements) of fp16 values; boxes cover both planes.
// Elements outside are read as zero.
inline int tensor_map_planes(CUtensorMap* map, const void* base, int64_t rows, int64_t cols, int64_t ld, int64_t plane,
                             uint32_t box_cols, uint32_t box_rows, CUtensorMapSwizzle swizzle) {
  const EncodeTiled f = encode_tiled();
  if (!f) return (int)cudaErrorNotSupported;
  const cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, 2};
  const cuuint64_t strides[2] = {(cuuint64_t)ld * 2, (cuuint64_t)plane * 2};
  const cuuint32_t box[3] = {box_cols, box_rows, 2}, step[3] = {1, 1, 1};
  const CUresult r = f(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(base), dims, strides, box, step,
                       CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                       CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : (int)cudaErrorInvalidValue;
}

}  // namespace kn

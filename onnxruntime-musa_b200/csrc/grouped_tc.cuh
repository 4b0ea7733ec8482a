// PTX wrappers and tables shared by the tensor-core kernels of the expert products and the
// adapter projection (grouped_tc.cu, grouped_small.cu).
#pragma once

#include <atomic>

#include "grouped.h"

namespace moe {

__device__ __forceinline__ void tma_load_3d_pair(void* dst, const CUtensorMap* map, uint32_t bar,
                                                 int c0, int c1, int c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1), "r"(c2)
      : "memory");
}

// 16 TMEM lanes x 32 columns (four 16 x 8 blocks): block j, lane l of the warp holds rows
// l/4 (v[4j], v[4j+1]) and l/4 + 8 (v[4j+2], v[4j+3]) of columns 8j + 2(l%4) + {0, 1} --
// the accumulator fragment of mma.m16n8k16.
__device__ __forceinline__ void tmem_ld_frag4(uint32_t taddr, float (&v)[16]) {
  uint32_t r[16];
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x4.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]),
        "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}

// Four 8 x 8 blocks of 16-bit elements to shared memory; lane 8i + t gives the address of
// row t of block i (16 bytes).  _t: each block transposed.
__device__ __forceinline__ void stmatrix4(uint32_t addr, uint32_t a, uint32_t b, uint32_t c,
                                          uint32_t d) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(addr),
               "r"(a), "r"(b), "r"(c), "r"(d)
               : "memory");
}
__device__ __forceinline__ void stmatrix4_t(uint32_t addr, uint32_t a, uint32_t b, uint32_t c,
                                            uint32_t d) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(addr),
               "r"(a), "r"(b), "r"(c), "r"(d)
               : "memory");
}

// Descriptor of an MN-major operand tile written by TMA with 128-byte swizzling: blocks of
// 64 contiguous MN elements (128 B) by kRows contraction rows, `mn_stride` bytes from one
// 64-element block to the next, 1024 B from one 8-row group of the contraction to the next.
__device__ __forceinline__ uint64_t smem_desc_mn_sw128(uint32_t saddr, uint32_t mn_stride) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((saddr >> 4) & 0x3FFF);
  d |= static_cast<uint64_t>(mn_stride >> 4) << 16;
  d |= static_cast<uint64_t>(1024 >> 4) << 32;
  d |= static_cast<uint64_t>(1) << 46;
  d |= static_cast<uint64_t>(2) << 61;
  return d;
}
// Instruction-descriptor bits of MN-major A / B operands.
constexpr uint32_t kIdescAMn = 1u << 15;
constexpr uint32_t kIdescBMn = 1u << 16;

// Rows [x, y) of each group and the prefix of its tile counts, in shared memory.
struct GroupTable {
  int2* rows;   // [E]
  int* tiles;   // [E + 1]
};

// Filled by one full warp.  offsets == nullptr: one group of all rows.  Offsets are clamped
// to [0, rows] and a group never ends before it begins, whatever the caller's array holds.
__device__ __forceinline__ void build_group_table(const int32_t* offsets, int E, int rows,
                                                  int tile_rows, const GroupTable& t) {
  const int lane = threadIdx.x & 31;
  int carry = 0;
  for (int base = 0; base < E; base += 32) {
    const int e = base + lane;
    int n = 0;
    if (e < E) {
      int b = 0, c = rows;
      if (offsets != nullptr) {
        b = min(max(__ldg(offsets + e), 0), rows);
        c = max(min(max(__ldg(offsets + e + 1), 0), rows), b);
      }
      t.rows[e] = make_int2(b, c);
      n = (c - b + tile_rows - 1) / tile_rows;
    }
    int incl = n;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, incl, d);
      if (lane >= d) incl += v;
    }
    if (e < E) t.tiles[e] = carry + incl - n;
    carry += __shfl_sync(0xffffffffu, incl, 31);
  }
  if (lane == 0) t.tiles[E] = carry;
}

// Largest e with tiles[e] * per <= L (the group that holds tile L).
__device__ __forceinline__ int find_group(const int* tiles, int E, int per, int L) {
  int lo = 0, hi = E - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (tiles[mid] * per <= L) lo = mid; else hi = mid - 1;
  }
  return lo;
}

template <typename T> struct TcFormat;
template <> struct TcFormat<__half> { static constexpr uint32_t kId = 0; };
template <> struct TcFormat<__nv_bfloat16> { static constexpr uint32_t kId = 1; };

// Raises a kernel's dynamic shared memory limit once per device (the attribute belongs to
// the device's context; a race between first callers repeats an idempotent call).
struct SmemOptIn {
  std::atomic<uint64_t> done{0};
  template <typename K>
  cudaError_t set(K* kernel, int bytes) {
    int dev = 0;
    cudaError_t st = cudaGetDevice(&dev);
    if (st != cudaSuccess) return st;
    const uint64_t bit = dev < 64 ? uint64_t{1} << dev : 0;
    if (done.load(std::memory_order_relaxed) & bit) return cudaSuccess;
    st = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (st == cudaSuccess) done.fetch_or(bit, std::memory_order_relaxed);
    return st;
  }
};

// 128-byte-swizzled map of 64-column boxes over [dim2][dim1][dim0] (dim0 contiguous).
bool grouped_map(CUtensorMap* m, int dtype, const void* ptr, int64_t dim0, int64_t dim1,
                 int64_t dim2, int box1);

}  // namespace moe

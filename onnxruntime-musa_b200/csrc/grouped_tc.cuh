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

// The reverse of tmem_ld_frag4; tmem_st_wait() before anyone else reads.
__device__ __forceinline__ void tmem_st_frag4(uint32_t taddr, const float (&v)[16]) {
  uint32_t r[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) r[i] = __float_as_uint(v[i]);
  asm volatile(
      "tcgen05.st.sync.aligned.16x256b.x4.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

// Most slices (of 64 contraction entries) that one accumulator takes: 16384 entries.  tcgen05
// cuts products off when it aligns them to the running sum, always towards zero, so a long sum
// of one sign drifts: 2^19 rows in one accumulator came out 0.4% low, eight half steps of fp16.
// 1024 steps of 16 entries lose at most 2^-12 of the magnitudes; longer contractions are added
// up from such segments in fp32, rounded to nearest.  It also bounds every wait on an
// accumulator: a segment is 256 slices of some 512 cycles, tens of microseconds.  (Shorter
// segments lose less, but most layers' contractions then pay for the extra pass over tensor
// memory: up to 16384 there is none.  The kernels that can add segments up are instantiations of
// their own, taken where a contraction may be longer: in the others that code, never run, cost 2
// to 5%, fc2 of 296 rows over 64 experts 38.2 -> 39.9 us.)
constexpr int kSegment = 256;
__host__ __device__ constexpr int segments_of(int slices) {
  return slices <= kSegment ? 1 : (slices + kSegment - 1) / kSegment;
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

// Reports a wait that ran out (a DeviceError) to the host: `word` is pinned host memory.
__device__ __forceinline__ void report_error(int* word, int code) {
  *reinterpret_cast<volatile int*>(word) = code;
  __threadfence_system();
}

// mbar_wait() by a whole warp: its lanes leave together, whichever of them ran out of time, so
// that what the warp does next as one (tensor memory loads, shuffles) stays whole.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity));
}
__device__ __forceinline__ bool warp_stopped(volatile int* abort_flag) {
  return __any_sync(0xffffffffu, *abort_flag);
}

// Before a CTA that gave up leaves: waits for the copies that may still be under way into its
// ring, in the order of the stages from the one that was waited for.  (A stage that was never
// asked for runs out of time too and ends this.)
__device__ __forceinline__ void drain_ring(uint64_t* full, int stages, int stage, uint32_t phase) {
  for (int k = 0; k < stages; ++k) {
    if (!mbar_wait(&full[stage], phase)) return;
    if (++stage == stages) { stage = 0; phase ^= 1; }
  }
}

// Parts from the other CTAs of a cluster, which send theirs (zeros) after a wait of their own ran
// out, too: this wait is four times as long, so that nobody's parts arrive after its CTA has left.
__device__ __forceinline__ bool wait_parts(uint64_t* bar) {
  for (int k = 0; k < 4; ++k)
    if (mbar_wait_cluster(bar, 0)) return true;
  return false;
}

// Rows [x, y) of each group and the prefix of its tile counts, in shared memory.
struct GroupTable {
  int2* rows;   // [E]
  int* tiles;   // [E + 1]
};

// Filled by one full warp.  offsets == nullptr: one group of all rows.  Offsets are clamped
// to [0, rows] and a group never ends before it begins, whatever the caller's array holds.
// A lane takes ceil(E / 32) adjacent groups, so that all loads
// are in flight together (a short kernel waits for this before anything else).
__device__ __forceinline__ void build_group_table(const int32_t* offsets, int E, int rows,
                                                  int tile_rows, const GroupTable& t) {
  constexpr int kPer = kMaxExperts / 32;
  const int lane = threadIdx.x & 31;
  if (offsets == nullptr) {
    if (lane == 0) {
      t.rows[0] = make_int2(0, rows);
      t.tiles[0] = 0;
      t.tiles[1] = (rows + tile_rows - 1) / tile_rows;
    }
    return;
  }
  const int per = (E + 31) >> 5, e0 = lane * per;
  int v[kPer + 1];
#pragma unroll
  for (int i = 0; i <= kPer; ++i)
    v[i] = i <= per && e0 + i <= E ? __ldg(offsets + e0 + i) : 0;
  int sum = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i)
    if (i < per && e0 + i < E) {
      const int b = min(max(v[i], 0), rows);
      const int c = max(min(v[i + 1], rows), b);
      t.rows[e0 + i] = make_int2(b, c);
      v[i] = (c - b + tile_rows - 1) / tile_rows;
      sum += v[i];
    }
  int incl = sum;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, incl, d);
    if (lane >= d) incl += u;
  }
  int at = incl - sum;
#pragma unroll
  for (int i = 0; i < kPer; ++i)
    if (i < per && e0 + i < E) {
      t.tiles[e0 + i] = at;
      at += v[i];
    }
  if (lane == 31) t.tiles[E] = incl;
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

// Launches with programmatic stream serialisation (unless MOE_B200_PDL=0): the kernel may start while the one before
// it on the stream drains, and calls pdl_wait() before it touches memory.  (Set up, barriers,
// tensor memory and descriptors then overlap the launch before: 2 us of a 10 us call.)
// `cluster` 0: the kernel's own.
template <typename... KArgs, typename... Args>
cudaError_t launch_overlapped(void (*kernel)(KArgs...), unsigned grid, int block, size_t smem,
                              int cluster, cudaStream_t s, Args&&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(static_cast<unsigned>(block));
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = static_cast<unsigned>(cluster);
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 0 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<KArgs>(args)...);
}

// 128-byte-swizzled map of 64-column boxes over [dim2][dim1][dim0] (dim0 contiguous).
bool grouped_map(CUtensorMap* m, int dtype, const void* ptr, int64_t dim0, int64_t dim1,
                 int64_t dim2, int box1);

}  // namespace moe

// Adapter projections of rows that follow different adapters: t[row] = A_a x[row].
//
// The second half, y += s_a B_a t, runs in the epilogue of the shared projection's kernels
// (grouped_simt.cu, grouped_small.cu, grouped_tc.cu), so y is written once and t stays in
// fp32.
//
// lora_shrink_tc_kernel (16-bit types): a CTA takes a chunk of adjacent rows and one split
// of K.  The A_a of the chunk's distinct adapters are stacked as the MMA's M (128 / r
// adapters a pass), its rows are the N, and each column keeps the lanes of its own adapter:
// rows need no sorting, and another adapter's values never reach a row.  One prompt in a
// chunk is one pass; a decode chunk of 8 rows is at most 8 adapters, read once each.
// Bound: the bytes of A_a (decode) and of x (prefill); the products are few.  The splits
// leave partial sums that the epilogue of the projection adds in order, which costs it
// splits * r floats a row and saves a join here.
#include <algorithm>

#include "grouped_tc.cuh"

namespace moe {
namespace {

constexpr int kWarps = 8;

// Any type and alignment: one CTA per row, a warp per rank entry, the lanes striding over
// K.  The row comes from L1 after the first warp's pass; A_a is read once per row.
template <typename T>
__global__ void __launch_bounds__(kWarps * 32)
lora_shrink_simt_kernel(const T* __restrict__ x, const T* __restrict__ a,
                        const int32_t* __restrict__ ids, int K, int rank, int adapters,
                        float* __restrict__ t) {
  const int64_t row = blockIdx.x;
  const int ad = ids[row];
  if (ad < 0 || ad >= adapters) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const T* xr = x + row * K;
  for (int j = warp; j < rank; j += kWarps) {
    const T* ar = a + (static_cast<int64_t>(ad) * rank + j) * K;
    float sum = 0.f;
#pragma unroll 4
    for (int k = lane; k < K; k += 32) sum = fmaf(to_f(ar[k]), to_f(xr[k]), sum);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    if (lane == 0) t[row * rank + j] = sum;
  }
}

__device__ int g_shrink_error;

constexpr int kBK = 64;
constexpr int kM = 128;
constexpr int kABytes = kM * kBK * 2;
constexpr int kMaxChunk = 64;
constexpr int kTcStages = 4;
constexpr int kTcThreads = 256;   // warp 0 TMA, warp 1 MMA, warps 4..7 epilogue

struct ShrinkParams {
  const int32_t* ids;
  float* t;
  int64_t rows;
  int K, rank, adapters;
  int chunk;      // rows of a CTA: 8 or 64
  int mma_n;      // max(chunk, 16)
  int splits;
  int stage_bytes;
};

__global__ void __launch_bounds__(kTcThreads)
lora_shrink_tc_kernel(const __grid_constant__ CUtensorMap map_x,
                      const __grid_constant__ CUtensorMap map_a, const uint32_t format,
                      const ShrinkParams p) {
  pdl_launch_dependents();  // the projection's main loop does not read t
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(ring + kTcStages * p.stage_bytes);
  uint64_t* empty = full + kTcStages;
  uint64_t* tfull = empty + kTcStages;   // [2]
  uint64_t* tempty = tfull + 2;          // [2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  __shared__ int s_id[kMaxChunk], s_first[kMaxChunk], s_slot[kMaxChunk], s_adapter[kMaxChunk];
  __shared__ int s_distinct;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int split = blockIdx.x % p.splits;
  const int64_t row0 = static_cast<int64_t>(blockIdx.x / p.splits) * p.chunk;
  const int n = static_cast<int>(min(static_cast<int64_t>(p.chunk), p.rows - row0));

  if (threadIdx.x == 0) {
    for (int s = 0; s < kTcStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&tfull[a], 1);
      mbar_init(&tempty[a], 4);
    }
    *abort_flag = 0;
    s_distinct = 0;
    fence_mbarrier_init();
  }
  const uint32_t tmem_cols = p.mma_n == 16 ? 32u : 2u * kMaxChunk;
  if (warp == 1) {
    tmem_alloc(tmem_slot, tmem_cols);
    tmem_relinquish();
  }
  // Distinct adapters of the chunk in order of first appearance.
  const int tok = static_cast<int>(threadIdx.x) - 64;  // warps 2 and 3
  const bool mine = tok >= 0 && tok < kMaxChunk;
  if (mine) {
    int id = -1;
    if (tok < n) {
      id = __ldg(p.ids + row0 + tok);
      if (id >= p.adapters) id = -1;
    }
    s_id[tok] = id;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (mine) {
    const int id = s_id[tok];
    int first = -1;
    if (id >= 0)
      for (first = 0; s_id[first] != id;) ++first;
    s_first[tok] = first;
  }
  __syncthreads();
  if (mine) {
    const int first = s_first[tok];
    int slot = -1;
    if (first >= 0) {
      slot = 0;
      for (int u = 0; u < first; ++u) slot += s_first[u] == u;
      if (first == tok) {
        s_adapter[slot] = s_id[tok];
        atomicAdd(&s_distinct, 1);
      }
    }
    s_slot[tok] = slot;
  }
  __syncthreads();
  const uint32_t tmem = *tmem_slot;

  const int rows_u = min(p.rank, kM);              // rows of one unit (adapter, rank block)
  const int blocks_u = (p.rank + kM - 1) / kM;     // rank blocks of an adapter
  const int per = kM / rows_u;                     // units of a pass
  const int units = s_distinct * blocks_u;
  const int passes = (units + per - 1) / per;
  const int slices = (p.K + kBK - 1) / kBK;
  const int s0 = static_cast<int>(static_cast<int64_t>(slices) * split / p.splits);
  const int s1 = static_cast<int>(static_cast<int64_t>(slices) * (split + 1) / p.splits);

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      for (int ps = 0; ps < passes && !*abort_flag; ++ps) {
        const int u0 = ps * per, nu = min(per, units - u0);
        for (int s = s0; s < s1; ++s) {
          if (!mbar_wait(&empty[stage], phase ^ 1)) {
            atomicExch(&g_shrink_error, kErrTimeoutProducer);
            *abort_flag = 1;
            break;
          }
          uint8_t* w = ring + stage * p.stage_bytes;
          mbar_arrive_expect_tx(&full[stage], (nu * rows_u + p.chunk) * kBK * 2);
          for (int u = 0; u < nu; ++u)
            tma_load_3d(w + u * rows_u * kBK * 2, &map_a, &full[stage], s * kBK,
                        ((u0 + u) % blocks_u) * kM, s_adapter[(u0 + u) / blocks_u]);
          tma_load_3d(w + kABytes, &map_x, &full[stage], s * kBK, static_cast<int>(row0), 0);
          if (++stage == kTcStages) { stage = 0; phase ^= 1; }
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      const uint32_t idesc = idesc_f16(format, kM, p.mma_n);
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int ps = 0; ps < passes && ok; ++ps) {
        const int acc = ps & 1;
        ok = mbar_wait(&tempty[acc], ((ps >> 1) & 1) ^ 1);
        tc_fence_after();
        for (int s = s0; s < s1 && ok; ++s) {
          ok = mbar_wait(&full[stage], phase);
          if (!ok) break;
          tc_fence_after();
          const uint32_t w = smem_u32(ring + stage * p.stage_bytes);
#pragma unroll
          for (int k = 0; k < kBK / 16; ++k)
            tc_mma_f16(tmem + acc * p.mma_n, smem_desc_k_sw128(w + k * 32),
                       smem_desc_k_sw128(w + kABytes + k * 32), idesc,
                       (s != s0 || k != 0) ? 1u : 0u);
          tc_commit(&empty[stage]);
          if (++stage == kTcStages) { stage = 0; phase ^= 1; }
        }
        tc_commit(&tfull[acc]);  // after a timeout too: it waits for the MMAs issued
      }
      if (!ok) {
        atomicExch(&g_shrink_error, kErrTimeoutMma);
        *abort_flag = 1;
      }
    }
  } else if (warp >= 4) {
    const int q = warp & 3;
    const int lane_row = q * 32 + lane;
    const int u = lane_row / rows_u, j0 = lane_row - u * rows_u;
    for (int ps = 0; ps < passes && !*abort_flag; ++ps) {
      const int acc = ps & 1;
      if (!mbar_wait(&tfull[acc], (ps >> 1) & 1)) {
        atomicExch(&g_shrink_error, kErrTimeoutEpilogue);
        *abort_flag = 1;
        break;
      }
      tc_fence_after();
      const int unit = ps * per + u;
      const int j = (unit % blocks_u) * kM + j0;
      const int slot = u < per && unit < units && j < p.rank ? unit / blocks_u : -2;
      float* dst = p.t + (static_cast<int64_t>(split) * p.rows + row0) * p.rank + j;
      for (int c = 0; c < n; c += 16) {
        float v[16];
        tmem_ld16(tmem + (static_cast<uint32_t>(q * 32) << 16) + acc * p.mma_n + c, v);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (c + i < n && s_slot[c + i] == slot)
            dst[static_cast<int64_t>(c + i) * p.rank] = s0 < s1 ? v[i] : 0.f;
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&tempty[acc]);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, tmem_cols);
  }
}

// Rows of a CTA: small chunks spread a decode batch (whose rows follow many adapters) over
// the GPU, tall ones read A_a once per 64 rows of a prompt.
int shrink_chunk(int64_t rows) { return rows <= 256 ? 8 : kMaxChunk; }

template <typename T>
cudaError_t shrink_simt(const LoraShrink& l, cudaStream_t s) {
  lora_shrink_simt_kernel<T><<<static_cast<unsigned>(l.rows), kWarps * 32, 0, s>>>(
      static_cast<const T*>(l.x), static_cast<const T*>(l.a), l.ids, l.K, l.rank, l.adapters, l.t);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_lora_shrink_simt(const LoraShrink& l, cudaStream_t s) {
  if (l.dtype == kDtF32) return shrink_simt<float>(l, s);
  if (l.dtype == kDtF16) return shrink_simt<__half>(l, s);
  if (l.dtype == kDtBF16) return shrink_simt<__nv_bfloat16>(l, s);
  return cudaErrorInvalidValue;
}

int lora_shrink_splits(int64_t rows, int K) {
  // Until about two CTAs an SM run, with at least two slices of K each.
  const int64_t chunks = (rows + shrink_chunk(rows) - 1) / shrink_chunk(rows);
  const int slices = (K + kBK - 1) / kBK;
  int splits = 1;
  while (splits < 8 && chunks * splits * 2 <= 296 && slices >= 4 * splits) splits *= 2;
  return splits;
}

bool lora_shrink_tc_supported(const LoraShrink& l) {
  if (l.dtype != kDtF16 && l.dtype != kDtBF16) return false;
  if (l.K % 8 != 0 || l.rank % 8 != 0) return false;
  auto aligned = [](const void* q) { return (reinterpret_cast<uintptr_t>(q) & 15) == 0; };
  return aligned(l.x) && aligned(l.a);
}

cudaError_t launch_lora_shrink_tc(const LoraShrink& l, cudaStream_t s) {
  ShrinkParams p{};
  p.ids = l.ids;
  p.t = l.t;
  p.rows = l.rows;
  p.K = l.K;
  p.rank = l.rank;
  p.adapters = l.adapters;
  p.chunk = shrink_chunk(l.rows);
  p.mma_n = std::max(p.chunk, 16);
  p.splits = l.splits;
  p.stage_bytes = kABytes + p.mma_n * kBK * 2;
  CUtensorMap mx, ma;
  if (!grouped_map(&mx, l.dtype, l.x, l.K, l.rows, 1, p.chunk) ||
      !grouped_map(&ma, l.dtype, l.a, l.K, l.rank, l.adapters, std::min(l.rank, kM)))
    return cudaErrorInvalidValue;
  const int smem = 1024 + kTcStages * p.stage_bytes + 256;
  static SmemOptIn opt_in;
  cudaError_t st = opt_in.set(lora_shrink_tc_kernel,
                              1024 + kTcStages * (kABytes + kMaxChunk * kBK * 2) + 256);
  if (st != cudaSuccess) return st;
  const int64_t ctas = (l.rows + p.chunk - 1) / p.chunk * p.splits;
  lora_shrink_tc_kernel<<<static_cast<unsigned>(ctas), kTcThreads, smem, s>>>(
      mx, ma, l.dtype == kDtBF16 ? 1u : 0u, p);
  return cudaGetLastError();
}

cudaError_t take_lora_error(int* err) {
  cudaError_t st = cudaMemcpyFromSymbol(err, g_shrink_error, sizeof(int));
  if (st != cudaSuccess || *err == 0) return st;
  const int zero = 0;
  return cudaMemcpyToSymbol(g_shrink_error, &zero, sizeof(int));
}

}  // namespace moe

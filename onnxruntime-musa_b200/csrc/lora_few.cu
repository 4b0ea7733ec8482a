// The adapter projection of a few rows (at most eight, and rows x rank <= 128) in one launch:
// the form for a request's next token.
//
// Two launches (lora.cu, then grouped_small.cu) make a chain: read A_a, hand t over, read B_a.
// For so few rows t is cheap enough to form again in every tile: a CTA that streams its
// share of a weight tile [128, K] also loads the same columns of the rows' A_a (r rows each,
// stacked: at most 128), and the tensor core multiplies both with the same x.  The cluster's
// CTAs split K; the leader receives the others' partial sums of the tile and of t in its
// shared memory, adds them in rank order, and adds s_a B_a t with FMAs in fp32 -- t is never
// rounded -- from the B rows that each thread (one output feature) fetched while the weights
// streamed.  Sums of more than one segment of slices (kSegment) are added up in the epilogue's
// registers.
// Bound: the weights' bytes; A_a adds rows x rank / 128 of them, from L2 after the first tile.
// Measured: one row, rank 16, [4096, 4096], bf16, 10.0 us in a replayed graph of calls on the same
// inputs (3.4 TB/s, from L2); 14.4 us a call in a loop, which is the host's pace.
#include <algorithm>

#include "grouped_tc.cuh"

namespace moe {
namespace {

constexpr int kBK = 64;
constexpr int kTileM = 128;
constexpr int kWBytes = kTileM * kBK * 2;
constexpr int kXRows = 8;                 // rows loaded (the MMA's N = 16 reads 16)
constexpr int kXBytes = 16 * kBK * 2;
constexpr int kThreads = 192;             // warp 0 TMA, warp 1 MMA, warps 2..5 epilogue
constexpr int kMaxStages = 6;
constexpr int kTmemCols = 32;             // the tile in columns 0..15, t in 16..31
// Parts of one sender: [quads][128] float4 of the tile (4 rows of a feature each), 128 floats
// of t.
__host__ __device__ constexpr int part_bytes(int quads) { return quads * kTileM * 16 + 128 * 4; }

struct FewParams {
  const void* b;
  const int32_t* ids;
  const float* scales;
  void* y;
  int rows, N, K, rank, adapters;
  int splits, stages, stage_bytes, a_bytes;
  int quads;  // ceil(rows / 4)
  int* error;
  int test_stall;
};

__device__ __forceinline__ void st_async_f4(uint32_t addr, float a, float b, float c, float d,
                                            uint32_t bar) {
  asm volatile(
      "st.async.shared::cluster.mbarrier::complete_tx::bytes.v4.f32 [%0], {%1, %2, %3, %4}, [%5];" ::
          "r"(addr), "f"(a), "f"(b), "f"(c), "f"(d), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void st_async_f1(uint32_t addr, float a, uint32_t bar) {
  asm volatile(
      "st.async.shared::cluster.mbarrier::complete_tx::bytes.f32 [%0], %1, [%2];" ::"r"(addr),
      "f"(a), "r"(bar)
      : "memory");
}

// SEG: a CTA may have more than one segment of slices.
template <typename T, bool SEG>
__global__ void __launch_bounds__(kThreads, 2)
lora_few_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x,
                const __grid_constant__ CUtensorMap map_a, const FewParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  // Behind the ring: the slack that the MMA on a short stack of A rows may read.
  uint8_t* parts = ring + p.stages * p.stage_bytes + (kWBytes - p.a_bytes);
  float* t = reinterpret_cast<float*>(parts + (p.splits - 1) * part_bytes(p.quads));  // [128]
  uint64_t* full = reinterpret_cast<uint64_t*>(t + 128);
  uint64_t* empty = full + kMaxStages;
  uint64_t* tfull = empty + kMaxStages;
  uint64_t* xfull = tfull + 1;
  uint64_t* sfull = xfull + 1;   // a segment that is not the last is complete
  uint64_t* sempty = sfull + 1;  // ... and has been read
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sempty + 1);
  static_assert((2 * kMaxStages + 4) * 8 + 4 <= 256, "barrier block");

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int S = p.splits;
  const int split = S == 1 ? 0 : static_cast<int>(cluster_ctarank());
  const int m0 = static_cast<int>(blockIdx.x) / S * kTileM;
  const int used = p.rows * p.rank;  // stacked rows of A

  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(tfull, 1);
    mbar_init(xfull, 1);
    mbar_init(sfull, 1);
    mbar_init(sempty, 4);
    fence_mbarrier_init();
    tma_prefetch_desc(&map_w);
    tma_prefetch_desc(&map_x);
    tma_prefetch_desc(&map_a);
    if (split == 0 && S > 1) mbar_arrive_expect_tx(xfull, (S - 1) * (p.quads * kTileM * 16 + used * 4));
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (S > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  pdl_wait();
  pdl_launch_dependents();  // this CTA holds its tensor memory
  const uint32_t tmem = *tmem_slot;
  // Adapter of row `lane`, -1 for none.
  int ad = lane < p.rows ? __ldg(p.ids + lane) : -1;
  if (ad >= p.adapters) ad = -1;
  const int slices = (p.K + kBK - 1) / kBK;

  if (warp == 0) {
    const int mine = __popc(__ballot_sync(0xffffffffu, ad >= 0));
    int stage = 0;
    uint32_t phase = 0;
    for (int s = p.test_stall ? slices : split; s < slices; s += S) {
      uint8_t* w = ring + stage * p.stage_bytes;
      int ok = 1;
      if (lane == 0) {
        ok = mbar_wait(&empty[stage], phase ^ 1);
        if (ok) {
          mbar_arrive_expect_tx(&full[stage],
                                kWBytes + kXRows * kBK * 2 + mine * p.rank * kBK * 2);
          tma_load_3d(w, &map_w, &full[stage], s * kBK, m0, 0);
          tma_load_3d(w + kWBytes + p.a_bytes, &map_x, &full[stage], s * kBK, 0, 0);
        } else {
          report_error(p.error, kErrTimeoutProducer);
        }
      }
      if (!__shfl_sync(0xffffffffu, ok, 0)) break;
      if (ad >= 0)
        tma_load_3d(w + kWBytes + lane * p.rank * kBK * 2, &map_a, &full[stage], s * kBK, 0, ad);
      if (++stage == p.stages) { stage = 0; phase ^= 1; }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      const uint32_t idesc = idesc_f16(TcFormat<T>::kId, kTileM, 16);
      int stage = 0, left = kSegment;  // slices until the segment is complete
      uint32_t phase = 0, seg = 0;
      bool gave_up = false;
      for (int s = split; s < slices; s += S) {
        bool ok = true;
        if (SEG && left == 0) {
          tc_commit(sfull);
          ok = mbar_wait(sempty, seg++ & 1);
          left = kSegment;
        }
        if (!ok || !mbar_wait(&full[stage], phase)) {
          report_error(p.error, kErrTimeoutMma);
          gave_up = true;
          break;
        }
        tc_fence_after();
        const uint32_t w = smem_u32(ring + stage * p.stage_bytes);
        const uint32_t x = w + kWBytes + p.a_bytes;
#pragma unroll
        for (int k = 0; k < kBK / 16; ++k) {
          const uint32_t more = (left != kSegment || k != 0) ? 1u : 0u;
          tc_mma_f16(tmem, smem_desc_k_sw128(w + k * 32), smem_desc_k_sw128(x + k * 32), idesc, more);
          tc_mma_f16(tmem + 16, smem_desc_k_sw128(w + kWBytes + k * 32),
                     smem_desc_k_sw128(x + k * 32), idesc, more);
        }
        --left;
        tc_commit(&empty[stage]);
        if (++stage == p.stages) { stage = 0; phase ^= 1; }
      }
      tc_commit(tfull);
      if (gave_up) drain_ring(full, p.stages, stage, phase);
    }
  }
  __syncwarp();

  // Epilogue: thread q * 32 + lane has output feature n, and row `me` of the stack of A.
  const bool epi = warp >= 2;
  const int q = warp & 3, me = q * 32 + lane, n = m0 + me;
  uint4 bq[16];  // B_a[n, :] of the rows one after the other, eight entries each
  if (epi && split == 0) {
    int row = 0, j = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int a = __shfl_sync(0xffffffffu, ad, row);
      bq[i] = make_uint4(0, 0, 0, 0);
      if (i * 8 < used && a >= 0 && n < p.N)
        bq[i] = __ldg(reinterpret_cast<const uint4*>(
            static_cast<const T*>(p.b) + (static_cast<int64_t>(a) * p.N + n) * p.rank + j));
      j += 8;
      if (j == p.rank) { j = 0; row = min(row + 1, 31); }
    }
  }
  const uint32_t lanes = tmem + (static_cast<uint32_t>(q * 32) << 16);
  const int row = me / p.rank;  // the row whose A entry this thread's is, and so its column
  float v[16], part_t = 0.f;
  auto fetch = [&] {
    float tv[16];
    tmem_ld16(lanes, v);
    tmem_ld16(lanes + 16, tv);
    tmem_ld_wait();
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (row == i) part_t = tv[i];
  };
  const int segments = SEG ? segments_of((slices - split + S - 1) / S) : 1;
  float sum[8] = {}, sum_t = 0.f;
  for (int seg = 0; epi && seg < segments - 1; ++seg) {
    if (!warp_wait(sfull, seg & 1)) break;  // (tfull will not complete either)
    tc_fence_after();
    fetch();
#pragma unroll
    for (int i = 0; i < 8; ++i) sum[i] += v[i];
    sum_t += part_t;
    tc_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(sempty);
  }
  const bool ok = warp_wait(tfull, 0);
  if (!ok) report_error(p.error, kErrTimeoutEpilogue);
  tc_fence_after();
  if (S > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  if (epi) {
    fetch();
    if (segments > 1) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] += sum[i];
      part_t += sum_t;
    }
    if (split >= slices || !ok) {  // nothing accumulated
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = 0.f;
      part_t = 0.f;
    }
    if (split != 0) {
      const uint32_t dst = mapa_shared(smem_u32(parts + (split - 1) * part_bytes(p.quads)), 0);
      const uint32_t bar = mapa_shared(smem_u32(xfull), 0);
      st_async_f4(dst + me * 16, v[0], v[1], v[2], v[3], bar);
      if (p.quads > 1) st_async_f4(dst + (kTileM + me) * 16, v[4], v[5], v[6], v[7], bar);
      if (me < used) st_async_f1(dst + p.quads * kTileM * 16 + me * 4, part_t, bar);
    }
  }
  if (split == 0 && epi) {
    if (S > 1 && !wait_parts(xfull)) report_error(p.error, kErrTimeoutEpilogue);
    for (int r = 1; r < S; ++r) {  // the parts in rank order
      const uint8_t* src = parts + (r - 1) * part_bytes(p.quads);
      const float4 a = *reinterpret_cast<const float4*>(src + me * 16);
      v[0] += a.x; v[1] += a.y; v[2] += a.z; v[3] += a.w;
      if (p.quads > 1) {
        const float4 b = *reinterpret_cast<const float4*>(src + (kTileM + me) * 16);
        v[4] += b.x; v[5] += b.y; v[6] += b.z; v[7] += b.w;
      }
      if (me < used)
        part_t += *reinterpret_cast<const float*>(src + p.quads * kTileM * 16 + me * 4);
    }
    if (me < used) t[me] = part_t;
    asm volatile("bar.sync 1, 128;" ::: "memory");
    // d[row] = sum_j B_a[n, j] t[row, j].
    float d[8] = {};
    int row = 0, j = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      if (i * 8 >= used) break;
      const T* e = reinterpret_cast<const T*>(&bq[i]);
      float sum = 0.f;
#pragma unroll
      for (int k = 0; k < 8; ++k) sum = fmaf(to_f(e[k]), t[i * 8 + k], sum);
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (k == row) d[k] += sum;
      j += 8;
      if (j == p.rank) { j = 0; ++row; }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (i >= p.rows) break;
      const int a = __shfl_sync(0xffffffffu, ad, i);
      const float y = a >= 0 ? fmaf(__ldg(p.scales + a), d[i], v[i]) : v[i];
      if (n < p.N) static_cast<T*>(p.y)[static_cast<int64_t>(i) * p.N + n] = from_f<T>(y);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

template <typename T>
cudaError_t launch_few(const GroupedArgs& g, const LoraShrink& l, const void* b, int num_sms,
                       cudaStream_t s) {
  FewParams p{};
  p.b = b;
  p.ids = l.ids;
  p.scales = l.scales;
  p.y = g.out;
  p.error = g.error;
  p.test_stall = g.test_stall;
  p.rows = static_cast<int>(g.rows);
  p.N = g.N;
  p.K = g.K;
  p.rank = l.rank;
  p.adapters = l.adapters;
  p.quads = (p.rows + 3) / 4;
  p.a_bytes = p.rows * p.rank * kBK * 2;
  p.stage_bytes = kWBytes + p.a_bytes + kXBytes;
  const int tiles = (g.N + kTileM - 1) / kTileM;
  const int slices = (g.K + kBK - 1) / kBK;
  // Two CTAs an SM, as in grouped_small.cu.
  p.splits = 1;
  while (p.splits < 8 && tiles * p.splits <= num_sms && slices >= 4 * p.splits) p.splits *= 2;
  const int fixed = 1024 + kWBytes - p.a_bytes + (p.splits - 1) * part_bytes(p.quads) + 512 + 256;
  p.stages = std::min(kMaxStages, (113 * 1024 - fixed) / p.stage_bytes);
  CUtensorMap mw, mx, ma;
  if (!grouped_map(&mw, g.dtype, g.w, g.K, g.N, 1, kTileM) ||
      !grouped_map(&mx, g.dtype, g.x, g.K, g.rows, 1, kXRows) ||
      !grouped_map(&ma, g.dtype, l.a, g.K, l.rank, l.adapters, l.rank))
    return cudaErrorInvalidValue;
  auto launch = [&](auto kernel, SmemOptIn& opt_in) {
    cudaError_t st = opt_in.set(kernel, 113 * 1024);
    if (st != cudaSuccess) return st;
    return launch_overlapped(kernel, static_cast<unsigned>(tiles * p.splits), kThreads,
                             fixed + p.stages * p.stage_bytes, p.splits, s, mw, mx, ma, p);
  };
  static SmemOptIn one, many;
  return segments_of((slices + p.splits - 1) / p.splits) > 1 ? launch(lora_few_kernel<T, true>, many)
                                                             : launch(lora_few_kernel<T, false>, one);
}

}  // namespace

bool lora_few_supported(int64_t rows, int64_t rank) { return rows <= 8 && rows * rank <= 128; }

cudaError_t launch_lora_few(const GroupedArgs& g, const LoraShrink& l, const void* b, int num_sms,
                            cudaStream_t s) {
  if (g.dtype == kDtF16) return launch_few<__half>(g, l, b, num_sms, s);
  if (g.dtype == kDtBF16) return launch_few<__nv_bfloat16>(g, l, b, num_sms, s);
  return cudaErrorInvalidValue;
}

}  // namespace moe

// Adapter projections of rows that follow different adapters: t[row] = A_a x[row].
//
// The second half, y += s_a B_a t, runs in the epilogue of the shared projection's kernels
// (grouped_simt.cu, grouped_small.cu, grouped_tc.cu), so y is written once.  t is summed in fp32;
// the FFMA kernels take it as it is, the tensor-core kernels in two 16-bit parts
// (grouped_lora.cuh says what those keep).
//
// lora_shrink_tc_kernel (16-bit types): a CTA takes a chunk of adjacent rows and one split
// of K.  The A_a of the chunk's distinct adapters are stacked as the MMA's M (128 / r
// adapters a pass), its rows are the N, and each column keeps the lanes of its own adapter:
// rows need no sorting, and another adapter's values never reach a row.  One prompt in a
// chunk is one pass; a decode chunk of 4 rows is at most 4 adapters, read once each.  A pass
// over more than one segment of slices (kSegment) takes an accumulator for each, which the
// epilogue adds up.
// Bound: the bytes of A_a (decode) and of x (prefill); the products are few.  The splits of
// a chunk are a cluster: each leaves its partial sums in shared memory, and each row's are
// added in rank order by one warp, which scales them and splits them into the 16-bit parts
// that the projection takes (grouped_lora.cuh).  Measured cold, K = 4096, bf16: 12.4 us for 64
// rows of 32 adapters of rank 16, 25 us for 4001 rows of 11 prompts, rank 64.
#include <algorithm>

#include "grouped_tc.cuh"

namespace moe {
namespace {

constexpr int kWarps = 8;

// Any type and alignment: a CTA takes kRows adjacent rows and kWarps rank entries, a warp
// each, the lanes striding over K.  One pass over an A row serves all rows that follow its
// adapter (rows of a prompt; A_a is what is read most).
constexpr int kRows = 4;
constexpr int kLaneFold = 32 * 512;  // contraction entries of 32 lanes' running sums

template <typename T>
__device__ __forceinline__ void load_vec(const T* p, int n, bool vec, float (&v)[4]) {
  if (vec && n >= 4) {
    if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<float4*>(v) = *reinterpret_cast<const float4*>(p);
    } else {
      const uint2 u = *reinterpret_cast<const uint2*>(p);
      const T* q = reinterpret_cast<const T*>(&u);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = to_f(q[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = i < n ? to_f(p[i]) : 0.f;
  }
}

template <typename T>
__global__ void __launch_bounds__(kWarps * 32)
lora_shrink_simt_kernel(const T* __restrict__ x, const T* __restrict__ a,
                        const int32_t* __restrict__ ids, const float* __restrict__ scales,
                        int64_t rows, int K, int rank, int adapters, bool vec,
                        float* __restrict__ t) {
  pdl_wait();
  pdl_launch_dependents();
  const int64_t row0 = static_cast<int64_t>(blockIdx.x) * kRows;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int j = blockIdx.y * kWarps + warp;
  if (j >= rank) return;
  int ad[kRows];
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    ad[i] = row0 + i < rows ? ids[row0 + i] : -1;
    if (ad[i] >= adapters) ad[i] = -1;
  }
#pragma unroll
  for (int f = 0; f < kRows; ++f) {
    // The first row of each adapter leads; the rows after it that follow the same join.
    bool lead = ad[f] >= 0;
#pragma unroll
    for (int i = 0; i < f; ++i) lead = lead && ad[i] != ad[f];
    if (!lead) continue;
    const T* ar = a + (static_cast<int64_t>(ad[f]) * rank + j) * K;
    float sum[kRows] = {}, folds[kRows] = {};
    for (int c0 = 0; c0 < K; c0 += kLaneFold) {
      const int c1 = min(c0 + kLaneFold, K);
#pragma unroll 8
      for (int k = c0 + lane * 4; k < c1; k += 128) {
        float w[4], v[4];
        load_vec(ar + k, K - k, vec, w);
#pragma unroll
        for (int i = f; i < kRows; ++i) {
          if (ad[i] != ad[f]) continue;
          load_vec(x + (row0 + i) * K + k, K - k, vec, v);
#pragma unroll
          for (int q = 0; q < 4; ++q) sum[i] = fmaf(w[q], v[q], sum[i]);
        }
      }
      if (K > kLaneFold) {  // sums of 512 entries, then a sum of those
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
          folds[i] += sum[i];
          sum[i] = 0.f;
        }
      }
    }
    if (K > kLaneFold) {
#pragma unroll
      for (int i = 0; i < kRows; ++i) sum[i] = folds[i];
    }
#pragma unroll
    for (int i = f; i < kRows; ++i) {
      if (ad[i] != ad[f]) continue;
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], d);
      if (lane == 0) t[(row0 + i) * rank + j] = scales[ad[f]] * sum[i];
    }
  }
}

constexpr int kBK = 64;
constexpr int kM = 128;
constexpr int kABytes = kM * kBK * 2;
constexpr int kMaxChunk = 64;
constexpr int kTcStages = 8;   // most stages of the ring
// Largest dynamic shared memory: align slack, ring, partial sums, barriers.
constexpr int kTcSmemMax = 1024 + 3 * (kABytes + kMaxChunk * kBK * 2) +
                           kMaxChunk * kLoraMaxRank * 4 + 256;
static_assert(1024 + 92 * 1024 + kABytes + 8 * kLoraMaxRank * 4 + 256 <= kTcSmemMax, "");
constexpr int kTcThreads = 192;   // warp 0 TMA, warp 1 MMA, warps 2..5 epilogue

struct ShrinkParams {
  const int32_t* ids;
  const float* scales;
  uint16_t* parts;
  float* row_scale;
  int* row_code;
  int64_t rows;
  int K, rank, adapters;
  int chunk;      // rows of a CTA: 4 or 64
  int mma_n;      // max(chunk, 16)
  int splits;
  int a_bytes;    // rows of A_a in a stage (the MMA reads on behind them, in other stages
                  // or the slack after the ring: lanes that nobody reads)
  int stages, stage_bytes;
  int* error;
  int test_stall;
};

__device__ __forceinline__ float4 ld_cluster_f4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}

// Two 16-bit parts of a value.  A finite value that would round to infinity takes the largest
// finite one and the rest; an infinity stays one part (its rest would be NaN).
template <typename T> constexpr float kMaxFinite = 65504.f;
template <> constexpr float kMaxFinite<__nv_bfloat16> = 3.3895313892515355e38f;
template <typename T>
__device__ __forceinline__ void split_part(float v, float& hi, float& lo) {
  hi = to_f(from_f<T>(v));
  lo = v - hi;
  if (isinf(hi)) {
    if (isfinite(v)) hi = copysignf(kMaxFinite<T>, v);
    lo = isfinite(v) ? v - hi : 0.f;
  }
}
template <typename T>
__device__ __forceinline__ void split_parts(const float4& v, uint2& hi, uint2& lo) {
  float h[4], l[4];
  split_part<T>(v.x, h[0], l[0]);
  split_part<T>(v.y, h[1], l[1]);
  split_part<T>(v.z, h[2], l[2]);
  split_part<T>(v.w, h[3], l[3]);
  hi = make_uint2(pack2<T>(h[0], h[1]), pack2<T>(h[2], h[3]));
  lo = make_uint2(pack2<T>(l[0], l[1]), pack2<T>(l[2], l[3]));
}

// SEG: a CTA may have more than one segment of slices.
template <typename T, bool SEG>
__global__ void __launch_bounds__(kTcThreads)
lora_shrink_tc_kernel(const __grid_constant__ CUtensorMap map_x,
                      const __grid_constant__ CUtensorMap map_a, const ShrinkParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  float* part = reinterpret_cast<float*>(ring + p.stages * p.stage_bytes + kABytes - p.a_bytes);  // [chunk][rank]
  uint64_t* full = reinterpret_cast<uint64_t*>(part + p.chunk * p.rank);
  uint64_t* empty = full + kTcStages;
  uint64_t* tfull = empty + kTcStages;   // [2]
  uint64_t* tempty = tfull + 2;          // [2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  __shared__ int s_id[kMaxChunk], s_first[kMaxChunk], s_slot[kMaxChunk], s_adapter[kMaxChunk];
  __shared__ int s_distinct;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int split = static_cast<int>(cluster_ctarank());
  const int64_t row0 = static_cast<int64_t>(blockIdx.x / p.splits) * p.chunk;
  const int n = static_cast<int>(min(static_cast<int64_t>(p.chunk), p.rows - row0));

  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) {
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
  pdl_wait();
  // Distinct adapters of the chunk in order of first appearance.
  const int tok = static_cast<int>(threadIdx.x) - 64;  // warps 2 and 3: a thread a row
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
  // The projection's main loop does not read the parts, so it may start now -- not before
  // this CTA holds its tensor memory, which the projection could otherwise take and keep
  // until this kernel is done.
  pdl_launch_dependents();
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
  const int segments = SEG ? segments_of(s1 - s0) : 1;

  if (warp == 0) {
    // Lane 0 waits for the slot and loads x; lane u loads the rows of unit u (up to 16 boxes
    // a slice: issued by one thread they took longer than the transfer).
    int stage = 0;
    uint32_t phase = 0;
    bool ok = p.test_stall == 0;
    for (int ps = 0; ps < passes && ok; ++ps) {
      const int u0 = ps * per, nu = min(per, units - u0);
      const int unit = u0 + lane;
      const bool mine_u = lane < nu;
      const int a_row = mine_u ? (unit % blocks_u) * kM : 0;
      const int a_id = mine_u ? s_adapter[unit / blocks_u] : 0;
      for (int s = s0; s < s1; ++s) {
        uint8_t* w = ring + stage * p.stage_bytes;
        if (lane == 0) {
          ok = mbar_wait(&empty[stage], phase ^ 1);
          if (ok) {
            mbar_arrive_expect_tx(&full[stage], (nu * rows_u + p.chunk) * kBK * 2);
            tma_load_3d(w + p.a_bytes, &map_x, &full[stage], s * kBK, static_cast<int>(row0), 0);
          } else {
            report_error(p.error, kErrTimeoutProducer);
            *abort_flag = 1;
          }
        }
        ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
        if (!ok) break;
        if (mine_u)
          tma_load_3d(w + lane * rows_u * kBK * 2, &map_a, &full[stage], s * kBK, a_row, a_id);
        if (++stage == p.stages) { stage = 0; phase ^= 1; }
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      const uint32_t idesc = idesc_f16(TcFormat<T>::kId, kM, p.mma_n);
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int fill = 0; fill < passes * segments && ok; ++fill) {
        const int acc = fill & 1;
        ok = mbar_wait(&tempty[acc], ((fill >> 1) & 1) ^ 1);
        tc_fence_after();
        const int first = SEG ? s0 + fill % segments * kSegment : s0;
        const int stop = SEG ? min(first + kSegment, s1) : s1;
        for (int s = first; s < stop && ok; ++s) {
          ok = mbar_wait(&full[stage], phase);
          if (!ok) break;
          tc_fence_after();
          const uint32_t w = smem_u32(ring + stage * p.stage_bytes);
#pragma unroll
          for (int k = 0; k < kBK / 16; ++k)
            tc_mma_f16(tmem + acc * p.mma_n, smem_desc_k_sw128(w + k * 32),
                       smem_desc_k_sw128(w + p.a_bytes + k * 32), idesc,
                       (s != first || k != 0) ? 1u : 0u);
          tc_commit(&empty[stage]);
          if (++stage == p.stages) { stage = 0; phase ^= 1; }
        }
        tc_commit(&tfull[acc]);  // after a timeout too: it waits for the MMAs issued
      }
      if (!ok) {
        report_error(p.error, kErrTimeoutMma);
        *abort_flag = 1;
        drain_ring(full, p.stages, stage, phase);
      }
    }
  } else {
    const int q = warp & 3;
    const int lane_row = q * 32 + lane;
    const int u = lane_row / rows_u, j0 = lane_row - u * rows_u;
    for (int fill = 0; fill < passes * segments && !warp_stopped(abort_flag); ++fill) {
      const int acc = fill & 1, ps = fill / segments;
      const bool more = fill % segments != 0;  // adds to the segments before
      const int unit = ps * per + u;
      const int j = (unit % blocks_u) * kM + j0;
      const int slot = u < per && unit < units && j < p.rank ? unit / blocks_u : -2;
      uint64_t own = 0;  // the rows that follow this lane's adapter
      for (int i = 0; i < n; ++i)
        if (s_slot[i] == slot) own |= uint64_t{1} << i;
      if (!warp_wait(&tfull[acc], (fill >> 1) & 1)) {
        report_error(p.error, kErrTimeoutEpilogue);
        *abort_flag = 1;
        break;
      }
      tc_fence_after();
      for (int c = 0; c < n; c += 16) {
        float v[16];
        tmem_ld16(tmem + (static_cast<uint32_t>(q * 32) << 16) + acc * p.mma_n + c, v);
        tmem_ld_wait();
        const unsigned bits = static_cast<unsigned>(own >> c);
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (bits & (1u << i)) {
            float& t = part[(c + i) * p.rank + j];
            t = (more ? t : 0.f) + (s0 < s1 ? v[i] : 0.f);
          }
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
  cluster_sync();  // every split's partial sums are in its `part`
  // Row i of the chunk is finished by CTA i % splits, one warp a row; a lane takes granules
  // of four entries.
  for (int i = split + p.splits * warp; i < n; i += p.splits * (kTcThreads / 32)) {
    if (s_slot[i] < 0) {
      if (lane == 0) p.row_code[row0 + i] = -1;
      continue;
    }
    const float sc = __ldg(p.scales + s_id[i]);
    float4 v[2];
    float m = 0.f;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int j = 4 * (lane + 32 * h);
      v[h] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (j < p.rank) {
        const uint32_t at = smem_u32(part + i * p.rank + j);
        float4 w[8];
#pragma unroll
        for (int r = 0; r < 8; ++r)
          w[r] = r < p.splits ? ld_cluster_f4(mapa_shared(at, r)) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int r = 0; r < 8; ++r) {
          v[h].x += w[r].x; v[h].y += w[r].y; v[h].z += w[r].z; v[h].w += w[r].w;
        }
        v[h].x *= sc; v[h].y *= sc; v[h].z *= sc; v[h].w *= sc;
      }
      auto size = [](float t) { return isfinite(t) ? fabsf(t) : 0.f; };  // (no scale helps others)
      m = fmaxf(m, fmaxf(fmaxf(size(v[h].x), size(v[h].y)), fmaxf(size(v[h].z), size(v[h].w))));
    }
    int code = s_id[i];
    if (std::is_same<T, __half>::value) {
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
      float down = 1.f;
      // Inside [2^-8, 2^15) the parts keep 16 bits of the row's largest finite entry as they are.
      if ((m > 0.f && m < 0.00390625f) || m >= 32768.f) {
        const int e = min(max((__float_as_int(m) >> 23) - 127, -120), 120);
        const float up = __int_as_float((127 - e) << 23);
        down = __int_as_float((127 + e) << 23);
        code |= kLoraScaled;
#pragma unroll
        for (int h = 0; h < 2; ++h) { v[h].x *= up; v[h].y *= up; v[h].z *= up; v[h].w *= up; }
      }
      if (lane == 0) p.row_scale[row0 + i] = down;
    }
    if (lane == 0) p.row_code[row0 + i] = code;
    uint16_t* dst = p.parts + (row0 + i) * p.rank;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int j = 4 * (lane + 32 * h);
      if (j < p.rank) {
        uint2 hi, lo;
        split_parts<T>(v[h], hi, lo);
        *reinterpret_cast<uint2*>(dst + j) = hi;
        *reinterpret_cast<uint2*>(dst + j + p.rows * p.rank) = lo;
      }
    }
  }
  cluster_sync();  // no CTA leaves while another reads its part
}

// Rows of a CTA: small chunks spread a decode batch (whose rows follow many adapters) over
// the GPU, tall ones read A_a once per 64 rows of a prompt.
int shrink_chunk(int64_t rows) { return rows <= 256 ? 4 : kMaxChunk; }

template <typename T>
cudaError_t shrink_simt(const LoraShrink& l, float* t, cudaStream_t s) {
  const bool vec = l.K % 4 == 0 &&
                   (reinterpret_cast<uintptr_t>(l.x) | reinterpret_cast<uintptr_t>(l.a)) %
                           (4 * sizeof(T)) == 0;
  return launch_dependent(pdl_enabled(), lora_shrink_simt_kernel<T>,
                          dim3(static_cast<unsigned>((l.rows + kRows - 1) / kRows),
                               (l.rank + kWarps - 1) / kWarps),
                          dim3(kWarps * 32), 0, s, static_cast<const T*>(l.x),
                          static_cast<const T*>(l.a), l.ids, l.scales, l.rows, l.K, l.rank,
                          l.adapters, vec, t);
}

template <typename T>
cudaError_t shrink_tc(const LoraShrink& l, uint16_t* parts, float* row_scale, int* row_code,
                      int num_sms, cudaStream_t s) {
  ShrinkParams p{};
  p.ids = l.ids;
  p.scales = l.scales;
  p.parts = parts;
  p.row_scale = row_scale;
  p.row_code = row_code;
  p.rows = l.rows;
  p.K = l.K;
  p.rank = l.rank;
  p.adapters = l.adapters;
  p.error = l.error;
  p.test_stall = l.test_stall;
  p.chunk = shrink_chunk(l.rows);
  p.mma_n = std::max(p.chunk, 16);
  // A stage holds the adapters that a chunk can have (one token: r rows), so that a short
  // K is in flight as a whole.  Small chunks stay at 56 KB, which fits an SM beside two CTAs of
  // the projection; of tall ones with the partial sums of rank 64, two fit an SM.
  const int unit = std::min(l.rank, kM);
  p.a_bytes = static_cast<int>(std::min<int64_t>(kM / unit, std::min<int64_t>(l.rows, p.chunk))) *
              unit * kBK * 2;
  p.stage_bytes = p.a_bytes + p.mma_n * kBK * 2;
  p.stages = p.chunk == kMaxChunk ? 3 : std::max(2, std::min(kTcStages, 40 * 1024 / p.stage_bytes));
  // Splits: until about two CTAs an SM run, with at least two slices of K each.
  const int64_t chunks = (l.rows + p.chunk - 1) / p.chunk;
  const int slices = (l.K + kBK - 1) / kBK;
  p.splits = 1;
  while (p.splits < 8 && chunks * p.splits <= num_sms && slices >= 4 * p.splits) p.splits *= 2;
  CUtensorMap mx, ma;
  if (!grouped_map(&mx, l.dtype, l.x, l.K, l.rows, 1, p.chunk) ||
      !grouped_map(&ma, l.dtype, l.a, l.K, l.rank, l.adapters, std::min(l.rank, kM)))
    return cudaErrorInvalidValue;
  const size_t smem =
      1024 + p.stages * p.stage_bytes + kABytes - p.a_bytes + p.chunk * p.rank * 4 + 256;
  auto launch = [&](auto kernel, SmemOptIn& opt_in) {
    cudaError_t st = opt_in.set(kernel, kTcSmemMax);
    if (st != cudaSuccess) return st;
    return launch_overlapped(kernel, static_cast<unsigned>(chunks * p.splits), kTcThreads, smem,
                             p.splits, s, mx, ma, p);
  };
  static SmemOptIn one, many;
  return segments_of((slices + p.splits - 1) / p.splits) > 1
             ? launch(lora_shrink_tc_kernel<T, true>, many)
             : launch(lora_shrink_tc_kernel<T, false>, one);
}

}  // namespace

cudaError_t launch_lora_shrink_simt(const LoraShrink& l, float* t, cudaStream_t s) {
  if (l.dtype == kDtF32) return shrink_simt<float>(l, t, s);
  if (l.dtype == kDtF16) return shrink_simt<__half>(l, t, s);
  if (l.dtype == kDtBF16) return shrink_simt<__nv_bfloat16>(l, t, s);
  return cudaErrorInvalidValue;
}

bool lora_shrink_tc_supported(const LoraShrink& l) {
  if (l.dtype != kDtF16 && l.dtype != kDtBF16) return false;
  if (l.K % 8 != 0 || l.rank % 8 != 0) return false;
  auto aligned = [](const void* q) { return (reinterpret_cast<uintptr_t>(q) & 15) == 0; };
  return aligned(l.x) && aligned(l.a);
}

cudaError_t launch_lora_shrink_tc(const LoraShrink& l, uint16_t* parts, float* row_scale,
                                  int* row_code, int num_sms, cudaStream_t s) {
  if (l.dtype == kDtF16) return shrink_tc<__half>(l, parts, row_scale, row_code, num_sms, s);
  if (l.dtype == kDtBF16)
    return shrink_tc<__nv_bfloat16>(l, parts, row_scale, row_code, num_sms, s);
  return cudaErrorInvalidValue;
}

}  // namespace moe

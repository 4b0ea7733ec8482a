// The expert products and the adapter projection for few rows per group: streaming the
// weights.
//
// y[p] = W[e] x[p] with a handful of rows reads every weight once for a few products; the
// floor is the weights' bytes over the HBM rate, and what decides is how many bytes are in
// flight.  So a tile is 128 features x all rows of the group (<= the tile cap), as
// D[feature, row] (weights are the MMA's M = 128, rows its N = 16 .. 256), and the
// contraction is split over a cluster of 1..8 CTAs so that the tiles of a call fill the
// GPU: each CTA streams its share of the slices through a TMA ring of about 100 KB (two
// CTAs an SM, 200 KB in flight) into one tcgen05 accumulator.  The partial sums are joined
// through distributed shared memory -- 8-row blocks of the accumulator go to the CTA that
// owns the block, which adds them in rank order -- so there is no global workspace, no
// counter to clear, no second launch, and the result is the same bits on every call.
// Measured: 8 rows over 8 experts of [768, 2048], bf16, 8.6 us in a replayed graph of calls on the same
// inputs (2.9 TB/s, from L2: the latency of a launch, a ring fill and a join); 9.9 us a call in a
// loop, which is the host's pace.
//
// The adapter term (LORA) does not wait for the product: while the weights stream, the
// epilogue warps form it for the blocks that they will finish and park it in the other half
// of the CTA's tensor memory.
//
// A CTA with more than one segment of slices (kSegment) hands its accumulator to the epilogue
// warps after each but the last; they keep the sum of the segments in the other half.
#include <algorithm>

#include "grouped_lora.cuh"

namespace moe {
namespace {

constexpr int kBK = 64;
constexpr int kTileM = 128;
constexpr int kWBytes = kTileM * kBK * 2;
constexpr int kThreads = 320;                    // warp 0 TMA, warp 1 MMA, warps 2.. epilogue
constexpr int kMaxStages = 8;
constexpr int kStageRow = 64;                    // bytes of a staged output row
constexpr int kEpiBytes = 8 * kStageRow;         // per warp
constexpr int kPartBytes = 4 * 8 * 32 * 4;       // one CTA's part of an 8-row block (fp32)
constexpr int kFixed = 1024 + 8 * kEpiBytes + 256 + kMaxExperts * 8 + (kMaxExperts + 1) * 4 + 12;

struct SmallParams {
  const int32_t* offsets;
  int64_t total_rows;
  int E;
  int m_dim, con;
  int m_tiles;
  int cap;            // most rows of a tile (16, 32, 64, 128 or 256)
  int box;            // rows of one TMA box of the rows operand: min(cap, 64)
  int splits;         // cluster size
  int stages, stage_bytes;
  int part_bytes;     // of the exchange behind the ring; 0: it reuses the ring
  uint32_t tmem_cols;
  void* out;
  int64_t ldo;
  LoraTerm lora;
  int* error;
  int test_stall;
};

__device__ __forceinline__ void tmem_ld_frag1(uint32_t taddr, float (&v)[4]) {
  uint32_t r[4];
  asm volatile("tcgen05.ld.sync.aligned.16x256b.x1.b32 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(taddr));
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tmem_st_frag1(uint32_t taddr, const float (&v)[4]) {
  asm volatile("tcgen05.st.sync.aligned.16x256b.x1.b32 [%0], {%1,%2,%3,%4};" ::"r"(taddr),
               "r"(__float_as_uint(v[0])), "r"(__float_as_uint(v[1])),
               "r"(__float_as_uint(v[2])), "r"(__float_as_uint(v[3]))
               : "memory");
}
// 16 bytes to another CTA's shared memory, counted on that CTA's barrier `bar`.
__device__ __forceinline__ void st_async_f4(uint32_t addr, const float (&v)[4], uint32_t bar) {
  asm volatile(
      "st.async.shared::cluster.mbarrier::complete_tx::bytes.v4.f32 [%0], {%1, %2, %3, %4}, [%5];" ::
          "r"(addr), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void cluster_arrive() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// SEG: a CTA may have more than one segment of slices.
template <typename T, int DIR, int LORA, bool SEG>
__global__ void __launch_bounds__(LORA > 0 ? 512 : kThreads, LORA > 0 ? 1 : 2)  // 128 / 96 registers
grouped_small_kernel(const __grid_constant__ CUtensorMap map_w,
                     const __grid_constant__ CUtensorMap map_x, const SmallParams p) {
  constexpr bool kAMn = DIR == kGmmGradInput;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* parts_buf = p.part_bytes ? ring + p.stages * p.stage_bytes : ring;
  uint8_t* stage_out = ring + p.stages * p.stage_bytes + p.part_bytes;
  uint64_t* full = reinterpret_cast<uint64_t*>(stage_out + 8 * kEpiBytes);
  uint64_t* empty = full + kMaxStages;
  uint64_t* tfull = empty + kMaxStages;
  uint64_t* xfull = tfull + 1;
  uint64_t* sfull = xfull + 1;   // a segment that is not the last is complete
  uint64_t* sempty = sfull + 1;  // ... and has been added to the sum
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sempty + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  static_assert((2 * kMaxStages + 4) * 8 + 8 <= 256, "barrier block");
  GroupTable table;
  table.rows = reinterpret_cast<int2*>(full + 32);
  table.tiles = reinterpret_cast<int*>(table.rows + kMaxExperts);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int split = p.splits == 1 ? 0 : static_cast<int>(cluster_ctarank());
  const int L = blockIdx.x / p.splits;

  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(tfull, 1);
    mbar_init(xfull, 1);
    mbar_init(sfull, 1);
    mbar_init(sempty, blockDim.x / 32 - 2);
    *abort_flag = 0;
    fence_mbarrier_init();
    tma_prefetch_desc(&map_w);
    tma_prefetch_desc(&map_x);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, p.tmem_cols);
    tmem_relinquish();
  }
  // The adapter projection's inputs were ready before the launch in front of it started;
  // its parts are awaited below.
  if (LORA == 0) pdl_wait();
  if (warp == 2)
    build_group_table(p.offsets, p.E, static_cast<int>(p.total_rows), p.cap, table);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_launch_dependents();  // this CTA holds its tensor memory: see launch_small
  const uint32_t tmem = *tmem_slot;
  if (L >= table.tiles[p.E] * p.m_tiles) {  // the grid is an upper bound; whole clusters leave
    if (warp == 1) tmem_dealloc(tmem, p.tmem_cols);
    return;
  }

  // From here on the cluster stays together; its CTAs' barriers are initialised.
  if (p.splits > 1 && p.part_bytes) cluster_arrive();

  // Tile: the row tiles of a weight tile run side by side (the weights then come from L2).
  const int e = find_group(table.tiles, p.E, p.m_tiles, L);
  const int nt_tiles = table.tiles[e + 1] - table.tiles[e];
  const int local = L - table.tiles[e] * p.m_tiles;
  const int m0 = (local / nt_tiles) * kTileM;
  const int2 gr = table.rows[e];
  const int h = ((gr.y - gr.x + nt_tiles - 1) / nt_tiles + 15) & ~15;
  const int row0 = gr.x + (local % nt_tiles) * h;
  const int n = min(h, gr.y - row0);
  const int nt = max((n + 15) & ~15, 16);
  const int slices = (p.con + kBK - 1) / kBK;
  // The CTAs of a cluster take the slices in turn: what they read at a time then lies side by
  // side in each weight row (2 to 4% on the streamed bytes).
  const int s0 = split, s1 = slices, ds = p.splits;
  const int segments = SEG ? segments_of((s1 - s0 + ds - 1) / ds) : 1;

  if (warp == 0 && lane == 0) {
    const int boxes = (nt + p.box - 1) / p.box;
    int stage = 0;
    uint32_t phase = 0;
    for (int s = p.test_stall ? s1 : s0; s < s1; s += ds) {
      if (!mbar_wait(&empty[stage], phase ^ 1)) {
        report_error(p.error, kErrTimeoutProducer);
        *abort_flag = 1;
        break;
      }
      uint8_t* w = ring + stage * p.stage_bytes;
      mbar_arrive_expect_tx(&full[stage], kWBytes + boxes * p.box * kBK * 2);
      const int c = s * kBK;
      if (kAMn) {
        tma_load_3d(w, &map_w, &full[stage], m0, c, e);
        tma_load_3d(w + kWBytes / 2, &map_w, &full[stage], m0 + 64, c, e);
      } else {
        tma_load_3d(w, &map_w, &full[stage], c, m0, e);
      }
      for (int j = 0; j < boxes; ++j)
        tma_load_3d(w + kWBytes + j * p.box * kBK * 2, &map_x, &full[stage], c,
                    row0 + j * p.box, 0);
      if (++stage == p.stages) { stage = 0; phase ^= 1; }
    }
  } else if (warp == 1 && lane == 0) {
    const uint32_t idesc = idesc_f16(TcFormat<T>::kId, kTileM, nt) | (kAMn ? kIdescAMn : 0);
    int stage = 0, left = kSegment;  // slices until the segment is complete
    uint32_t phase = 0, seg = 0;
    bool gave_up = false;
    for (int s = s0; s < s1; s += ds) {
      bool ok = true;
      if (SEG && left == 0) {
        tc_commit(sfull);
        if (LORA > 0) pdl_wait();  // the epilogue warps wait for the launch before
        ok = mbar_wait(sempty, seg++ & 1);
        left = kSegment;
      }
      if (!ok || !mbar_wait(&full[stage], phase)) {
        report_error(p.error, kErrTimeoutMma);
        *abort_flag = 1;
        gave_up = true;
        break;
      }
      tc_fence_after();
      const uint32_t w = smem_u32(ring + stage * p.stage_bytes);
#pragma unroll
      for (int k = 0; k < kBK / 16; ++k) {
        const uint64_t ad = kAMn ? smem_desc_mn_sw128(w + k * 2048, kWBytes / 2)
                                 : smem_desc_k_sw128(w + k * 32);
        tc_mma_f16(tmem, ad, smem_desc_k_sw128(w + kWBytes + k * 32), idesc,
                   (left != kSegment || k != 0) ? 1u : 0u);
      }
      --left;
      tc_commit(&empty[stage]);
      if (++stage == p.stages) { stage = 0; phase ^= 1; }
    }
    tc_commit(tfull);
    if (gave_up) drain_ring(full, p.stages, stage, phase);
  }
  __syncwarp();

  // Epilogue warp w reads TMEM lanes 32 (w % 4) ..; the warps of a lane quarter (two, or one
  // in a block of 192 threads) take turns with the 8-row blocks that this CTA owns (block b
  // belongs to CTA b % splits).
  const int S = p.splits;
  const int blocks = (n + 7) / 8;
  const int owned = blocks > split ? (blocks - split + S - 1) / S : 0;
  const bool epi = warp >= 2;
  const int q = warp & 3, pair = (warp - 2) >> 2, turns = (blockDim.x - 64) / 128;
  const int feat = m0 + q * 32;
  const uint32_t taddr = tmem + (static_cast<uint32_t>(q * 32) << 16);
  // Per block: the adapter term (of the owned blocks) and the segments before the last.
  const uint32_t tsum = taddr + p.cap;
  if (threadIdx.x == 64 && S > 1 && owned > 0)
    mbar_arrive_expect_tx(xfull, owned * (S - 1) * kPartBytes);
  if constexpr (LORA > 0) {
    if (epi && pair < owned) {
      // While the weights stream, a load takes microseconds: the fragments of B are under way
      // before the parts exist, and each block's parts before the block in front is done.
      // One copy of the code for all of it: a warp runs it a few times only, and fetching
      // instructions waits in the same queues (with gather and apply at three places each it
      // took 8 us longer).
      LoraBatch<T, LORA, 4 / LORA> batch;
      batch.clear();
      const int g = lane >> 2;
      int i = pair;
      int row = (i * S + split) * 8 + g;
      int ad = lora_adapter(p.lora, row0 + row, row < n);
      unsigned todo = __ballot_sync(0xffffffffu, ad >= 0);
      uint4 parts[LORA], parts_next[LORA];
      int row_next = 0, ad_next = -1;
      float lo[4] = {0.f, 0.f, 0.f, 0.f}, hi[4] = {0.f, 0.f, 0.f, 0.f};
      bool first = true, fresh = true;
#pragma unroll 1
      while (true) {
        batch.gather(p.lora, ad, todo, feat, p.m_dim);
        if (first) {
          pdl_wait();  // the packed parts come from the launch before this one
          lora_rows<LORA>(p.lora, p.total_rows, row0 + row, row < n, 0, parts);
          first = false;
        }
        if (fresh) {
          row_next = ((i + turns) * S + split) * 8 + g;
          const bool more = i + turns < owned && row_next < n;
          ad_next = lora_adapter(p.lora, row0 + row_next, more);
          lora_rows<LORA>(p.lora, p.total_rows, row0 + row_next, more, 0, parts_next);
          fresh = false;
        }
        batch.apply(p.lora, p.total_rows, ad, row0 + row, feat, p.m_dim, parts, lo, hi);
        if (todo != 0) continue;
        tmem_st_frag1(tsum + 8 * (i * S + split), lo);
        tmem_st_frag1(tsum + (16u << 16) + 8 * (i * S + split), hi);
        i += turns;
        if (i >= owned) break;
        row = row_next;
        ad = ad_next;
#pragma unroll
        for (int s = 0; s < LORA; ++s) parts[s] = parts_next[s];
        todo = __ballot_sync(0xffffffffu, ad >= 0);
#pragma unroll
        for (int j = 0; j < 4; ++j) lo[j] = hi[j] = 0.f;
        fresh = true;
      }
      tmem_st_wait();
    } else {
      pdl_wait();
    }
    __syncwarp();
  }

  for (int seg = 0; epi && seg < segments - 1; ++seg) {
    if (!warp_wait(sfull, seg & 1)) break;  // (tfull will not complete either)
    tc_fence_after();
    // Each warp adds what it will send or finish below.
    auto add = [&](int b, bool first) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t at = (static_cast<uint32_t>(16 * h) << 16) + 8 * b;
        float a[4], s[4] = {0.f, 0.f, 0.f, 0.f};
        tmem_ld_frag1(taddr + at, a);
        if (!first) tmem_ld_frag1(tsum + at, s);
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 4; ++j) s[j] += a[j];
        tmem_st_frag1(tsum + at, s);
      }
    };
    for (int b = pair; b < blocks; b += turns)
      if (b % S != split) add(b, seg == 0);
    for (int i = pair; i < owned; i += turns) add(i * S + split, LORA == 0 && seg == 0);
    tmem_st_wait();
    tc_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(sempty);
  }

  const bool ok = warp_wait(tfull, 0);
  if (!ok) {
    report_error(p.error, kErrTimeoutEpilogue);
    *abort_flag = 1;
  }
  tc_fence_after();
  const bool empty_part = s0 >= s1 || !ok;  // nothing accumulated: the part is zero
  if (S > 1) {
    if (p.part_bytes) {
      cluster_wait();  // every CTA of the cluster has initialised its barriers
    } else {
      cluster_sync();  // ... and its MMAs have read its ring, which takes the parts now
    }
    if (epi)
      for (int b = pair; b < blocks; b += turns) {
        const int owner = b % S;
        if (owner == split) continue;
        float lo[4] = {0.f, 0.f, 0.f, 0.f}, hi[4] = {0.f, 0.f, 0.f, 0.f};
        if (!empty_part) {
          tmem_ld_frag1(taddr + 8 * b, lo);
          tmem_ld_frag1(taddr + (16u << 16) + 8 * b, hi);
          tmem_ld_wait();
          if (segments > 1) {
            float slo[4], shi[4];
            tmem_ld_frag1(tsum + 8 * b, slo);
            tmem_ld_frag1(tsum + (16u << 16) + 8 * b, shi);
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 4; ++j) { lo[j] += slo[j]; hi[j] += shi[j]; }
          }
        }
        // Slot of this sender among the owner's S - 1, block b / S of the owner's.
        const int slot = split < owner ? split : split - 1;
        const uint32_t dst = smem_u32(parts_buf) + ((b / S) * (S - 1) + slot) * kPartBytes +
                             q * (kPartBytes / 4) + lane * 16;
        const uint32_t bar = mapa_shared(smem_u32(xfull), owner);
        st_async_f4(mapa_shared(dst, owner), lo, bar);
        st_async_f4(mapa_shared(dst + 512, owner), hi, bar);
      }
    if (owned > 0 && !wait_parts(xfull)) report_error(p.error, kErrTimeoutEpilogue);
  }

  uint8_t* buf = stage_out + (warp & 7) * kEpiBytes;
  const int st_row = lane & 7, st_blk = lane >> 3;
  const uint32_t st_addr =
      smem_u32(buf) + st_row * kStageRow + ((st_blk ^ ((st_row >> 1) & 3)) << 4);
  const int rd_row = lane >> 2, rd_blk = lane & 3;
  const uint8_t* rd_ptr = buf + rd_row * kStageRow + ((rd_blk ^ ((rd_row >> 1) & 3)) << 4);
  for (int i = pair; epi && i < owned; i += turns) {
    const int b = i * S + split;
    float lo[4] = {0.f, 0.f, 0.f, 0.f}, hi[4] = {0.f, 0.f, 0.f, 0.f};
    float own_lo[4] = {0.f, 0.f, 0.f, 0.f}, own_hi[4] = {0.f, 0.f, 0.f, 0.f};
    float add_lo[4] = {0.f, 0.f, 0.f, 0.f}, add_hi[4] = {0.f, 0.f, 0.f, 0.f};
    if (!empty_part) {
      tmem_ld_frag1(taddr + 8 * b, own_lo);
      tmem_ld_frag1(taddr + (16u << 16) + 8 * b, own_hi);
    }
    if (LORA > 0 || segments > 1) {
      tmem_ld_frag1(tsum + 8 * b, add_lo);
      tmem_ld_frag1(tsum + (16u << 16) + 8 * b, add_hi);
    }
    tmem_ld_wait();
    for (int r = 0; r < S; ++r) {  // the parts in rank order
      if (r == split) {
#pragma unroll
        for (int j = 0; j < 4; ++j) { lo[j] += own_lo[j]; hi[j] += own_hi[j]; }
      } else {
        const uint8_t* src = parts_buf + (i * (S - 1) + (r < split ? r : r - 1)) * kPartBytes +
                             q * (kPartBytes / 4) + lane * 16;
        const float4 a = *reinterpret_cast<const float4*>(src);
        const float4 c = *reinterpret_cast<const float4*>(src + 512);
        lo[0] += a.x; lo[1] += a.y; lo[2] += a.z; lo[3] += a.w;
        hi[0] += c.x; hi[1] += c.y; hi[2] += c.z; hi[3] += c.w;
      }
    }
    if (LORA > 0 || segments > 1) {
#pragma unroll
      for (int j = 0; j < 4; ++j) { lo[j] += add_lo[j]; hi[j] += add_hi[j]; }
    }
    stmatrix4_t(st_addr, pack2<T>(lo[0], lo[1]), pack2<T>(lo[2], lo[3]), pack2<T>(hi[0], hi[1]),
                pack2<T>(hi[2], hi[3]));
    __syncwarp();
    const uint4 w = *reinterpret_cast<const uint4*>(rd_ptr);
    const int row = 8 * b + rd_row, col = feat + 8 * rd_blk;
    if (row < n && col < p.m_dim)
      *reinterpret_cast<uint4*>(static_cast<T*>(p.out) +
                                static_cast<int64_t>(row0 + row) * p.ldo + col) = w;
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, p.tmem_cols);
  }
}

template <typename T, int DIR, int LORA>
cudaError_t launch_small(const GroupedArgs& g, const LoraTerm* lora, int num_sms, cudaStream_t s) {
  const int feat = DIR == kGmmForward ? g.N : g.K;
  SmallParams p{};
  p.offsets = g.offsets;
  p.total_rows = g.rows;
  p.E = g.E;
  p.m_dim = feat;
  p.con = DIR == kGmmForward ? g.K : g.N;
  p.m_tiles = (feat + kTileM - 1) / kTileM;
  p.out = g.out;
  p.ldo = feat;
  p.error = g.error;
  p.test_stall = g.test_stall;
  if (lora != nullptr) p.lora = *lora;
  // Tile cap: twice the mean rows per group (uneven groups then mostly stay one tile, and
  // their weights are streamed once), all of them when there is one group.
  const int64_t want = g.E == 1 ? g.rows : 2 * ((g.rows + g.E - 1) / g.E);
  p.cap = 16;
  while (p.cap < 256 && p.cap < want) p.cap *= 2;
  p.box = std::min(p.cap, 64);
  p.stage_bytes = kWBytes + p.cap * kBK * 2;
  // Tensor memory of the CTAs that fit an SM together never exceeds its 512 columns (a CTA
  // of these kernels takes at least 90 KB of shared memory per 256 columns), so an
  // allocation never waits for a CTA that waits for its own cluster.  (The second half: the
  // adapter term, the sum of the segments.)
  // The tile count lives on the device; each ragged group adds at most one.
  const int64_t tiles = (g.E == 1 ? (g.rows + p.cap - 1) / p.cap
                                  : g.rows / p.cap + std::min<int64_t>(g.rows, g.E)) *
                        p.m_tiles;
  // CTAs an SM: two, sharing its memory, up to 128 rows; one at 256.  (One alone with 130 KB
  // was slower: clusters of such CTAs do not all find room at once, 16.5 against 13.4 us for
  // 64 rows, 4096 x 4096.)  With adapters two have 192 threads, and of 32 or 64 rows 85 KB, which
  // leaves room for a CTA of the kernel that forms the parts, so that the weights stream
  // while that runs (up to 16 rows that has few CTAs, and more bytes in flight count).
  const int resident = p.cap > 128 ? 1 : 2;
  const int budget = (p.cap > 128 ? 220 : LORA > 0 && (p.cap == 32 || p.cap == 64) ? 86 : 113) * 1024;
  const int threads = LORA > 0 && resident == 2 ? 192 : kThreads;
  // Splits: until the grid fills these, with at least two slices each.  Clusters of eight CTAs
  // that each take an SM do not all find room at once (384 rows, [1024, 4096]: 21 us, by four
  // 14), except a few of them (192 rows: 11.6 us, by four 13.3).
  const int64_t fill = static_cast<int64_t>(num_sms) * resident;
  const int slices = (p.con + kBK - 1) / kBK;
  const int most = resident == 1 && tiles * 8 > 64 ? 4 : 8;
  p.splits = 1;
  while (p.splits < most && tiles * p.splits * 2 <= fill && slices >= 4 * p.splits) p.splits *= 2;
  const bool seg = segments_of((slices + p.splits - 1) / p.splits) > 1;
  p.tmem_cols = static_cast<uint32_t>(std::max(32, p.cap * (LORA > 0 || seg ? 2 : 1)));
  // The exchange has its own memory up to 64 rows (at most 28 KB); above, it reuses the ring
  // and the cluster meets once more before it.
  const int blocks_owned = (p.cap / 8 + p.splits - 1) / p.splits;
  p.part_bytes = p.cap <= 64 ? blocks_owned * (p.splits - 1) * kPartBytes : 0;
  p.stages = std::min(kMaxStages, (budget - kFixed - p.part_bytes) / p.stage_bytes);
  CUtensorMap mw, mx;
  if (!grouped_map(&mw, g.dtype, g.w, g.K, g.N, g.E, DIR == kGmmForward ? 128 : 64) ||
      !grouped_map(&mx, g.dtype, DIR == kGmmForward ? g.x : g.dy, p.con, g.rows, 1, p.box))
    return cudaErrorInvalidValue;
  const int smem = kFixed + p.stages * p.stage_bytes + p.part_bytes;
  auto launch = [&](auto kernel, SmemOptIn& opt_in) {
    cudaError_t st = opt_in.set(kernel, 227 * 1024);
    if (st != cudaSuccess) return st;
    return launch_overlapped(kernel, static_cast<unsigned>(tiles * p.splits), threads, smem,
                             p.splits, s, mw, mx, p);
  };
  static SmemOptIn one, many;
  return seg ? launch(grouped_small_kernel<T, DIR, LORA, true>, many)
             : launch(grouped_small_kernel<T, DIR, LORA, false>, one);
}

template <typename T>
cudaError_t launch_small_type(const GroupedArgs& g, const LoraTerm* lora, int num_sms,
                              cudaStream_t s) {
  // Register blocks of the adapter term: one step (ranks up to 16) of four adapters, or two
  // steps of two.
  if (lora != nullptr)
    return lora->steps == 1 ? launch_small<T, kGmmForward, 1>(g, lora, num_sms, s)
                            : launch_small<T, kGmmForward, 2>(g, lora, num_sms, s);
  if (g.dir == kGmmForward) return launch_small<T, kGmmForward, 0>(g, nullptr, num_sms, s);
  return launch_small<T, kGmmGradInput, 0>(g, nullptr, num_sms, s);
}

}  // namespace

cudaError_t launch_grouped_small(const GroupedArgs& g, const LoraTerm* lora, int num_sms,
                                 cudaStream_t s) {
  if (g.dir == kGmmGradWeight) return cudaErrorInvalidValue;
  if (g.dtype == kDtF16) return launch_small_type<__half>(g, lora, num_sms, s);
  if (g.dtype == kDtBF16) return launch_small_type<__nv_bfloat16>(g, lora, num_sms, s);
  return cudaErrorInvalidValue;
}

}  // namespace moe

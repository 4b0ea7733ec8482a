// The expert products on the 5th-generation tensor cores: 256 x 256 tiles by CTA pairs.
//
// All three products are one kernel that differs in which operand dimension lies contiguous
// in memory, so no operand is ever transposed in memory:
//                 M (256 per tile)      N (<= 256 per tile)   contraction
//   forward       W[e] rows n, K-major  x rows, K-major       K
//   grad_input    W[e] cols k, MN-major dy rows, K-major      N
//   grad_weight   dy cols n, MN-major   x cols k, MN-major    rows of e
// The ragged dimension (the rows of an expert) is the MMA's N in the first two: an expert's
// rows are cut into ceil(rows / 256) tiles of equal height rounded up to 16, so a tile
// computes at most 15 rows too many instead of up to 255; rows are columns of the
// accumulator, so what a tile reads beyond its expert only reaches columns that are not
// stored.  In grad_weight the ragged dimension is summed over: whole 16-row steps come from
// dy and x, and the last rows % 16 rows of each expert from a zero-padded copy
// (tail_kernel), because a neighbour's row in the step would be added (and a zero in only
// one operand would not stop its infinities).
//
// Per CTA: warp 0 TMA producer, warp 1 MMA issuer (leader CTA), warps 2..9 epilogue.  Each
// CTA stages its 128 of the 256 M entries and half of the N entries of a 64-deep slice
// (32 KB, six stages); two 256-column accumulators, so the epilogue of a tile overlaps the
// MMAs of the next.  Bound: the tensor pipe; a slice of the pair is 512 cycles of MMA
// for 64 KB from L2.  Measured in a replayed graph of ten calls: 131072 rows by a power law over
// 64 experts of [768, 2048], bf16, forward 337 us (1.22 PFLOP/s), both gradients 745 us (1.11); 8192
// rows over 8 experts of [4096, 14336], fp16, 769 us (1.25).  In long loops of calls the power
// limit takes 15 to 20%: 394, 866 and 892 us.
//
// Contractions of more than one segment (kSegment slices: grad_weight of more than 16384 rows of
// an expert, mostly) are added up in tensor memory: after each segment but the last the epilogue
// warps add the accumulator to a sum in the other accumulator's columns and leave the rounding
// error of that addition in the accumulator, where the next segment starts from it.  So the
// length of the sum does not show in the result, and no wait is longer than a segment.  Such a
// tile has both accumulators, and the tile after it waits for its epilogue.
//
// The adapter projection is the forward product of one group, and its adapter term more
// slices of the same accumulator where sixteen adjacent rows (counted from the tile's first)
// follow one adapter: B_a as the M operand, the rows' parts (grouped_lora.cuh) as the N
// operand, on the accumulator columns of the run of such rows.  Warp 10 finds the runs.  The
// rows in between -- sixteen that follow several adapters, fp16 rows scaled against overflow
// -- get it in the epilogue, which mma.sync makes slow beside tcgen05 (all of it there: 33 us
// a tile of 224 rows, rank 64, beside 24 us of MMA).
#include <algorithm>
#include <mutex>

#include "grouped_lora.cuh"

namespace moe {

namespace {

constexpr int kBK = 64;
constexpr int kTileM = 256;
constexpr int kTileN = 256;
constexpr int kStages = 6;
constexpr int kABytes = 128 * kBK * 2;
constexpr int kBBytes = 128 * kBK * 2;
constexpr int kBox = 64 * kBK * 2;       // one 64 x 64 box of a 16-bit operand
constexpr int kThreads = 320;
constexpr int kLoraThreads = 352;        // warp 10: the tile's runs of rows
constexpr int kEpiWarps = 8;
constexpr int kStageRow = 64;            // bytes of one staged output row (32 elements)
constexpr int kEpiBytes = 4 * 8 * kStageRow;  // per warp: four blocks of 8 rows
constexpr int kRaster = 8;               // M-fastest runs of this many tiles (L2 reuse)
constexpr int kTailRows = 16;
constexpr int kSmem = 1024 + kStages * (kABytes + kBBytes) + kEpiWarps * kEpiBytes + 384 +
                      kMaxExperts * 8 + (kMaxExperts + 1) * 4;
static_assert(kSmem <= 227 * 1024, "shared memory of the pair kernel");

struct PairParams {
  const int32_t* offsets;
  int rows, E;
  int m_dim;      // extent of the M side (features; grad_weight: N)
  int n_dim;      // grad_weight: K
  int con;        // contraction length (not grad_weight)
  int m_tiles, n_tiles;
  int tile_rows;   // most rows of a tile (forward, grad_input)
  void* out;
  int64_t ldo;
  LoraTerm lora;
  int rank_blocks;  // of 64
  int* error;
  int test_stall;
};

struct PairTile {
  int e;
  int m0;          // first entry of the M side
  int n0;          // first row (forward, grad_input) or column of x (grad_weight)
  int n;           // valid N entries
  int nt;          // MMA N
  int blocks;      // 64-deep slices
  int begin, cnt;  // grad_weight: the expert's rows
};

// Position `local` of an a x b grid walked in runs of kRaster of the first coordinate: the
// 74 tiles that run at a time then share few operand slices of either side.
__device__ __forceinline__ void raster(int local, int a, int b, int& i, int& j) {
  const int run = local / (kRaster * b), in = local - run * kRaster * b;
  const int w = min(kRaster, a - run * kRaster);
  j = in / w;
  i = run * kRaster + in - j * w;
}

template <int DIR>
__device__ __forceinline__ PairTile pair_tile(int L, const GroupTable& g, const PairParams& p) {
  PairTile t;
  if (DIR == kGmmGradWeight) {
    const int per = p.m_tiles * p.n_tiles;
    t.e = L / per;
    int i, j;
    raster(L - t.e * per, p.m_tiles, p.n_tiles, i, j);
    t.m0 = i * kTileM;
    t.n0 = j * kTileN;
    t.n = min(kTileN, p.n_dim - t.n0);
    t.nt = kTileN;
    t.begin = g.rows[t.e].x;
    t.cnt = g.rows[t.e].y - t.begin;
    const int rem = t.cnt % kBK;
    t.blocks = t.cnt / kBK + (rem >= kTailRows ? 1 : 0) + (rem % kTailRows ? 1 : 0);
  } else {
    t.e = find_group(g.tiles, p.E, p.m_tiles, L);
    const int nt = g.tiles[t.e + 1] - g.tiles[t.e];
    int i, j;
    raster(L - g.tiles[t.e] * p.m_tiles, nt, p.m_tiles, i, j);
    const int2 r = g.rows[t.e];
    const int h = ((r.y - r.x + nt - 1) / nt + 15) & ~15;
    t.m0 = j * kTileM;
    t.n0 = r.x + i * h;
    t.n = min(h, r.y - t.n0);
    t.nt = (t.n + 15) & ~15;
    t.blocks = (p.con + kBK - 1) / kBK;
    t.begin = t.cnt = 0;
  }
  return t;
}

// Tile of turn `i`: rounds of one tile per pair, walked forth and back.  (Tiles of grad_weight
// cost what their expert has rows; walked forth only, the first pairs got the dearer tile of
// every round: 366 us against 337 for 16384 tokens over 64 experts by a power law, [768, 2048].
// Claiming tiles from a counter took 349 us, and 301 against 235 for a short batch, whose tiles
// are two slices long.)
__device__ __forceinline__ int turn_tile(int i, int pair, int npairs) {
  return i * npairs + ((i & 1) ? npairs - 1 - pair : pair);
}

// Adapter projection: what a group of sixteen rows follows -- an adapter, none (-1), several
// (kMixedCode; also rows scaled against overflow) or, past the last row, anything.
constexpr int kMixedCode = -2;
constexpr int kAnyCode = -3;
__device__ __forceinline__ int join_codes(int a, int b) {
  return a == b || b == kAnyCode ? a : a == kAnyCode ? b : kMixedCode;
}
// Runs of groups that follow the same adapter, in order.
struct RunWalk {
  const volatile int* code_of;
  int groups, at = 0;
  int code = -1, begin = 0, count = 0;
  __device__ RunWalk(const volatile int* c, int n) : code_of(c), groups(n) {}
  __device__ __forceinline__ bool next() {
    while (at < groups && code_of[at] < 0) ++at;
    if (at >= groups) return false;
    begin = at;
    code = code_of[at];
    while (at < groups && code_of[at] == code) ++at;
    count = at - begin;
    return true;
  }
};
__device__ __forceinline__ void fence_proxy_async_all() {
  asm volatile("fence.proxy.async;" ::: "memory");
}

// Adds the 32 lanes x 32 columns of an accumulator at `acc` to the sum at `sum` and leaves the
// rounding error of each addition (exact, by the six operations of a two-sum) in the
// accumulator; a sum that is not finite leaves none.  After the last segment the whole sum goes
// to the accumulator.
__device__ __forceinline__ void add_segment(uint32_t acc, uint32_t sum, bool first, bool last) {
#pragma unroll
  for (int h = 0; h < 2; ++h, acc += 16u << 16, sum += 16u << 16) {
    float a[16], s[16];
    tmem_ld_frag4(acc, a);
    if (!first) tmem_ld_frag4(sum, s);
    tmem_ld_wait();
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      if (first) {
        s[j] = a[j];
        a[j] = 0.f;
      } else {
        const float t = __fadd_rn(s[j], a[j]), u = __fsub_rn(t, s[j]);
        const float e = __fadd_rn(__fsub_rn(s[j], __fsub_rn(t, u)), __fsub_rn(a[j], u));
        s[j] = t;
        a[j] = last ? t : isfinite(t) ? e : 0.f;
      }
    }
    if (!last) tmem_st_frag4(sum, s);
    tmem_st_frag4(acc, a);
  }
}

// MMA steps of 16 in slice `b` of the tile.
template <int DIR>
__device__ __forceinline__ int block_steps(const PairTile& t, int b) {
  if (DIR != kGmmGradWeight) return kBK / 16;
  const int left = t.cnt - b * kBK;
  if (left >= kBK) return kBK / 16;
  // Behind the full slices: the whole steps of the remainder, then the padded tail.
  return left >= kTailRows && b == t.cnt / kBK ? left / kTailRows : 1;
}
// True for the slice that holds the padded tail of the expert.
__device__ __forceinline__ bool is_tail(const PairTile& t, int b) {
  return t.cnt % kTailRows != 0 && b == t.blocks - 1;
}

// LORA: 16-entry steps of the rank per register block of the adapter term, 0 without one.
// SEG: contractions may have more than one segment.
template <typename T, int DIR, int LORA, bool SEG>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(LORA > 0 ? kLoraThreads : kThreads, 1)
grouped_pair_kernel(const __grid_constant__ CUtensorMap map_a,
                    const __grid_constant__ CUtensorMap map_b,
                    const __grid_constant__ CUtensorMap map_at,
                    const __grid_constant__ CUtensorMap map_bt, const PairParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* sA = smem;
  uint8_t* sB = smem + kStages * kABytes;
  uint8_t* stage_out = sB + kStages * kBBytes;
  uint64_t* bars = reinterpret_cast<uint64_t*>(stage_out + kEpiWarps * kEpiBytes);
  uint64_t* full = bars;
  uint64_t* empty = bars + kStages;
  uint64_t* tfull = bars + 2 * kStages;
  uint64_t* tempty = tfull + 2;
  uint64_t* done = tempty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  // Adapter projection: what each 16-row group of a tile follows, for the tile of turn i in
  // slot i % 2.
  uint64_t* cfull = done + 2;
  uint64_t* cempty = cfull + 2;
  volatile int* codes = reinterpret_cast<volatile int*>(cempty + 2);  // [2][16]
  static_assert((2 * kStages + 10) * 8 + 2 * 16 * 4 <= 384, "barrier block");
  GroupTable table;
  table.rows = reinterpret_cast<int2*>(bars + 48);
  table.tiles = reinterpret_cast<int*>(table.rows + kMaxExperts);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&tfull[a], 1);
      mbar_init(&tempty[a], 2 * kEpiWarps);
      mbar_init(&cfull[a], 1);
      mbar_init(&cempty[a], kEpiWarps + (leader ? 2 : 1));  // and the producer, the MMA warp
    }
    mbar_init(done, 1);
    *abort_flag = 0;
    fence_mbarrier_init();
    tma_prefetch_desc(&map_a);
    tma_prefetch_desc(&map_b);
  }
  if (warp == 1) {
    tmem_alloc_pair(tmem_slot, 2 * kTileN);
    tmem_relinquish_pair();
  }
  // The adapter projection's inputs were ready before the launch in front of it started;
  // its parts are awaited by the epilogue.
  if (LORA == 0) pdl_wait();
  if (warp == 2) build_group_table(p.offsets, p.E, p.rows, p.tile_rows, table);
  tc_fence_before();
  __syncthreads();
  cluster_sync();  // both CTAs' barriers are initialised before any remote signal
  tc_fence_after();
  pdl_launch_dependents();
  const uint32_t tmem_base = *tmem_slot;
  const int total =
      DIR == kGmmGradWeight ? p.E * p.m_tiles * p.n_tiles : table.tiles[p.E] * p.m_tiles;
  const int pair = blockIdx.x >> 1, npairs = gridDim.x >> 1;
  constexpr bool kAMn = DIR != kGmmForward;
  constexpr bool kBMn = DIR == kGmmGradWeight;

  if (warp == 0) {
    // ------------------------------------------------------------- TMA producer
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      for (int i = 0;; ++i) {
        const int L = turn_tile(i, pair, npairs);
        if (L >= total || *abort_flag || p.test_stall) break;
        const PairTile t = pair_tile<DIR>(L, table, p);
        const int a0 = t.m0 + static_cast<int>(rank) * 128;
        // Rows of this CTA's half of the MMA's N, in boxes of 64.
        const int half = t.nt / 2;
        const int b0 = t.n0 + static_cast<int>(rank) * half;
        const int b_boxes = DIR == kGmmGradWeight ? 2 : (half + 63) / 64;
        for (int b = 0; b < t.blocks; ++b) {
          if (!mbar_wait(&empty[stage], phase ^ 1)) {
            report_error(p.error, kErrTimeoutProducer);
            *abort_flag = 1;
            break;
          }
          const bool tail = DIR == kGmmGradWeight && is_tail(t, b);
          const uint32_t bar = mapa_shared(smem_u32(&full[stage]), 0);
          if (leader)
            mbar_arrive_expect_tx(&full[stage], tail ? 2 * 4 * kTailRows * 128
                                                     : 2 * (kABytes + b_boxes * kBox));
          uint8_t* da = sA + stage * kABytes;
          uint8_t* db = sB + stage * kBBytes;
          const int c = b * kBK;
          if (DIR == kGmmForward) {
            tma_load_3d_pair(da, &map_a, bar, c, a0, t.e);
          } else if (DIR == kGmmGradInput) {
            tma_load_3d_pair(da, &map_a, bar, a0, c, t.e);
            tma_load_3d_pair(da + kBox, &map_a, bar, a0 + 64, c, t.e);
          } else {
            const CUtensorMap* m = tail ? &map_at : &map_a;
            const int r = tail ? t.e * kTailRows : t.begin + c;
            tma_load_3d_pair(da, m, bar, a0, r, 0);
            tma_load_3d_pair(da + kBox, m, bar, a0 + 64, r, 0);
          }
          if (DIR == kGmmGradWeight) {
            const CUtensorMap* m = tail ? &map_bt : &map_b;
            const int r = tail ? t.e * kTailRows : t.begin + c;
            tma_load_3d_pair(db, m, bar, b0, r, 0);
            tma_load_3d_pair(db + kBox, m, bar, b0 + 64, r, 0);
          } else {
            for (int j = 0; j < b_boxes; ++j)
              tma_load_3d_pair(db + j * kBox, &map_b, bar, c, b0 + j * 64, 0);
          }
          if (++stage == kStages) { stage = 0; phase ^= 1; }
        }
        if (LORA > 0) {
          if (i == 0) {  // the parts come from the launch before
            pdl_wait();
            fence_proxy_async_all();
          }
          if (!mbar_wait(&cfull[i & 1], (i >> 1) & 1)) {
            report_error(p.error, kErrTimeoutProducer);
            *abort_flag = 1;
          }
          RunWalk w(codes + (i & 1) * 16, (t.n + 15) / 16);
          while (!*abort_flag && w.next()) {
            const int rows_half = w.count * 8;  // this CTA's half of the run's rows
            const int boxes = (rows_half + 63) / 64;
            const int r0 = t.n0 + w.begin * 16 + static_cast<int>(rank) * rows_half;
            for (int b = 0; b < 2 * p.rank_blocks; ++b) {
              if (!mbar_wait(&empty[stage], phase ^ 1)) {
                report_error(p.error, kErrTimeoutProducer);
                *abort_flag = 1;
                break;
              }
              const uint32_t bar = mapa_shared(smem_u32(&full[stage]), 0);
              if (leader) mbar_arrive_expect_tx(&full[stage], 2 * (kABytes + boxes * kBox));
              tma_load_3d_pair(sA + stage * kABytes, &map_at, bar, (b >> 1) * kBK, a0, w.code);
              for (int j = 0; j < boxes; ++j)
                tma_load_3d_pair(sB + stage * kBBytes + j * kBox, &map_bt, bar, (b >> 1) * kBK,
                                 r0 + j * 64, b & 1);
              if (++stage == kStages) { stage = 0; phase ^= 1; }
            }
          }
          mbar_arrive(&cempty[i & 1]);
        }
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------- MMA issuer (leader CTA only)
    if (lane == 0 && leader) {
      int stage = 0;
      uint32_t phase = 0;
      uint32_t fills = 0;   // bit a: parity of accumulator a's next fill
      bool both = false;    // the tile before has its sum in the other accumulator
      auto drained = [&](int a) { return mbar_wait(&tempty[a], (fills >> a & 1) ^ 1); };
      bool complete = false;
      for (int i = 0;; ++i) {
        const int L = turn_tile(i, pair, npairs);
        complete = L >= total;
        if (complete || *abort_flag) break;
        const PairTile t = pair_tile<DIR>(L, table, p);
        const uint32_t idesc = idesc_f16(TcFormat<T>::kId, kTileM, t.nt) |
                               (kAMn ? kIdescAMn : 0) | (kBMn ? kIdescBMn : 0);
        const int acc = i & 1;
        if (!drained(acc) || (SEG && both && !drained(acc ^ 1))) {
          report_error(p.error, kErrTimeoutMma);
          *abort_flag = 1;
          break;
        }
        tc_fence_after();
        const uint32_t d = tmem_base + acc * kTileN;
        bool ok = true;
        both = t.blocks > kSegment;
        for (int b = 0; b < t.blocks; ++b) {
          if (SEG && b != 0 && b % kSegment == 0) {  // a segment is complete: the epilogue takes it
            tc_commit_pair(&tfull[acc], 0x3);
            fills ^= 1u << acc;
            if (LORA > 0 && i == 0) pdl_wait();  // the epilogue does
            ok = drained(acc);
            tc_fence_after();
          }
          if (!ok || !mbar_wait(&full[stage], phase)) {
            report_error(p.error, kErrTimeoutMma);
            *abort_flag = 1;
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t a = smem_u32(sA + stage * kABytes);
          const uint32_t bb = smem_u32(sB + stage * kBBytes);
          const int steps = block_steps<DIR>(t, b);
#pragma unroll
          for (int k = 0; k < kBK / 16; ++k) {
            if (k >= steps) break;
            // 16 contraction entries on: 32 bytes along a K-major row, 16 rows of 128
            // bytes of an MN-major block.
            const uint64_t ad = kAMn ? smem_desc_mn_sw128(a + k * 2048, kBox)
                                     : smem_desc_k_sw128(a + k * 32);
            const uint64_t bd = kBMn ? smem_desc_mn_sw128(bb + k * 2048, kBox)
                                     : smem_desc_k_sw128(bb + k * 32);
            tc_mma_f16_pair(d, ad, bd, idesc, (b | k) != 0 ? 1u : 0u);
          }
          tc_commit_pair(&empty[stage], 0x3);
          if (++stage == kStages) { stage = 0; phase ^= 1; }
        }
        if (LORA > 0 && ok) {
          // What the rows follow comes from the launch before, which may take longer than any
          // wait on a barrier counts: that launch is waited for first.
          if (i == 0) pdl_wait();
          ok = mbar_wait(&cfull[i & 1], (i >> 1) & 1);
          RunWalk w(codes + (i & 1) * 16, (t.n + 15) / 16);
          while (ok && w.next()) {
            const uint32_t run_desc = idesc_f16(TcFormat<T>::kId, kTileM, w.count * 16);
            for (int b = 0; b < 2 * p.rank_blocks && ok; ++b) {
              ok = mbar_wait(&full[stage], phase);
              if (!ok) break;
              tc_fence_after();
              const uint32_t a = smem_u32(sA + stage * kABytes);
              const uint32_t bb = smem_u32(sB + stage * kBBytes);
              const int left = p.lora.rank - (b >> 1) * kBK;
#pragma unroll
              for (int k = 0; k < kBK / 16; ++k) {
                if (k * 16 >= left) break;
                tc_mma_f16_pair(d + w.begin * 16, smem_desc_k_sw128(a + k * 32),
                                smem_desc_k_sw128(bb + k * 32), run_desc, 1u);
              }
              tc_commit_pair(&empty[stage], 0x3);
              if (++stage == kStages) { stage = 0; phase ^= 1; }
            }
          }
          mbar_arrive(&cempty[i & 1]);
          if (!ok) {
            report_error(p.error, kErrTimeoutMma);
            *abort_flag = 1;
          }
        }
        if (!ok) break;
        tc_commit_pair(&tfull[acc], 0x3);
        fills ^= 1u << acc;
      }
      tc_commit_pair(done, 0x1);
      mbar_wait(done, 0);
      // (Copies into either CTA count on these barriers.)
      if (!complete) drain_ring(full, kStages, stage, phase);
    }
  } else if (LORA > 0 && warp == 2 + kEpiWarps) {
    // ------------------------------------- what the tile's rows follow (both CTAs)
    pdl_wait();
    for (int i = 0;; ++i) {
      const int L = turn_tile(i, pair, npairs);
      if (L >= total || warp_stopped(abort_flag)) break;
      const PairTile t = pair_tile<DIR>(L, table, p);
      if (!warp_wait(&cempty[i & 1], ((i >> 1) & 1) ^ 1)) {
        report_error(p.error, kErrTimeoutProducer);
        *abort_flag = 1;
        break;
      }
      // Eight rows a lane, then the two lanes of a group.
      int code = kAnyCode;
      for (int k = 0; k < 8; ++k) {
        const int r = lane * 8 + k;
        code = join_codes(code, r < t.n ? p.lora.row_code[t.n0 + r] : kAnyCode);
      }
      code = join_codes(code, __shfl_xor_sync(0xffffffffu, code, 1));
      if (code >= kLoraScaled) code = kMixedCode;
      if ((lane & 1) == 0) codes[(i & 1) * 16 + lane / 2] = code;
      __syncwarp();
      if (lane == 0) mbar_arrive(&cfull[i & 1]);
    }
  } else {
    // ----------------------------------------------------- epilogue (both CTAs)
    const int q = warp & 3;               // TMEM lane quarter of this warp
    const int first = warp < 6 ? 0 : 32;  // its 32-column chunks: every other one
    uint8_t* buf = stage_out + (warp - 2) * kEpiBytes;
    // stmatrix row addresses: lane 8i + t is row t of block i; 16-byte granules are XORed
    // with the row so that neither the blocks nor the 16-byte reads conflict.
    const int st_row = lane & 7, st_blk = lane >> 3;
    const uint32_t st_addr =
        smem_u32(buf) + st_row * kStageRow + ((st_blk ^ ((st_row >> 1) & 3)) << 4);
    const int rd_row = lane >> 2, rd_blk = lane & 3;
    const uint8_t* rd_ptr = buf + rd_row * kStageRow + ((rd_blk ^ ((rd_row >> 1) & 3)) << 4);
    T* out = static_cast<T*>(p.out);
    if (LORA > 0) pdl_wait();
    uint32_t fills = 0;  // as the MMA warp's
    for (int i = 0;; ++i) {
      const int L = turn_tile(i, pair, npairs);
      if (L >= total || warp_stopped(abort_flag)) break;
      const PairTile t = pair_tile<DIR>(L, table, p);
      const int acc = i & 1, segments = SEG ? segments_of(t.blocks) : 1;
      const uint32_t taddr =
          tmem_base + (static_cast<uint32_t>(q * 32) << 16) + acc * kTileN;
      const uint32_t tsum = taddr + (acc ? -kTileN : kTileN);  // sum of the segments before
      bool ok = true;
      for (int seg = 0; ok && seg < segments; ++seg) {
        ok = warp_wait(&tfull[acc], fills >> acc & 1);
        fills ^= 1u << acc;
        tc_fence_after();
        if (!ok || segments == 1) break;
        for (int c = first; c < t.n; c += 64)
          add_segment(taddr + c, tsum + c, seg == 0, seg == segments - 1);
        tmem_st_wait();
        if (seg == segments - 1) break;
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(mapa_shared(smem_u32(&tempty[acc]), 0));
      }
      if (!ok) {
        report_error(p.error, kErrTimeoutEpilogue);
        *abort_flag = 1;
        break;
      }
      const int m = t.m0 + static_cast<int>(rank) * 128 + q * 32;  // first M entry of the warp
      const bool zero = DIR == kGmmGradWeight && t.cnt == 0;  // an expert without rows
      auto release = [&] {  // this warp has read the accumulator
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(mapa_shared(smem_u32(&tempty[acc]), 0));
      };
      auto fetch = [&](int c, float (&lo)[16], float (&hi)[16]) {
        tmem_ld_frag4(taddr + c, lo);
        tmem_ld_frag4(taddr + (16u << 16) + c, hi);
      };
      // Stores 32 columns of the accumulator, c .. c + 31: four 8 x 32 blocks go through the
      // warp's staging memory and leave as 16-byte pieces of 64-byte rows.  The four go
      // together, so their latencies overlap.
      auto store = [&](int c, float (&lo)[16], float (&hi)[16]) {
        __syncwarp();  // the staged blocks before have been read
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (DIR == kGmmGradWeight) {
            // Eight M rows (block j of the 32) x 32 columns.
            const float(&v)[16] = j < 2 ? lo : hi;
            const int o = (j & 1) * 2;
            stmatrix4(st_addr + j * 8 * kStageRow, pack2<T>(v[o], v[o + 1]),
                      pack2<T>(v[4 + o], v[5 + o]), pack2<T>(v[8 + o], v[9 + o]),
                      pack2<T>(v[12 + o], v[13 + o]));
          } else {
            // Eight rows of the output (accumulator columns) x 32 features, transposed.
            stmatrix4_t(st_addr + j * 8 * kStageRow, pack2<T>(lo[4 * j], lo[4 * j + 1]),
                        pack2<T>(lo[4 * j + 2], lo[4 * j + 3]), pack2<T>(hi[4 * j], hi[4 * j + 1]),
                        pack2<T>(hi[4 * j + 2], hi[4 * j + 3]));
          }
        }
        __syncwarp();
        uint4 w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
          w[j] = *reinterpret_cast<const uint4*>(rd_ptr + j * 8 * kStageRow);
        if (DIR == kGmmGradWeight) {
          const int row = m + rd_row, col = c + 8 * rd_blk;
          T* dst = out + (static_cast<int64_t>(t.e) * p.m_dim + row) * p.ldo + t.n0 + col;
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (row + 8 * j < p.m_dim && col < t.n)
              *reinterpret_cast<uint4*>(dst + 8 * j * p.ldo) = w[j];
        } else {
          const int row = c + rd_row, col = m + 8 * rd_blk;
          T* dst = out + static_cast<int64_t>(t.n0 + row) * p.ldo + col;
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (row + 8 * j < t.n && col < p.m_dim)
              *reinterpret_cast<uint4*>(dst + 8 * j * p.ldo) = w[j];
        }
      };
      if constexpr (LORA > 0) {
        LoraFrags<LORA> frags;  // of this tile's features
        if (!warp_wait(&cfull[i & 1], (i >> 1) & 1)) {
          report_error(p.error, kErrTimeoutEpilogue);
          *abort_flag = 1;
          break;
        }
        for (int c = first; c < t.n; c += 64) {
          const volatile int* code = codes + (i & 1) * 16 + c / 16;
          const bool mixed0 = code[0] == kMixedCode, mixed1 = code[1] == kMixedCode;
          // The rows' parts are fetched ahead of the accumulators: one trip to L2 a chunk
          // instead of one a row block.
          int ads = -1;
          uint4 parts[4][LORA];
          if (mixed0 || mixed1) {
            if (c + lane < t.n) {
              const int rc = p.lora.row_code[t.n0 + c + lane];
              ads = rc < 0 ? -1 : rc & (kLoraScaled - 1);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int row = c + 8 * j + (lane >> 2);
              lora_rows<LORA>(p.lora, p.rows, t.n0 + row, row < t.n, 0, parts[j]);
            }
          }
          float lo[16], hi[16];
          fetch(c, lo, hi);
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (j < 2 ? !mixed0 : !mixed1) continue;
            float dl[4], dh[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) { dl[k] = lo[4 * j + k]; dh[k] = hi[4 * j + k]; }
            lora_add<T, LORA>(p.lora, p.rows, __shfl_sync(0xffffffffu, ads, 8 * j + (lane >> 2)),
                              t.n0 + c + 8 * j + (lane >> 2), m, p.m_dim, parts[j], frags, dl, dh);
#pragma unroll
            for (int k = 0; k < 4; ++k) { lo[4 * j + k] = dl[k]; hi[4 * j + k] = dh[k]; }
          }
          store(c, lo, hi);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&cempty[i & 1]);
        release();
      } else {
        // The next columns are on their way from tensor memory while these are stored, and
        // the accumulator goes back before the last ones are.
        float lo[16] = {}, hi[16] = {}, lo2[16] = {}, hi2[16] = {};
        int c = first;
        if (c < t.n && !zero) fetch(c, lo, hi);
        tmem_ld_wait();
        if (c >= t.n) release();
        while (c < t.n) {
          if (c + 64 < t.n) {
            if (!zero) fetch(c + 64, lo2, hi2);
          } else {
            release();
          }
          store(c, lo, hi);
          c += 64;
          if (c >= t.n) break;
          tmem_ld_wait();
          if (c + 64 < t.n) {
            if (!zero) fetch(c + 64, lo, hi);
          } else {
            release();
          }
          store(c, lo2, hi2);
          c += 64;
          tmem_ld_wait();
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  cluster_sync();  // no CTA leaves while its peer may still signal it or read its smem
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, 2 * kTileN);
  }
}

// The last cnt % 16 rows of each expert's dy and x, padded with zero rows to 16, as
// [E][16][N] and [E][16][K] (16-byte vectors; N and K are multiples of 8).
__global__ void __launch_bounds__(256)
tail_kernel(const int32_t* __restrict__ offsets, int rows, const uint4* __restrict__ dy, int nv,
            const uint4* __restrict__ x, int kv, uint4* __restrict__ ty, uint4* __restrict__ tx) {
  pdl_wait();
  pdl_launch_dependents();
  const int e = blockIdx.y;
  const int begin = min(max(__ldg(offsets + e), 0), rows);
  const int end = max(min(max(__ldg(offsets + e + 1), 0), rows), begin);
  const int rem = (end - begin) % kTailRows, r0 = end - rem;
  if (rem == 0) return;  // no tail slice reads this expert's part
  const int per = nv + kv;
  for (int i = blockIdx.x * 256 + threadIdx.x; i < kTailRows * per; i += gridDim.x * 256) {
    const int r = i / per, c = i - r * per;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (c < nv) {
      if (r < rem) v = dy[static_cast<int64_t>(r0 + r) * nv + c];
      ty[(static_cast<int64_t>(e) * kTailRows + r) * nv + c] = v;
    } else {
      if (r < rem) v = x[static_cast<int64_t>(r0 + r) * kv + c - nv];
      tx[(static_cast<int64_t>(e) * kTailRows + r) * kv + c - nv] = v;
    }
  }
}

using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                                   const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                   const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                   CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_fn() {
  static EncodeTiledFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* q = nullptr;
    cudaDriverEntryPointQueryResult r;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &q, cudaEnableDefault, &r) ==
            cudaSuccess &&
        r == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiledFn>(q);
  });
  return fn;
}

size_t tail_bytes(int64_t E, int64_t width) {
  return (static_cast<size_t>(E) * kTailRows * static_cast<size_t>(width) * 2 + 255) & ~size_t{255};
}

// Tile height for one group of `rows`: the tiles run in rounds of one per SM pair, and a
// round that is nearly empty costs a whole one, so the height (a multiple of 16) is the one
// with the shortest rounds x slice time.  A slice takes 2 h cycles of MMA or, below about
// 215 rows, the (16 KB + 64 h) bytes a CTA reads from L2 at some 70 a cycle.  (4001 rows,
// 4096 features: 224 instead of 256, four rounds of 224 rows instead of 3.5 that cost four.)
int tile_rows_one_group(int64_t rows, int m_tiles, int pairs) {
  int best = kTileN;
  double best_cost = 1e300;
  for (int h = kTileN; h >= 128; h -= 16) {
    const int64_t tiles = (rows + h - 1) / h * m_tiles;
    const double cost = static_cast<double>((tiles + pairs - 1) / pairs) *
                        std::max(2.0 * h, (16384.0 + 64.0 * h) / 70.0);
    if (cost < best_cost) {
      best_cost = cost;
      best = h;
    }
  }
  return best;
}

template <typename T, int DIR, int LORA, bool SEG>
cudaError_t launch_pair(const GroupedArgs& g, const LoraTerm* lora, int num_sms, cudaStream_t s) {
  CUtensorMap ma, mb, mat, mbt;
  PairParams p{};
  p.offsets = g.offsets;
  p.rows = static_cast<int>(g.rows);
  p.E = g.E;
  p.out = g.out;
  p.error = g.error;
  p.test_stall = g.test_stall;
  if (LORA > 0) p.lora = *lora;
  bool ok;
  if (DIR == kGmmGradWeight) {
    auto* ty = static_cast<uint8_t*>(g.workspace);
    uint8_t* tx = ty + tail_bytes(g.E, g.N);
    p.m_dim = g.N;
    p.n_dim = g.K;
    p.ldo = g.K;
    p.n_tiles = (g.K + kTileN - 1) / kTileN;
    ok = grouped_map(&ma, g.dtype, g.dy, g.N, g.rows, 1, 64) &&
         grouped_map(&mb, g.dtype, g.x, g.K, g.rows, 1, 64) &&
         grouped_map(&mat, g.dtype, ty, g.N, static_cast<int64_t>(g.E) * kTailRows, 1, kTailRows) &&
         grouped_map(&mbt, g.dtype, tx, g.K, static_cast<int64_t>(g.E) * kTailRows, 1, kTailRows);
    if (!ok) return cudaErrorInvalidValue;
    const int vecs = kTailRows * (g.N + g.K) / 8;
    cudaError_t st = launch_dependent(pdl_enabled(), tail_kernel,
                                      dim3(std::min(32, (vecs + 255) / 256), g.E), dim3(256), 0, s, g.offsets,
                                      p.rows, static_cast<const uint4*>(g.dy), g.N / 8,
                                      static_cast<const uint4*>(g.x), g.K / 8,
                                      reinterpret_cast<uint4*>(ty), reinterpret_cast<uint4*>(tx));
    if (st != cudaSuccess) return st;
  } else {
    const int feat = DIR == kGmmForward ? g.N : g.K;
    p.m_dim = feat;
    p.con = DIR == kGmmForward ? g.K : g.N;
    p.ldo = feat;
    ok = grouped_map(&ma, g.dtype, g.w, g.K, g.N, g.E, DIR == kGmmForward ? 128 : 64) &&
         grouped_map(&mb, g.dtype, DIR == kGmmForward ? g.x : g.dy, p.con, g.rows, 1, 64);
    if (!ok) return cudaErrorInvalidValue;
    mat = ma;
    mbt = mb;
    if (LORA > 0) {
      p.rank_blocks = (lora->rank + kBK - 1) / kBK;
      if (!grouped_map(&mat, g.dtype, lora->b, lora->rank, g.N, lora->adapters, 128) ||
          !grouped_map(&mbt, g.dtype, lora->parts, lora->rank, g.rows, 2, 64))
        return cudaErrorInvalidValue;
    }
    p.tile_rows = kTileN;
    if (g.E == 1) p.tile_rows = tile_rows_one_group(g.rows, (feat + kTileM - 1) / kTileM, num_sms / 2);
  }
  p.m_tiles = (p.m_dim + kTileM - 1) / kTileM;
  const int64_t tiles =
          DIR == kGmmGradWeight
              ? static_cast<int64_t>(g.E) * p.m_tiles * p.n_tiles
              : (g.E == 1 ? (g.rows + p.tile_rows - 1) / p.tile_rows
                         : g.rows / p.tile_rows + std::min<int64_t>(g.rows, g.E)) *
                    p.m_tiles;
  static SmemOptIn opt_in;
  cudaError_t st = opt_in.set(grouped_pair_kernel<T, DIR, LORA, SEG>, kSmem);
  if (st != cudaSuccess) return st;
  const int64_t pairs = std::min<int64_t>(tiles, num_sms / 2);
  return launch_overlapped(grouped_pair_kernel<T, DIR, LORA, SEG>, static_cast<unsigned>(2 * pairs),
                           LORA > 0 ? kLoraThreads : kThreads, kSmem, 0, s, ma, mb, mat, mbt, p);
}

template <typename T, int DIR, int LORA>
cudaError_t launch_pair_seg(const GroupedArgs& g, const LoraTerm* lora, int num_sms,
                            cudaStream_t s) {
  // The rows of an expert are known on the device only.
  const int64_t con = DIR == kGmmForward ? g.K : DIR == kGmmGradInput ? g.N : g.rows;
  return con <= kSegment * kBK ? launch_pair<T, DIR, LORA, false>(g, lora, num_sms, s)
                               : launch_pair<T, DIR, LORA, true>(g, lora, num_sms, s);
}

template <typename T>
cudaError_t launch_pair_type(const GroupedArgs& g, const LoraTerm* lora, int num_sms,
                             cudaStream_t s) {
  // Ranks up to 16 keep one step in registers, larger ones blocks of four.
  if (lora != nullptr)
    return lora->steps == 1 ? launch_pair_seg<T, kGmmForward, 1>(g, lora, num_sms, s)
                            : launch_pair_seg<T, kGmmForward, 4>(g, lora, num_sms, s);
  if (g.dir == kGmmForward) return launch_pair_seg<T, kGmmForward, 0>(g, nullptr, num_sms, s);
  if (g.dir == kGmmGradInput) return launch_pair_seg<T, kGmmGradInput, 0>(g, nullptr, num_sms, s);
  return launch_pair_seg<T, kGmmGradWeight, 0>(g, nullptr, num_sms, s);
}

}  // namespace

bool grouped_map(CUtensorMap* m, int dtype, const void* ptr, int64_t dim0, int64_t dim1,
                 int64_t dim2, int box1) {
  EncodeTiledFn enc = encode_fn();
  if (enc == nullptr) return false;
  cuuint64_t dims[3] = {static_cast<cuuint64_t>(dim0), static_cast<cuuint64_t>(dim1),
                        static_cast<cuuint64_t>(dim2)};
  cuuint64_t strides[2] = {dims[0] * 2, dims[0] * dims[1] * 2};
  cuuint32_t box[3] = {kBK, static_cast<cuuint32_t>(box1), 1};
  cuuint32_t es[3] = {1, 1, 1};
  return enc(m, dtype == kDtBF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
             3, const_cast<void*>(ptr), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

size_t grouped_tc_workspace(int dtype, GroupedDir dir, int64_t N, int64_t K, int64_t E) {
  if (dir != kGmmGradWeight || dtype == kDtF32 || N % 8 != 0 || K % 8 != 0) return 0;
  return tail_bytes(E, N) + tail_bytes(E, K);
}

bool grouped_tc_supported(const GroupedArgs& g) {
  if (g.dtype != kDtF16 && g.dtype != kDtBF16) return false;
  if (g.N % 8 != 0 || g.K % 8 != 0) return false;
  auto aligned = [](const void* q) { return (reinterpret_cast<uintptr_t>(q) & 15) == 0; };
  // A direction's unused operand is NULL and so aligned.
  return aligned(g.x) && aligned(g.dy) && aligned(g.w) && aligned(g.out);
}

cudaError_t launch_grouped_pair(const GroupedArgs& g, const LoraTerm* lora, int num_sms,
                                cudaStream_t s) {
  if (g.dtype == kDtF16) return launch_pair_type<__half>(g, lora, num_sms, s);
  if (g.dtype == kDtBF16) return launch_pair_type<__nv_bfloat16>(g, lora, num_sms, s);
  return cudaErrorInvalidValue;
}

}  // namespace moe

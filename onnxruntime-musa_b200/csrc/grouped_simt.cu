// The expert products and the adapter projection on the FP32 pipes, for every size,
// alignment and float type; the 16-bit tensor-core kernels (grouped_tc.cu) take the
// operands that TMA can address, this file the rest and all of fp32 (TF32 would round
// the operands to 11 bits, 2^13 times the rounding of an fp32 result).
//
// Mathematics: one tile C[m, n] = sum_c A(m, c) B(n, c) per CTA, summed in ascending c in
// fp32, kFold entries at a time and then those sums, each of whose roundings starts the next kFold:
// one running sum rounds at the magnitude it has reached, and a grad_input over 10696 entries was
// off from float64 by 1.3e-6, relative, where a blocked product is off by 4.7e-7 and this one now
// by 4.1e-7; grad_weight of 2^25 equal rows was off by 1.7e-4 before the roundings were kept, and
// the number of rows shows in the result no more.  (Price: 735 -> 783 us
// for 4096 rows, 8 experts of [2048, 2048] fp32.  Four other placements of the folds -- shared
// memory, the end of the slice loop, its prologue again for each fold -- took 790 to 890.)
// The three directions differ only in where the contraction index lies:
//   forward      A = x rows  (c contiguous)   B = W[e][n, c]  (c contiguous)
//   grad_input   A = dy rows (c contiguous)   B = W[e][c, n]  (n contiguous)
//   grad_weight  A = dy[c, m] (m contiguous)  B = x[c, n]     (n contiguous), c = rows of e
// Bound: FFMA issue.  Each thread owns TM x TN sums, so a step of c costs TM + TN shared
// loads for TM * TN FMAs; the next slice is loaded to registers while the current one is
// multiplied (double-buffered shared memory, one barrier per slice).  A call with few tiles
// waits for memory instead, slice after slice; there the contraction is split over a cluster
// of up to four CTAs, whose partial sums meet in distributed shared memory: each owns some of
// the tile's rows and adds the parts in rank order.
#include <algorithm>

#include "grouped_tc.cuh"

namespace moe {
namespace {

constexpr int kThreads = 256;
constexpr int kFold = 512;  // contraction entries per running sum

struct SimtParams {
  const void* a;
  const void* b;
  void* out;
  const int32_t* offsets;
  int64_t rows;
  int N, K, E;
  int a_vec, b_vec;  // 4-element loads are aligned and rows are a multiple of 4 long
  int splits;        // cluster size along the contraction
  LoraTerm lora;
};

__device__ __forceinline__ int group_begin(const int32_t* off, int e, int rows) {
  const int v = off == nullptr ? 0 : __ldg(off + e);
  return min(max(v, 0), rows);
}
__device__ __forceinline__ int group_end(const int32_t* off, int e, int rows, int begin) {
  const int v = off == nullptr ? rows : __ldg(off + e + 1);
  return max(min(max(v, 0), rows), begin);
}

struct Tile {
  int e, index, begin, end;
};

// Tile `L` of the list that holds, expert by expert, ceil(rows_e / tile_rows) tiles;
// false when the list is shorter.  Called by all NT threads, each of kMaxExperts / NT experts.
template <int NT>
__device__ bool find_tile(const int32_t* off, int E, int rows, int tile_rows, int L, Tile* out) {
  constexpr int kPer = (kMaxExperts + NT - 1) / NT;
  __shared__ int s_warp[NT / 32];
  __shared__ Tile s_tile;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int begin[kPer], end[kPer], n[kPer], sum = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int e = threadIdx.x * kPer + i;
    begin[i] = end[i] = n[i] = 0;
    if (e < E) {
      begin[i] = group_begin(off, e, rows);
      end[i] = group_end(off, e, rows, begin[i]);
      n[i] = (end[i] - begin[i] + tile_rows - 1) / tile_rows;
    }
    sum += n[i];
  }
  int incl = sum;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, incl, d);
    if (lane >= d) incl += v;
  }
  if (lane == 31) s_warp[warp] = incl;
  if (threadIdx.x == 0) s_tile.e = -1;
  __syncthreads();
  int first = incl - sum;
  for (int w = 0; w < warp; ++w) first += s_warp[w];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    if (n[i] > 0 && L >= first && L < first + n[i]) {
      s_tile.e = threadIdx.x * kPer + i;
      s_tile.index = L - first;
      s_tile.begin = begin[i];
      s_tile.end = end[i];
    }
    first += n[i];
  }
  __syncthreads();
  *out = s_tile;
  return s_tile.e >= 0;
}

// Four consecutive elements p[0..3], the first `n` of them valid, as fp32.
template <typename T>
__device__ __forceinline__ float4 load4(const T* p, int n, int vec) {
  float v[4] = {0.f, 0.f, 0.f, 0.f};
  if (n >= 4 && vec) {
    if constexpr (sizeof(T) == 4) {
      return __ldg(reinterpret_cast<const float4*>(p));
    } else {
      const uint2 u = __ldg(reinterpret_cast<const uint2*>(p));
      const T* q = reinterpret_cast<const T*>(&u);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = to_f(q[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < n) v[i] = to_f(p[i]);
  }
  return make_float4(v[0], v[1], v[2], v[3]);
}

// One operand's slice: X rows x kDepth contraction entries into s[kDepth][X + pad].  CONTIG_C: element (i, c)
// at p[i * ld + c], else at p[c * ld + i]; i < ni and c < nc are valid.
template <typename T, int X, int kDepth, bool CONTIG_C, int NT>
struct Slice {
  static constexpr int kPitch = X + 4;
  static constexpr int kAll = X * kDepth / 4;
  static constexpr int kQuads = (kAll + NT - 1) / NT;
  float4 v[kQuads];

  __device__ __forceinline__ void load(const T* p, int64_t ld, int ni, int c0, int nc, int vec) {
#pragma unroll
    for (int j = 0; j < kQuads; ++j) {
      const int q = threadIdx.x + j * NT;
      if (kAll % NT != 0 && q >= kAll) continue;
      if (CONTIG_C) {
        const int i = q / (kDepth / 4), c = c0 + (q % (kDepth / 4)) * 4;
        v[j] = i < ni && c < nc ? load4<T>(p + i * ld + c, nc - c, vec)
                                : make_float4(0.f, 0.f, 0.f, 0.f);
      } else {
        const int c = c0 + q / (X / 4), i = (q % (X / 4)) * 4;
        v[j] = c < nc && i < ni ? load4<T>(p + c * ld + i, ni - i, vec)
                                : make_float4(0.f, 0.f, 0.f, 0.f);
      }
    }
  }
  __device__ __forceinline__ void store(float* s) const {
#pragma unroll
    for (int j = 0; j < kQuads; ++j) {
      const int q = threadIdx.x + j * NT;
      if (kAll % NT != 0 && q >= kAll) continue;
      if (CONTIG_C) {
        const int i = q / (kDepth / 4), c = (q % (kDepth / 4)) * 4;
        s[(c + 0) * kPitch + i] = v[j].x;
        s[(c + 1) * kPitch + i] = v[j].y;
        s[(c + 2) * kPitch + i] = v[j].z;
        s[(c + 3) * kPitch + i] = v[j].w;
      } else {
        const int c = q / (X / 4), i = (q % (X / 4)) * 4;
        *reinterpret_cast<float4*>(s + c * kPitch + i) = v[j];
      }
    }
  }
};

// Two fp32 values in a register pair, and the packed FMA on them (each half rounds as fmaf).
__device__ __forceinline__ uint64_t pair2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpair2(uint64_t v, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

// CTAs an SM: four of up to 64 rows, two of 128.  (64 x 64 tiles by 128 threads of 8 x 4 sums:
// by 256 of 4 x 4, which load twice as much of shared memory for an FMA, 2000 rows in 4 groups of
// [1111, 999] took 182 us in grad_input against 147; five CTAs an SM spill, 161.  128 x 128 by 128
// threads of 16 x 8 took 817 us against 792 at 4096 rows, [2048, 2048], and spills when split.)
__host__ __device__ constexpr int resident(int tm, int nt) { return tm * nt / 16 <= 64 ? 4 : 2; }

// CTA tile (TY TM) x (16 TN) of NT = 16 TY threads, TN a multiple of 4 and TM too or 1: thread
// (ty, tx) owns rows ty * 4 + 4 TY i + [0, 4) (TM = 1: row ty) and columns tx * 4 + 64 j + [0, 4).
// SPLIT: the contraction may be split over a cluster; LORA: with the adapter term.  (Both in
// every kernel spilled registers in the main loop of the 128 x 128 tiles: 10% of its time.)
template <typename T, int DIR, int TM, int TN, int NT, bool SPLIT, bool LORA>
__global__ void __launch_bounds__(NT, resident(TM, NT))
grouped_simt_kernel(const SimtParams p) {
  constexpr int TY = NT / 16, BM = TY * TM, BN = 16 * TN;
  constexpr int kDepth = BM <= 64 ? 32 : 16;
  constexpr bool kAC = DIR != kGmmGradWeight;  // contraction contiguous in A
  constexpr bool kBC = DIR == kGmmForward;
  using SA = Slice<T, BM, kDepth, kAC, NT>;
  using SB = Slice<T, BN, kDepth, kBC, NT>;
  constexpr int kSlice = kDepth * (SA::kPitch + SB::kPitch);
  __shared__ __align__(16) float operands[2 * kSlice];
  auto sa = [&](int buf) { return operands + buf * kSlice; };
  auto sb = [&](int buf) { return operands + buf * kSlice + kDepth * SA::kPitch; };

  pdl_wait();
  const int rows = static_cast<int>(p.rows);
  const T* a;
  const T* b;
  T* out;
  int64_t lda, ldb, ldo;
  int nm, nn, nc, row0 = 0;  // valid rows, columns and contraction length of this tile
  const int col0 = (DIR == kGmmGradWeight ? blockIdx.x : blockIdx.y) * BN;
  if (DIR == kGmmGradWeight) {
    const int e = blockIdx.z / p.splits, m0 = blockIdx.y * BM;
    const int begin = group_begin(p.offsets, e, rows);
    nc = group_end(p.offsets, e, rows, begin) - begin;
    lda = p.N;
    ldb = ldo = p.K;
    a = static_cast<const T*>(p.a) + begin * lda + m0;
    b = static_cast<const T*>(p.b) + begin * ldb + col0;
    out = static_cast<T*>(p.out) + (static_cast<int64_t>(e) * p.N + m0) * ldo + col0;
    nm = p.N - m0;
    nn = p.K - col0;
  } else {
    Tile t;
    if (!find_tile<NT>(p.offsets, p.E, rows, BM, blockIdx.x, &t)) return;
    const int feat = DIR == kGmmForward ? p.N : p.K;
    nc = DIR == kGmmForward ? p.K : p.N;
    row0 = t.begin + t.index * BM;
    lda = nc;
    ldb = p.K;
    ldo = feat;
    a = static_cast<const T*>(p.a) + row0 * lda;
    b = static_cast<const T*>(p.b) + static_cast<int64_t>(t.e) * p.N * p.K +
        (DIR == kGmmForward ? static_cast<int64_t>(col0) * p.K : col0);
    out = static_cast<T*>(p.out) + row0 * ldo + col0;
    nm = t.end - row0;
    nn = feat - col0;
  }
  nm = min(nm, BM);
  nn = min(nn, BN);

  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const bool busy = (ty & ~1) * (TM == 1 ? 1 : 4) < nm;  // some row of this warp is valid
  uint64_t acc2[TM][TN / 2];  // two adjacent columns each
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN / 2; ++j) acc2[i][j] = 0;

  SA fa;
  SB fb;
  // This CTA's slices (all of them unless the contraction is split).
  const int S = SPLIT ? p.splits : 1;
  const int me = S > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const int all = (nc + kDepth - 1) / kDepth;
  const int from = all * me / S, slices = all * (me + 1) / S;
  if (slices > from) {
    fa.load(a, lda, nm, from * kDepth, nc, p.a_vec);
    fb.load(b, ldb, nn, from * kDepth, nc, p.b_vec);
    fa.store(sa(from & 1));
    fb.store(sb(from & 1));
  }
  __syncthreads();
  // (Registers are full, and with the folds in shared memory, 64 KB of it, 4000 rows, [700, 700],
  // 100 adapters of rank 128 took 1433 us against 954: so they wait in local memory, where the
  // hidden address keeps them.)
  constexpr int kFoldSlices = kFold / kDepth;
  float4 waiting[TM * TN / 4];
  auto each_fold = [&](auto&& op) {
    float4* folds = waiting;
    asm volatile("" : "+l"(folds)::"memory");
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; j += 4)
        op(folds[i * (TN / 4) + j / 4], acc2[i][j / 2], acc2[i][j / 2 + 1]);
  };
  // The sum of the folds `f` and the next one.  `more` follow: that sum waits and its rounding
  // error, exact by a two-sum, is what the next fold starts from (none beside an infinity).
  auto add_fold = [](float& f, float& a, bool more) {
    const float t = __fadd_rn(f, a), u = __fsub_rn(t, f);
    const float e = __fadd_rn(__fsub_rn(f, __fsub_rn(t, u)), __fsub_rn(a, u));
    f = t;
    a = !more ? t : isfinite(t) ? e : 0.f;
  };
#pragma unroll 1
  for (int s = from; s < slices;) {
    const int first = s, stop = min(s + kFoldSlices, slices);
    for (; s < stop; ++s) {
      const int cur = s & 1;
      if (s + 1 < slices) {
        fa.load(a, lda, nm, (s + 1) * kDepth, nc, p.a_vec);
        fb.load(b, ldb, nn, (s + 1) * kDepth, nc, p.b_vec);
      }
      const float *a_now = sa(cur), *b_now = sb(cur);
      if (busy) {
#pragma unroll
        for (int c = 0; c < kDepth; ++c) {
          float ra[TM];
          uint64_t rb[TN / 2];
          if constexpr (TM == 1) {
            ra[0] = a_now[c * SA::kPitch + ty];
          } else {
#pragma unroll
            for (int i = 0; i < TM; i += 4)
              *reinterpret_cast<float4*>(ra + i) =
                  *reinterpret_cast<const float4*>(&a_now[c * SA::kPitch + ty * 4 + i * TY]);
          }
#pragma unroll
          for (int j = 0; j < TN; j += 4)
            *reinterpret_cast<ulonglong2*>(rb + j / 2) =
                *reinterpret_cast<const ulonglong2*>(&b_now[c * SB::kPitch + tx * 4 + j * 16]);
#pragma unroll
          for (int i = 0; i < TM; ++i) {
            const uint64_t aa = pair2(ra[i], ra[i]);
#pragma unroll
            for (int j = 0; j < TN / 2; ++j) acc2[i][j] = fma2(aa, rb[j], acc2[i][j]);
          }
        }
      }
      if (s + 1 < slices) {
        fa.store(sa(cur ^ 1));
        fb.store(sb(cur ^ 1));
      }
      __syncthreads();
    }
    const bool more = stop < slices;
    if (first > from) {
      each_fold([&](float4& f, uint64_t& u, uint64_t& v) {
        float a, b, c, d;
        unpair2(u, a, b);
        unpair2(v, c, d);
        add_fold(f.x, a, more);
        add_fold(f.y, b, more);
        add_fold(f.z, c, more);
        add_fold(f.w, d, more);
        u = pair2(a, b);
        v = pair2(c, d);
      });
    } else if (more) {
      each_fold([](float4& f, uint64_t& u, uint64_t& v) {
        unpair2(u, f.x, f.y);
        unpair2(v, f.z, f.w);
        u = v = 0;
      });
    }
  }

  float acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; j += 4) {
      unpair2(acc2[i][j / 2], acc[i][j], acc[i][j + 1]);
      unpair2(acc2[i][j / 2 + 1], acc[i][j + 2], acc[i][j + 3]);
    }

  if (SPLIT && S > 1) {
    // The cluster's parts: row i of each thread goes to CTA i S / TM (TM = 1: the thread's row to CTA ty % S), which
    // adds the parts in rank order; four columns at a time.
    float4* parts = reinterpret_cast<float4*>(operands);  // [S - 1][rows owned][256]
    static_assert(sizeof(operands) >= 3 * ((TM + 3) / 4) * NT * 16, "parts fit the operands");
    const int per = TM == 1 ? 1 : TM / S;
#pragma unroll
    for (int j = 0; j < TN; j += 4) {
      cluster_sync();  // every CTA has read its slices, or the parts of the columns before
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        const int owner = TM == 1 ? ty % S : i / per;
        if (owner == me) continue;
        const int slot = me < owner ? me : me - 1;
        const uint32_t at = smem_u32(parts + (slot * per + i % per) * NT + threadIdx.x);
        asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(
                         mapa_shared(at, owner)),
                     "f"(acc[i][j]), "f"(acc[i][j + 1]), "f"(acc[i][j + 2]), "f"(acc[i][j + 3])
                     : "memory");
      }
      cluster_sync();
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        if ((TM == 1 ? ty % S : i / per) != me) continue;
        float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int r = 0; r < S; ++r) {
          const float4 v =
              r == me ? make_float4(acc[i][j], acc[i][j + 1], acc[i][j + 2], acc[i][j + 3])
                      : parts[((r < me ? r : r - 1) * per + i % per) * NT + threadIdx.x];
          sum.x += v.x; sum.y += v.y; sum.z += v.z; sum.w += v.w;
        }
        acc[i][j] = sum.x; acc[i][j + 1] = sum.y; acc[i][j + 2] = sum.z; acc[i][j + 3] = sum.w;
      }
    }
  }

  // Whether this CTA finishes row i of each thread.
  auto owned = [&](int i) { return S == 1 || (TM == 1 ? ty % S : i * S / TM) == me; };
  auto row_of = [&](int i) { return TM == 1 ? ty : ty * 4 + (i / 4) * 4 * TY + (i & 3); };
  if constexpr (LORA) {
    // The adapter term (t holds s_a A_a x).  Rows of other adapters skip an adapter's FMAs, so
    // that what it holds (an infinity, say) stays with its own rows.
    __shared__ int s_ad[BM], s_list[BM];
    __shared__ int s_count;
    if (threadIdx.x == 0) s_count = 0;
    const int r = p.lora.rank;
    for (int m = threadIdx.x; m < BM; m += NT) {
      const int id = m < nm ? __ldg(p.lora.ids + row0 + m) : -1;
      s_ad[m] = id >= 0 && id < p.lora.adapters ? id : -1;
    }
    __syncthreads();
    for (int m = threadIdx.x; m < BM; m += NT) {
      const int id = s_ad[m];
      int k = 0;
      if (id >= 0)
        while (s_ad[k] != id) ++k;
      if (id >= 0 && k == m) s_list[atomicAdd(&s_count, 1)] = id;
    }
    __syncthreads();
    const float* t = p.lora.t + static_cast<int64_t>(row0) * r;
    const T* b0 = static_cast<const T*>(p.lora.b) + static_cast<int64_t>(col0) * r;
    const int64_t per = static_cast<int64_t>(p.N) * r;
    const bool tv = r % 4 == 0;
    const bool bv = tv && reinterpret_cast<uintptr_t>(p.lora.b) % (4 * sizeof(T)) == 0;
    if (s_count > 4) {
      // Many adapters (decode): each thread walks its own rows' t and B.
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        const int m = row_of(i);
        if (!owned(i) || s_ad[m] < 0) continue;
        const T* bb = b0 + s_ad[m] * per;
        for (int q = 0; q < r; q += 4) {
          const float4 u = load4<float>(t + static_cast<int64_t>(m) * r + q, r - q, tv);
#pragma unroll
          for (int j = 0; j < TN; ++j) {
            const int n = tx * 4 + (j / 4) * 64 + (j & 3);
            if (n >= nn) continue;
            const float4 v = load4<T>(bb + static_cast<int64_t>(n) * r + q, r - q, bv);
            acc[i][j] = fmaf(u.x, v.x, fmaf(u.y, v.y, fmaf(u.z, v.z, fmaf(u.w, v.w, acc[i][j]))));
          }
        }
      }
    } else {
      // Few (prompts): slices of t against B_a, adapter by adapter.  (A row's sums come from one
      // adapter, so the list's order does not show.)
      Slice<float, BM, kDepth, true, NT> ft;
      Slice<T, BN, kDepth, true, NT> fl;
      const float *a_now = sa(0), *b_now = sb(0);
      for (int d = 0; d < s_count; ++d) {
        const int ad = s_list[d];
        for (int c0 = 0; c0 < r; c0 += kDepth) {
          ft.load(t, r, nm, c0, r, tv);
          fl.load(b0 + ad * per, r, nn, c0, r, bv);
          __syncthreads();
          ft.store(sa(0));
          fl.store(sb(0));
          __syncthreads();
          const int depth = min(kDepth, r - c0);
          for (int c = 0; c < depth; ++c) {
#pragma unroll
            for (int i = 0; i < TM; ++i) {
              const float u = a_now[c * SA::kPitch + row_of(i)];
              if (owned(i) && s_ad[row_of(i)] == ad) {
#pragma unroll
                for (int j = 0; j < TN; ++j)
                  acc[i][j] = fmaf(u, b_now[c * SB::kPitch + tx * 4 + (j / 4) * 64 + (j & 3)],
                                   acc[i][j]);
              }
            }
          }
        }
      }
    }
  }

#pragma unroll
  for (int i = 0; i < TM; ++i) {
    if (!owned(i)) continue;
    const int m = row_of(i);
    if (m >= nm) continue;
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      const int n = tx * 4 + (j / 4) * 64 + (j & 3);
      if (n < nn) out[m * ldo + n] = from_f<T>(acc[i][j]);
    }
  }
}

// Forward product of groups of a few rows: streaming the weights through the lanes.  A warp
// takes kGemvCols output features and up to kGemvRows rows of the group at a time; its lanes
// stride over the contraction, four entries each, and meet in a butterfly sum.  Bound: the
// weights' bytes (a 64-row tile of the kernel above would multiply 64 rows whatever the group
// has: 97 us for one row of [4096, 4096] fp32).  A lane sums kFold entries at a time, as the tiles
// do: 32768 equal ones in one sum were off by 3e-4.
constexpr int kGemvRows = 8;
constexpr int kGemvCols = 2;
constexpr int kLaneFold = 32 * kFold;  // contraction entries of 32 lanes' running sums

template <typename T>
__global__ void __launch_bounds__(kThreads)
grouped_gemv_kernel(const SimtParams p) {
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int rows = static_cast<int>(p.rows), e = blockIdx.y, K = p.K;
  const int begin = group_begin(p.offsets, e, rows), end = group_end(p.offsets, e, rows, begin);
  const int n0 = (blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5)) * kGemvCols;
  if (n0 >= p.N) return;
  const T* w0 = static_cast<const T*>(p.b) + (static_cast<int64_t>(e) * p.N + n0) * K;
  const T* x = static_cast<const T*>(p.a);
  for (int r0 = begin; r0 < end; r0 += kGemvRows) {
    const int nr = min(kGemvRows, end - r0);
    float acc[kGemvCols][kGemvRows] = {}, folds[kGemvCols][kGemvRows] = {};
    const T* xr = x + static_cast<int64_t>(r0) * K;
    auto take_fold = [&] {
#pragma unroll
      for (int j = 0; j < kGemvCols; ++j)
#pragma unroll
        for (int i = 0; i < kGemvRows; ++i) {
          folds[j][i] += acc[j][i];
          acc[j][i] = 0.f;
        }
    };
    for (int c0 = 0; c0 < K; c0 += kLaneFold) {
      const int c1 = min(c0 + kLaneFold, K);
      if (c0 > 0) take_fold();
#pragma unroll 4
      for (int c = c0 + lane * 4; c < c1; c += 128) {
        float4 w[kGemvCols];
#pragma unroll
        for (int j = 0; j < kGemvCols; ++j)
          w[j] = n0 + j < p.N ? load4<T>(w0 + static_cast<int64_t>(j) * K + c, K - c, p.b_vec)
                              : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int i = 0; i < kGemvRows; ++i) {
          if (i >= nr) break;
          const float4 v = load4<T>(xr + static_cast<int64_t>(i) * K + c, K - c, p.a_vec);
#pragma unroll
          for (int j = 0; j < kGemvCols; ++j) {
            acc[j][i] = fmaf(w[j].x, v.x, acc[j][i]);
            acc[j][i] = fmaf(w[j].y, v.y, acc[j][i]);
            acc[j][i] = fmaf(w[j].z, v.z, acc[j][i]);
            acc[j][i] = fmaf(w[j].w, v.w, acc[j][i]);
          }
        }
      }
    }
    if (K > kLaneFold) {
      take_fold();
#pragma unroll
      for (int j = 0; j < kGemvCols; ++j)
#pragma unroll
        for (int i = 0; i < kGemvRows; ++i) acc[j][i] = folds[j][i];
    }
    if (p.lora.t != nullptr) {  // y += B_a t, the lanes striding over the rank
      const int r = p.lora.rank;
#pragma unroll
      for (int i = 0; i < kGemvRows; ++i) {
        if (i >= nr) break;
        const int ad = __ldg(p.lora.ids + r0 + i);
        if (ad < 0 || ad >= p.lora.adapters) continue;
        const float* t = p.lora.t + static_cast<int64_t>(r0 + i) * r;
        const T* bb = static_cast<const T*>(p.lora.b) + (static_cast<int64_t>(ad) * p.N + n0) * r;
        for (int q = lane; q < r; q += 32) {
          const float tq = t[q];
#pragma unroll
          for (int j = 0; j < kGemvCols; ++j)
            if (n0 + j < p.N) acc[j][i] = fmaf(to_f(bb[j * r + q]), tq, acc[j][i]);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < kGemvRows; ++i) {
      if (i >= nr) break;
#pragma unroll
      for (int j = 0; j < kGemvCols; ++j) {
        float v = acc[j][i];
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
        if (lane == 0 && n0 + j < p.N)
          static_cast<T*>(p.out)[static_cast<int64_t>(r0 + i) * p.N + n0 + j] = from_f<T>(v);
      }
    }
  }
}

template <typename T>
cudaError_t launch_gemv(const SimtParams& p, cudaStream_t s) {
  const int per = kThreads / 32 * kGemvCols;
  return launch_dependent(pdl_enabled(), grouped_gemv_kernel<T>, dim3((p.N + per - 1) / per, p.E),
                          dim3(kThreads), 0, s, p);
}

template <typename T, int DIR, int TM, int TN, int NT, bool LORA>
cudaError_t launch_tile(const GroupedArgs& g, SimtParams p, int num_sms, cudaStream_t s) {
  constexpr int BM = NT / 16 * TM, BN = 16 * TN;
  dim3 grid;
  p.splits = 1;
  int64_t tiles, con;
  if (DIR == kGmmGradWeight) {
    grid = dim3((g.K + BN - 1) / BN, (g.N + BM - 1) / BM, g.E);
    tiles = static_cast<int64_t>(grid.x) * grid.y * grid.z;
    con = g.rows / g.E;
  } else {
    // The tile count lives on the device; ragged groups add at most one tile each.
    const int feat = DIR == kGmmForward ? g.N : g.K;
    const int64_t rows_tiles = g.rows / BM + std::min<int64_t>(g.rows, g.E);
    grid = dim3(static_cast<unsigned>(rows_tiles), (feat + BN - 1) / BN, 1);
    tiles = rows_tiles * grid.y;
    con = DIR == kGmmForward ? g.K : g.N;
  }
  // Split until the SMs' resident CTAs run (four, of 128 x 128 tiles two), with a contraction
  // of at least 64 each.
  const int64_t fill = static_cast<int64_t>(num_sms) * resident(TM, NT);
  while (p.splits < 4 && tiles * p.splits * 2 <= fill && con >= 128 * p.splits) p.splits *= 2;
  grid.z *= p.splits;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(NT);
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = 1;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = static_cast<unsigned>(p.splits);
  cfg.attrs = attr;
  cfg.numAttrs = p.splits > 1 ? 2 : 1;
  if (BM <= 64 || p.splits > 1)
    return cudaLaunchKernelEx(&cfg, grouped_simt_kernel<T, DIR, TM, TN, NT, true, LORA>, p);
  return cudaLaunchKernelEx(&cfg, grouped_simt_kernel<T, DIR, TM, TN, NT, BM <= 64, LORA>, p);
}

template <typename T, int DIR, bool LORA>
cudaError_t launch_dir(const GroupedArgs& g, const LoraTerm* lora, int num_sms, cudaStream_t s) {
  SimtParams p{};
  p.a = DIR == kGmmForward ? g.x : g.dy;
  p.b = DIR == kGmmGradWeight ? g.x : g.w;
  p.out = g.out;
  p.offsets = g.offsets;
  p.rows = g.rows;
  p.N = g.N;
  p.K = g.K;
  p.E = g.E;
  auto vec = [](const void* q, int ld) {
    return ld % 4 == 0 && reinterpret_cast<uintptr_t>(q) % (4 * sizeof(T)) == 0 ? 1 : 0;
  };
  p.a_vec = vec(p.a, DIR == kGmmForward ? g.K : g.N);
  p.b_vec = vec(p.b, g.K);
  if (lora != nullptr) p.lora = *lora;
  if constexpr (DIR == kGmmForward) {
    if (g.rows <= (g.E == 1 ? kGemvRows : 4 * static_cast<int64_t>(g.E))) return launch_gemv<T>(p, s);
  }
  // 128 x 128 tiles where groups fill them and they, split four ways, fill the GPU (each thread
  // then does 64 FMAs per 16 shared loads instead of 32 per 12); else 64 x 64, and 16 rows for
  // groups of a few rows, which multiply less padding.  Several groups pad the tall tiles more
  // and want twice as many of them (fp32, 128 : 64 rows, us: 500 rows in 4 groups, grad_input of
  // [1024, 2048] 112 : 94, of [640, 2048] 75 : 60; one group of 1000 rows, [1024, 1024], 67 : 72;
  // below 148 tiles the small ones won in every case measured, 4 groups [1024, 2048] 116 : 104).
  const int64_t feat = DIR == kGmmForward ? g.N : g.K;
  const int64_t big = DIR == kGmmGradWeight
                          ? static_cast<int64_t>(g.E) * ((g.N + 127) / 128) * ((g.K + 127) / 128)
                          : ((g.rows + 127) / 128) * ((feat + 127) / 128);
  const int64_t height = DIR == kGmmGradWeight ? g.N : g.rows / g.E;
  // (With element-wise loads the small tiles win until the big ones fill the GPU unsplit.)
  const int64_t ways = p.a_vec && p.b_vec ? 4 : 1;
  const bool twice = ways == 4 && g.E > 1 && DIR != kGmmGradWeight;
  if (height >= 96 && feat >= 96 && (twice ? ways * big > 2 * num_sms : ways * big >= num_sms))
    return launch_tile<T, DIR, 8, 8, 256, LORA>(g, p, num_sms, s);
  if constexpr (DIR != kGmmGradWeight) {
    if (g.rows <= 16 * static_cast<int64_t>(g.E)) return launch_tile<T, DIR, 1, 4, 256, LORA>(g, p, num_sms, s);
  }
  return launch_tile<T, DIR, 8, 4, 128, LORA>(g, p, num_sms, s);
}

template <typename T>
cudaError_t launch_type(const GroupedArgs& g, const LoraTerm* lora, int num_sms, cudaStream_t s) {
  if (lora != nullptr) return launch_dir<T, kGmmForward, true>(g, lora, num_sms, s);
  if (g.dir == kGmmForward) return launch_dir<T, kGmmForward, false>(g, nullptr, num_sms, s);
  if (g.dir == kGmmGradInput) return launch_dir<T, kGmmGradInput, false>(g, nullptr, num_sms, s);
  return launch_dir<T, kGmmGradWeight, false>(g, nullptr, num_sms, s);
}

}  // namespace

cudaError_t launch_grouped_simt(const GroupedArgs& g, const LoraTerm* lora, int num_sms,
                                cudaStream_t s) {
  if (g.dtype == kDtF32) return launch_type<float>(g, lora, num_sms, s);
  if (g.dtype == kDtF16) return launch_type<__half>(g, lora, num_sms, s);
  if (g.dtype == kDtBF16) return launch_type<__nv_bfloat16>(g, lora, num_sms, s);
  return cudaErrorInvalidValue;
}

}  // namespace moe

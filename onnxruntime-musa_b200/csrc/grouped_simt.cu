// The expert products and the adapter projection on the FP32 pipes, for every size,
// alignment and float type; the 16-bit tensor-core kernels (grouped_tc.cu) take the
// operands that TMA can address, this file the rest and all of fp32 (TF32 would round
// the operands to 11 bits, 2^13 times the rounding of an fp32 result).
//
// Mathematics: one tile C[m, n] = sum_c A(m, c) B(n, c) per CTA, summed in ascending c in
// fp32.  The three directions differ only in where the contraction index lies:
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
// false when the list is shorter.  Called by all kThreads (>= E) threads.
__device__ bool find_tile(const int32_t* off, int E, int rows, int tile_rows, int L, Tile* out) {
  __shared__ int s_warp[kThreads / 32];
  __shared__ Tile s_tile;
  const int e = threadIdx.x, lane = e & 31, warp = e >> 5;
  int begin = 0, end = 0, n = 0;
  if (e < E) {
    begin = group_begin(off, e, rows);
    end = group_end(off, e, rows, begin);
    n = (end - begin + tile_rows - 1) / tile_rows;
  }
  int incl = n;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, incl, d);
    if (lane >= d) incl += v;
  }
  if (lane == 31) s_warp[warp] = incl;
  if (e == 0) s_tile.e = -1;
  __syncthreads();
  int base = 0;
  for (int w = 0; w < warp; ++w) base += s_warp[w];
  const int first = base + incl - n;
  if (n > 0 && L >= first && L < first + n) {
    s_tile.e = e;
    s_tile.index = L - first;
    s_tile.begin = begin;
    s_tile.end = end;
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
template <typename T, int X, int kDepth, bool CONTIG_C>
struct Slice {
  static constexpr int kPitch = X + 4;
  static constexpr int kAll = X * kDepth / 4;
  static constexpr int kQuads = (kAll + kThreads - 1) / kThreads;
  float4 v[kQuads];

  __device__ __forceinline__ void load(const T* p, int64_t ld, int ni, int c0, int nc, int vec) {
#pragma unroll
    for (int j = 0; j < kQuads; ++j) {
      const int q = threadIdx.x + j * kThreads;
      if (kAll % kThreads != 0 && q >= kAll) continue;
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
      const int q = threadIdx.x + j * kThreads;
      if (kAll % kThreads != 0 && q >= kAll) continue;
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

// CTA tile (16 TM) x (16 TN), TN a multiple of 4 and TM too or 1: thread (ty, tx) owns rows
// ty * 4 + 64 i + [0, 4) (TM = 1: row ty) and columns tx * 4 + 64 j + [0, 4).
template <typename T, int DIR, int TM, int TN>
__global__ void __launch_bounds__(kThreads, TM <= 4 ? 4 : 2)
grouped_simt_kernel(const SimtParams p) {
  constexpr int BM = 16 * TM, BN = 16 * TN;
  constexpr int kDepth = TM <= 4 ? 32 : 16;
  constexpr bool kAC = DIR != kGmmGradWeight;  // contraction contiguous in A
  constexpr bool kBC = DIR == kGmmForward;
  using SA = Slice<T, BM, kDepth, kAC>;
  using SB = Slice<T, BN, kDepth, kBC>;
  __shared__ __align__(16) float sa[2][kDepth * SA::kPitch];
  __shared__ __align__(16) float sb[2][kDepth * SB::kPitch];

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
    if (!find_tile(p.offsets, p.E, rows, BM, blockIdx.x, &t)) return;
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
  constexpr bool kSplit = TM <= 4;
  const int S = kSplit ? p.splits : 1;
  const int me = S > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const int all = (nc + kDepth - 1) / kDepth;
  const int from = all * me / S, slices = all * (me + 1) / S;
  if (slices > from) {
    fa.load(a, lda, nm, from * kDepth, nc, p.a_vec);
    fb.load(b, ldb, nn, from * kDepth, nc, p.b_vec);
    fa.store(sa[0]);
    fb.store(sb[0]);
  }
  __syncthreads();
  for (int s = from; s < slices; ++s) {
    const int cur = (s - from) & 1;
    if (s + 1 < slices) {
      fa.load(a, lda, nm, (s + 1) * kDepth, nc, p.a_vec);
      fb.load(b, ldb, nn, (s + 1) * kDepth, nc, p.b_vec);
    }
    if (busy) {
#pragma unroll
      for (int c = 0; c < kDepth; ++c) {
        float ra[TM];
        uint64_t rb[TN / 2];
        if constexpr (TM == 1) {
          ra[0] = sa[cur][c * SA::kPitch + ty];
        } else {
#pragma unroll
          for (int i = 0; i < TM; i += 4)
            *reinterpret_cast<float4*>(ra + i) =
                *reinterpret_cast<const float4*>(&sa[cur][c * SA::kPitch + ty * 4 + i * 16]);
        }
#pragma unroll
        for (int j = 0; j < TN; j += 4)
          *reinterpret_cast<ulonglong2*>(rb + j / 2) =
              *reinterpret_cast<const ulonglong2*>(&sb[cur][c * SB::kPitch + tx * 4 + j * 16]);
#pragma unroll
        for (int i = 0; i < TM; ++i) {
          const uint64_t aa = pair2(ra[i], ra[i]);
#pragma unroll
          for (int j = 0; j < TN / 2; ++j) acc2[i][j] = fma2(aa, rb[j], acc2[i][j]);
        }
      }
    }
    if (s + 1 < slices) {
      fa.store(sa[cur ^ 1]);
      fb.store(sb[cur ^ 1]);
    }
    __syncthreads();
  }

  float acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN / 2; ++j) unpair2(acc2[i][j], acc[i][2 * j], acc[i][2 * j + 1]);

  if constexpr (kSplit) {
    if (S > 1) {
      // Row i of each thread's four goes to CTA i S / 4 (TM = 1: the thread's row to CTA
      // ty % S), which adds the parts in rank order.
      float4* parts = reinterpret_cast<float4*>(&sb[0][0]);  // [S - 1][rows owned][256]
      static_assert(sizeof(sb) >= 3 * kThreads * 16, "parts fit the operand slices");
      const int per = TM == 1 ? 1 : TM / S;
      cluster_sync();  // every CTA has read its slices
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        const int owner = TM == 1 ? ty % S : i / per;
        if (owner == me) continue;
        const int slot = me < owner ? me : me - 1;
        const uint32_t at = smem_u32(parts + (slot * per + i % per) * kThreads + threadIdx.x);
        asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(
                         mapa_shared(at, owner)),
                     "f"(acc[i][0]), "f"(acc[i][1]), "f"(acc[i][2]), "f"(acc[i][3])
                     : "memory");
      }
      cluster_sync();
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        if ((TM == 1 ? ty % S : i / per) != me) continue;
        float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int r = 0; r < S; ++r) {
          const float4 v = r == me ? make_float4(acc[i][0], acc[i][1], acc[i][2], acc[i][3])
                                   : parts[((r < me ? r : r - 1) * per + i % per) * kThreads +
                                           threadIdx.x];
          sum.x += v.x; sum.y += v.y; sum.z += v.z; sum.w += v.w;
        }
        acc[i][0] = sum.x; acc[i][1] = sum.y; acc[i][2] = sum.z; acc[i][3] = sum.w;
      }
    }
  }

#pragma unroll
  for (int i = 0; i < TM; ++i) {
    if (kSplit && S > 1 && (TM == 1 ? ty % S : i * S / TM) != me) continue;
    const int m = TM == 1 ? ty : ty * 4 + (i / 4) * 64 + (i & 3);
    if (m >= nm) continue;
    if (DIR == kGmmForward && p.lora.t != nullptr) {
      // y += s_a * sum_j t[row, j] B_a[n, j].
      const int row = row0 + m, ad = __ldg(p.lora.ids + row), r = p.lora.rank;
      if (ad >= 0 && ad < p.lora.adapters) {
        float d[TN];
#pragma unroll
        for (int j = 0; j < TN; ++j) d[j] = 0.f;
        const T* bb = static_cast<const T*>(p.lora.b) + static_cast<int64_t>(ad) * p.N * r;
        for (int q = 0; q < r; ++q) {
          const float t = __ldg(p.lora.t + static_cast<int64_t>(row) * r + q);
#pragma unroll
          for (int j = 0; j < TN; ++j) {
            const int n = tx * 4 + (j / 4) * 64 + (j & 3);
            if (n < nn) d[j] = fmaf(t, to_f(bb[static_cast<int64_t>(col0 + n) * r + q]), d[j]);
          }
        }
        const float sc = __ldg(p.lora.scales + ad);
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = fmaf(sc, d[j], acc[i][j]);
      }
    }
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      const int n = tx * 4 + (j / 4) * 64 + (j & 3);
      if (n < nn) out[m * ldo + n] = from_f<T>(acc[i][j]);
    }
  }
}

template <typename T, int DIR, int TM, int TN>
cudaError_t launch_tile(const GroupedArgs& g, SimtParams p, cudaStream_t s) {
  constexpr int BM = 16 * TM, BN = 16 * TN;
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
  // Split until about four CTAs an SM run, with at least two slices of 32 each.
  if (TM <= 4)
    while (p.splits < 4 && tiles * p.splits * 2 <= 4 * 148 && con >= 128 * p.splits) p.splits *= 2;
  grid.z *= p.splits;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(kThreads);
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = 1;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = static_cast<unsigned>(p.splits);
  cfg.attrs = attr;
  cfg.numAttrs = p.splits > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, grouped_simt_kernel<T, DIR, TM, TN>, p);
}

template <typename T, int DIR>
cudaError_t launch_dir(const GroupedArgs& g, const LoraTerm* lora, cudaStream_t s) {
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
  // 128 x 128 tiles once they fill the GPU twice over (each thread then does 64 FMAs per
  // 16 shared loads instead of 16 per 8); below that the 64 x 64 tiles' four times as many
  // CTAs win.  Groups of a few rows take tiles of 16 rows, which multiply less padding.
  const int64_t feat = DIR == kGmmForward ? g.N : g.K;
  const int64_t big = DIR == kGmmGradWeight
                          ? static_cast<int64_t>(g.E) * ((g.N + 127) / 128) * ((g.K + 127) / 128)
                          : (g.rows / 128) * ((feat + 127) / 128);
  if (big >= 2 * 148) return launch_tile<T, DIR, 8, 8>(g, p, s);
  if constexpr (DIR != kGmmGradWeight) {
    if (g.rows <= 16 * static_cast<int64_t>(g.E)) return launch_tile<T, DIR, 1, 4>(g, p, s);
  }
  return launch_tile<T, DIR, 4, 4>(g, p, s);
}

template <typename T>
cudaError_t launch_type(const GroupedArgs& g, const LoraTerm* lora, cudaStream_t s) {
  if (g.dir == kGmmForward) return launch_dir<T, kGmmForward>(g, lora, s);
  if (g.dir == kGmmGradInput) return launch_dir<T, kGmmGradInput>(g, lora, s);
  return launch_dir<T, kGmmGradWeight>(g, lora, s);
}

}  // namespace

cudaError_t launch_grouped_simt(const GroupedArgs& g, const LoraTerm* lora, cudaStream_t s) {
  static_assert(kThreads >= kMaxExperts, "find_tile needs a thread per expert");
  if (g.dtype == kDtF32) return launch_type<float>(g, lora, s);
  if (g.dtype == kDtF16) return launch_type<__half>(g, lora, s);
  if (g.dtype == kDtBF16) return launch_type<__nv_bfloat16>(g, lora, s);
  return cudaErrorInvalidValue;
}

}  // namespace moe

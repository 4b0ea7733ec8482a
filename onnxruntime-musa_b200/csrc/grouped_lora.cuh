// The adapter term in the epilogue of the tensor-core kernels:
//   acc[n, t] += s_a * sum_j B_a[n, j] t[t, j],   a = the adapter of row t,
// on accumulator fragments as tmem_ld_frag* delivers them (32 features x 8 rows per warp).
//
// The rank-sized intermediate enters mma.m16n8k16 as the sum of two 16-bit parts,
// hi = round(s_a t) and lo = round(s_a t - hi).  In bf16 they keep an entry to 2^-16 of itself (half
// a step, 2^-8, of a rest that is at most 2^-8 of it); one part would leave an error of half an
// output step of the term itself.  In fp16 to 2^-22 of itself (2^-11 twice), but not below 2^-25,
// half the type's smallest step: rows whose largest finite entry lies outside [2^-8, 2^15) are first
// scaled by a power of two to |s_a t| < 2 (t may exceed fp16's range), undone on the fp32 sum,
// so that floor is at most 2^-17 of the row's largest entry.  (Every row scaled would hold it at 2^-25,
// but sixteen rows with a scaled one among them go through mma.sync in the pair kernel's epilogue,
// whose price stands there.)
// The shrink kernel (lora.cu) forms the parts.
// The eight rows of a fragment may follow different adapters: the products of each adapter
// among them are formed for all eight columns in a sum of their own, and a column takes
// only its own adapter's, so nothing of another adapter (an infinity, say) reaches a row.
#pragma once

#include "grouped_tc.cuh"

namespace moe {

__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                          uint32_t a3, uint32_t b0, uint32_t b1, __half) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                          uint32_t a3, uint32_t b0, uint32_t b1, __nv_bfloat16) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Fragments of 16 STEPS columns of one adapter's B for a warp's 32 features, kept while
// the rows follow the same adapter (a prompt's rows all do).
template <int STEPS>
struct LoraFrags {
  int adapter = -1;
  uint2 f[STEPS][4];  // features g, g + 8, g + 16, g + 24 (g = lane / 4)

  template <typename T>
  __device__ __forceinline__ void load(const LoraTerm& l, int a, int s0, int n0, int N) {
    const int lane = threadIdx.x & 31;
    const int g = lane >> 2, c = lane & 3;
    const T* b = static_cast<const T*>(l.b) + static_cast<int64_t>(a) * N * l.rank;
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      const int j = (s0 + s) * 16 + 4 * c;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int n = n0 + g + 8 * i;
        f[s][i] = j < l.rank && n < N
                      ? __ldg(reinterpret_cast<const uint2*>(b + static_cast<int64_t>(n) * l.rank + j))
                      : make_uint2(0, 0);
      }
    }
  }
};

// The parts of row `row` for this lane, 16 STEPS entries from step s0 on: entries
// 4 (l % 4) + [0, 4) of each step as {hi, hi, lo, lo}.  (The order of the entries inside a
// step is free as long as both operands agree, and four in a row make the loads wide.)
template <int STEPS>
__device__ __forceinline__ void lora_rows(const LoraTerm& l, int64_t rows, int64_t row, bool ok,
                                          int s0, uint4 (&v)[STEPS]) {
  const int j = s0 * 16 + 4 * (threadIdx.x & 3);
  const uint16_t* q = l.parts + row * l.rank + j;
#pragma unroll
  for (int s = 0; s < STEPS; ++s) {
    uint2 hi = make_uint2(0, 0), lo = make_uint2(0, 0);
    if (ok && j + 16 * s < l.rank) {
      hi = *reinterpret_cast<const uint2*>(q + 16 * s);
      lo = *reinterpret_cast<const uint2*>(q + 16 * s + rows * l.rank);
    }
    v[s] = make_uint4(hi.x, hi.y, lo.x, lo.y);
  }
}

// Adapter of row `row` (-1: none).
__device__ __forceinline__ int lora_adapter(const LoraTerm& l, int64_t row, bool ok) {
  const int a = ok ? __ldg(l.ids + row) : -1;
  return a < l.adapters ? max(a, -1) : -1;
}

// Adds the adapter term of eight rows and features n0 .. n0 + 31 to lo (features 0..15) and
// hi (16..31).  This lane's row (of the fragment's column l / 4): adapter `ad`, number
// `row`, its first 16 STEPS entries `v`.
template <typename T, int STEPS>
__device__ __forceinline__ void lora_add(const LoraTerm& l, int64_t rows, int ad, int64_t row,
                                         int n0, int N,
                                         const uint4 (&v)[STEPS], LoraFrags<STEPS>& fr,
                                         float (&lo)[4], float (&hi)[4]) {
  unsigned todo = __ballot_sync(0xffffffffu, ad >= 0);
  if (todo == 0) return;
  const int c = threadIdx.x & 3;
  const int ad0 = __shfl_sync(0xffffffffu, ad, 8 * c);      // adapters of this lane's two
  const int ad1 = __shfl_sync(0xffffffffu, ad, 8 * c + 4);  // accumulator columns
  float f0 = 1.f, f1 = 1.f;
  if (std::is_same<T, __half>::value) {
    const float f = ad >= 0 ? l.row_scale[row] : 1.f;
    f0 = __shfl_sync(0xffffffffu, f, 8 * c);
    f1 = __shfl_sync(0xffffffffu, f, 8 * c + 4);
  }
  while (todo != 0) {
    const int a = __shfl_sync(0xffffffffu, ad, __ffs(todo) - 1);
    todo &= ~__ballot_sync(0xffffffffu, ad == a);
    float d[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll 1
    for (int s0 = 0; s0 < l.steps; s0 += STEPS) {
      uint4 w[STEPS];
      if (s0 == 0) {
        if (fr.adapter != a || l.steps > STEPS) fr.template load<T>(l, a, 0, n0, N);
#pragma unroll
        for (int s = 0; s < STEPS; ++s) w[s] = v[s];
      } else {
        fr.template load<T>(l, a, s0, n0, N);
        lora_rows<STEPS>(l, rows, row, ad >= 0, s0, w);
      }
#pragma unroll
      for (int s = 0; s < STEPS; ++s) {
        if (s0 + s >= l.steps) break;
        const uint2(&f)[4] = fr.f[s];
        mma_16816(d[0], f[0].x, f[1].x, f[0].y, f[1].y, w[s].x, w[s].y, T());
        mma_16816(d[1], f[2].x, f[3].x, f[2].y, f[3].y, w[s].x, w[s].y, T());
        mma_16816(d[0], f[0].x, f[1].x, f[0].y, f[1].y, w[s].z, w[s].w, T());
        mma_16816(d[1], f[2].x, f[3].x, f[2].y, f[3].y, w[s].z, w[s].w, T());
      }
    }
    fr.adapter = a;
    if (ad0 == a) {
      lo[0] = fmaf(f0, d[0][0], lo[0]);
      lo[2] = fmaf(f0, d[0][2], lo[2]);
      hi[0] = fmaf(f0, d[1][0], hi[0]);
      hi[2] = fmaf(f0, d[1][2], hi[2]);
    }
    if (ad1 == a) {
      lo[1] = fmaf(f1, d[0][1], lo[1]);
      lo[3] = fmaf(f1, d[0][3], lo[3]);
      hi[1] = fmaf(f1, d[1][1], hi[1]);
      hi[3] = fmaf(f1, d[1][3], hi[3]);
    }
  }
}

// The same for rows that may follow many adapters (decode): the fragments of BATCH adapters
// are fetched together, so a block of eight adapters waits for memory 8 / BATCH times
// instead of eight; gather() may run before the rows' parts exist.
template <typename T, int STEPS, int BATCH>
struct LoraBatch {
  int a[BATCH];              // adapters whose fragments are held, -1: none
  LoraFrags<STEPS> fr[BATCH];

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int k = 0; k < BATCH; ++k) a[k] = -1;
  }
  // The first BATCH adapters of `todo` (lanes whose row still waits for its adapter `ad`).
  __device__ __forceinline__ void gather(const LoraTerm& l, int ad, unsigned& todo, int n0, int N) {
#pragma unroll
    for (int k = 0; k < BATCH; ++k) {
      int next = -1;
      if (todo != 0) {
        next = __shfl_sync(0xffffffffu, ad, __ffs(todo) - 1);
        todo &= ~__ballot_sync(0xffffffffu, ad == next);
        if (next != a[k] || l.steps > STEPS) fr[k].template load<T>(l, next, 0, n0, N);
      }
      a[k] = next;
    }
  }
  static __device__ __forceinline__ void step(const uint2 (&f)[4], const uint4& w,
                                              float (&d)[2][4]) {
    mma_16816(d[0], f[0].x, f[1].x, f[0].y, f[1].y, w.x, w.y, T());
    mma_16816(d[1], f[2].x, f[3].x, f[2].y, f[3].y, w.x, w.y, T());
    mma_16816(d[0], f[0].x, f[1].x, f[0].y, f[1].y, w.z, w.w, T());
    mma_16816(d[1], f[2].x, f[3].x, f[2].y, f[3].y, w.z, w.w, T());
  }
  // The sums of the held adapters: each column is set from its own adapter only.
  __device__ __forceinline__ void apply(const LoraTerm& l, int64_t rows, int ad, int64_t row, int n0,
                                        int N, const uint4 (&v)[STEPS], float (&lo)[4], float (&hi)[4]) {
    const int c = threadIdx.x & 3;
    const int ad0 = __shfl_sync(0xffffffffu, ad, 8 * c);
    const int ad1 = __shfl_sync(0xffffffffu, ad, 8 * c + 4);
    float f0 = 1.f, f1 = 1.f;
    if (std::is_same<T, __half>::value) {
      const float f = ad >= 0 ? l.row_scale[row] : 1.f;
      f0 = __shfl_sync(0xffffffffu, f, 8 * c);
      f1 = __shfl_sync(0xffffffffu, f, 8 * c + 4);
    }
#pragma unroll
    for (int k = 0; k < BATCH; ++k) {
      if (a[k] < 0) break;
      float d[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
      for (int s = 0; s < STEPS; ++s) step(fr[k].f[s], v[s], d);
      if (STEPS > 1) {  // (one step is all of a rank up to 16)
#pragma unroll 1
        for (int s0 = STEPS; s0 < l.steps; s0 += STEPS) {
          uint4 w[STEPS];
          fr[k].template load<T>(l, a[k], s0, n0, N);
          lora_rows<STEPS>(l, rows, row, ad >= 0, s0, w);
#pragma unroll
          for (int s = 0; s < STEPS; ++s) step(fr[k].f[s], w[s], d);
        }
      }
      if (ad0 == a[k]) {
        lo[0] = f0 * d[0][0];
        lo[2] = f0 * d[0][2];
        hi[0] = f0 * d[1][0];
        hi[2] = f0 * d[1][2];
      }
      if (ad1 == a[k]) {
        lo[1] = f1 * d[0][1];
        lo[3] = f1 * d[0][3];
        hi[1] = f1 * d[1][1];
        hi[3] = f1 * d[1][3];
      }
    }
  }
};

}  // namespace moe

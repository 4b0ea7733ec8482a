// The adapter term in the epilogue of the tensor-core kernels:
//   acc[n, t] += s_a * sum_j B_a[n, j] t[t, j],   a = the adapter of row t,
// on accumulator fragments as tmem_ld_frag* delivers them (32 features x 8 rows per warp).
//
// The rank-sized intermediate t is fp32 and enters mma.m16n8k16 as the sum of two 16-bit
// parts, hi = round(t) and lo = round(t - hi), which keeps 16 (bf16) or 22 (fp16) of its
// bits; one part would leave an error of half an output step of the term itself.  fp16
// rows are first scaled by a power of two to |t| < 2 (t may exceed fp16's range), undone
// on the fp32 sum.
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

template <typename T>
__device__ __forceinline__ void split16(float v, float& hi, float& lo) {
  hi = to_f(from_f<T>(v));
  lo = v - hi;
}

// Sum over the splits of t[row, j .. j+3] (j a multiple of 4; j < rank).
__device__ __forceinline__ float4 lora_t4(const LoraTerm& l, int64_t rows, int64_t row, int j) {
  const float* q = l.t + row * l.rank + j;
  float4 v = *reinterpret_cast<const float4*>(q);
  for (int s = 1; s < l.splits; ++s) {
    q += rows * l.rank;
    const float4 w = *reinterpret_cast<const float4*>(q);
    v.x += w.x; v.y += w.y; v.z += w.z; v.w += w.w;
  }
  return v;
}

// Adds the adapter term of rows row0 .. row0 + 7 (those < row_end) and features n0 .. n0 + 31
// to lo (features 0..15) and hi (16..31).  Contraction entries are dealt to the lanes four
// in a row (lane % 4 holds entries 4 (l % 4) + [0, 4) of a step in both operands): the order
// inside a step is free, and the loads become 8 and 16 bytes wide.
template <typename T>
__device__ __forceinline__ void lora_add(const LoraTerm& l, int64_t rows, int row0, int row_end,
                                         int n0, int N, float (&lo)[4], float (&hi)[4]) {
  const int lane = threadIdx.x & 31;
  const int g = lane >> 2, c = lane & 3;
  const int row = row0 + g;
  int ad = -1;
  if (row < row_end) {
    ad = __ldg(l.ids + row);
    if (ad >= l.adapters) ad = -1;
  }
  const int ad0 = __shfl_sync(0xffffffffu, ad, 8 * c);      // adapters of this lane's two
  const int ad1 = __shfl_sync(0xffffffffu, ad, 8 * c + 4);  // accumulator columns
  unsigned todo = __ballot_sync(0xffffffffu, ad >= 0);
  if (todo == 0) return;
  const int steps = (l.rank + 15) / 16;
  float up = 1.f, down = 1.f;  // fp16: 2^-e and 2^e of this lane's row
  if (std::is_same<T, __half>::value) {
    float m = 0.f;
    if (ad >= 0)
      for (int s = 0; s < steps; ++s) {
        const int j = s * 16 + 4 * c;
        if (j < l.rank) {
          const float4 v = lora_t4(l, rows, row, j);
          m = fmaxf(m, fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w))));
        }
      }
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
    if (m > 0.f && m < __int_as_float(0x7f800000)) {
      const int e = min(max((__float_as_int(m) >> 23) - 127, -120), 120);
      up = __int_as_float((127 - e) << 23);
      down = __int_as_float((127 + e) << 23);
    }
  }
  const float down0 = __shfl_sync(0xffffffffu, down, 8 * c);
  const float down1 = __shfl_sync(0xffffffffu, down, 8 * c + 4);
  while (todo != 0) {
    const int a = __shfl_sync(0xffffffffu, ad, __ffs(todo) - 1);
    todo &= ~__ballot_sync(0xffffffffu, ad == a);
    const T* b = static_cast<const T*>(l.b) + static_cast<int64_t>(a) * N * l.rank;
    float d[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll 2
    for (int s = 0; s < steps; ++s) {
      const int j = s * 16 + 4 * c;
      const bool in = j < l.rank;
      uint2 f[4];  // features g, g + 8, g + 16, g + 24
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int n = n0 + g + 8 * i;
        f[i] = in && n < N
                   ? __ldg(reinterpret_cast<const uint2*>(b + static_cast<int64_t>(n) * l.rank + j))
                   : make_uint2(0, 0);
      }
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      if (in && ad == a) v = lora_t4(l, rows, row, j);
      float h0, h1, h2, h3, r0, r1, r2, r3;
      split16<T>(v.x * up, h0, r0);
      split16<T>(v.y * up, h1, r1);
      split16<T>(v.z * up, h2, r2);
      split16<T>(v.w * up, h3, r3);
      const uint32_t bh0 = pack2<T>(h0, h1), bh1 = pack2<T>(h2, h3);
      const uint32_t bl0 = pack2<T>(r0, r1), bl1 = pack2<T>(r2, r3);
      mma_16816(d[0], f[0].x, f[1].x, f[0].y, f[1].y, bh0, bh1, T());
      mma_16816(d[1], f[2].x, f[3].x, f[2].y, f[3].y, bh0, bh1, T());
      mma_16816(d[0], f[0].x, f[1].x, f[0].y, f[1].y, bl0, bl1, T());
      mma_16816(d[1], f[2].x, f[3].x, f[2].y, f[3].y, bl0, bl1, T());
    }
    const float sc = __ldg(l.scales + a);
    if (ad0 == a) {
      lo[0] += sc * (d[0][0] * down0);
      lo[2] += sc * (d[0][2] * down0);
      hi[0] += sc * (d[1][0] * down0);
      hi[2] += sc * (d[1][2] * down0);
    }
    if (ad1 == a) {
      lo[1] += sc * (d[0][1] * down1);
      lo[3] += sc * (d[0][3] * down1);
      hi[1] += sc * (d[1][1] * down1);
      hi[3] += sc * (d[1][3] * down1);
    }
  }
}

}  // namespace moe

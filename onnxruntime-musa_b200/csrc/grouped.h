// Internal launch interface of the expert products (grouped_matmul and its gradients) and
// of the adapter projection (lora_matmul).  Not part of the public C ABI.
#pragma once

#include "moe_kernels.h"

namespace moe {

// Which of the three products of y[p] = W[e(p)] x[p] is formed.  `feat` is the output
// feature side, `con` the contraction; W is [E, N, K].
enum GroupedDir : int {
  kGmmForward = 0,     // y  [R, N]    = x [R, K] W[e]^T          feat = N, con = K
  kGmmGradInput = 1,   // dx [R, K]    = dy [R, N] W[e]           feat = K, con = N
  kGmmGradWeight = 2,  // dW [E, N, K] = dy_e^T x_e               con = the rows of e
};

struct GroupedArgs {
  int dtype;
  GroupedDir dir;
  int64_t rows;            // R
  int N, K, E;
  const void* x;           // [R, K]   (forward, grad_weight)
  const void* dy;          // [R, N]   (grad_input, grad_weight)
  const void* w;           // [E, N, K] (forward, grad_input)
  const int32_t* offsets;  // [E + 1]; nullptr: one group of all rows (E = 1)
  void* out;
  void* workspace = nullptr;  // grad_weight on tensor cores: padded row tails
  int* error = nullptr;       // where the tensor-core kernels report a wait that ran out
  int test_stall = 0;         // test hook: their producers issue no loads
};

// The adapter term of lora_matmul, added to the forward product of one group.
struct LoraTerm {
  int rank;               // r
  int adapters;           // L
  const void* b;          // [L, N, r]
  const int32_t* ids;     // [rows]; outside [0, L): no adapter
  // FFMA kernels: t = s_a A_a x in fp32, [rows][rank].
  const float* t;
  // Tensor-core kernels: s_a t in two 16-bit parts, [2][rows][rank] (grouped_lora.cuh);
  // fp16: the power of two that each row's parts are to be scaled by; and each row's adapter,
  // -1 for none, with kLoraScaled set where that power is not 1.
  const uint16_t* parts;
  int steps;              // ceil(rank / 16)
  const float* row_scale;
  const int* row_code;
};

// Largest feature and contraction length, and most rows, of a call (index arithmetic of
// the kernels: tile numbers and TMA coordinates in 32 bits, offsets in 64).
constexpr int64_t kGmmMaxDim = 1 << 20;
constexpr int64_t kGmmMaxRows = 1 << 30;
constexpr int kLoraMaxRank = 256;
constexpr int kLoraScaled = 1 << 24;  // above every adapter number

// t[row, j] = sum_k A_a[j, k] x[row, k] for rows with an adapter a (others are left).
struct LoraShrink {
  int dtype;
  int64_t rows;
  int K, rank, adapters;
  const void* x;           // [rows, K]
  const void* a;           // [L, r, K]
  const int32_t* ids;
  const float* scales;     // [L]
  int* error;              // as GroupedArgs
  int test_stall;
};
// Any type and alignment: s_a t in fp32, [rows][rank].
cudaError_t launch_lora_shrink_simt(const LoraShrink& l, float* t, cudaStream_t s);
// 16-bit types, K and rank multiples of 8, 16-byte aligned x and a: the parts of
// LoraTerm, its row_scale and row_code.
bool lora_shrink_tc_supported(const LoraShrink& l);
cudaError_t launch_lora_shrink_tc(const LoraShrink& l, uint16_t* parts, float* row_scale,
                                  int* row_code, int num_sms, cudaStream_t s);

// Tensor-core path: 16-bit types, N and K multiples of 8, 16-byte aligned buffers.
bool grouped_tc_supported(const GroupedArgs& g);
size_t grouped_tc_workspace(int dtype, GroupedDir dir, int64_t N, int64_t K, int64_t E);
// 256 x 256 tiles by CTA pairs, and weight streaming for few rows per group (not
// grad_weight).  `lora` (forward, one group, rank % 8 == 0) may be nullptr; its parts
// are awaited with pdl_wait().
cudaError_t launch_grouped_pair(const GroupedArgs& g, const LoraTerm* lora, int num_sms,
                                cudaStream_t s);
cudaError_t launch_grouped_small(const GroupedArgs& g, const LoraTerm* lora, int num_sms,
                                 cudaStream_t s);

// The whole adapter projection of a few rows in one launch (same types, sizes and alignment as
// the two launches; b: lora_b).
bool lora_few_supported(int64_t rows, int64_t rank);
cudaError_t launch_lora_few(const GroupedArgs& g, const LoraShrink& l, const void* b, int num_sms,
                            cudaStream_t s);

// FFMA kernels: any size, alignment and float type.
cudaError_t launch_grouped_simt(const GroupedArgs& g, const LoraTerm* lora, int num_sms,
                                cudaStream_t s);

}  // namespace moe

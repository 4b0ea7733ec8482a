// C entries of the expert products (moe_b200_grouped_matmul*) and the adapter projection
// (moe_b200_lora_matmul): argument checks and the choice of kernel.
#include <algorithm>
#include <atomic>
#include <cstdlib>
#include <cstring>
#include <initializer_list>
#include <mutex>

#include "../../include/moe_b200.h"
#include "grouped.h"

namespace {

using moe::set_error;

bool float_type(int32_t dt) {
  return dt == moe::kDtF32 || dt == moe::kDtF16 || dt == moe::kDtBF16;
}

int cuda_status(cudaError_t st, const char* what) {
  if (st == cudaSuccess) return MOE_B200_OK;
  return set_error(MOE_B200_EP_FAIL, "%s: %s", what, cudaGetErrorString(st));
}

int check_shape(const char* what, int32_t dtype, int64_t rows, int64_t n, int64_t k,
                int64_t groups, const char* group_name, int64_t max_groups) {
  if (!float_type(dtype))
    return set_error(MOE_B200_NOT_IMPLEMENTED, "%s: unsupported dtype %d", what, dtype);
  if (rows < 0 || rows > moe::kGmmMaxRows)
    return set_error(MOE_B200_INVALID_ARGUMENT, "%s: num_rows=%lld must be in [0, %lld]", what,
                     static_cast<long long>(rows), static_cast<long long>(moe::kGmmMaxRows));
  if (n < 1 || n > moe::kGmmMaxDim || k < 1 || k > moe::kGmmMaxDim)
    return set_error(MOE_B200_INVALID_ARGUMENT, "%s: n=%lld and k=%lld must be in [1, %lld]", what,
                     static_cast<long long>(n), static_cast<long long>(k),
                     static_cast<long long>(moe::kGmmMaxDim));
  if (groups < 1 || groups > max_groups)
    return set_error(MOE_B200_INVALID_ARGUMENT, "%s: %s=%lld must be in [1, %lld]", what,
                     group_name, static_cast<long long>(groups),
                     static_cast<long long>(max_groups));
  return MOE_B200_OK;
}

// Every buffer must be aligned to its element size (the kernels pick wider loads by the
// alignment they find).
int check_pointers(const char* what, int32_t dtype, const void* const* ptrs, int n,
                   const void* const* words, int nw) {
  const uintptr_t es = static_cast<uintptr_t>(moe::dtype_bytes(dtype));
  for (int i = 0; i < n + nw; ++i) {
    const void* q = i < n ? ptrs[i] : words[i - n];
    if (q == nullptr)
      return set_error(MOE_B200_INVALID_ARGUMENT, "%s: buffers must be non-NULL", what);
    if (reinterpret_cast<uintptr_t>(q) % (i < n ? es : 4) != 0)
      return set_error(MOE_B200_INVALID_ARGUMENT,
                       "%s: buffers must be aligned to their element size", what);
  }
  return MOE_B200_OK;
}

struct Range {
  const void* at;
  int64_t bytes;
};

// What a call writes must not lie in what it reads: tiles finish in any order.
int check_overlap(const char* what, const Range& written, std::initializer_list<Range> others) {
  const uintptr_t w = reinterpret_cast<uintptr_t>(written.at);
  for (const Range& r : others) {
    const uintptr_t q = reinterpret_cast<uintptr_t>(r.at);
    if (w < q + static_cast<uintptr_t>(r.bytes) && q < w + static_cast<uintptr_t>(written.bytes))
      return set_error(MOE_B200_INVALID_ARGUMENT,
                       "%s: outputs and the workspace must not overlap other buffers", what);
  }
  return MOE_B200_OK;
}

int sm_count() {
  static std::atomic<int> counts[64];
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  n = counts[dev].load(std::memory_order_relaxed);
  if (n == 0) {
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 148;
    counts[dev].store(n, std::memory_order_relaxed);
  }
  return n;
}

bool env_flag(const char* name) {
  const char* v = std::getenv(name);
  return v != nullptr && v[0] != '\0' && std::strcmp(v, "0") != 0;
}

// Words of pinned host memory in which kernels report a wait that ran out: one for every device,
// which the next call on it looks at (and moe_b200_take_device_error), and some that traced calls
// take in turn, so that each finds its own error.  Allocated once, for the life of the process
// (a captured graph keeps the address); nullptr if that fails.
constexpr int kDevices = 64, kTracedCalls = 64;
std::atomic<int*> g_error_words{nullptr};

int* error_words() {
  int* words = g_error_words.load(std::memory_order_acquire);
  if (words != nullptr) return words;
  static std::mutex mutex;
  std::lock_guard<std::mutex> lock(mutex);
  words = g_error_words.load(std::memory_order_acquire);
  if (words != nullptr) return words;
  // The first call may be captured: allocating is no work on a stream, so it may be done then.
  cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
  if (cudaThreadExchangeStreamCaptureMode(&mode) != cudaSuccess) return nullptr;
  void* at = nullptr;
  const cudaError_t st = cudaHostAlloc(&at, (kDevices + kTracedCalls) * sizeof(int),
                                       cudaHostAllocPortable | cudaHostAllocMapped);
  cudaThreadExchangeStreamCaptureMode(&mode);
  if (st != cudaSuccess) return nullptr;
  words = static_cast<int*>(at);
  std::fill(words, words + kDevices + kTracedCalls, 0);
  g_error_words.store(words, std::memory_order_release);
  return words;
}

int* device_word(int* words) {
  int dev = 0;
  return words + (cudaGetDevice(&dev) == cudaSuccess && dev > 0 ? dev % kDevices : 0);
}

// Reads and clears a word; the store of a kernel may come at any time.
int take_word(int* word) {
  return *static_cast<volatile int*>(word) == 0 ? 0 : __atomic_exchange_n(word, 0, __ATOMIC_ACQ_REL);
}

struct Call {
  int* error;   // the kernels' word
  bool traced;  // MOE_B200_TRACE_SYNC: wait for the call and report its own error (not of a captured
                // call, which has not run when it returns: its replays report as untraced calls)
  int stall;    // MOE_B200_TEST_STALL: the tensor-core kernels' producers issue no loads
};

// In front of a call's launches.  An earlier call whose wait ran out has left its output
// incomplete and nobody has been told: this one reports it and does nothing.
int begin(const char* what, Call* c, cudaStream_t s) {
  int* words = error_words();
  if (words == nullptr)
    return set_error(MOE_B200_EP_FAIL, "%s: no pinned host memory for the error words", what);
  c->error = device_word(words);
  const int err = take_word(c->error);
  if (err != 0)
    return set_error(MOE_B200_EP_FAIL,
                     "%s: an earlier expert product or adapter projection on this device gave up "
                     "waiting and its output is incomplete (device error code %d); this call was "
                     "not made", what, err);
  c->stall = env_flag("MOE_B200_TEST_STALL") ? 1 : 0;
  if (env_flag("MOE_B200_TRACE_SYNC")) {
    cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
    const int rc = cuda_status(cudaStreamIsCapturing(s, &capture), what);
    if (rc != MOE_B200_OK) return rc;
    c->traced = capture == cudaStreamCaptureStatusNone;
  }
  if (c->traced) {
    static std::atomic<unsigned> turn{0};
    c->error = words + kDevices + turn.fetch_add(1, std::memory_order_relaxed) % kTracedCalls;
    take_word(c->error);
  }
  return MOE_B200_OK;
}

// Behind them.
int finish(const char* what, const Call& c, cudaStream_t s) {
  if (!c.traced) return MOE_B200_OK;
  const int rc = cuda_status(cudaStreamSynchronize(s), what);
  if (rc != MOE_B200_OK) return rc;
  const int err = take_word(c.error);
  return err == 0 ? MOE_B200_OK : set_error(MOE_B200_EP_FAIL, "%s: device error code %d", what, err);
}

// The CTA-pair kernel or the weight-streaming kernel, by what was measured (bf16, us, forward /
// grad_input, streaming : pair):
//   8 experts [4096, 4096]   64 rows each 49 : 52 / 45 : 50, 96 rows 60 : 54 / 61 : 51,
//                            256 rows 95 : 75 / 99 : 82
//   64 experts [768, 2048]   16 rows each 41.2 : 41.0 / 44.5 : 38.6 (a contraction of 768)
//   1 group [4096, 4096]     192 rows 14.7 : 25.0, 1024 rows 34 : 30
// The pair kernel needs tiles for the SM pairs; then it wins from about 80 rows a group, and
// with short contractions for any number, because it is persistent (the streaming kernel pays
// its start-up for every tile).
bool use_pair(const moe::GroupedArgs& g, int sms) {
  if (g.dir == moe::kGmmGradWeight) return true;
  const int64_t feat = g.dir == moe::kGmmForward ? g.N : g.K;
  const int64_t con = g.dir == moe::kGmmForward ? g.K : g.N;
  const int64_t groups = std::min<int64_t>(g.rows, g.E), per = g.rows / groups;
  const int64_t tiles = (per + 255) / 256 * groups * ((feat + 255) / 256);
  const int pairs = sms / 2;
  return (per >= 80 && tiles >= pairs * 3 / 4) || (con <= 2048 && tiles >= 2 * pairs);
}

cudaError_t launch_tc(const moe::GroupedArgs& g, const moe::LoraTerm* lora, cudaStream_t s) {
  const int sms = sm_count();
  return use_pair(g, sms) ? moe::launch_grouped_pair(g, lora, sms, s)
                          : moe::launch_grouped_small(g, lora, sms, s);
}

int run_grouped(const char* what, moe::GroupedArgs& g, cudaStream_t s) {
  Call call{};
  int rc = begin(what, &call, s);
  if (rc != MOE_B200_OK) return rc;
  g.error = call.error;
  g.test_stall = call.stall;
  const cudaError_t st = moe::grouped_tc_supported(g) ? launch_tc(g, nullptr, s)
                                                      : moe::launch_grouped_simt(g, nullptr, sm_count(), s);
  rc = cuda_status(st, what);
  return rc != MOE_B200_OK ? rc : finish(what, call, s);
}

// Workspace of lora_matmul: four bytes per row and rank entry (two 16-bit parts, or t in
// fp32), then a float and an int per row.
size_t lora_parts_bytes(int64_t rows, int64_t rank) {
  return (static_cast<size_t>(rows) * static_cast<size_t>(rank) * 4 + 15) & ~size_t{15};
}
size_t lora_bytes(int64_t rows, int64_t rank) {
  return lora_parts_bytes(rows, rank) + static_cast<size_t>(rows) * 8;
}

}  // namespace

extern "C" {

int moe_b200_take_device_error(int32_t* code) {
  static const char* kWhat = "take_device_error";
  if (code == nullptr)
    return set_error(MOE_B200_INVALID_ARGUMENT, "%s: code must be non-NULL", kWhat);
  int* words = g_error_words.load(std::memory_order_acquire);
  *code = words == nullptr ? 0 : take_word(device_word(words));
  return MOE_B200_OK;
}

int moe_b200_grouped_matmul(int32_t dtype, int64_t num_rows, int64_t n, int64_t k,
                            int64_t num_experts, const void* x, const void* weights,
                            const int32_t* expert_offsets, void* y, void* stream) {
  static const char* kWhat = "grouped_matmul";
  moe::clear_stale_cuda_error();
  int rc = check_shape(kWhat, dtype, num_rows, n, k, num_experts, "num_experts", moe::kMaxExperts);
  if (rc != MOE_B200_OK || num_rows == 0) return rc;
  const void* ptrs[] = {x, weights, y};
  const void* words[] = {expert_offsets};
  rc = check_pointers(kWhat, dtype, ptrs, 3, words, 1);
  if (rc != MOE_B200_OK) return rc;
  const int64_t es = moe::dtype_bytes(dtype);
  rc = check_overlap(kWhat, {y, num_rows * n * es},
                     {{x, num_rows * k * es}, {weights, num_experts * n * k * es},
                      {expert_offsets, (num_experts + 1) * 4}});
  if (rc != MOE_B200_OK) return rc;
  moe::GroupedArgs g{};
  g.dtype = dtype;
  g.dir = moe::kGmmForward;
  g.rows = num_rows;
  g.N = static_cast<int>(n);
  g.K = static_cast<int>(k);
  g.E = static_cast<int>(num_experts);
  g.x = x;
  g.w = weights;
  g.offsets = expert_offsets;
  g.out = y;
  return run_grouped(kWhat, g, static_cast<cudaStream_t>(stream));
}

int moe_b200_grouped_matmul_grad_input(int32_t dtype, int64_t num_rows, int64_t n, int64_t k,
                                       int64_t num_experts, const void* dy, const void* weights,
                                       const int32_t* expert_offsets, void* dx, void* stream) {
  static const char* kWhat = "grouped_matmul_grad_input";
  moe::clear_stale_cuda_error();
  int rc = check_shape(kWhat, dtype, num_rows, n, k, num_experts, "num_experts", moe::kMaxExperts);
  if (rc != MOE_B200_OK || num_rows == 0) return rc;
  const void* ptrs[] = {dy, weights, dx};
  const void* words[] = {expert_offsets};
  rc = check_pointers(kWhat, dtype, ptrs, 3, words, 1);
  if (rc != MOE_B200_OK) return rc;
  const int64_t es = moe::dtype_bytes(dtype);
  rc = check_overlap(kWhat, {dx, num_rows * k * es},
                     {{dy, num_rows * n * es}, {weights, num_experts * n * k * es},
                      {expert_offsets, (num_experts + 1) * 4}});
  if (rc != MOE_B200_OK) return rc;
  moe::GroupedArgs g{};
  g.dtype = dtype;
  g.dir = moe::kGmmGradInput;
  g.rows = num_rows;
  g.N = static_cast<int>(n);
  g.K = static_cast<int>(k);
  g.E = static_cast<int>(num_experts);
  g.dy = dy;
  g.w = weights;
  g.offsets = expert_offsets;
  g.out = dx;
  return run_grouped(kWhat, g, static_cast<cudaStream_t>(stream));
}

int moe_b200_grouped_matmul_grad_weight_workspace_size(int32_t dtype, int64_t n, int64_t k,
                                                       int64_t num_experts, size_t* bytes) {
  static const char* kWhat = "grouped_matmul_grad_weight_workspace_size";
  int rc = check_shape(kWhat, dtype, 0, n, k, num_experts, "num_experts", moe::kMaxExperts);
  if (rc != MOE_B200_OK) return rc;
  if (bytes == nullptr)
    return set_error(MOE_B200_INVALID_ARGUMENT, "%s: bytes must be non-NULL", kWhat);
  *bytes = moe::grouped_tc_workspace(dtype, moe::kGmmGradWeight, n, k, num_experts);
  return MOE_B200_OK;
}

int moe_b200_grouped_matmul_grad_weight(int32_t dtype, int64_t num_rows, int64_t n, int64_t k,
                                        int64_t num_experts, const void* x, const void* dy,
                                        const int32_t* expert_offsets, void* dw, void* workspace,
                                        size_t workspace_bytes, void* stream) {
  static const char* kWhat = "grouped_matmul_grad_weight";
  moe::clear_stale_cuda_error();
  int rc = check_shape(kWhat, dtype, num_rows, n, k, num_experts, "num_experts", moe::kMaxExperts);
  if (rc != MOE_B200_OK) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (num_rows == 0) {  // no rows: every expert's gradient is zero
    const void* out[] = {dw};
    rc = check_pointers(kWhat, dtype, out, 1, nullptr, 0);
    if (rc != MOE_B200_OK) return rc;
    return cuda_status(cudaMemsetAsync(dw, 0,
                                       static_cast<size_t>(num_experts) * n * k *
                                           moe::dtype_bytes(dtype), s),
                       kWhat);
  }
  const void* ptrs[] = {x, dy, dw};
  const void* words[] = {expert_offsets};
  rc = check_pointers(kWhat, dtype, ptrs, 3, words, 1);
  if (rc != MOE_B200_OK) return rc;
  size_t need = 0;
  rc = moe_b200_grouped_matmul_grad_weight_workspace_size(dtype, n, k, num_experts, &need);
  if (rc != MOE_B200_OK) return rc;
  if (workspace_bytes < need || (need > 0 && (workspace == nullptr ||
                                              reinterpret_cast<uintptr_t>(workspace) % 256 != 0)))
    return set_error(MOE_B200_INVALID_ARGUMENT,
                     "%s: workspace must be 256-byte aligned and hold %zu bytes", kWhat, need);
  const int64_t es = moe::dtype_bytes(dtype);
  const Range in[] = {{x, num_rows * k * es}, {dy, num_rows * n * es},
                      {expert_offsets, (num_experts + 1) * 4}};
  const Range ws = {workspace, static_cast<int64_t>(need)};
  rc = check_overlap(kWhat, {dw, num_experts * n * k * es}, {in[0], in[1], in[2], ws});
  if (rc == MOE_B200_OK) rc = check_overlap(kWhat, ws, {in[0], in[1], in[2]});
  if (rc != MOE_B200_OK) return rc;
  moe::GroupedArgs g{};
  g.dtype = dtype;
  g.dir = moe::kGmmGradWeight;
  g.rows = num_rows;
  g.N = static_cast<int>(n);
  g.K = static_cast<int>(k);
  g.E = static_cast<int>(num_experts);
  g.x = x;
  g.dy = dy;
  g.offsets = expert_offsets;
  g.out = dw;
  g.workspace = workspace;
  return run_grouped(kWhat, g, s);
}

int moe_b200_lora_matmul_workspace_size(int32_t dtype, int64_t num_rows, int64_t rank,
                                        size_t* bytes) {
  static const char* kWhat = "lora_matmul_workspace_size";
  int rc = check_shape(kWhat, dtype, num_rows, 1, 1, rank, "rank", moe::kLoraMaxRank);
  if (rc != MOE_B200_OK) return rc;
  if (bytes == nullptr)
    return set_error(MOE_B200_INVALID_ARGUMENT, "%s: bytes must be non-NULL", kWhat);
  *bytes = lora_bytes(num_rows, rank);
  return MOE_B200_OK;
}

int moe_b200_lora_matmul(int32_t dtype, int64_t num_rows, int64_t n, int64_t k,
                         int64_t num_adapters, int64_t rank, const void* x, const void* weight,
                         const void* lora_a, const void* lora_b, const int32_t* adapter_ids,
                         const float* scales, void* y, void* workspace, size_t workspace_bytes,
                         void* stream) {
  static const char* kWhat = "lora_matmul";
  moe::clear_stale_cuda_error();
  int rc = check_shape(kWhat, dtype, num_rows, n, k, num_adapters, "num_adapters",
                       moe::kGmmMaxDim);
  if (rc != MOE_B200_OK) return rc;
  if (rank < 1 || rank > moe::kLoraMaxRank)
    return set_error(MOE_B200_INVALID_ARGUMENT, "%s: rank=%lld must be in [1, %d]", kWhat,
                     static_cast<long long>(rank), moe::kLoraMaxRank);
  if (num_rows == 0) return MOE_B200_OK;
  const void* ptrs[] = {x, weight, lora_a, lora_b, y};
  const void* words[] = {adapter_ids, scales};
  rc = check_pointers(kWhat, dtype, ptrs, 5, words, 2);
  if (rc != MOE_B200_OK) return rc;
  const size_t need = lora_bytes(num_rows, rank);
  if (workspace_bytes < need || workspace == nullptr ||
      reinterpret_cast<uintptr_t>(workspace) % 256 != 0)
    return set_error(MOE_B200_INVALID_ARGUMENT,
                     "%s: workspace must be 256-byte aligned and hold %zu bytes", kWhat, need);
  const int64_t es = moe::dtype_bytes(dtype);
  const Range in[] = {{x, num_rows * k * es}, {weight, n * k * es},
                      {lora_a, num_adapters * rank * k * es},
                      {lora_b, num_adapters * n * rank * es}, {adapter_ids, num_rows * 4},
                      {scales, num_adapters * 4}};
  const Range ws = {workspace, static_cast<int64_t>(need)};
  rc = check_overlap(kWhat, {y, num_rows * n * es}, {in[0], in[1], in[2], in[3], in[4], in[5], ws});
  if (rc == MOE_B200_OK) rc = check_overlap(kWhat, ws, {in[0], in[1], in[2], in[3], in[4], in[5]});
  if (rc != MOE_B200_OK) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  Call call{};
  rc = begin(kWhat, &call, s);
  if (rc != MOE_B200_OK) return rc;
  moe::LoraShrink l{};
  l.dtype = dtype;
  l.rows = num_rows;
  l.K = static_cast<int>(k);
  l.rank = static_cast<int>(rank);
  l.adapters = static_cast<int>(num_adapters);
  l.x = x;
  l.a = lora_a;
  l.ids = adapter_ids;
  l.scales = scales;
  l.error = call.error;
  l.test_stall = call.stall;
  moe::GroupedArgs g{};
  g.dtype = dtype;
  g.dir = moe::kGmmForward;
  g.rows = num_rows;
  g.N = static_cast<int>(n);
  g.K = static_cast<int>(k);
  g.E = 1;
  g.x = x;
  g.w = weight;
  g.out = y;
  g.error = call.error;
  g.test_stall = call.stall;
  const bool a16 = (reinterpret_cast<uintptr_t>(lora_b) & 15) == 0;
  const bool tc = moe::grouped_tc_supported(g) && moe::lora_shrink_tc_supported(l) && a16;
  if (tc && moe::lora_few_supported(num_rows, rank)) {
    rc = cuda_status(moe::launch_lora_few(g, l, lora_b, sm_count(), s), kWhat);
    return rc != MOE_B200_OK ? rc : finish(kWhat, call, s);
  }
  moe::LoraTerm term{};
  term.rank = l.rank;
  term.adapters = l.adapters;
  term.b = lora_b;
  term.ids = adapter_ids;
  cudaError_t st;
  if (tc) {
    auto* parts = static_cast<uint16_t*>(workspace);
    auto* row_scale = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) +
                                               lora_parts_bytes(num_rows, rank));
    auto* row_code = reinterpret_cast<int*>(row_scale + num_rows);
    st = moe::launch_lora_shrink_tc(l, parts, row_scale, row_code, sm_count(), s);
    term.parts = parts;
    term.steps = static_cast<int>((rank + 15) / 16);
    term.row_scale = row_scale;
    term.row_code = row_code;
  } else {
    auto* t = static_cast<float*>(workspace);
    st = moe::launch_lora_shrink_simt(l, t, s);
    term.t = t;
  }
  rc = cuda_status(st, kWhat);
  if (rc != MOE_B200_OK) return rc;
  rc = cuda_status(tc ? launch_tc(g, &term, s) : moe::launch_grouped_simt(g, &term, sm_count(), s), kWhat);
  return rc != MOE_B200_OK ? rc : finish(kWhat, call, s);
}

}  // extern "C"

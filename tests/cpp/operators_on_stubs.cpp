// The entry points of hc_ops.cu on a library whose launches are only counted: what they refuse, without a GPU.
// Built by tests/test_entry_points_host.py with the host compiler, together with hc_ops.cu itself.
#include <mutex>
#include <string>

#include "../../honeycrisp_b200/csrc/common.cuh"

static std::mutex mu;
static std::string message;
static int enqueued = 0;

extern "C" {
int stub_enqueued() { int n = enqueued; enqueued = 0; return n; }
const char* stub_message() { return message.c_str(); }
cudaError_t cudaGetDevice(int* d) { *d = 0; return cudaSuccess; }
cudaError_t cudaSetDevice(int) { return cudaSuccess; }
cudaError_t cudaMemsetAsync(void*, int, size_t, cudaStream_t) { enqueued++; return cudaSuccess; }
}

namespace hc {
std::mutex& ctx_mutex(hc_ctx*) { return mu; }
cudaStream_t ctx_stream(hc_ctx*) { return nullptr; }
unsigned int* ctx_status_word(hc_ctx*) { return nullptr; }
int ctx_sm_count(hc_ctx*) { return 148; }
int ctx_device(hc_ctx*) { return 0; }
hc_status ctx_fail(hc_ctx*, hc_status s, const char* m) { message = m; return s; }
hc_status ctx_cuda_fail(hc_ctx*, cudaError_t, const char* m) { message = m; return HC_ERR_CUDA; }
void ctx_note_launch(hc_ctx*, const LaunchRecord&, int64_t) {}
void ctx_count_launches(hc_ctx*, int) {}
void tc_forget_predecessor(cudaStream_t) {}
hc_status ctx_scratch(hc_ctx*, size_t, void** p) { *p = (void*)256; return HC_OK; }
hc_status ctx_build_problem(hc_ctx*, hc_dtype, int64_t, const void*, int, const void*, int, int, int64_t, int64_t, int64_t, void*, GemmProblem*) { return HC_OK; }
hc_status ctx_run_problem(hc_ctx*, const GemmProblem&, int64_t) { enqueued++; return HC_OK; }
cudaError_t launch_grouped(const GroupedProblem&, cudaStream_t, unsigned int*, void*, size_t, int, LaunchRecord*, size_t*) { enqueued++; return cudaSuccess; }
size_t activation_grad_scratch(hc_dtype, int64_t, int64_t) { return 1; }
size_t layer_norm_grad_scratch(hc_dtype, int64_t, int64_t, int) { return 1; }
cudaError_t launch_activation_grad(hc_dtype, int, const void*, const void*, int64_t, int64_t, void*, float*, float*, int*, cudaStream_t) { enqueued++; return cudaSuccess; }
cudaError_t launch_layer_norm(hc_dtype, hc_dtype, const void*, const void*, const void*, int64_t, int64_t, float, void*, float*, float*, int, cudaStream_t) { enqueued++; return cudaSuccess; }
cudaError_t launch_layer_norm_grad(hc_dtype, hc_dtype, const void*, const void*, const void*, const float*, const float*, int64_t, int64_t, void*, void*, void*, float*, int, int*, cudaStream_t) { enqueued++; return cudaSuccess; }
cudaError_t launch_adamw(const hc_adamw_tensor*, int64_t, const AdamWFactors&, int*, cudaStream_t) { enqueued++; return cudaSuccess; }
}  // namespace hc

// One AdamW step over many tensors in one launch (for every kMaxTensors of them):
//   m = b1 m + (1 - b1) g      v = b2 v + (1 - b2) g^2
//   p = p (1 - lr wd) - lr (m / c1) / (sqrt(v / c2) + eps),   c = 1 - b^step
// in float32 whatever the parameter's and gradient's types, p rounded once.  HBM-bound: it reads p, g, m, v and writes
// p, m, v and, for layers that compute in float16 on float32 master weights, a float16 copy of p.
//
// The tensors' table travels as a kernel parameter, so nothing is copied to the device and a graph holds the table.
// Every tensor is cut into chunks of kChunk elements; CTA i takes chunk i and finds its tensor by bisection over the
// table's first chunks.
#include "common.cuh"
#include "epilogue.cuh"
#include "stream_order.cuh"

namespace hc {
namespace {

constexpr int kMaxTensors = 448;          // 448 x 56 bytes: below the 32764 bytes of kernel parameters
constexpr int kThreads = 256;
constexpr int kChunk = kThreads * 16;     // elements a CTA updates

struct AdamTensor {
  void* p;
  const void* g;
  float *m, *v;
  __half* copy;
  int64_t count;
  uint32_t first_chunk;
  uint16_t p_half, g_half;
};
struct AdamJob {
  AdamTensor t[kMaxTensors];
  int n;
  AdamWFactors f;
};
static_assert(sizeof(AdamJob) <= 32764, "kernel parameters");

__device__ __forceinline__ float adam_one(const AdamWFactors& f, float g, float& m, float& v, float p) {
  m = fmaf(f.beta1, m, f.one_minus_beta1 * g);
  v = fmaf(f.beta2, v, f.one_minus_beta2 * g * g);
  return p * f.decay - f.lr * (m * f.inv_c1) / (sqrtf(v * f.inv_c2) + f.epsilon);
}

__global__ void __launch_bounds__(kThreads) adamw_kernel(const __grid_constant__ AdamJob j) {
  pdl_wait();
  int lo = 0, hi = j.n - 1;
  while (lo < hi) {   // the last tensor whose first chunk is not beyond this CTA's
    const int mid = (lo + hi + 1) / 2;
    if (j.t[mid].first_chunk <= blockIdx.x) lo = mid;
    else hi = mid - 1;
  }
  const AdamTensor& t = j.t[lo];
  const int64_t base = (int64_t)(blockIdx.x - t.first_chunk) * kChunk;
  const int n = (int)min((int64_t)kChunk, t.count - base);
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const int64_t k = base + i;
    const float g = t.g_half ? __half2float(((const __half*)t.g)[k]) : ((const float*)t.g)[k];
    const float p = t.p_half ? __half2float(((const __half*)t.p)[k]) : ((const float*)t.p)[k];
    float m = t.m[k], v = t.v[k];
    const float q = adam_one(j.f, g, m, v, p);
    t.m[k] = m;
    t.v[k] = v;
    if (t.p_half) ((__half*)t.p)[k] = __float2half_rn(q);
    else ((float*)t.p)[k] = q;
    if (t.copy) t.copy[k] = __float2half_rn(q);
  }
}

}  // namespace

cudaError_t launch_adamw(const hc_adamw_tensor* tensors, int64_t count, const AdamWFactors& f, int* launches, cudaStream_t stream) {
  *launches = 0;
  AdamJob j;
  j.f = f;
  int64_t i = 0;
  while (i < count) {
    j.n = 0;
    uint64_t chunks = 0;
    for (; i < count && j.n < kMaxTensors; i++) {
      const hc_adamw_tensor& a = tensors[i];
      if (a.count == 0) continue;
      const uint64_t c = ((uint64_t)a.count + kChunk - 1) / kChunk;
      if (c > 2147483647ull) return cudaErrorInvalidValue;
      if (chunks + c > 2147483647ull) break;
      AdamTensor& t = j.t[j.n++];
      t.p = a.param; t.g = a.grad; t.m = a.moment1; t.v = a.moment2; t.copy = (__half*)a.param_copy; t.count = a.count;
      t.first_chunk = (uint32_t)chunks;
      t.p_half = a.param_dtype == HC_F16; t.g_half = a.grad_dtype == HC_F16;
      chunks += c;
    }
    if (j.n == 0) continue;
    void* args[] = {(void*)&j};
    cudaError_t e = launch_behind((const void*)adamw_kernel, args, dim3((unsigned)chunks), dim3(kThreads), 0, stream);
    if (e != cudaSuccess) return e;
    *launches += 1;
  }
  return cudaSuccess;
}

}  // namespace hc

// One AdamW step over many tensors in one launch (for every kMaxTensors of them):
//   m = b1 m + (1 - b1) g      v = b2 v + (1 - b2) g^2
//   p = p (1 - lr wd) - lr (m / c1) / (sqrt(v / c2) + eps),   c = 1 - b^step
// in float32 whatever the parameter's and gradient's types, p rounded once.  HBM-bound: it reads p, g, m, v and writes
// p, m, v and, for layers that compute in float16 on float32 master weights, a float16 copy of p.
//
// The tensors' table travels as a kernel parameter, so nothing is copied to the device and a graph holds the table.
// Every tensor is cut into chunks of kChunk elements; CTA i takes chunk i and finds its tensor by bisection over the
// table's first chunks.
#include <cstring>

#include "common.cuh"
#include "epilogue.cuh"
#include "stream_order.cuh"

namespace hc {
namespace {

constexpr int kMaxTensors = 448;          // 448 x 56 bytes: below the 32764 bytes of kernel parameters
constexpr int kThreads = 256;
constexpr int kQuads = 2;                 // groups of four elements a thread updates
constexpr int kChunk = kThreads * kQuads * 4;

struct AdamTensor {
  void* p;
  const void* g;
  float *m, *v;
  __half* copy;
  int64_t count;
  uint32_t first_chunk;
  uint8_t p_half, g_half;
  uint8_t head;      // elements in front of the first one that vector accesses may take; 255: none may
  uint8_t unused;
};
// The table as a kernel parameter, in three sizes: the launch copies all of it.
template <int kMax>
struct AdamJob {
  AdamTensor t[kMax];
  int n;
  AdamWFactors f;
};
static_assert(sizeof(AdamJob<kMaxTensors>) <= 32764, "kernel parameters");

__device__ __forceinline__ float adam_one(const AdamWFactors& f, float g, float& m, float& v, float p) {
  m = fmaf(f.beta1, m, f.one_minus_beta1 * g);
  v = fmaf(f.beta2, v, f.one_minus_beta2 * g * g);
  return p * f.decay - f.lr * (m * f.inv_c1) / (sqrtf(v * f.inv_c2) + f.epsilon);
}

__device__ __forceinline__ void adam_element(const AdamWFactors& f, const AdamTensor& t, int64_t k) {
  const float g = t.g_half ? __half2float(((const __half*)t.g)[k]) : ((const float*)t.g)[k];
  const float p = t.p_half ? __half2float(((const __half*)t.p)[k]) : ((const float*)t.p)[k];
  float m = t.m[k], v = t.v[k];
  const float q = adam_one(f, g, m, v, p);
  t.m[k] = m;
  t.v[k] = v;
  if (t.p_half) ((__half*)t.p)[k] = __float2half_rn(q);
  else ((float*)t.p)[k] = q;
  if (t.copy) t.copy[k] = __float2half_rn(q);
}

__device__ __forceinline__ float4 load_four(const void* p, int half, int64_t k) {
  if (!half) return __ldcs((const float4*)((const float*)p + k));
  const uint2 u = __ldcs((const uint2*)((const __half*)p + k));
  const float2 a = __half22float2(*(const __half2*)&u.x), b = __half22float2(*(const __half2*)&u.y);
  return make_float4(a.x, a.y, b.x, b.y);
}
__device__ __forceinline__ void store_four(void* p, int half, int64_t k, const float4& x) {
  if (!half) {
    __stcs((float4*)((float*)p + k), x);
  } else {
    const __half2 a = __floats2half2_rn(x.x, x.y), b = __floats2half2_rn(x.z, x.w);
    __stcs((uint2*)((__half*)p + k), make_uint2(*(const uint32_t*)&a, *(const uint32_t*)&b));
  }
}

// A CTA updates kChunk elements of one tensor.  All of a thread's quads are read before the first is written, which
// keeps eight loads in flight, of 16 bytes each (8 of float16); the few elements around the aligned quads go one by one.
template <int kMax>
__global__ void __launch_bounds__(kThreads) adamw_kernel(const __grid_constant__ AdamJob<kMax> j) {
  int lo = 0, hi = j.n - 1;
  while (lo < hi) {   // the last tensor whose first chunk is not beyond this CTA's
    const int mid = (lo + hi + 1) / 2;
    if (j.t[mid].first_chunk <= blockIdx.x) lo = mid;
    else hi = mid - 1;
  }
  const AdamTensor& t = j.t[lo];
  const int64_t base = (int64_t)(blockIdx.x - t.first_chunk) * kChunk;
  const int n = (int)min((int64_t)kChunk, t.count - base);
  pdl_wait();
  if (t.head == 255) {
    for (int i = threadIdx.x; i < n; i += kThreads) adam_element(j.f, t, base + i);
    return;
  }
  const int head = min((int)t.head, n), quads = (n - head) / 4, tail = head + quads * 4;
  const int64_t first = base + head;
  float4 g[kQuads], p[kQuads], m[kQuads], v[kQuads];
#pragma unroll
  for (int i = 0; i < kQuads; i++) {
    const int q = threadIdx.x + i * kThreads;
    if (q < quads) {
      g[i] = load_four(t.g, t.g_half, first + q * 4);
      p[i] = load_four(t.p, t.p_half, first + q * 4);
      m[i] = load_four(t.m, 0, first + q * 4);
      v[i] = load_four(t.v, 0, first + q * 4);
    }
  }
#pragma unroll
  for (int i = 0; i < kQuads; i++) {
    const int q = threadIdx.x + i * kThreads;
    if (q < quads) {
      p[i].x = adam_one(j.f, g[i].x, m[i].x, v[i].x, p[i].x);
      p[i].y = adam_one(j.f, g[i].y, m[i].y, v[i].y, p[i].y);
      p[i].z = adam_one(j.f, g[i].z, m[i].z, v[i].z, p[i].z);
      p[i].w = adam_one(j.f, g[i].w, m[i].w, v[i].w, p[i].w);
      store_four(t.p, t.p_half, first + q * 4, p[i]);
      store_four(t.m, 0, first + q * 4, m[i]);
      store_four(t.v, 0, first + q * 4, v[i]);
      if (t.copy) store_four(t.copy, 1, first + q * 4, p[i]);
    }
  }
  if ((int)threadIdx.x < head) adam_element(j.f, t, base + threadIdx.x);
  if ((int)threadIdx.x < n - tail) adam_element(j.f, t, base + tail + threadIdx.x);
}

// Elements in front of the first quad that lies on four-element boundaries of every buffer; 255 where they disagree.
uint8_t head_of(const hc_adamw_tensor& a) {
  const int pe = a.param_dtype == HC_F16 ? 2 : 4, ge = a.grad_dtype == HC_F16 ? 2 : 4;
  const int at = (int)((uintptr_t)a.moment1 / 4 % 4);
  const bool same = (int)((uintptr_t)a.moment2 / 4 % 4) == at && (int)((uintptr_t)a.param / pe % 4) == at &&
                    (int)((uintptr_t)a.grad / ge % 4) == at && (!a.param_copy || (int)((uintptr_t)a.param_copy / 2 % 4) == at);
  return same ? (uint8_t)((4 - at) % 4) : 255;
}

template <int kMax>
cudaError_t launch_sized(const AdamJob<kMaxTensors>& all, int64_t chunks, cudaStream_t stream) {
  AdamJob<kMax> j;
  memcpy(j.t, all.t, sizeof(AdamTensor) * (size_t)all.n);
  j.n = all.n;
  j.f = all.f;
  void* args[] = {(void*)&j};
  return launch_behind((const void*)adamw_kernel<kMax>, args, dim3((unsigned)chunks), dim3(kThreads), 0, stream);
}

}  // namespace

cudaError_t launch_adamw(const hc_adamw_tensor* tensors, int64_t count, const AdamWFactors& f, int* launches, cudaStream_t stream) {
  *launches = 0;
  AdamJob<kMaxTensors> j;
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
      t.head = head_of(a);
      chunks += c;
    }
    if (j.n == 0) continue;
    cudaError_t e = j.n <= 24 ? launch_sized<24>(j, (int64_t)chunks, stream)
                    : j.n <= 96 ? launch_sized<96>(j, (int64_t)chunks, stream) : launch_sized<kMaxTensors>(j, (int64_t)chunks, stream);
    if (e != cudaSuccess) return e;
    *launches += 1;
  }
  return cudaSuccess;
}

}  // namespace hc

// Layer normalisation over the last axis, forward and backward.
//
//   mean = sum(x) / n      rstd = 1 / sqrt(sum((x - mean)^2) / n + epsilon)      h = (x - mean) rstd
//   out  = h w + b
//   dx   = rstd (g w - mean(g w) - h mean(g w h))      dw = sum_rows g h      db = sum_rows g
//
// All sums are float32; the variance is summed from the differences, a second pass over values that are still in
// registers, so that a large mean does not cancel.  HBM-bound.
#include "common.cuh"
#include "epilogue.cuh"
#include "stream_order.cuh"

namespace hc {
namespace {

struct NormJob {
  const void* x;
  const void* grad;     // backward
  const void* w;        // parameters: null for ones / zeros
  const void* b;
  void* out;            // forward: out; backward: dx (may be null)
  float* mean;          // forward: may be null; backward: inputs
  float* rstd;
  int64_t rows, cols;
  float epsilon;
  int param_half;
};

__device__ __forceinline__ float param_at(const void* p, int64_t c, int half) {
  return half ? __half2float(((const __half*)p)[c]) : ((const float*)p)[c];
}

// Sum over the kThreads of a row (a warp, or a whole block); every thread gets it.  `slot` alternates between
// successive sums of a block, so that one barrier each is enough.
template <int kThreads, int kN>
__device__ __forceinline__ void row_sum(float (&v)[kN], float (*scratch)[kN][32], int& slot) {
#pragma unroll
  for (int i = 0; i < kN; i++)
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
  if (kThreads > 32) {
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    if (lane == 0)
#pragma unroll
      for (int i = 0; i < kN; i++) scratch[slot][i][warp] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kN; i++) {
      v[i] = lane < kThreads / 32 ? scratch[slot][i][lane] : 0.0f;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
    }
    slot ^= 1;
  }
}

// One row at a time for kThreads threads, any length and alignment: the row is read again for every sum.
template <typename T>
__global__ void __launch_bounds__(256) norm_forward_any_kernel(const NormJob j) {
  __shared__ float scratch[2][1][32];
  pdl_wait();
  int slot = 0;
  const float inv_n = 1.0f / (float)j.cols;
  for (int64_t row = blockIdx.x; row < j.rows; row += gridDim.x) {
    const T* x = (const T*)j.x + row * j.cols;
    T* out = (T*)j.out + row * j.cols;
    float s[1] = {0.0f};
    for (int64_t c = threadIdx.x; c < j.cols; c += 256) s[0] += widen_f<T>(x[c]);
    row_sum<256, 1>(s, scratch, slot);
    const float mean = s[0] * inv_n;
    s[0] = 0.0f;
    for (int64_t c = threadIdx.x; c < j.cols; c += 256) {
      const float d = widen_f<T>(x[c]) - mean;
      s[0] += d * d;
    }
    row_sum<256, 1>(s, scratch, slot);
    const float rstd = 1.0f / sqrtf(s[0] * inv_n + j.epsilon);
    for (int64_t c = threadIdx.x; c < j.cols; c += 256) {
      float y = (widen_f<T>(x[c]) - mean) * rstd;
      if (j.w) y *= param_at(j.w, c, j.param_half);
      if (j.b) y += param_at(j.b, c, j.param_half);
      out[c] = narrow_f<T>(y);
    }
    if (threadIdx.x == 0) {
      if (j.mean) j.mean[row] = mean;
      if (j.rstd) j.rstd[row] = rstd;
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(256) norm_dx_any_kernel(const NormJob j) {
  __shared__ float scratch[2][2][32];
  pdl_wait();
  int slot = 0;
  const float inv_n = 1.0f / (float)j.cols;
  for (int64_t row = blockIdx.x; row < j.rows; row += gridDim.x) {
    const T* x = (const T*)j.x + row * j.cols;
    const T* g = (const T*)j.grad + row * j.cols;
    T* out = (T*)j.out + row * j.cols;
    const float mean = j.mean[row], rstd = j.rstd[row];
    float s[2] = {0.0f, 0.0f};
    for (int64_t c = threadIdx.x; c < j.cols; c += 256) {
      const float h = (widen_f<T>(x[c]) - mean) * rstd;
      const float gw = widen_f<T>(g[c]) * (j.w ? param_at(j.w, c, j.param_half) : 1.0f);
      s[0] += gw;
      s[1] += gw * h;
    }
    row_sum<256, 2>(s, scratch, slot);
    const float m0 = s[0] * inv_n, m1 = s[1] * inv_n;
    for (int64_t c = threadIdx.x; c < j.cols; c += 256) {
      const float h = (widen_f<T>(x[c]) - mean) * rstd;
      const float gw = widen_f<T>(g[c]) * (j.w ? param_at(j.w, c, j.param_half) : 1.0f);
      out[c] = narrow_f<T>(rstd * (gw - m0 - h * m1));
    }
  }
}

// dw and db: a CTA owns a strip of columns and a run of rows, as the activation gradient's does.
template <typename T, int kW>
__global__ void __launch_bounds__(256) norm_params_kernel(const NormJob j, float* partial, int64_t rows_per_run, int64_t runs) {
  pdl_wait();
  pdl_release();
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int64_t col = ((int64_t)blockIdx.x * 32 + lane) * kW;
  const int64_t row0 = (int64_t)blockIdx.y * rows_per_run, row1 = min(j.rows, row0 + rows_per_run);
  float dw[kW], db[kW];
#pragma unroll
  for (int e = 0; e < kW; e++) dw[e] = db[e] = 0.0f;
  if (col < j.cols) {
#pragma unroll 4
    for (int64_t r = row0 + warp; r < row1; r += 8) {
      const int64_t at = r * j.cols + col;
      float x[kW], g[kW];
      if constexpr (kW == 1) {
        x[0] = widen_f<T>(((const T*)j.x)[at]);
        g[0] = widen_f<T>(((const T*)j.grad)[at]);
      } else {
        Pack16<T>::widen(*(const uint4*)((const T*)j.x + at), x);
        Pack16<T>::widen(*(const uint4*)((const T*)j.grad + at), g);
      }
      const float mean = j.mean[r], rstd = j.rstd[r];
#pragma unroll
      for (int e = 0; e < kW; e++) {
        db[e] += g[e];
        dw[e] += g[e] * ((x[e] - mean) * rstd);
      }
    }
  }
  __shared__ float tile[2][8][32 * kW];
#pragma unroll
  for (int e = 0; e < kW; e++) {
    tile[0][warp][lane * kW + e] = dw[e];
    tile[1][warp][lane * kW + e] = db[e];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 64 * kW; i += 256) {
    const int which = i / (32 * kW), k = i % (32 * kW);
    const int64_t c = (int64_t)blockIdx.x * 32 * kW + k;
    if (c >= j.cols) continue;
    float s = 0.0f;
#pragma unroll
    for (int w = 0; w < 8; w++) s += tile[which][w][k];
    partial[((int64_t)which * runs + blockIdx.y) * j.cols + c] = s;
  }
}

unsigned row_grid(int64_t rows) { return (unsigned)(rows < 148 * 64 ? rows : 148 * 64); }

}  // namespace

cudaError_t launch_layer_norm(hc_dtype dtype, hc_dtype param_dtype, const void* x, const void* w, const void* b, int64_t rows,
                              int64_t cols, float epsilon, void* out, float* mean, float* rstd, cudaStream_t stream) {
  NormJob j = {x, nullptr, w, b, out, mean, rstd, rows, cols, epsilon, param_dtype == HC_F16};
  void* args[] = {(void*)&j};
  const void* fn = dtype == HC_F16 ? (const void*)norm_forward_any_kernel<__half> : (const void*)norm_forward_any_kernel<float>;
  return launch_behind(fn, args, dim3(row_grid(rows)), dim3(256), 0, stream);
}

size_t layer_norm_grad_scratch(hc_dtype dtype, int64_t rows, int64_t cols) {
  const RunSplit v = split_runs(rows, cols, 32 * (dtype == HC_F16 ? 8 : 4)), n = split_runs(rows, cols, 32);
  return 2 * (size_t)(v.runs > n.runs ? v.runs : n.runs) * (size_t)cols * 4;
}

cudaError_t launch_layer_norm_grad(hc_dtype dtype, hc_dtype param_dtype, const void* grad, const void* x, const void* w,
                                   const float* mean, const float* rstd, int64_t rows, int64_t cols, void* dx, void* dw, void* db,
                                   float* scratch, int* launches, cudaStream_t stream) {
  NormJob j = {x, grad, w, nullptr, dx, (float*)mean, (float*)rstd, rows, cols, 0.0f, param_dtype == HC_F16};
  *launches = 0;
  if (dx && rows > 0) {
    void* args[] = {(void*)&j};
    const void* fn = dtype == HC_F16 ? (const void*)norm_dx_any_kernel<__half> : (const void*)norm_dx_any_kernel<float>;
    cudaError_t e = launch_behind(fn, args, dim3(row_grid(rows)), dim3(256), 0, stream);
    if (e != cudaSuccess) return e;
    *launches += 1;
  }
  if (!dw && !db) return cudaSuccess;
  const int64_t eb = dtype == HC_F16 ? 2 : 4;
  const bool vec = (((uintptr_t)x | (uintptr_t)grad) & 15) == 0 && (cols * eb) % 16 == 0;
  const RunSplit s = split_runs(rows, cols, 32 * (vec ? (int)(16 / eb) : 1));
  if (s.strips > 2147483647LL) return cudaErrorInvalidValue;
  const void* fn = dtype == HC_F16 ? (vec ? (const void*)norm_params_kernel<__half, 8> : (const void*)norm_params_kernel<__half, 1>)
                                   : (vec ? (const void*)norm_params_kernel<float, 4> : (const void*)norm_params_kernel<float, 1>);
  int64_t per = s.rows_per_run, runs = s.runs;
  void* args[] = {(void*)&j, (void*)&scratch, (void*)&per, (void*)&runs};
  cudaError_t e = launch_behind(fn, args, dim3((unsigned)s.strips, (unsigned)s.runs), dim3(256), 0, stream);
  if (e != cudaSuccess) return e;
  // one partial matrix stack for dw, one for db; a gradient that is not wanted is not stored
  if (dw) e = launch_sum_runs(scratch, s.runs, cols, dw, db, param_dtype == HC_F16, stream);
  else e = launch_sum_runs(scratch + s.runs * cols, s.runs, cols, db, nullptr, param_dtype == HC_F16, stream);
  *launches += 2;
  return e;
}

}  // namespace hc

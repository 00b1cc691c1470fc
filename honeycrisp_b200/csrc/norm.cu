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

// Sum over the kThreads of a row (a warp, or several whole ones); every thread of the row gets it.  `slot` alternates
// between successive sums, so that one barrier each is enough.  With more than one row a CTA (kRows), a row of several
// warps has a named barrier of its own.
template <int kThreads, int kRows, int kN>
__device__ __forceinline__ void row_sum(float (&v)[kN], float (*scratch)[kN][32], int& slot) {
#pragma unroll
  for (int i = 0; i < kN; i++)
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
  if (kThreads > 32) {
    constexpr int kWarps = kThreads / 32;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, first = warp / kWarps * kWarps;
    if (lane == 0)
#pragma unroll
      for (int i = 0; i < kN; i++) scratch[slot][i][warp] = v[i];
    if (kRows == 1) __syncthreads();
    else asm volatile("bar.sync %0, %1;" ::"r"(1 + warp / kWarps), "n"(kThreads) : "memory");
#pragma unroll
    for (int i = 0; i < kN; i++) {
      v[i] = lane < kWarps ? scratch[slot][i][first + lane] : 0.0f;
#pragma unroll
      for (int o = kWarps / 2; o > 0; o >>= 1) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
      if (kWarps < 32) v[i] = __shfl_sync(0xffffffffu, v[i], 0);
    }
    slot ^= 1;
  }
}

// kC pieces of kW consecutive elements of a row, kThreads pieces apart: 16 bytes each, or single elements where rows are
// not 16-byte multiples.  What lies past the row's end reads as zero.
template <typename T, int kW, int kC>
struct Piece {
  static constexpr int E = kW * kC;
  uint4 raw[kW == 1 ? 1 : kC];
  T one[kW == 1 ? kC : 1];
  template <int kThreads>
  __device__ __forceinline__ void load(const T* row, int64_t cols, int t) {
#pragma unroll
    for (int c = 0; c < kC; c++) {
      const int64_t at = (int64_t)(t + c * kThreads) * kW;
      if constexpr (kW == 1) one[c] = at < cols ? row[at] : (T)0.0f;
      else raw[c] = at < cols ? __ldcs((const uint4*)(row + at)) : make_uint4(0, 0, 0, 0);
    }
  }
  __device__ __forceinline__ void widen(float (&x)[E]) const {
    if constexpr (kW == 1) {
#pragma unroll
      for (int c = 0; c < kC; c++) x[c] = widen_f<T>(one[c]);
    } else {
#pragma unroll
      for (int c = 0; c < kC; c++) {
        float v[kW];
        Pack16<T>::widen(raw[c], v);
#pragma unroll
        for (int e = 0; e < kW; e++) x[c * kW + e] = v[e];
      }
    }
  }
  template <int kThreads>
  __device__ __forceinline__ static void store(T* row, int64_t cols, int t, const float (&x)[E]) {
#pragma unroll
    for (int c = 0; c < kC; c++) {
      const int64_t at = (int64_t)(t + c * kThreads) * kW;
      if (at >= cols) continue;
      if constexpr (kW == 1) {
        row[at] = narrow_f<T>(x[c]);
      } else {
        float v[kW];
#pragma unroll
        for (int e = 0; e < kW; e++) v[e] = x[c * kW + e];
        *(uint4*)(row + at) = Pack16<T>::narrow(v);
      }
    }
  }
  template <int kThreads>
  __device__ __forceinline__ static void load_params(const void* p, int half, float other, int64_t cols, int t, float (&x)[E]) {
#pragma unroll
    for (int c = 0; c < kC; c++)
#pragma unroll
      for (int e = 0; e < kW; e++) {
        const int64_t at = (int64_t)(t + c * kThreads) * kW + e;
        x[c * kW + e] = at >= cols ? 0.0f : p ? param_at(p, at, half) : other;
      }
  }
};

// A row lives in the registers of kThreads threads, kRows rows side by side in a CTA; CTAs walk the rows, keeping the
// parameters and reading the next row while the sums of this one are made.
template <typename T, int kW, int kC, int kThreads, int kRows>
__global__ void __launch_bounds__(kThreads* kRows) norm_forward_kernel(const NormJob j) {
  typedef Piece<T, kW, kC> P;
  constexpr int E = P::E;
  __shared__ float scratch[2][1][32];
  pdl_wait();
  const int t = threadIdx.x % kThreads;
  const int64_t stride = (int64_t)gridDim.x * kRows;
  int64_t row = (int64_t)blockIdx.x * kRows + threadIdx.x / kThreads;
  if (row >= j.rows) return;   // whole rows leave together; their barriers are their own
  const float inv_n = 1.0f / (float)j.cols;
  P next;
  next.template load<kThreads>((const T*)j.x + row * j.cols, j.cols, t);
  float w[E], b[E];
  P::template load_params<kThreads>(j.w, j.param_half, 1.0f, j.cols, t, w);
  P::template load_params<kThreads>(j.b, j.param_half, 0.0f, j.cols, t, b);
  int slot = 0;
  for (; row < j.rows; row += stride) {
    float x[E];
    next.widen(x);
    // (`out` may be x's buffer: rows ahead are still unwritten, they belong to this CTA)
    if (row + stride < j.rows) next.template load<kThreads>((const T*)j.x + (row + stride) * j.cols, j.cols, t);
    float s[1] = {0.0f};
#pragma unroll
    for (int e = 0; e < E; e++) s[0] += x[e];
    row_sum<kThreads, kRows, 1>(s, scratch, slot);
    const float mean = s[0] * inv_n;
    s[0] = 0.0f;
#pragma unroll
    for (int c = 0; c < kC; c++)
#pragma unroll
      for (int e = 0; e < kW; e++) {
        const int i = c * kW + e;
        x[i] -= mean;
        if ((int64_t)(t + c * kThreads) * kW < j.cols) s[0] += x[i] * x[i];
      }
    row_sum<kThreads, kRows, 1>(s, scratch, slot);
    const float rstd = 1.0f / sqrtf(s[0] * inv_n + j.epsilon);
#pragma unroll
    for (int e = 0; e < E; e++) x[e] = fmaf(x[e] * rstd, w[e], b[e]);
    P::template store<kThreads>((T*)j.out + row * j.cols, j.cols, t, x);
    if (t == 0) {
      if (j.mean) j.mean[row] = mean;
      if (j.rstd) j.rstd[row] = rstd;
    }
  }
}

// Backward in one pass: dx of a row from its two sums, and the columns' sums for dw and db kept in registers while the CTA
// walks its rows.  At the end each CTA leaves one row of the partial matrices [2][CTAs][cols], which sum_runs_kernel adds
// in order.  The grid, and so the order of the sums, depends on shape, alignment and device alone.
template <typename T, int kW, int kC, int kThreads, int kRows>
__global__ void __launch_bounds__(kThreads* kRows, (kThreads * kRows * kW * kC <= 4096) ? 2 : 1)
norm_backward_kernel(const NormJob j, float* partial) {
  typedef Piece<T, kW, kC> P;
  constexpr int E = P::E;
  __shared__ float scratch[2][2][32];
  extern __shared__ float columns[];   // kRows > 1: [2][kRows][kThreads * E]
  pdl_wait();
  pdl_release();   // the kernel behind sums the partial matrices and waits for this one
  const int t = threadIdx.x % kThreads, sub = threadIdx.x / kThreads;
  const int64_t stride = (int64_t)gridDim.x * kRows;
  const float inv_n = 1.0f / (float)j.cols;
  float w[E], dw[E], db[E];
  P::template load_params<kThreads>(j.w, j.param_half, 1.0f, j.cols, t, w);
#pragma unroll
  for (int e = 0; e < E; e++) dw[e] = db[e] = 0.0f;
  int64_t row = (int64_t)blockIdx.x * kRows + sub;
  P nx, ng;
  float nmean = 0.0f, nrstd = 0.0f;
  auto fetch = [&](int64_t r) {
    nx.template load<kThreads>((const T*)j.x + r * j.cols, j.cols, t);
    ng.template load<kThreads>((const T*)j.grad + r * j.cols, j.cols, t);
    nmean = j.mean[r];
    nrstd = j.rstd[r];
  };
  if (row < j.rows) fetch(row);
  int slot = 0;
  for (; row < j.rows; row += stride) {
    float h[E], g[E];
    nx.widen(h);
    ng.widen(g);
    const float mean = nmean, rstd = nrstd;
    if (row + stride < j.rows) fetch(row + stride);
    float s[2] = {0.0f, 0.0f};
#pragma unroll
    for (int e = 0; e < E; e++) {
      h[e] = (h[e] - mean) * rstd;   // past the row's end g is zero, and so is all that follows from it
      db[e] += g[e];
      dw[e] = fmaf(g[e], h[e], dw[e]);
      g[e] *= w[e];
      s[0] += g[e];
      s[1] = fmaf(g[e], h[e], s[1]);
    }
    row_sum<kThreads, kRows, 2>(s, scratch, slot);
    if (j.out) {
      const float m0 = s[0] * inv_n, m1 = s[1] * inv_n;
#pragma unroll
      for (int e = 0; e < E; e++) g[e] = rstd * (g[e] - m0 - h[e] * m1);
      P::template store<kThreads>((T*)j.out + row * j.cols, j.cols, t, g);
    }
  }
  if (!partial) return;
  float* to[2] = {partial + (int64_t)blockIdx.x * j.cols, partial + ((int64_t)gridDim.x + blockIdx.x) * j.cols};
  if (kRows == 1) {
#pragma unroll
    for (int c = 0; c < kC; c++)
#pragma unroll
      for (int e = 0; e < kW; e++) {
        const int64_t at = (int64_t)(t + c * kThreads) * kW + e;
        if (at < j.cols) { to[0][at] = dw[c * kW + e]; to[1][at] = db[c * kW + e]; }
      }
  } else {
    constexpr int N = kThreads * E;
#pragma unroll
    for (int c = 0; c < kC; c++)
#pragma unroll
      for (int e = 0; e < kW; e++) {
        const int at = (t + c * kThreads) * kW + e;
        columns[sub * N + at] = dw[c * kW + e];
        columns[(kRows + sub) * N + at] = db[c * kW + e];
      }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * N; i += kThreads * kRows) {
      const int which = i / N, at = i % N;
      if (at >= j.cols) continue;
      float v = 0.0f;
#pragma unroll
      for (int r = 0; r < kRows; r++) v += columns[(which * kRows + r) * N + at];
      to[which][at] = v;
    }
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
    row_sum<256, 1, 1>(s, scratch, slot);
    const float mean = s[0] * inv_n;
    s[0] = 0.0f;
    for (int64_t c = threadIdx.x; c < j.cols; c += 256) {
      const float d = widen_f<T>(x[c]) - mean;
      s[0] += d * d;
    }
    row_sum<256, 1, 1>(s, scratch, slot);
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
    row_sum<256, 1, 2>(s, scratch, slot);
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

// One register form: pieces of kW elements, kW * kC elements a thread, kThreads threads a row, kRows rows a CTA.
struct NormForm {
  const void* fn;
  int threads, rows, elements;   // of a row; rows a CTA; elements a thread
};
template <typename T, int kW, int kE, int kThreads, int kRows>
NormForm forward_form() { return {(const void*)norm_forward_kernel<T, kW, kE / kW, kThreads, kRows>, kThreads, kRows, kE}; }
template <typename T, int kW, int kE, int kThreads, int kRows>
NormForm backward_form() { return {(const void*)norm_backward_kernel<T, kW, kE / kW, kThreads, kRows>, kThreads, kRows, kE}; }

// The fewest threads whose registers hold a row: eight elements each up to 4096 columns, more beyond; rows of up to 256
// columns take a warp each.  None beyond what a CTA holds.
template <typename T, int kW>
NormForm pick_forward(int64_t cols) {
  if (cols <= 256) return forward_form<T, kW, 8, 32, 8>();
  if (cols <= 1024) return forward_form<T, kW, 8, 128, 2>();
  if (cols <= 2048) return forward_form<T, kW, 8, 256, 1>();
  if (cols <= 4096) return forward_form<T, kW, 8, 512, 1>();
  if (cols <= 8192) return forward_form<T, kW, 8, 1024, 1>();
  if (cols <= 16384) return forward_form<T, kW, 16, 1024, 1>();
  return {nullptr, 0, 0, 0};
}
template <typename T, int kW>
NormForm pick_backward(int64_t cols) {
  if (cols <= 256) return backward_form<T, kW, 8, 32, 8>();
  if (cols <= 1024) return backward_form<T, kW, 8, 128, 2>();
  if (cols <= 2048) return backward_form<T, kW, 8, 256, 1>();
  if (cols <= 4096) return backward_form<T, kW, 8, 512, 1>();
  if (cols <= 8192) return backward_form<T, kW, 16, 512, 1>();
  return {nullptr, 0, 0, 0};
}
bool sixteen(const void* a, const void* b, const void* c, int64_t row_bytes) {
  return (((uintptr_t)a | (uintptr_t)b | (uintptr_t)c) & 15) == 0 && row_bytes % 16 == 0;
}
// CTAs that walk the rows: as many as are resident (2048 threads an SM, of which the registers of eight elements a thread
// allow half in the backward pass).
int64_t walkers(const NormForm& f, int64_t rows, int sm_count, int threads_per_sm) {
  const int per_sm = threads_per_sm / (f.threads * f.rows) > 0 ? threads_per_sm / (f.threads * f.rows) : 1;
  const int64_t need = (rows + f.rows - 1) / f.rows, most = (int64_t)sm_count * per_sm;
  return need < most ? (need > 0 ? need : 1) : most;
}

}  // namespace

cudaError_t launch_layer_norm(hc_dtype dtype, hc_dtype param_dtype, const void* x, const void* w, const void* b, int64_t rows,
                              int64_t cols, float epsilon, void* out, float* mean, float* rstd, int sm_count, cudaStream_t stream) {
  NormJob j = {x, nullptr, w, b, out, mean, rstd, rows, cols, epsilon, param_dtype == HC_F16};
  void* args[] = {(void*)&j};
  const bool half = dtype == HC_F16, vec = sixteen(x, out, nullptr, cols * (half ? 2 : 4));
  const NormForm f = half ? (vec ? pick_forward<__half, 8>(cols) : pick_forward<__half, 1>(cols))
                          : (vec ? pick_forward<float, 4>(cols) : pick_forward<float, 1>(cols));
  if (f.fn)
    return launch_behind(f.fn, args, dim3((unsigned)walkers(f, rows, sm_count, 2048)), dim3(f.threads * f.rows), 0, stream);
  const void* fn = half ? (const void*)norm_forward_any_kernel<__half> : (const void*)norm_forward_any_kernel<float>;
  return launch_behind(fn, args, dim3(row_grid(rows)), dim3(256), 0, stream);
}

namespace {
NormForm backward_of(hc_dtype dtype, const void* grad, const void* x, const void* dx, int64_t cols) {
  const bool half = dtype == HC_F16, vec = sixteen(x, grad, dx, cols * (half ? 2 : 4));
  return half ? (vec ? pick_backward<__half, 8>(cols) : pick_backward<__half, 1>(cols))
              : (vec ? pick_backward<float, 4>(cols) : pick_backward<float, 1>(cols));
}
}  // namespace

size_t layer_norm_grad_scratch(hc_dtype dtype, int64_t rows, int64_t cols, int sm_count) {
  const NormForm f = backward_of(dtype, nullptr, nullptr, nullptr, cols);   // the grid depends on cols, not on alignment
  if (f.fn) return 2 * (size_t)walkers(f, rows, sm_count, 1024) * (size_t)cols * 4;
  const RunSplit v = split_runs(rows, cols, 32 * (dtype == HC_F16 ? 8 : 4)), n = split_runs(rows, cols, 32);
  return 2 * (size_t)(v.runs > n.runs ? v.runs : n.runs) * (size_t)cols * 4;
}

cudaError_t launch_layer_norm_grad(hc_dtype dtype, hc_dtype param_dtype, const void* grad, const void* x, const void* w,
                                   const float* mean, const float* rstd, int64_t rows, int64_t cols, void* dx, void* dw, void* db,
                                   float* scratch, int sm_count, int* launches, cudaStream_t stream) {
  NormJob j = {x, grad, w, nullptr, dx, (float*)mean, (float*)rstd, rows, cols, 0.0f, param_dtype == HC_F16};
  *launches = 0;
  const NormForm f = backward_of(dtype, grad, x, dx, cols);
  if (f.fn) {
    const int64_t ctas = walkers(f, rows, sm_count, 1024);
    float* partial = dw || db ? scratch : nullptr;
    void* args[] = {(void*)&j, (void*)&partial};
    const size_t smem = f.rows > 1 ? 2 * (size_t)f.rows * f.threads * f.elements * sizeof(float) : 0;
    cudaError_t e = launch_behind(f.fn, args, dim3((unsigned)ctas), dim3(f.threads * f.rows), smem, stream);
    if (e != cudaSuccess) return e;
    *launches += 1;
    if (!partial) return cudaSuccess;
    *launches += 1;
    const bool half = param_dtype == HC_F16;
    return dw ? launch_sum_runs(partial, ctas, cols, dw, db, half, stream)
              : launch_sum_runs(partial + ctas * cols, ctas, cols, db, nullptr, half, stream);
  }
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

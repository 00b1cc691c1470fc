// The gradient through an activation, with the bias gradient of the layer in front of it:
//   dpre = grad * act'(pre),   bias_grad[c] = sum over rows of the unrounded dpre.
//
// One pass over the two inputs, HBM-bound: 3 tensors of traffic.  A CTA owns a strip of columns (one 16-byte
// chunk for each of 32 lanes) and a run of rows that its eight warps walk side by side; the float32 sums of its columns stay
// in registers until the end, are combined through shared memory and go to a partial matrix [row runs, columns] that a second
// kernel sums in ascending order.  The split depends on the shape alone, so a repeat gives the same bits.
#include "common.cuh"
#include "epilogue.cuh"
#include "stream_order.cuh"

namespace hc {
namespace {

constexpr int kLanes = 32, kWarps = 8;

// kW: columns per lane; a 16-byte chunk, or 1 where rows are not 16-byte multiples.
template <typename T, int kW, bool kSum, int kAct>
__global__ void __launch_bounds__(kLanes * kWarps) activation_grad_kernel(const T* grad, const T* pre, T* dpre, float* partial,
                                                                          int64_t rows, int64_t cols, int64_t rows_per_run) {
  pdl_wait();
  if (kSum) pdl_release();   // the kernel behind sums the partial matrix and waits for this one
  const int lane = threadIdx.x % kLanes, warp = threadIdx.x / kLanes;
  const int64_t col = ((int64_t)blockIdx.x * kLanes + lane) * kW;
  const int64_t row0 = (int64_t)blockIdx.y * rows_per_run, row1 = min(rows, row0 + rows_per_run);
  float sum[kW];
#pragma unroll
  for (int e = 0; e < kW; e++) sum[e] = 0.0f;
  auto use = [&](int64_t at, float (&x)[kW], const float (&z)[kW]) {
    act_scale_t<kAct, sizeof(T) == 2, kW>(x, z);
    if (kSum)
#pragma unroll
      for (int e = 0; e < kW; e++) sum[e] += x[e];
    if constexpr (kW == 1) dpre[at] = narrow_f<T>(x[0]);
    else *(uint4*)(dpre + at) = Pack16<T>::narrow(x);
  };
  // Rows of both inputs travel ahead of their use (dpre may be one of the inputs, so the compiler cannot move a load across a
  // store by itself; a thread's rows ahead are its own and still unwritten).  16-byte chunks wait in shared memory, where each
  // thread reads back what it copied itself, three rows ahead; single elements in registers, eight rows at a time.
  if constexpr (kW > 1) {
    constexpr int kDepth = 4;
    __shared__ uint4 queue[kDepth][2][kLanes * kWarps];
    if (col < cols) {
      const int64_t step = kWarps * cols;
      const int mine = (int)((row1 - row0 - warp + kWarps - 1) / kWarps);   // rows of this warp (negative: none)
      const T *g_at = grad + (row0 + warp) * cols + col, *z_at = pre + (row0 + warp) * cols + col;
      auto fetch = [&](int i) {
        if (i < mine) {
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(&queue[i % kDepth][0][threadIdx.x])), "l"(g_at + i * step) : "memory");
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(&queue[i % kDepth][1][threadIdx.x])), "l"(z_at + i * step) : "memory");
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
      };
#pragma unroll
      for (int i = 0; i < kDepth - 1; i++) fetch(i);
#pragma unroll 1
      for (int i = 0; i < mine; i++) {
        fetch(i + kDepth - 1);
        asm volatile("cp.async.wait_group %0;" ::"n"(kDepth - 1) : "memory");
        float x[kW], z[kW];
        Pack16<T>::widen(queue[i % kDepth][0][threadIdx.x], x);
        Pack16<T>::widen(queue[i % kDepth][1][threadIdx.x], z);
        use((row0 + warp + (int64_t)i * kWarps) * cols + col, x, z);
      }
    }
  } else if (col < cols) {
    constexpr int kAhead = 8;
    int64_t r0 = row0 + warp;
    for (; r0 + (kAhead - 1) * kWarps < row1; r0 += kAhead * kWarps) {
      T graw[kAhead], zraw[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; i++) {
        graw[i] = grad[(r0 + i * kWarps) * cols + col];
        zraw[i] = pre[(r0 + i * kWarps) * cols + col];
      }
#pragma unroll
      for (int i = 0; i < kAhead; i++) {
        float x[1] = {widen_f<T>(graw[i])};
        const float z[1] = {widen_f<T>(zraw[i])};
        use((r0 + i * kWarps) * cols + col, x, z);
      }
    }
    // the last rows one by one, in code of their own: a short input runs only these few instructions
#pragma unroll 1
    for (; r0 < row1; r0 += kWarps) {
      float x[1] = {widen_f<T>(grad[r0 * cols + col])};
      const float z[1] = {widen_f<T>(pre[r0 * cols + col])};
      use(r0 * cols + col, x, z);
    }
  }
  if (kSum) {
    __shared__ float tile[kWarps][kLanes * kW];
#pragma unroll
    for (int e = 0; e < kW; e++) tile[warp][lane * kW + e] = sum[e];
    __syncthreads();
    for (int i = threadIdx.x; i < kLanes * kW; i += kLanes * kWarps) {
      const int64_t c = (int64_t)blockIdx.x * kLanes * kW + i;
      if (c >= cols) continue;
      float s = 0.0f;
#pragma unroll
      for (int w = 0; w < kWarps; w++) s += tile[w][i];
      partial[(int64_t)blockIdx.y * cols + c] = s;
    }
  }
}

// out[c] = sum over runs of partial[run][c], for one or two stacks of partial matrices: 32 columns a CTA, each of 32 warps sums every
// 32nd run, the 32 sums are added in order.
constexpr int kSumWarps = 32;
__global__ void __launch_bounds__(32 * kSumWarps) sum_runs_kernel(const float* partial, int64_t runs, int64_t cols, void* out0, void* out1,
                                                                  int half) {
  pdl_wait();
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int64_t c = (int64_t)blockIdx.x * 32 + lane;
  const float* src = partial + (int64_t)blockIdx.y * runs * cols;
  void* out = blockIdx.y == 0 ? out0 : out1;
  float s = 0.0f;
  if (c < cols)
#pragma unroll 8
    for (int64_t r = warp; r < runs; r += kSumWarps) s += src[r * cols + c];
  __shared__ float tile[kSumWarps][33];
  tile[warp][lane] = s;
  __syncthreads();
  if (warp == 0 && c < cols && out) {
#pragma unroll
    for (int w = 1; w < kSumWarps; w++) s += tile[w][lane];
    if (half) ((__half*)out)[c] = __float2half_rn(s);
    else ((float*)out)[c] = s;
  }
}

}  // namespace

RunSplit split_runs(int64_t rows, int64_t cols, int cols_per_cta) {
  // About eight CTAs for each of 148 SMs, runs of at least 16 rows (two for every warp); up to 64 rows are one run, whose sums
  // need no second kernel.
  RunSplit s;
  s.strips = (cols + cols_per_cta - 1) / cols_per_cta;
  int64_t runs = (148 * 8 + s.strips - 1) / s.strips;
  if (runs > (rows + 15) / 16) runs = (rows + 15) / 16;
  if (rows <= 64) runs = 1;
  if (runs < 1) runs = 1;
  s.rows_per_run = (rows + runs - 1) / runs;
  s.rows_per_run = (s.rows_per_run + 7) / 8 * 8;
  if (s.rows_per_run < 8) s.rows_per_run = 8;   // no rows: one run that sums nothing
  s.runs = (rows + s.rows_per_run - 1) / s.rows_per_run;
  if (s.runs < 1) s.runs = 1;
  return s;
}

cudaError_t launch_sum_runs(const float* partial, int64_t runs, int64_t cols, void* out0, void* out1, bool half, cudaStream_t stream) {
  int h = half ? 1 : 0;
  void* args[] = {(void*)&partial, (void*)&runs, (void*)&cols, (void*)&out0, (void*)&out1, (void*)&h};
  return launch_behind((const void*)sum_runs_kernel, args, dim3((unsigned)((cols + 31) / 32), out1 ? 2 : 1), dim3(32 * kSumWarps), 0,
                       stream);
}

namespace {
template <typename T, int kAct>
const void* kernel_of(bool vec, bool sum) {
  constexpr int W = Pack16<T>::W;
  return vec ? (sum ? (const void*)activation_grad_kernel<T, W, true, kAct> : (const void*)activation_grad_kernel<T, W, false, kAct>)
             : (sum ? (const void*)activation_grad_kernel<T, 1, true, kAct> : (const void*)activation_grad_kernel<T, 1, false, kAct>);
}
template <typename T>
cudaError_t launch_typed(const void* grad, const void* pre, int64_t rows, int64_t cols, void* dpre, float* bias_grad,
                         float* partial, bool vec, const RunSplit& s, int act, int* launches, cudaStream_t stream) {
  const void* fn = nullptr;
  switch (act) {
    case HC_ACT_RELU: fn = kernel_of<T, HC_ACT_RELU>(vec, bias_grad); break;
    case HC_ACT_GELU: fn = kernel_of<T, HC_ACT_GELU>(vec, bias_grad); break;
    case HC_ACT_GELU_TANH: fn = kernel_of<T, HC_ACT_GELU_TANH>(vec, bias_grad); break;
    case HC_ACT_SILU: fn = kernel_of<T, HC_ACT_SILU>(vec, bias_grad); break;
    default: fn = kernel_of<T, HC_ACT_NONE>(vec, bias_grad); break;
  }
  int64_t per = s.rows_per_run;
  void* args[] = {(void*)&grad, (void*)&pre, (void*)&dpre, (void*)&partial, (void*)&rows, (void*)&cols, (void*)&per};
  cudaError_t e = launch_behind(fn, args, dim3((unsigned)s.strips, (unsigned)s.runs), dim3(kLanes * kWarps), 0, stream);
  if (e != cudaSuccess) return e;
  *launches = 1;
  if (!bias_grad || s.runs == 1) return e;   // one run's partial matrix is the sum
  *launches = 2;
  return launch_sum_runs(partial, s.runs, cols, bias_grad, nullptr, false, stream);
}
bool rows_of_16_bytes(const void* a, const void* b, const void* c, int64_t row_bytes) {
  return (((uintptr_t)a | (uintptr_t)b | (uintptr_t)c) & 15) == 0 && row_bytes % 16 == 0;
}
}  // namespace

size_t activation_grad_scratch(hc_dtype dtype, int64_t rows, int64_t cols) {
  // alignment decides between a 16-byte chunk and one column a lane, and with it the split: room for either
  const RunSplit v = split_runs(rows, cols, kLanes * (dtype == HC_F16 ? 8 : 4)), n = split_runs(rows, cols, kLanes);
  return (size_t)(v.runs > n.runs ? v.runs : n.runs) * (size_t)cols * 4;
}

cudaError_t launch_activation_grad(hc_dtype dtype, int act, const void* grad, const void* pre, int64_t rows, int64_t cols,
                                   void* dpre, float* bias_grad, float* scratch, int* launches, cudaStream_t stream) {
  *launches = 0;
  const int64_t eb = dtype == HC_F16 ? 2 : 4;
  const bool vec = rows_of_16_bytes(grad, pre, dpre, cols * eb);
  const RunSplit s = split_runs(rows, cols, kLanes * (vec ? (int)(16 / eb) : 1));
  if (s.strips > 2147483647LL || s.runs > 65535) return cudaErrorInvalidValue;
  if (s.runs == 1) scratch = bias_grad;
  return dtype == HC_F16 ? launch_typed<__half>(grad, pre, rows, cols, dpre, bias_grad, scratch, vec, s, act, launches, stream)
                         : launch_typed<float>(grad, pre, rows, cols, dpre, bias_grad, scratch, vec, s, act, launches, stream);
}

}  // namespace hc

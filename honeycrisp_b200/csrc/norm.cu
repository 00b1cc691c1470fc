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

// kN sums at once over the kThreads of a row (a warp, or several whole ones); every thread of the row gets them all.  The
// butterfly halves the values while it halves the lanes (a lane keeps one half and sends the other), so that eight sums
// take nine shuffles, not forty; lane i * 32 / kN ends with sum i, and a shuffle for each sum hands them to all.  `slot` alternates
// between successive calls, so that one barrier each is enough; with more than one row group a CTA (kRows), each has a named barrier of its own.
template <int kThreads, int kRows, int kN>
__device__ __forceinline__ void row_sum(float (&v)[kN], float (*scratch)[kN][32], int& slot) {
  constexpr int kShare = 32 / kN;   // lanes that end with the same sum
  const int lane = threadIdx.x % 32;
  int o = 16;
#pragma unroll
  for (int n = kN / 2; n >= 1; n >>= 1) {
    const bool up = (lane & o) != 0;
#pragma unroll
    for (int i = 0; i < n; i++) {
      const float send = up ? v[i] : v[i + n], keep = up ? v[i + n] : v[i];
      v[i] = keep + __shfl_xor_sync(0xffffffffu, send, o);
    }
    o >>= 1;
  }
  float x = v[0];
#pragma unroll
  for (int k = kShare / 2; k > 0; k >>= 1) x += __shfl_xor_sync(0xffffffffu, x, k);
  if (kThreads > 32) {
    constexpr int kWarps = kThreads / 32;
    const int warp = threadIdx.x / 32, first = warp / kWarps * kWarps;
    if (lane % kShare == 0) scratch[slot][lane / kShare][warp] = x;
    if (kRows == 1) __syncthreads();
    else asm volatile("bar.sync %0, %1;" ::"r"(1 + warp / kWarps), "n"(kThreads) : "memory");
    x = 0.0f;
#pragma unroll
    for (int w = 0; w < kWarps; w += kShare)
      if (w + lane % kShare < kWarps) x += scratch[slot][lane / kShare][first + w + lane % kShare];
#pragma unroll
    for (int k = kShare / 2; k > 0; k >>= 1) x += __shfl_xor_sync(0xffffffffu, x, k);
    slot ^= 1;
  }
#pragma unroll
  for (int i = 0; i < kN; i++) v[i] = __shfl_sync(0xffffffffu, x, i * kShare);
}

// kC pieces of kW consecutive elements of a row, kThreads pieces apart: 16 bytes each, or single elements where rows are
// not 16-byte multiples.  What lies past the row's end reads as zero.
//
// Rows come through a queue of kSlots rows.  16-byte pieces travel by asynchronous copies into shared memory, from which each
// thread reads back only what it copied itself, so the queue needs neither registers nor barriers; single elements wait
// in registers, one batch of kBatch rows ahead.
template <typename T, int kW, int kC, int kThreads, int kRows, int kBatch, int kSlots>
struct RowQueue {
  static constexpr int E = kW * kC;
  static constexpr bool kAsync = kW > 1;
  static constexpr uint32_t kPiece = kThreads * kRows * 16, kSlot = kC * kPiece;   // bytes from piece to piece, from row to row
  static constexpr size_t bytes = kAsync ? (size_t)kSlots * kSlot : 0;
  uint32_t base;
  bool inside[kC];   // the piece lies inside the row
  T held[kAsync ? 1 : kBatch * kC];

  __device__ __forceinline__ void init(void* smem, int64_t cols, int t) {
    base = (uint32_t)__cvta_generic_to_shared(smem) + threadIdx.x * 16;
#pragma unroll
    for (int c = 0; c < kC; c++) inside[c] = (int64_t)(t + c * kThreads) * kW < cols;
  }
  // Row r of a batch; `src`: this thread's first piece of it.
  __device__ __forceinline__ void fetch(const T* src, int r, uint32_t batch, bool live) {
#pragma unroll
    for (int c = 0; c < kC; c++) {
      if constexpr (kAsync) {
        if (live && inside[c])
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(base + (batch * kBatch + r) * kSlot + c * kPiece), "l"(src + c * kThreads * kW) : "memory");
      } else {
        T v = (T)0.0f;
        if (live && inside[c]) v = src[c * kThreads];
        held[r * kC + c] = v;
      }
    }
  }
  __device__ __forceinline__ void take(int r, uint32_t batch, bool live, float (&x)[E]) const {
#pragma unroll
    for (int c = 0; c < kC; c++) {
      if constexpr (kAsync) {
        uint4 u = make_uint4(0, 0, 0, 0);
        if (live && inside[c])
          asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w)
                       : "r"(base + (batch * kBatch + r) * kSlot + c * kPiece) : "memory");
        float v[kW];
        Pack16<T>::widen(u, v);
#pragma unroll
        for (int e = 0; e < kW; e++) x[c * kW + e] = v[e];
      } else {
        x[c] = widen_f<T>(held[r * kC + c]);
      }
    }
  }
  // `dst`: where this thread's first piece of the row goes.
  __device__ __forceinline__ void store(T* dst, const float (&x)[E]) const {
#pragma unroll
    for (int c = 0; c < kC; c++) {
      if (!inside[c]) continue;
      if constexpr (kAsync) {
        float v[kW];
#pragma unroll
        for (int e = 0; e < kW; e++) v[e] = x[c * kW + e];
        *(uint4*)(dst + c * kThreads * kW) = Pack16<T>::narrow(v);
      } else {
        dst[c * kThreads] = narrow_f<T>(x[c]);
      }
    }
  }
};
__device__ __forceinline__ void queue_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kPending>
__device__ __forceinline__ void queue_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(kPending) : "memory"); }

template <int kW, int kC, int kThreads>
__device__ __forceinline__ void load_params(const void* p, int half, float other, int64_t cols, int t, float (&x)[kW * kC]) {
#pragma unroll
  for (int c = 0; c < kC; c++)
#pragma unroll
    for (int e = 0; e < kW; e++) {
      const int64_t at = (int64_t)(t + c * kThreads) * kW + e;
      x[c * kW + e] = at >= cols ? 0.0f : p ? param_at(p, at, half) : other;
    }
}

// Batches in a queue: what `budget` bytes of shared memory hold, two to four.
constexpr int queue_batches(int batch_bytes, int budget) {
  return budget / batch_bytes < 2 ? 2 : budget / batch_bytes > 4 ? 4 : budget / batch_bytes;
}

// A row lives in the registers of kThreads threads, kRows row groups side by side in a CTA, each with its own barrier; CTAs
// walk the rows, kBatch at a time for each group.
// What a row costs is the latency of its two sums, so rows in flight count: 32 elements a thread put eight rows of 4096 on an
// SM where eight elements a thread put two (16384 x 4096 float16: 62 us with two, 51 with eight), and short rows
// share their sums' shuffles in batches.  With 32 elements the parameters would take the registers, so they lie in shared
// memory, in planes of 16 bytes a lane; with eight or 16 they stay in registers.
template <typename T, int kW, int kC, int kThreads, int kRows, int kBatch>
struct ForwardLayout {
  static constexpr int kBatches = queue_batches(kBatch * kThreads * kRows * kC * 16, 65536);
  typedef RowQueue<T, kW, kC, kThreads, kRows, kBatch, kBatches * kBatch> Q;
  static constexpr bool kShared = kW * kC > 16;
  static constexpr size_t smem = Q::bytes + (kShared ? 2 * (size_t)kThreads * kW * kC * 4 : 0);   // the parameters behind the queue
};
template <typename T, int kW, int kC, int kThreads, int kRows, int kBatch>
__global__ void __launch_bounds__(kThreads* kRows, kThreads* kRows <= 512 ? 2 : 1) norm_forward_kernel(const NormJob j) {
  typedef ForwardLayout<T, kW, kC, kThreads, kRows, kBatch> L;
  typedef typename L::Q Q;
  constexpr int E = Q::E, D = L::kBatches;
  constexpr int V = kW >= 4 ? 4 : 1, PLANES = E / V;   // a plane holds V consecutive elements of every thread
  __shared__ float scratch[2][kBatch][32];
  extern __shared__ __align__(16) unsigned char queue_mem[];
  pdl_wait();
  const int t = threadIdx.x % kThreads;
  const int rows = (int)j.rows, stride = (int)gridDim.x * kRows * kBatch;
  int row = ((int)blockIdx.x * kRows + (int)(threadIdx.x / kThreads)) * kBatch;
  const float inv_n = 1.0f / (float)j.cols;
  const T* src = (const T*)j.x + row * j.cols + t * kW;
  T* dst = (T*)j.out + row * j.cols + t * kW;
  const int64_t step = stride * j.cols;
  Q q;
  q.init(queue_mem, j.cols, t);
  auto fetch = [&](const T* from, int first, uint32_t batch) {
#pragma unroll
    for (int r = 0; r < kBatch; r++) q.fetch(from + r * j.cols, r, batch, first + r < rows);
    queue_commit();
  };
#pragma unroll
  for (int d = 0; d < (Q::kAsync ? D - 1 : 1); d++) fetch(src + d * step, row + d * stride, d);
  float* shared_w = (float*)(queue_mem + Q::bytes);
  float* shared_b = shared_w + kThreads * E;
  float w[L::kShared ? 1 : E], b[L::kShared ? 1 : E];
  if constexpr (L::kShared) {
    for (int i = threadIdx.x; i < kThreads * E; i += kThreads * kRows) {
      // element i of the row: piece i / kW, which thread piece % kThreads keeps as its (piece / kThreads)-th
      const int piece = i / kW, e = i % kW, c = piece / kThreads, owner = piece % kThreads;
      const int to = (((c * kW + e) / V) * kThreads + owner) * V + e % V;
      shared_w[to] = i >= j.cols ? 0.0f : j.w ? param_at(j.w, i, j.param_half) : 1.0f;
      shared_b[to] = i >= j.cols ? 0.0f : j.b ? param_at(j.b, i, j.param_half) : 0.0f;
    }
    __syncthreads();
  } else {
    load_params<kW, kC, kThreads>(j.w, j.param_half, 1.0f, j.cols, t, w);
    load_params<kW, kC, kThreads>(j.b, j.param_half, 0.0f, j.cols, t, b);
  }
  int slot = 0;
  uint32_t at = 0;
  for (; row < rows; row += stride, src += step, dst += step) {   // whole groups leave together; their barriers are their own
    float x[kBatch][E], s[kBatch], mean[kBatch];
    // (`out` may be x's buffer: the rows ahead are still unwritten, they belong to these threads)
    if constexpr (Q::kAsync) {
      fetch(src + (D - 1) * step, row + (D - 1) * stride, at == 0 ? D - 1 : at - 1);
      queue_wait<D - 1>();
    }
#pragma unroll
    for (int r = 0; r < kBatch; r++) {
      q.take(r, at, row + r < rows, x[r]);
      s[r] = 0.0f;
#pragma unroll
      for (int e = 0; e < E; e++) s[r] += x[r][e];
    }
    at = at + 1 == D ? 0 : at + 1;
    if constexpr (!Q::kAsync) fetch(src + step, row + stride, 0);
    row_sum<kThreads, kRows, kBatch>(s, scratch, slot);
#pragma unroll
    for (int r = 0; r < kBatch; r++) {
      mean[r] = s[r] * inv_n;
      s[r] = 0.0f;
#pragma unroll
      for (int c = 0; c < kC; c++)
#pragma unroll
        for (int e = 0; e < kW; e++) {
          const int i = c * kW + e;
          x[r][i] -= mean[r];
          if (q.inside[c]) s[r] = fmaf(x[r][i], x[r][i], s[r]);
        }
    }
    row_sum<kThreads, kRows, kBatch>(s, scratch, slot);
#pragma unroll
    for (int r = 0; r < kBatch; r++) {
      const float rstd = 1.0f / sqrtf(s[r] * inv_n + j.epsilon);
      if (row + r >= rows) continue;
      if constexpr (L::kShared) {
#pragma unroll
        for (int k = 0; k < PLANES; k++) {
          const float* pw = shared_w + (k * kThreads + t) * V;
          const float* pb = shared_b + (k * kThreads + t) * V;
          if constexpr (V == 4) {
            const float4 a = *(const float4*)pw, c = *(const float4*)pb;
            x[r][k * 4] = fmaf(x[r][k * 4] * rstd, a.x, c.x);
            x[r][k * 4 + 1] = fmaf(x[r][k * 4 + 1] * rstd, a.y, c.y);
            x[r][k * 4 + 2] = fmaf(x[r][k * 4 + 2] * rstd, a.z, c.z);
            x[r][k * 4 + 3] = fmaf(x[r][k * 4 + 3] * rstd, a.w, c.w);
          } else {
            x[r][k] = fmaf(x[r][k] * rstd, *pw, *pb);
          }
        }
      } else {
#pragma unroll
        for (int e = 0; e < E; e++) x[r][e] = fmaf(x[r][e] * rstd, w[e], b[e]);
      }
      q.store(dst + r * j.cols, x[r]);
      if (t == 0) {
        if (j.mean) j.mean[row + r] = mean[r];
        if (j.rstd) j.rstd[row + r] = rstd;
      }
    }
  }
}

// Backward in one pass: dx of a row from its two sums, and the columns' sums for dw and db kept in registers while the CTA
// walks its rows, kBatch of them at a time: one round of sums, whose latency no other work of the CTA hides, serves them all.
// At the end each CTA leaves one row of the partial matrices [2][CTAs][cols], which sum_runs_kernel adds in order.  The grid,
// and so the order of the sums, depends on shape, alignment and device alone.
// h is (x - mean) rstd, the difference first: x rstd - mean rstd, one instruction for a pair where this takes two, is off by 2^-24 |mean| rstd,
// which on rows whose mean is thousands of times their spread is thousands of times the rounding of h.
template <typename T, int kW, int kC, int kThreads, int kRows, int kBatch>
struct BackwardLayout {
  static constexpr int kBatches = queue_batches(2 * kBatch * kThreads * kRows * kC * 16, kThreads * kRows > 256 ? 131072 : 65536);   // 128 KB an SM
  typedef RowQueue<T, kW, kC, kThreads, kRows, kBatch, kBatches * kBatch> Q;
  static constexpr size_t sums = kRows > 1 ? 2 * (size_t)kRows * kThreads * kW * kC * sizeof(float) : 0;
  static constexpr size_t smem = 2 * Q::bytes > sums ? 2 * Q::bytes : sums;
};
template <typename T, int kW, int kC, int kThreads, int kRows, int kBatch>
__global__ void __launch_bounds__(kThreads* kRows, kThreads * kRows <= 256 ? 2 : 1) norm_backward_kernel(const NormJob j, float* partial) {
  typedef BackwardLayout<T, kW, kC, kThreads, kRows, kBatch> L;
  typedef typename L::Q Q;
  constexpr int E = Q::E, D = L::kBatches;
  __shared__ float scratch[2][2 * kBatch][32];
  extern __shared__ __align__(16) unsigned char queue_mem[];
  pdl_wait();
  pdl_release();   // the kernel behind sums the partial matrices and waits for this one
  const int t = threadIdx.x % kThreads, sub = threadIdx.x / kThreads;
  const int rows = (int)j.rows, stride = (int)gridDim.x * kRows * kBatch;
  const float inv_n = 1.0f / (float)j.cols;
  int row = ((int)blockIdx.x * kRows + sub) * kBatch;
  const int64_t step = stride * j.cols, first_at = row * j.cols + t * kW;
  const T *src_x = (const T*)j.x + first_at, *src_g = (const T*)j.grad + first_at;
  T* dst = (T*)j.out + first_at;
  Q qx, qg;
  qx.init(queue_mem, j.cols, t);
  qg.init(queue_mem + Q::bytes, j.cols, t);
  auto fetch = [&](int64_t ahead, int first, uint32_t batch) {
#pragma unroll
    for (int r = 0; r < kBatch; r++) {
      qx.fetch(src_x + ahead + r * j.cols, r, batch, first + r < rows);
      qg.fetch(src_g + ahead + r * j.cols, r, batch, first + r < rows);
    }
    queue_commit();
  };
#pragma unroll
  for (int d = 0; d < (Q::kAsync ? D - 1 : 1); d++) fetch(d * step, row + d * stride, d);
  float mean_at[kBatch], rstd_at[kBatch];
  auto statistics = [&](int first) {
#pragma unroll
    for (int r = 0; r < kBatch; r++) {
      mean_at[r] = first + r < rows ? j.mean[first + r] : 0.0f;
      rstd_at[r] = first + r < rows ? j.rstd[first + r] : 0.0f;
    }
  };
  statistics(row);
  // Elements in pairs: the pass is bound by instructions as much as by memory, and a pair costs one of each kind.
  constexpr int P = E / 2;
  float2 w[P], dw[P], db[P];
  {
    float all[E];
    load_params<kW, kC, kThreads>(j.w, j.param_half, 1.0f, j.cols, t, all);
#pragma unroll
    for (int e = 0; e < P; e++) {
      w[e] = make_float2(all[2 * e], all[2 * e + 1]);
      dw[e] = db[e] = make_float2(0.0f, 0.0f);
    }
  }
  int slot = 0;
  uint32_t at = 0;
  for (; row < rows; row += stride, src_x += step, src_g += step, dst += step) {
    float2 h[kBatch][P], g[kBatch][P];
    if constexpr (Q::kAsync) {
      fetch((D - 1) * step, row + (D - 1) * stride, at == 0 ? D - 1 : at - 1);
      queue_wait<D - 1>();
    }
#pragma unroll
    for (int r = 0; r < kBatch; r++) {
      float xv[E], gv[E];
      qx.take(r, at, row + r < rows, xv);
      qg.take(r, at, row + r < rows, gv);
#pragma unroll
      for (int e = 0; e < P; e++) {
        h[r][e] = make_float2(xv[2 * e], xv[2 * e + 1]);
        g[r][e] = make_float2(gv[2 * e], gv[2 * e + 1]);
      }
    }
    at = at + 1 == D ? 0 : at + 1;
    if constexpr (!Q::kAsync) fetch(step, row + stride, 0);
    float rstd[kBatch], s[2 * kBatch];
#pragma unroll
    for (int r = 0; r < kBatch; r++) {
      rstd[r] = rstd_at[r];
      const float2 scale = both(rstd[r]), off = both(-mean_at[r]);
      float2 s0 = both(0.0f), s1 = both(0.0f);
#pragma unroll
      for (int e = 0; e < P; e++) {
        h[r][e] = mul2(add2(h[r][e], off), scale);   // past the row's end g is zero, and so is all that follows from it
        db[e] = add2(db[e], g[r][e]);
        dw[e] = fma2(g[r][e], h[r][e], dw[e]);
        g[r][e] = mul2(g[r][e], w[e]);
        s0 = add2(s0, g[r][e]);
        s1 = fma2(g[r][e], h[r][e], s1);
      }
      s[2 * r] = s0.x + s0.y;
      s[2 * r + 1] = s1.x + s1.y;
    }
    statistics(row + stride);
    row_sum<kThreads, kRows, 2 * kBatch>(s, scratch, slot);
    if (j.out) {
#pragma unroll
      for (int r = 0; r < kBatch; r++) {
        if (row + r >= rows) continue;
        const float2 scale = both(rstd[r]), m0 = both(-s[2 * r] * inv_n), m1 = both(-s[2 * r + 1] * inv_n);
        float out[E];
#pragma unroll
        for (int e = 0; e < P; e++) {
          const float2 v = mul2(scale, fma2(h[r][e], m1, add2(g[r][e], m0)));
          out[2 * e] = v.x;
          out[2 * e + 1] = v.y;
        }
        qx.store(dst + r * j.cols, out);
      }
    }
  }
  if (!partial) return;
  auto of = [](const float2 (&v)[P], int e) { return e & 1 ? v[e / 2].y : v[e / 2].x; };
  float* to[2] = {partial + (int64_t)blockIdx.x * j.cols, partial + ((int64_t)gridDim.x + blockIdx.x) * j.cols};
  if (kRows == 1) {
#pragma unroll
    for (int c = 0; c < kC; c++)
#pragma unroll
      for (int e = 0; e < kW; e++) {
        const int64_t k = (int64_t)(t + c * kThreads) * kW + e;
        if (k < j.cols) { to[0][k] = of(dw, c * kW + e); to[1][k] = of(db, c * kW + e); }
      }
  } else {
    constexpr int N = kThreads * E;
    float* columns = (float*)queue_mem;   // [2][kRows][N], over the queue
    queue_wait<0>();
    __syncthreads();
#pragma unroll
    for (int c = 0; c < kC; c++)
#pragma unroll
      for (int e = 0; e < kW; e++) {
        const int k = (t + c * kThreads) * kW + e;
        columns[sub * N + k] = of(dw, c * kW + e);
        columns[(kRows + sub) * N + k] = of(db, c * kW + e);
      }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * N; i += kThreads * kRows) {
      const int which = i / N, k = i % N;
      if (k >= j.cols) continue;
      float v = 0.0f;
#pragma unroll
      for (int r = 0; r < kRows; r++) v += columns[(which * kRows + r) * N + k];
      to[which][k] = v;
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

// One register form: pieces of kW elements, kE elements a thread, kThreads threads a row, kRows rows a CTA.
struct NormForm {
  const void* fn;
  int block, rows;   // threads and rows of a CTA
  size_t smem;
  int per_sm;        // CTAs an SM holds
};
// What registers a thread and shared memory allow.
constexpr int resident(int block, int registers, size_t smem) {
  const int by_registers = 65536 / (registers * block), by_smem = (int)(232448 / (smem + 2048));
  return by_registers < by_smem ? (by_registers > 0 ? by_registers : 1) : (by_smem > 0 ? by_smem : 1);
}
template <typename T, int kW, int kE, int kThreads, int kRows, int kBatch>
NormForm forward_form() {
  typedef ForwardLayout<T, kW, kE / kW, kThreads, kRows, kBatch> L;
  static_assert(L::smem + 2048 <= 232448, "more shared memory than one CTA can have");
  return {(const void*)norm_forward_kernel<T, kW, kE / kW, kThreads, kRows, kBatch>, kThreads * kRows, kRows * kBatch, L::smem,
          resident(kThreads * kRows, kThreads * kRows > 256 ? 64 : kE * kBatch > 8 ? 128 : 72, L::smem)};
}
template <typename T, int kW, int kE, int kThreads, int kRows, int kBatch>
NormForm backward_form() {
  typedef BackwardLayout<T, kW, kE / kW, kThreads, kRows, kBatch> L;
  static_assert(L::smem + 2048 <= 232448, "more shared memory than one CTA can have");
  return {(const void*)norm_backward_kernel<T, kW, kE / kW, kThreads, kRows, kBatch>, kThreads * kRows, kRows * kBatch, L::smem,
          resident(kThreads * kRows, kThreads * kRows > 512 ? 64 : 128, L::smem)};
}
cudaError_t launch_form(const NormForm& f, void** args, int64_t ctas, cudaStream_t stream) {
  if (f.smem > 49152) {   // more than a kernel may have unasked, on the current device
    cudaError_t e = cudaFuncSetAttribute(f.fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)f.smem);
    if (e != cudaSuccess) return e;
  }
  return launch_behind(f.fn, args, dim3((unsigned)ctas), dim3(f.block), f.smem, stream);
}

// Rows of up to 256 columns take a warp each.  float16 in 16-byte pieces: as few threads as hold the row at 32 elements a
// thread; eight elements a thread where there are fewer rows than two for each SM, and for float32 and single elements, whose rows
// bring enough bytes or instructions of their own (16384 x 4096 float32: 86 us with eight, 98 with 32).
template <typename T, int kW>
NormForm pick_forward(int64_t rows, int64_t cols, int sm_count) {
  if (cols <= 256) return forward_form<T, kW, 8, 32, 8, kW == 1 ? 1 : 4>();
  if constexpr (kW == 8)
    if (rows > 2 * sm_count) {
      if (cols <= 1024) return forward_form<T, kW, 32, 32, 8, 1>();
      if (cols <= 2048) return forward_form<T, kW, 32, 64, 8, 1>();
      if (cols <= 4096) return forward_form<T, kW, 32, 128, 4, 1>();
      if (cols <= 8192) return forward_form<T, kW, 32, 256, 4, 1>();
    }
  if (cols <= 1024) return forward_form<T, kW, 8, 128, 2, 1>();
  if (cols <= 2048) return forward_form<T, kW, 8, 256, 1, 1>();
  if (cols <= 4096) return forward_form<T, kW, 8, 512, 1, 1>();
  if (cols <= 8192) return forward_form<T, kW, 8, 1024, 1, 1>();
  if (cols <= 16384) return forward_form<T, kW, 16, 1024, 1, 1>();
  return {nullptr, 0, 0, 0, 0};
}
template <typename T, int kW>
NormForm pick_backward(int64_t cols) {
  constexpr int kBatch = kW == 8 ? 4 : 2;   // 64 KB of rows on the way either way, but for single elements
  if (cols <= 256) return backward_form<T, kW, 8, 32, 8, kBatch>();
  if (cols <= 1024) return backward_form<T, kW, 8, 128, 2, kBatch>();
  if (cols <= 2048) return backward_form<T, kW, 8, 256, 1, kBatch>();
  if (cols <= 4096) return backward_form<T, kW, 8, 512, 1, kBatch>();
  if (cols <= 8192) return backward_form<T, kW, 8, 1024, 1, 1>();
  return {nullptr, 0, 0, 0, 0};
}
bool sixteen(const void* a, const void* b, const void* c, int64_t row_bytes) {
  return (((uintptr_t)a | (uintptr_t)b | (uintptr_t)c) & 15) == 0 && row_bytes % 16 == 0;
}
// CTAs that walk the rows: as many as are resident.
int64_t walkers(const NormForm& f, int64_t rows, int sm_count) {
  const int64_t need = (rows + f.rows - 1) / f.rows, most = (int64_t)sm_count * f.per_sm;
  return need < most ? (need > 0 ? need : 1) : most;
}
}  // namespace

cudaError_t launch_layer_norm(hc_dtype dtype, hc_dtype param_dtype, const void* x, const void* w, const void* b, int64_t rows,
                              int64_t cols, float epsilon, void* out, float* mean, float* rstd, int sm_count, cudaStream_t stream) {
  NormJob j = {x, nullptr, w, b, out, mean, rstd, rows, cols, epsilon, param_dtype == HC_F16};
  void* args[] = {(void*)&j};
  const bool half = dtype == HC_F16, vec = sixteen(x, out, nullptr, cols * (half ? 2 : 4));
  const NormForm f = half ? (vec ? pick_forward<__half, 8>(rows, cols, sm_count) : pick_forward<__half, 1>(rows, cols, sm_count))
                          : (vec ? pick_forward<float, 4>(rows, cols, sm_count) : pick_forward<float, 1>(rows, cols, sm_count));
  if (f.fn && rows < (1ll << 30))   // 32-bit row numbers, with room for the queue ahead
    return launch_form(f, args, walkers(f, rows, sm_count), stream);
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
  if (f.fn && rows < (1ll << 30)) return 2 * (size_t)sm_count * 2 * (size_t)cols * 4;   // at most two CTAs an SM (128 registers, 256 threads at least), whatever the alignment
  const RunSplit v = split_runs(rows, cols, 32 * (dtype == HC_F16 ? 8 : 4)), n = split_runs(rows, cols, 32);
  return 2 * (size_t)(v.runs > n.runs ? v.runs : n.runs) * (size_t)cols * 4;
}

cudaError_t launch_layer_norm_grad(hc_dtype dtype, hc_dtype param_dtype, const void* grad, const void* x, const void* w,
                                   const float* mean, const float* rstd, int64_t rows, int64_t cols, void* dx, void* dw, void* db,
                                   float* scratch, int sm_count, int* launches, cudaStream_t stream) {
  NormJob j = {x, grad, w, nullptr, dx, (float*)mean, (float*)rstd, rows, cols, 0.0f, param_dtype == HC_F16};
  *launches = 0;
  const NormForm f = backward_of(dtype, grad, x, dx, cols);
  if (f.fn && rows < (1ll << 30)) {
    const int64_t ctas = walkers(f, rows, sm_count);
    float* partial = dw || db ? scratch : nullptr;
    void* args[] = {(void*)&j, (void*)&partial};
    cudaError_t e = launch_form(f, args, ctas, stream);
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

// Products of up to eight rows, with the fused epilogue: the form of a Linear layer that serves a few tokens.
//
// Bound by reading the weights once.  Each weight is read by one thread, widened, and multiplied by all rows on the CUDA
// cores; the contraction is cut so that about three CTAs an SM have 16-byte loads in flight, and the parts go to float32 partial
// matrices that the kernel behind sums in ascending order, with the epilogue.
// Where it is taken (skinny_preferred), measured at 4096 x 16384 weights: float32, which the tensor cores take as two halves
// written by a pass of their own (4 rows: 47 us here, 200 there); weights that TMA cannot address, which would be copied whole
// first (4 rows of 4095 x 16383 float16: 44 us, 101); one row of float16 (8192 x 8192 24.1 us here, 30.5 there; 4096 x 16384 23.5,
// 26.7; 1000 x 50264 19.6, 25.0; 4096 x 1024 10.5, 10.0).  Two to eight rows of float16 are the tensor cores' (4 rows of the
// 4096 x 16384: 48 us here, 26.7 there).
// It also takes the small products of few rows that one 128 x 128 CUDA-core tile would walk alone (1024 x 1024, one row:
// 12 us for 305).
#include "epilogue.cuh"
#include "stream_order.cuh"

namespace hc {
namespace {

constexpr int kMaxChunk = 1024;   // contracted indices a CTA takes, held widened in shared memory

struct SkinnyJob {
  const void *x, *w;
  float* ws;            // [parts][M][ws_ld]
  int64_t ldx, ldw, N, K, ws_ld;
  int chunk;            // contracted indices a part
};

// Rows of x, widened, in shared memory: xs[k][m] for the column-wise form, xs[m][k] (pitch kMaxChunk) for the row-wise one.
template <typename T, int kM, bool kRowWise>
__device__ __forceinline__ void stage_x(float* xs, const T* x, int64_t ldx, int rows, int n) {
  for (int i = threadIdx.x; i < kM * n; i += 256) {
    const int m = i / n, k = i - m * n;
    xs[kRowWise ? m * kMaxChunk + k : k * kM + m] = m < rows ? widen_f<T>(x[m * ldx + k]) : 0.0f;
  }
}
template <int kM>
__device__ __forceinline__ void read_x(const float* xs, int k, float (&x)[kM]) {
  if constexpr (kM % 4 == 0) {
#pragma unroll
    for (int q = 0; q < kM / 4; q++) {
      const float4 v = *(const float4*)(xs + k * kM + q * 4);
      x[q * 4] = v.x; x[q * 4 + 1] = v.y; x[q * 4 + 2] = v.z; x[q * 4 + 3] = v.w;
    }
  } else {
#pragma unroll
    for (int m = 0; m < kM; m++) x[m] = xs[k * kM + m];
  }
}

// w stored [K][N], from the CTA's first row and column on: a thread owns eight columns (adjacent where 16-byte loads allow it,
// else 64 apart, so that a warp's loads are adjacent), four groups of 64 threads take every fourth of the `n` rows.
template <typename T, int kM, bool kVec, bool kGroups>
__device__ __forceinline__ void walk_columns(const T* w, int64_t ldw, int64_t cols, const float* xs, int n, float (&acc)[kM][8]) {
  const int tx = threadIdx.x % 64, ky = threadIdx.x / 64;
  w += kVec ? tx * 8 : tx;
  // Rows whose loads are under way together.  Single elements of few rows want more of them (4095 x 16383 float16: one row 55.7 us with
  // two, 38.5 with four; four rows 44.7, 55.9); float32 chunks of three or four rows fewer, which lets a third CTA onto an SM (4096 x
  // 16384, four rows: 55.9 us with four, 47.4 with two), and of more rows as many as fit two CTAs (eight rows: 63.6, 76.5), except
  // beside the other forms of a kernel for groups, whose registers they set (64 groups of 1024 x 4096 over two rows: 232 us, 162).
  constexpr int kAhead = kVec ? (sizeof(T) == 2 ? 8 : kM <= 2 || (kM > 4 && !kGroups) ? 4 : 2) : kM <= 2 ? 4 : 2;
  auto row = [&](int k, const float (&v)[8]) {
    float x[kM];
    read_x<kM>(xs, k, x);
#pragma unroll
    for (int m = 0; m < kM; m++)
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        const float2 s = fma2(both(x[m]), make_float2(v[e], v[e + 1]), make_float2(acc[m][e], acc[m][e + 1]));
        acc[m][e] = s.x;
        acc[m][e + 1] = s.y;
      }
  };
  for (int kb = ky; kb < n; kb += 4 * kAhead) {
    if constexpr (kVec) {
      constexpr int kPieces = sizeof(T) == 2 ? 1 : 2;
      const bool in = tx * 8 < cols;
      uint4 u[kAhead][kPieces];
#pragma unroll
      for (int i = 0; i < kAhead; i++)
#pragma unroll
        for (int q = 0; q < kPieces; q++)
          u[i][q] = kb + 4 * i < n && in ? __ldcs((const uint4*)(w + (int64_t)(kb + 4 * i) * ldw) + q) : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int i = 0; i < kAhead; i++) {
        if (kb + 4 * i >= n) break;
        float v[8];
#pragma unroll
        for (int q = 0; q < kPieces; q++) {
          float part[8 / kPieces];
          Pack16<T>::widen(u[i][q], part);
#pragma unroll
          for (int e = 0; e < 8 / kPieces; e++) v[q * (8 / kPieces) + e] = part[e];
        }
        row(kb + 4 * i, v);
      }
    } else {
      T u[kAhead][8];
#pragma unroll
      for (int i = 0; i < kAhead; i++)
#pragma unroll
        for (int e = 0; e < 8; e++) {
          T t = (T)0.0f;
          if (kb + 4 * i < n && tx + 64 * e < cols) t = w[(int64_t)(kb + 4 * i) * ldw + 64 * e];
          u[i][e] = t;
        }
#pragma unroll
      for (int i = 0; i < kAhead; i++) {
        if (kb + 4 * i >= n) break;
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = widen_f<T>(u[i][e]);
        row(kb + 4 * i, v);
      }
    }
  }
}
// The four groups' sums through shared memory (over the staged rows); `out(m, column of the strip, sum)` for the first group's.
template <int kM, bool kVec, typename F>
__device__ __forceinline__ void join_columns(float* red, const float (&acc)[kM][8], F&& out) {
  const int tx = threadIdx.x % 64, ky = threadIdx.x / 64;
  __syncthreads();
  if (ky > 0)
#pragma unroll
    for (int m = 0; m < kM; m++)
#pragma unroll
      for (int e = 0; e < 8; e++) red[((ky - 1) * kM + m) * 512 + e * 64 + tx] = acc[m][e];
  __syncthreads();
  if (ky == 0)
#pragma unroll
    for (int m = 0; m < kM; m++)
#pragma unroll
      for (int e = 0; e < 8; e++) {
        float s = acc[m][e];
#pragma unroll
        for (int g = 0; g < 3; g++) s += red[(g * kM + m) * 512 + e * 64 + tx];
        out(m, kVec ? tx * 8 + e : tx + 64 * e, s);
      }
}

// w stored [N][K], from a warp's first of four columns on: a lane takes eight adjacent contracted indices (or eight 32 apart).
constexpr int kCols = 4;
template <typename T, int kM, bool kVec>
__device__ __forceinline__ void walk_rows(const T* w0, int64_t ldw, int64_t cols, const float* xs0, int n, float (&acc)[kCols][kM]) {
  const int lane = threadIdx.x % 32;
#pragma unroll 2
  for (int kb = 0; kb < n; kb += 256) {
    float v[kCols][8];
    const T* w = w0 + kb;
    if constexpr (kVec) {
      constexpr int kPieces = sizeof(T) == 2 ? 1 : 2, E = 8 / kPieces;
      uint4 u[kCols][kPieces];
#pragma unroll
      for (int c = 0; c < kCols; c++)
#pragma unroll
        for (int q = 0; q < kPieces; q++)
          u[c][q] = c < cols && kb + lane * 8 < n ? __ldcs((const uint4*)(w + c * ldw + lane * 8) + q) : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int c = 0; c < kCols; c++)
#pragma unroll
        for (int q = 0; q < kPieces; q++) {
          float part[E];
          Pack16<T>::widen(u[c][q], part);
#pragma unroll
          for (int e = 0; e < E; e++) v[c][q * E + e] = part[e];
        }
    } else {
      T u[kCols][8];
#pragma unroll
      for (int c = 0; c < kCols; c++)
#pragma unroll
        for (int e = 0; e < 8; e++) {
          T t = (T)0.0f;
          if (c < cols && kb + lane + 32 * e < n) t = w[c * ldw + lane + 32 * e];
          u[c][e] = t;
        }
#pragma unroll
      for (int c = 0; c < kCols; c++)
#pragma unroll
        for (int e = 0; e < 8; e++) v[c][e] = widen_f<T>(u[c][e]);
    }
#pragma unroll
    for (int m = 0; m < kM; m++) {
      float x[8];
      const float* xs = xs0 + m * kMaxChunk + kb;
      if (kVec && kb + lane * 8 < n) {   // n is a multiple of eight here
        const float4 a = *(const float4*)(xs + lane * 8), b = *(const float4*)(xs + lane * 8 + 4);
        x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
      } else {
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = !kVec && kb + lane + 32 * e < n ? xs[lane + 32 * e] : 0.0f;   // beyond, the buffer holds nothing
      }
#pragma unroll
      for (int c = 0; c < kCols; c++)
#pragma unroll
        for (int e = 0; e < 8; e++) acc[c][m] = fmaf(x[e], v[c][e], acc[c][m]);
    }
  }
}
// The lanes' sums: the butterfly halves the values while it halves the lanes, so that 32 of them take 31 shuffles, not 160.
template <int kM, typename F>
__device__ __forceinline__ void join_rows(float (&acc)[kCols][kM], F&& out) {
  constexpr int kV = kCols * kM, kN = kV <= 4 ? 4 : kV <= 8 ? 8 : kV <= 16 ? 16 : 32, kShare = 32 / kN;   // lanes that end with the same sum
  const int lane = threadIdx.x % 32;
  float v[kN];
#pragma unroll
  for (int i = 0; i < kN; i++) v[i] = i < kV ? acc[i < kV ? i / kM : 0][i % kM] : 0.0f;
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
  const int i = lane / kShare;
  if (lane % kShare == 0 && i < kV) out(i % kM, i / kM, x);
}
template <int kA, int kB>
__device__ __forceinline__ void clear(float (&acc)[kA][kB]) {
#pragma unroll
  for (int a = 0; a < kA; a++)
#pragma unroll
    for (int b = 0; b < kB; b++) acc[a][b] = 0.0f;
}

template <typename T, int kM, bool kVec>
__global__ void __launch_bounds__(256) skinny_columns_kernel(const SkinnyJob j) {
  extern __shared__ __align__(16) float smem[];
  pdl_wait();
  pdl_release();
  const int64_t k0 = (int64_t)blockIdx.y * j.chunk, col0 = (int64_t)blockIdx.x * 512;
  const int n = (int)min((int64_t)j.chunk, j.K - k0);
  stage_x<T, kM, false>(smem, (const T*)j.x + k0, j.ldx, kM, n);
  __syncthreads();
  float acc[kM][8];
  clear(acc);
  walk_columns<T, kM, kVec, false>((const T*)j.w + k0 * j.ldw + col0, j.ldw, j.N - col0, smem, n, acc);
  join_columns<kM, kVec>(smem, acc, [&](int m, int c, float s) {
    if (col0 + c < j.N) j.ws[((int64_t)blockIdx.y * kM + m) * j.ws_ld + col0 + c] = s;
  });
}

template <typename T, int kM, bool kVec>
__global__ void __launch_bounds__(256) skinny_rows_kernel(const SkinnyJob j, int columns_per_warp) {
  extern __shared__ __align__(16) float smem[];
  pdl_wait();
  pdl_release();
  const int warp = threadIdx.x / 32;
  const int64_t k0 = (int64_t)blockIdx.y * j.chunk;
  const int n = (int)min((int64_t)j.chunk, j.K - k0);
  stage_x<T, kM, true>(smem, (const T*)j.x + k0, j.ldx, kM, n);
  __syncthreads();
  const int64_t first = ((int64_t)blockIdx.x * 8 + warp) * columns_per_warp;
  for (int64_t c0 = first; c0 < min(first + columns_per_warp, j.N); c0 += kCols) {
    float acc[kCols][kM];
    clear(acc);
    walk_rows<T, kM, kVec>((const T*)j.w + c0 * j.ldw + k0, j.ldw, j.N - c0, smem, n, acc);
    join_rows<kM>(acc, [&](int m, int c, float s) {
      if (c0 + c < j.N) j.ws[((int64_t)blockIdx.y * kM + m) * j.ws_ld + c0 + c] = s;
    });
  }
}

// result = epilogue(sum over parts of ws[part][M][ws_ld]).  A lane takes four columns of a row; the CTA's warps (up to eight) take
// every eighth part each, and their sums are added in order.  One thread walking all the parts, as where the tensor cores' few
// parts are summed, would wait for them in turn (one row of 4096 x 1024 float32, 128 parts: 18.1 us for the product, 11.2 here).
struct PartsJob {
  const float* ws;
  void* out;
  int64_t M, N, ws_ld, ldc;
  int parts, vec_ok;
  FusedEpilogue fe;
};
constexpr int kPartWarps = 8;
template <typename T>
__global__ void __launch_bounds__(32 * kPartWarps) sum_parts_kernel(const PartsJob j) {
  __shared__ float4 tile[kPartWarps][32];
  pdl_release();
  pdl_wait();
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, warps = blockDim.x / 32;
  const int64_t quads = j.ws_ld / 4, i = (int64_t)blockIdx.x * 32 + lane;
  const int64_t row = i / quads, n = (i - row * quads) * 4;
  float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  if (row < j.M) {
    const float* src = j.ws + row * j.ws_ld + n;
    const int64_t pitch = j.M * j.ws_ld;
#pragma unroll 4
    for (int z = warp; z < j.parts; z += warps) {
      const float4 v = __ldcg((const float4*)(src + z * pitch));
      acc.x += v.x; acc.y += v.y; acc.z += v.z; acc.w += v.w;
    }
  }
  if (warp > 0) tile[warp][lane] = acc;
  __syncthreads();
  if (warp > 0 || row >= j.M) return;
  for (int w = 1; w < warps; w++) {
    const float4 v = tile[w][lane];
    acc.x += v.x; acc.y += v.y; acc.z += v.z; acc.w += v.w;
  }
  const int valid = (int)min((int64_t)4, j.N - n);
  float x[4] = {acc.x, acc.y, acc.z, acc.w};
  const int64_t off = row * j.ldc + n;
  fused_direct<T, 4>(j.fe, off, n, valid, x);
  T* dst = (T*)j.out + off;
  T r[4];
#pragma unroll
  for (int e = 0; e < 4; e++) r[e] = narrow_f<T>(x[e]);
  if (valid == 4 && j.vec_ok) {
    if (sizeof(T) == 2) *(uint2*)dst = *(const uint2*)r;
    else *(uint4*)dst = *(const uint4*)r;
  } else {
    for (int e = 0; e < valid; e++) dst[e] = r[e];
  }
}

template <typename T, int kM>
const void* pick(bool rows_form, bool vec) {
  if (rows_form) return vec ? (const void*)skinny_rows_kernel<T, kM, true> : (const void*)skinny_rows_kernel<T, kM, false>;
  return vec ? (const void*)skinny_columns_kernel<T, kM, true> : (const void*)skinny_columns_kernel<T, kM, false>;
}
template <typename T>
const void* pick_rows(int64_t m, bool rows_form, bool vec) {
  switch (m) {
    case 1: return pick<T, 1>(rows_form, vec);
    case 2: return pick<T, 2>(rows_form, vec);
    case 3: return pick<T, 3>(rows_form, vec);
    case 4: return pick<T, 4>(rows_form, vec);
    case 5: return pick<T, 5>(rows_form, vec);
    case 6: return pick<T, 6>(rows_form, vec);
    case 7: return pick<T, 7>(rows_form, vec);
    default: return pick<T, 8>(rows_form, vec);
  }
}

struct SkinnyPlan { int64_t strips, parts; int chunk, columns_per_warp; int64_t ws_ld; size_t ws_bytes; };
SkinnyPlan plan_skinny(const GemmProblem& p, int sm_count) {
  SkinnyPlan s;
  const int64_t target = 3 * (int64_t)sm_count;
  s.columns_per_warp = 4;
  int64_t least;   // contracted indices a part is worth
  if (p.b_mn_major) {
    s.strips = (p.N + 511) / 512;
    least = 32;
  } else {
    // columns a warp takes: as many as still leave two CTAs an SM, so that the staged rows serve more than one pass
    while (s.columns_per_warp < 64 && (p.N + 16 * s.columns_per_warp - 1) / (16 * s.columns_per_warp) >= 2 * sm_count) s.columns_per_warp *= 2;
    s.strips = (p.N + 8 * s.columns_per_warp - 1) / (8 * s.columns_per_warp);
    least = 256;
  }
  int64_t parts = target / (s.strips > 0 ? s.strips : 1);
  if (parts > (p.K + least - 1) / least) parts = (p.K + least - 1) / least;
  const int64_t most = (p.K + kMaxChunk - 1) / kMaxChunk;   // parts that hold as much as a CTA can
  // Where more CTAs are needed than run at once, the column-wise form takes whole rounds of them, just filled (8192 x 28672 float16,
  // one row: 94 us with 448 CTAs, 72 with 840); the row-wise form, whose CTAs are shorter, loses by it (16384 x 4096 28.4, 32.5).
  if (parts < most) parts = p.b_mn_major ? (most * s.strips + target - 1) / target * target / s.strips : most;
  if (parts < 1) parts = 1;
  int64_t chunk = (p.K + parts - 1) / parts;
  chunk = (chunk + 7) / 8 * 8;   // parts start where 16-byte loads of a row do
  if (chunk > kMaxChunk) chunk = kMaxChunk;
  s.chunk = (int)chunk;
  s.parts = (p.K + chunk - 1) / chunk;
  s.ws_ld = (p.N + 3) & ~(int64_t)3;
  s.ws_bytes = (size_t)(s.parts * p.M * s.ws_ld) * 4;
  return s;
}

}  // namespace

bool skinny_fits(const GemmProblem& p) {
  return p.fused && p.batch == 1 && p.M >= 1 && p.M <= 8 && !p.a_mn_major && p.K >= 1 && p.K < (1ll << 25) && p.N < (1ll << 31) - 1024;
}

bool skinny_preferred(const GemmProblem& p) {
  const bool addressable = ((uintptr_t)p.B & 15) == 0 && (p.ldb * 2) % 16 == 0;
  return p.dtype == HC_F32 || !addressable || p.M == 1;
}

// ---- the same for groups of rows -------------------------------------------------------------------------------------------
namespace {

// A tile is eight rows of a group by a strip of its matrix (512 columns, or 64 of the row-wise form); the table is
// group_setup_kernel's.  The whole contraction is walked, in chunks of the staged rows.
struct FewJob {
  const void *a, *b;
  void* out;
  int64_t inner, cols;
  GroupTiles t;
  int strips;
};
template <typename T, bool kVec, bool kRowWise, int kM>
__device__ __forceinline__ void few_tile(const FewJob& j, float* smem, int g, int64_t row0, int rows, int strip) {
  const T* x = (const T*)j.a + row0 * j.inner;
  const T* w = (const T*)j.b + (int64_t)g * j.inner * j.cols;
  T* out = (T*)j.out + row0 * j.cols;
  if constexpr (!kRowWise) {
    const int64_t col0 = (int64_t)strip * 512;
    float acc[kM][8];
    clear(acc);
    for (int64_t k0 = 0; k0 < j.inner; k0 += kMaxChunk) {
      const int n = (int)min((int64_t)kMaxChunk, j.inner - k0);
      __syncthreads();
      stage_x<T, kM, false>(smem, x + k0, j.inner, rows, n);
      __syncthreads();
      walk_columns<T, kM, kVec, true>(w + k0 * j.cols + col0, j.cols, j.cols - col0, smem, n, acc);
    }
    join_columns<kM, kVec>(smem, acc, [&](int m, int c, float s) {
      if (m < rows && col0 + c < j.cols) out[m * j.cols + col0 + c] = narrow_f<T>(s);
    });
  } else {
    const int64_t first = (int64_t)strip * 64 + threadIdx.x / 32 * 8;
    float acc[2][kCols][kM];
#pragma unroll
    for (int q = 0; q < 2; q++) clear(acc[q]);
    for (int64_t k0 = 0; k0 < j.inner; k0 += kMaxChunk) {
      const int n = (int)min((int64_t)kMaxChunk, j.inner - k0);
      __syncthreads();
      stage_x<T, kM, true>(smem, x + k0, j.inner, rows, n);
      __syncthreads();
#pragma unroll
      for (int q = 0; q < 2; q++)
        if (first + 4 * q < j.cols) walk_rows<T, kM, kVec>(w + (first + 4 * q) * j.inner + k0, j.inner, j.cols - first - 4 * q, smem, n, acc[q]);
    }
#pragma unroll
    for (int q = 0; q < 2; q++)
      join_rows<kM>(acc[q], [&](int m, int c, float s) {
        if (m < rows && first + 4 * q + c < j.cols) out[m * j.cols + first + 4 * q + c] = narrow_f<T>(s);
      });
  }
}
template <typename T, bool kVec, bool kRowWise>
__global__ void __launch_bounds__(256) few_rows_kernel(const FewJob j) {
  extern __shared__ __align__(16) float smem[];
  pdl_wait();
  int lo = 0, hi = j.t.groups - 1;
  if ((int)blockIdx.x >= j.t.first_tile[j.t.groups]) return;   // the grid is for the most tiles there could be
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (j.t.first_tile[mid] <= (int)blockIdx.x) lo = mid;
    else hi = mid - 1;
  }
  const int r = (int)blockIdx.x - j.t.first_tile[lo], chunk = r / j.strips, strip = r - chunk * j.strips;
  const int64_t row0 = j.t.start[lo] + 8 * chunk;
  const int rows = min(8, (int)(j.t.end[lo] - row0));
  if (rows <= 2) few_tile<T, kVec, kRowWise, 2>(j, smem, lo, row0, rows, strip);
  else if (rows <= 4) few_tile<T, kVec, kRowWise, 4>(j, smem, lo, row0, rows, strip);
  else few_tile<T, kVec, kRowWise, 8>(j, smem, lo, row0, rows, strip);
}

// Weight gradient: a CTA's 32 x 512 outputs, eight by eight a thread, summed over the group's rows 16 at a time from shared
// memory.  Bound by writing the result, as long as the rows are few.
template <typename T, bool kVec>
__global__ void __launch_bounds__(256) few_weight_grad_kernel(const void* a, const void* b, void* out, int64_t rows, int64_t cols, GroupTiles t) {
  __shared__ __align__(16) float as[16][32], bs[16][512];
  pdl_wait();
  const int g = blockIdx.z, tx = threadIdx.x % 64, ty = threadIdx.x / 64;
  const int64_t i0 = (int64_t)blockIdx.y * 32, j0 = (int64_t)blockIdx.x * 512;
  const int start = t.start[g], n = t.end[g] - start;
  float acc[8][8];
  clear(acc);
  for (int r0 = 0; r0 < n; r0 += 16) {
    const int nr = min(16, n - r0);
    __syncthreads();
    for (int i = threadIdx.x; i < nr * 32; i += 256) {
      const int r = i / 32, c = i % 32;
      as[r][c] = i0 + c < rows ? widen_f<T>(((const T*)a)[(start + r0 + r) * rows + i0 + c]) : 0.0f;
    }
    for (int i = threadIdx.x; i < nr * 512; i += 256) {
      const int r = i / 512, c = i % 512;
      bs[r][c] = j0 + c < cols ? widen_f<T>(((const T*)b)[(start + r0 + r) * cols + j0 + c]) : 0.0f;
    }
    __syncthreads();
    for (int r = 0; r < nr; r++) {
      float x[8], v[8];
#pragma unroll
      for (int e = 0; e < 8; e++) {
        x[e] = as[r][ty * 8 + e];
        v[e] = bs[r][kVec ? tx * 8 + e : tx + 64 * e];
      }
#pragma unroll
      for (int p = 0; p < 8; p++)
#pragma unroll
        for (int e = 0; e < 8; e++) acc[p][e] = fmaf(x[p], v[e], acc[p][e]);
    }
  }
  T* dst = (T*)out + (int64_t)g * rows * cols;
#pragma unroll
  for (int p = 0; p < 8; p++) {
    const int64_t i = i0 + ty * 8 + p;
    if (i >= rows) break;
    if constexpr (kVec) {
      if (j0 + tx * 8 >= cols) continue;
      constexpr int W = Pack16<T>::W;
#pragma unroll
      for (int q = 0; q < 8 / W; q++) {
        float v[W];
#pragma unroll
        for (int e = 0; e < W; e++) v[e] = acc[p][q * W + e];
        *(uint4*)(dst + i * cols + j0 + tx * 8 + q * W) = Pack16<T>::narrow(v);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; e++)
        if (j0 + tx + 64 * e < cols) dst[i * cols + j0 + tx + 64 * e] = narrow_f<T>(acc[p][e]);
    }
  }
}

template <typename T>
cudaError_t launch_few_typed(const GroupedProblem& p, const GroupTiles& t, int64_t tiles, cudaStream_t stream) {
  if (p.weight_grad) {
    const bool vec = ((uintptr_t)p.out & 15) == 0 && p.cols % 8 == 0;
    const void *a = p.a, *b = p.b;
    void* out = p.out;
    int64_t rows = p.rows, cols = p.cols;
    void* args[] = {(void*)&a, (void*)&b, (void*)&out, (void*)&rows, (void*)&cols, (void*)&t};
    return launch_behind(vec ? (const void*)few_weight_grad_kernel<T, true> : (const void*)few_weight_grad_kernel<T, false>, args,
                         dim3((unsigned)((cols + 511) / 512), (unsigned)((rows + 31) / 32), (unsigned)p.groups), dim3(256), 0, stream);
  }
  const int64_t ld = p.trans_b ? p.inner : p.cols;
  const bool vec = ((uintptr_t)p.b & 15) == 0 && ld % 8 == 0;
  FewJob j = {p.a, p.b, p.out, p.inner, p.cols, t, few_strips(p)};
  void* args[] = {(void*)&j};
  const void* fn = p.trans_b ? (const void*)few_rows_kernel<T, false, true> : (const void*)few_rows_kernel<T, false, false>;
  if constexpr (sizeof(T) == 4)   // float16 that 16-byte loads can read is the tensor cores'
    if (vec) fn = p.trans_b ? (const void*)few_rows_kernel<T, true, true> : (const void*)few_rows_kernel<T, true, false>;
  return launch_behind(fn, args, dim3((unsigned)tiles), dim3(256), 49152, stream);   // eight staged rows; three groups' sums
}

}  // namespace

int few_strips(const GroupedProblem& p) { return (int)((p.cols + (p.trans_b ? 63 : 511)) / (p.trans_b ? 64 : 512)); }

// Groups of few rows, on the average (the offsets are not known to the host).  Forward: where the tensor cores would first have the
// weights copied or split, which reads and writes them once more each (57 experts of 1049 x 2832 float32, two rows each:
// 545 us there, 148 here); weight gradient: while a sum over the rows costs less than writing the result
// (104 groups of 312 x 1251 float32 over nine rows in all: 331 us there, 34 here), but for float16 that TMA can address (64 groups of
// 1024 x 4096 over two rows each: 128 us there, 150 here).
bool few_preferred(const GroupedProblem& p) {
  const int64_t eb = p.dtype == HC_F16 ? 2 : 4, mean = (p.total_rows + p.groups - 1) / p.groups;
  if (p.weight_grad) {
    const bool by_tma = p.rows % 8 == 0 && p.cols % 8 == 0 && (((uintptr_t)p.a | (uintptr_t)p.b | (uintptr_t)p.out) & 15) == 0;
    return (p.rows + 31) / 32 <= 65535 && (p.dtype == HC_F32 ? mean <= 16 : mean <= 8 && !by_tma);
  }
  const int64_t ld = p.trans_b ? p.inner : p.cols;
  const bool addressable = ((uintptr_t)p.b & 15) == 0 && (ld * eb) % 16 == 0;
  return mean <= 8 && p.inner > 0 && (p.dtype == HC_F32 || !addressable);
}

cudaError_t launch_few(const GroupedProblem& p, const GroupTiles& t, int64_t tiles, cudaStream_t stream) {
  return p.dtype == HC_F16 ? launch_few_typed<__half>(p, t, tiles, stream) : launch_few_typed<float>(p, t, tiles, stream);
}

cudaError_t launch_skinny(const GemmProblem& p, cudaStream_t stream, void* scratch, size_t scratch_bytes, int sm_count, LaunchRecord* rec,
                          size_t* scratch_needed) {
  const SkinnyPlan s = plan_skinny(p, sm_count);
  *scratch_needed = s.ws_bytes;
  if (!scratch || scratch_bytes < s.ws_bytes) return cudaErrorInvalidValue;
  if (s.strips > 2147483647LL || s.parts > 65535) return cudaErrorInvalidValue;
  const int64_t eb = p.dtype == HC_F16 ? 2 : 4;
  const bool vec = ((uintptr_t)p.B & 15) == 0 && (p.ldb * eb) % 16 == 0 && (p.b_mn_major ? p.N : p.K) % 8 == 0;
  SkinnyJob j = {p.A, p.B, (float*)scratch, p.lda, p.ldb, p.N, p.K, s.ws_ld, s.chunk};
  int per_warp = s.columns_per_warp;
  void* args[] = {(void*)&j, (void*)&per_warp};
  const bool rows_form = !p.b_mn_major;
  const void* fn = p.dtype == HC_F16 ? pick_rows<__half>(p.M, rows_form, vec) : pick_rows<float>(p.M, rows_form, vec);
  // the staged rows, and over them the groups' sums
  const size_t staged = (size_t)p.M * (rows_form ? kMaxChunk : s.chunk) * 4, sums = rows_form ? 0 : (size_t)p.M * 3 * 512 * 4;
  *rec = LaunchRecord();
  rec->kernel = HC_KERNEL_SIMT;
  rec->tile_m = (int)p.M; rec->tile_n = rows_form ? 8 * s.columns_per_warp : 512; rec->tile_k = s.chunk; rec->stages = 1;
  rec->grid = (int)s.strips; rec->block = 256; rec->tiles = s.strips * s.parts; rec->scratch_bytes = s.ws_bytes;
  cudaError_t e = launch_behind(fn, args, dim3((unsigned)s.strips, (unsigned)s.parts), dim3(256), staged > sums ? staged : sums, stream);
  if (e != cudaSuccess) return e;
  rec->launches = 2;
  PartsJob sum = {(const float*)scratch, p.C, p.M, p.N, s.ws_ld, p.ldc, (int)s.parts, ((uintptr_t)p.C & (4 * eb - 1)) == 0 && p.ldc % 4 == 0, p.fe};
  void* sum_args[] = {(void*)&sum};
  const int warps = s.parts < kPartWarps ? (int)s.parts : kPartWarps;
  const int64_t blocks = (p.M * (s.ws_ld / 4) + 31) / 32;
  return launch_behind(p.dtype == HC_F16 ? (const void*)sum_parts_kernel<__half> : (const void*)sum_parts_kernel<float>, sum_args,
                       dim3((unsigned)blocks), dim3(32 * warps), 0, stream);
}

}  // namespace hc

// Products of up to eight rows, with the fused epilogue: the form of a Linear layer that serves a few tokens.
//
// Bound by reading the weights once.  Each weight is read by one thread, widened, and multiplied by all rows on the CUDA
// cores; the contraction is cut so that about three CTAs an SM have 16-byte loads in flight, and the parts go to float32 partial
// matrices that the kernel behind sums in ascending order, with the epilogue.
// Where it is taken (skinny_preferred), measured at 4096 x 16384 weights: float32, which the tensor cores take as two halves
// written by a pass of their own (4 rows: 57 us here, 200 there); weights that TMA cannot address, which would be copied whole
// first (4 rows of 4095 x 16383 float16: 48 us, 271); one row of float16 (25.7 us whatever the activation, 26 to 28 there;
// the floor is 20.5).  Two to eight rows of float16 are the tensor cores' (4 rows: 48 us here, 26 there).
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

template <typename T, int kM>
__device__ __forceinline__ void stage_x(const SkinnyJob& j, float* xs, int64_t k0, int n, bool k_inner) {
  // xs[k][m] for the column-wise kernel, xs[m][k] for the row-wise one
  for (int i = threadIdx.x; i < kM * n; i += 256) {
    const int m = i / n, k = i - m * n;
    xs[k_inner ? m * kMaxChunk + k : k * kM + m] = widen_f<T>(((const T*)j.x)[m * j.ldx + k0 + k]);
  }
}

// w stored [K][N]: a thread owns eight columns (adjacent where 16-byte loads allow it, else 64 apart, so that a warp's loads
// are adjacent), four groups of 64 threads take every fourth row of the part.
template <typename T, int kM, bool kVec>
__global__ void __launch_bounds__(256) skinny_columns_kernel(const SkinnyJob j) {
  extern __shared__ __align__(16) float smem[];
  pdl_wait();
  pdl_release();
  const int tx = threadIdx.x % 64, ky = threadIdx.x / 64;
  const int64_t k0 = (int64_t)blockIdx.y * j.chunk;
  const int n = (int)min((int64_t)j.chunk, j.K - k0);
  const int64_t col0 = (int64_t)blockIdx.x * 512;
  stage_x<T, kM>(j, smem, k0, n, false);
  __syncthreads();
  float acc[kM][8];
#pragma unroll
  for (int m = 0; m < kM; m++)
#pragma unroll
    for (int e = 0; e < 8; e++) acc[m][e] = 0.0f;
  const T* w = (const T*)j.w + k0 * j.ldw + col0 + (kVec ? tx * 8 : tx);
  bool in[kVec ? 1 : 8];
  if (kVec) in[0] = col0 + tx * 8 < j.N;
  else
#pragma unroll
    for (int e = 0; e < 8; e++) in[e % (kVec ? 1 : 8)] = col0 + tx + 64 * e < j.N;
  constexpr int kAhead = kVec ? (sizeof(T) == 2 ? 8 : 4) : 2;   // rows whose loads are under way together
  auto row = [&](int k, const float (&v)[8]) {
    float x[kM];
#pragma unroll
    for (int m = 0; m < kM; m++) x[m] = smem[k * kM + m];
#pragma unroll
    for (int m = 0; m < kM; m++)
#pragma unroll
      for (int e = 0; e < 8; e++) acc[m][e] = fmaf(x[m], v[e], acc[m][e]);
  };
  for (int kb = ky; kb < n; kb += 4 * kAhead) {
    if constexpr (kVec) {
      constexpr int kPieces = sizeof(T) == 2 ? 1 : 2;
      uint4 u[kAhead][kPieces];
#pragma unroll
      for (int i = 0; i < kAhead; i++)
#pragma unroll
        for (int q = 0; q < kPieces; q++)
          u[i][q] = kb + 4 * i < n && in[0] ? __ldcs((const uint4*)(w + (int64_t)(kb + 4 * i) * j.ldw) + q) : make_uint4(0, 0, 0, 0);
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
          if (kb + 4 * i < n && in[e]) t = w[(int64_t)(kb + 4 * i) * j.ldw + 64 * e];
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
  // the four groups' sums, over the rows in shared memory
  __syncthreads();
  float* red = smem;   // [3][kM][512]
  if (ky > 0)
#pragma unroll
    for (int m = 0; m < kM; m++)
#pragma unroll
      for (int e = 0; e < 8; e++) red[((ky - 1) * kM + m) * 512 + (kVec ? e * 64 + tx : tx + 64 * e)] = acc[m][e];
  __syncthreads();
  if (ky > 0) return;
#pragma unroll
  for (int m = 0; m < kM; m++)
#pragma unroll
    for (int e = 0; e < 8; e++) {
      float s = acc[m][e];
#pragma unroll
      for (int g = 0; g < 3; g++) s += red[(g * kM + m) * 512 + e * 64 + tx];
      const int64_t col = col0 + (kVec ? tx * 8 + e : tx + 64 * e);
      if (col < j.N) j.ws[((int64_t)blockIdx.y * kM + m) * j.ws_ld + col] = s;
    }
}

// w stored [N][K]: a warp takes four columns at a time along the part, a lane eight adjacent contracted indices (or eight 32 apart).
template <typename T, int kM, bool kVec>
__global__ void __launch_bounds__(256) skinny_rows_kernel(const SkinnyJob j, int columns_per_warp) {
  extern __shared__ __align__(16) float smem[];
  pdl_wait();
  pdl_release();
  constexpr int kCols = 4;
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int64_t k0 = (int64_t)blockIdx.y * j.chunk;
  const int n = (int)min((int64_t)j.chunk, j.K - k0);
  stage_x<T, kM>(j, smem, k0, n, true);
  __syncthreads();
  const int64_t first = ((int64_t)blockIdx.x * 8 + warp) * columns_per_warp;
  for (int64_t c0 = first; c0 < min(first + columns_per_warp, j.N); c0 += kCols) {
    float acc[kCols][kM];
#pragma unroll
    for (int c = 0; c < kCols; c++)
#pragma unroll
      for (int m = 0; m < kM; m++) acc[c][m] = 0.0f;
#pragma unroll 2
    for (int kb = 0; kb < n; kb += 256) {
      float v[kCols][8];
      const T* w = (const T*)j.w + c0 * j.ldw + k0 + kb;
      if constexpr (kVec) {
        constexpr int kPieces = sizeof(T) == 2 ? 1 : 2, E = 8 / kPieces;
        uint4 u[kCols][kPieces];
#pragma unroll
        for (int c = 0; c < kCols; c++)
#pragma unroll
          for (int q = 0; q < kPieces; q++)
            u[c][q] = c0 + c < j.N && kb + lane * 8 < n ? __ldcs((const uint4*)(w + c * j.ldw + lane * 8) + q) : make_uint4(0, 0, 0, 0);
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
            if (c0 + c < j.N && kb + lane + 32 * e < n) t = w[c * j.ldw + lane + 32 * e];
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
        const float* xs = smem + m * kMaxChunk + kb;
#pragma unroll
        for (int e = 0; e < 8; e++) {
          const int at = kVec ? lane * 8 + e : lane + 32 * e;
          x[e] = kb + at < n ? xs[at] : 0.0f;   // beyond the part the buffer holds nothing
        }
#pragma unroll
        for (int c = 0; c < kCols; c++)
#pragma unroll
          for (int e = 0; e < 8; e++) acc[c][m] = fmaf(x[e], v[c][e], acc[c][m]);
      }
    }
#pragma unroll
    for (int c = 0; c < kCols; c++)
#pragma unroll
      for (int m = 0; m < kM; m++) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) acc[c][m] += __shfl_xor_sync(0xffffffffu, acc[c][m], o);
        if (lane == c * kM + m && c0 + c < j.N) j.ws[((int64_t)blockIdx.y * kM + m) * j.ws_ld + c0 + c] = acc[c][m];
      }
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
  if (parts < (p.K + kMaxChunk - 1) / kMaxChunk) parts = (p.K + kMaxChunk - 1) / kMaxChunk;
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
  return launch_sum_parts(p, (const float*)scratch, s.ws_ld, (int)s.parts, stream);
}

}  // namespace hc

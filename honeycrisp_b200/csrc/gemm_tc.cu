// Dense products on the tensor-core kernel of tc_kernel.cuh: choice of the tile shape and of a cut
// of the contraction, work area, prepared launches, and the kernel that sums the parts of a cut
// contraction.
#include "tc_kernel.cuh"

namespace hc {
namespace {

// Self-test of the bounded wait: one thread waits on a barrier that nothing will ever arrive
// on, with a short limit, through the same wait routine the GEMM kernel uses.  The wait gives
// up, the status word gets its bit, and the kernel returns normally.
__global__ void wait_probe_kernel(unsigned int* status, unsigned long long limit_ns) {
  __shared__ __align__(8) uint64_t bar;
  __shared__ int abort_flag;
  if (threadIdx.x == 0) {
    abort_flag = 0;
    mbar_init(smem_u32(&bar), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    if (!mbar_wait_slow(smem_u32(&bar), 0, &abort_flag, limit_ns)) atomicOr(status, kDevTimeoutSelfTest);
  }
}

// Second half of a cut contraction: result = round(sum over parts, ascending, of the float32
// partial matrices) (+ bias, as a second rounded operation for float16, exactly like the
// epilogue of the uncut kernel).  Four columns per thread; the partial matrices have a row pitch
// that is a multiple of four floats, so every load is one aligned float4.
struct ReduceJob {
  const float* ws;
  void* C;
  const void* bias;
  int64_t M, N, ws_ld, batch, ldc, strideC;
  int parts, vec_ok;
  FusedEpilogue fe;    // kFusedSum only
};

template <bool kHalf, bool kFusedSum = false>
__global__ void __launch_bounds__(256) splitk_reduce_kernel(const ReduceJob j) {
  pdl_release();
  pdl_wait();
  const int64_t groups = j.ws_ld / 4;
  const int64_t total = j.batch * j.M * groups;
  const int64_t part_stride = j.M * j.ws_ld;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t g = i % groups, row = (i / groups) % j.M, mat = i / (groups * j.M);
    const int64_t n = g * 4;
    const float* src = j.ws + (mat * j.parts) * part_stride + row * j.ws_ld + n;
    float4 acc = __ldcg((const float4*)src);
    for (int z = 1; z < j.parts; z++) {
      const float4 v = __ldcg((const float4*)(src + z * part_stride));
      acc.x = __fadd_rn(acc.x, v.x); acc.y = __fadd_rn(acc.y, v.y);
      acc.z = __fadd_rn(acc.z, v.z); acc.w = __fadd_rn(acc.w, v.w);
    }
    float x[4] = {acc.x, acc.y, acc.z, acc.w};
    const int valid = (int)min((int64_t)4, j.N - n);
    if (kFusedSum) {
      typedef typename std::conditional<kHalf, __half, float>::type T;
      const int64_t off = mat * j.strideC + row * j.ldc + n;
      fused_direct<T, 4>(j.fe, off, n, valid, x);
      T* dst = (T*)j.C + off;
      T r[4];
#pragma unroll
      for (int e = 0; e < 4; e++) r[e] = narrow_f<T>(x[e]);
      if (valid == 4 && j.vec_ok) {
        if (kHalf) *(uint2*)dst = *(const uint2*)r;
        else *(uint4*)dst = *(const uint4*)r;
      } else {
        for (int e = 0; e < valid; e++) dst[e] = r[e];
      }
    } else if (kHalf) {
      __half h[4];
#pragma unroll
      for (int e = 0; e < 4; e++) {
        h[e] = __float2half_rn(x[e]);
        if (j.bias && e < valid)
          h[e] = __float2half_rn(__fadd_rn(__half2float(h[e]), __half2float(((const __half*)j.bias)[n + e])));
      }
      __half* dst = (__half*)j.C + mat * j.strideC + row * j.ldc + n;
      if (valid == 4 && j.vec_ok) {
        *(uint2*)dst = *(const uint2*)h;
      } else {
        for (int e = 0; e < valid; e++) dst[e] = h[e];
      }
    } else {
      if (j.bias)
#pragma unroll
        for (int e = 0; e < 4; e++)
          if (e < valid) x[e] = __fadd_rn(x[e], ((const float*)j.bias)[n + e]);
      float* dst = (float*)j.C + mat * j.strideC + row * j.ldc + n;
      if (valid == 4 && j.vec_ok) {
        *(float4*)dst = make_float4(x[0], x[1], x[2], x[3]);
      } else {
        for (int e = 0; e < valid; e++) dst[e] = x[e];
      }
    }
  }
}

}  // namespace

cudaError_t launch_wait_probe(cudaStream_t stream, unsigned int* status_word, unsigned long long limit_ns) {
  wait_probe_kernel<<<1, 32, 0, stream>>>(status_word, limit_ns);
  return cudaGetLastError();
}

// Any product of sane size runs on the tensor cores: operands TMA cannot address directly
// (unaligned base, pitches that are not 16-byte multiples) are repacked into the work area first
// - the float32 split does that anyway - and a result TMA cannot address is stored from registers.
bool tc_supported(const GemmProblem& p) {
  if (p.M <= 0 || p.N <= 0 || p.K <= 0 || p.batch <= 0) return false;
  if (p.M >= (1ll << 31) - 256 || p.N >= (1ll << 31) - 256 || p.K >= (1ll << 31) - 256 || p.batch >= (1ll << 31))
    return false;
  return encode_fn() != nullptr;
}

// float32 products: the lo halves of both operands are stored compactly, with the leading
// dimension rounded up to four elements so TMA can address them.  The hi half is the operand
// where it lies; only an operand TMA cannot address (base or pitches not multiples of 16 bytes)
// is also copied, into the same compact layout.
struct SplitLayout {
  int64_t a_rows, a_width, a_ld, a_mat, b_rows, b_width, b_ld, b_mat;
  size_t a_bytes, b_bytes;   // of one compact array
  bool a_copy, b_copy;       // the operand needs a TMA-addressable copy as its hi half
};
static SplitLayout split_layout(const GemmProblem& p) {
  SplitLayout s;
  s.a_rows = p.a_mn_major ? p.K : p.M; s.a_width = p.a_mn_major ? p.M : p.K;
  s.b_rows = p.b_mn_major ? p.K : p.N; s.b_width = p.b_mn_major ? p.N : p.K;
  s.a_ld = round4(s.a_width); s.b_ld = round4(s.b_width);
  s.a_mat = s.a_rows * s.a_ld; s.b_mat = s.b_rows * s.b_ld;
  s.a_bytes = ((size_t)(s.a_mat * p.batch) * 4 + 255) & ~(size_t)255;
  s.b_bytes = ((size_t)(s.b_mat * p.batch) * 4 + 255) & ~(size_t)255;
  s.a_copy = !operand_ok(p.A, 4, p.lda, p.strideA, p.batch, p.M, p.K);
  s.b_copy = !operand_ok(p.B, 4, p.ldb, p.strideB, p.batch, p.N, p.K);
  return s;
}

// float16 operands that need repacking: packed copy with the leading dimension rounded to 8.
struct RepackLayout {
  bool a, b;
  int64_t a_rows, a_width, a_ld, a_mat, b_rows, b_width, b_ld, b_mat;
  size_t a_bytes, b_bytes;
};
static RepackLayout repack_layout(const GemmProblem& p) {
  RepackLayout r;
  r.a = !operand_ok(p.A, 2, p.lda, p.strideA, p.batch, p.M, p.K);
  r.b = !operand_ok(p.B, 2, p.ldb, p.strideB, p.batch, p.N, p.K);
  r.a_rows = p.a_mn_major ? p.K : p.M; r.a_width = p.a_mn_major ? p.M : p.K;
  r.b_rows = p.b_mn_major ? p.K : p.N; r.b_width = p.b_mn_major ? p.N : p.K;
  r.a_ld = (r.a_width + 7) & ~7ll; r.b_ld = (r.b_width + 7) & ~7ll;
  r.a_mat = r.a_rows * r.a_ld; r.b_mat = r.b_rows * r.b_ld;
  r.a_bytes = r.a ? (((size_t)(r.a_mat * p.batch) * 2 + 255) & ~(size_t)255) : 0;
  r.b_bytes = r.b ? (((size_t)(r.b_mat * p.batch) * 2 + 255) & ~(size_t)255) : 0;
  return r;
}

// ---- choice of tile shape and of a cut of the contraction ------------------------------------
struct TcPlan {
  int shape = SHAPE_PAIR;
  int slabs = 1;            // k slabs per pipeline slot
  int splits = 1;           // parts of the contraction (1: none)
  int kb_per_split = 0;     // slots per part
  int64_t ws_ld = 0;        // row pitch (floats) of one partial matrix
  size_t ws_bytes = 0;      // float32 partial sums: splits x batch x M x ws_ld
};

constexpr size_t kMaxSplitWorkspace = 256ull << 20;

// The cost model.  A shape costs (waves of tiles over the SMs) x (clocks per tile); the clocks
// per 64-wide k block of each float16 shape are measured on large products (relative to 600 for
// the 256x256 pair), plus a fixed cost per tile for refilling the pipeline.  Large tiles move the
// fewest operand bytes per flop and win whenever there are enough tiles to fill the SMs; for small
// products the small pair shapes spread the work over more SMs, which shortens the one wave there
// is.  Only the 256x512 shape cannot hide the result drain behind the next tile.
// When even the smallest shape leaves most SMs idle and the contraction is long (the weight
// gradient of a small Linear layer: few outputs, many tokens), the contraction is cut into up to
// 16 parts that run as separate tiles into float32 partial matrices, summed in ascending part
// order by a second kernel (splitk_reduce_kernel): deterministic, and float16 still rounds once.
// float32 (3xTF32, 12 MMAs per 32-wide slab) goes through the same model with its own clocks.
TcPlan plan_tc(const GemmProblem& p, int sm_count, bool may_split, const Tunables& tun) {
  const bool f32 = p.dtype == HC_F32;
  const int BK = f32 ? 32 : 64;
  const int dbg = debug_flags();
  const int kslabs = (int)((p.K + BK - 1) / BK);
  // A block of a larger product is planned as the whole product.
  const int64_t M = p.plan_M > 0 ? p.plan_M : p.M, N = p.plan_N > 0 ? p.plan_N : p.N;
  const bool pairs_ok = M > BM && !(dbg & 4);
  struct Cand { int shape; bool ok; int rows, cols, slots, slabs; double clk_per_slab, drain_per_tile; bool splittable; };
  const double drain = 2400.0, refill = 300.0;
  const int pair_slots = sm_count / 2;
  Cand cands[SHAPE_COUNT - 1];
  int n_cands = 0;
  if (!f32) {
    // A fused epilogue takes longer than the half-by-half drain of the 512-wide tile hides.
    const bool wide_ok = pairs_ok && N >= 1024 && kslabs >= tun.wide_min_kb && !p.fused;
    cands[n_cands++] = {SHAPE_WIDE, wide_ok, 256, 512, pair_slots, 1, 1140.0, drain, false};
    cands[n_cands++] = {SHAPE_PAIR, pairs_ok && N > 128, 256, 256, pair_slots, 1, 600.0, 0.0, true};
    cands[n_cands++] = {SHAPE_C1_256, N > 128, 128, 256, sm_count, 1, 680.0, 0.0, false};
    cands[n_cands++] = {SHAPE_C1_128, true, 128, 128, sm_count, 2, 410.0, 0.0, true};
    cands[n_cands++] = {SHAPE_PAIR_128, pairs_ok && N > 64, 256, 128, pair_slots, 2, 340.0, 0.0, true};
    // 32 columns of B per CTA: half a 128-byte row of an MN-major box, which the copy cannot split
    cands[n_cands++] = {SHAPE_PAIR_64, pairs_ok && !p.b_mn_major, 256, 64, pair_slots, 2, 265.0, 0.0, true};
  } else {
    // float32 (3xTF32): 12 MMAs per 32-wide slab; clocks per slab measured the same way.  The small
    // pair shapes need the windowed epilogue (they are not built for the no-window debug mode).
    const bool small_ok = pairs_ok && !(dbg & 2);
    cands[n_cands++] = {SHAPE_WIDE, false, 256, 512, pair_slots, 1, 0.0, 0.0, false};
    // The fused epilogue's unrolled blocks do not fit the registers beside 128 running sums a thread, so it
    // takes the 128-wide tiles (4100 x 1000 x 4100 with GELU: 309 us on 256-wide tiles, 181 on these).
    cands[n_cands++] = {SHAPE_PAIR, pairs_ok && N > 128 && !p.fused, 256, 256, pair_slots, 1, 1700.0, 0.0, true};
    cands[n_cands++] = {SHAPE_C1_256, N > 128 && !p.fused, 128, 256, sm_count, 1, 1900.0, 0.0, true};
    cands[n_cands++] = {SHAPE_C1_128, true, 128, 128, sm_count, 1, 1130.0, 0.0, true};
    cands[n_cands++] = {SHAPE_PAIR_128, small_ok && N > 64, 256, 128, pair_slots, 1, 950.0, 0.0, true};
    cands[n_cands++] = {SHAPE_PAIR_64, small_ok, 256, 64, pair_slots, 1, 615.0, 0.0, true};
  }
  const int forced = tun.shape;
  const int forced_splits = tun.splits;   // 1: never cut; n > 1: cut into n where possible
  int choices[8] = {1, 2, 3, 4, 6, 8, 12, 16};
  int n_choices = 8;
  if (forced_splits > 1) { choices[0] = forced_splits > 64 ? 64 : forced_splits; n_choices = 1; }
  TcPlan best;
  double best_cost = -1.0;
  for (int ci = 0; ci < n_cands; ci++) {
    const Cand& c = cands[ci];
    if (!c.ok || c.slots < 1) continue;
    if (forced >= 1 && forced < SHAPE_COUNT && cands[forced - 1].ok && c.shape != forced) continue;
    const int64_t tiles = ((M + c.rows - 1) / c.rows) * ((N + c.cols - 1) / c.cols) * p.batch;
    const int kslots = (kslabs + c.slabs - 1) / c.slabs;
    const int64_t ws_ld = (p.N + 3) & ~3ll;   // of this block
    // (matrix index x parts must stay a 32-bit tensor-map coordinate)
    const bool can_split = may_split && c.splittable && !p.no_split && forced_splits != 1 && p.batch < (1ll << 24);
    for (int i = 0; i < n_choices; i++) {
      int want = can_split ? choices[i] : 1;
      if (want > kslots) want = kslots;
      if (want < 1) want = 1;
      int per = (kslots + want - 1) / want;
      if (want > 1 && forced_splits <= 1 && per * c.slabs < 8) break;   // at least 8 slabs per part
      if (want > 1 && forced_splits <= 1 && tiles >= c.slots) break;    // a full wave needs no cut
      const int parts = (kslots + per - 1) / per;
      const size_t ws = parts > 1 ? (size_t)parts * p.batch * p.M * ws_ld * 4 : 0;
      // the limit applies to the whole product, so that a block of it is cut like the whole
      if (parts > 1 && (size_t)parts * p.batch * M * ((N + 3) & ~3ll) * 4 > kMaxSplitWorkspace) break;
      const int64_t units = tiles * parts;
      const int64_t waves = (units + c.slots - 1) / c.slots;
      double cost = (double)waves * ((double)per * c.slabs * c.clk_per_slab + c.drain_per_tile + refill) +
                    (c.drain_per_tile > 0 ? 0.0 : drain);
      if (parts > 1) cost += 2500.0 + (double)ws / 3000.0;   // the second launch and its traffic
      if (best_cost < 0 || cost < best_cost) {
        best_cost = cost;
        best.shape = c.shape; best.slabs = c.slabs; best.splits = parts; best.kb_per_split = per;
        best.ws_ld = ws_ld; best.ws_bytes = ws;
      }
      if (!can_split) break;
    }
  }
  return best;
}

static size_t operand_scratch_bytes(const GemmProblem& p) {
  if (p.dtype != HC_F32) {
    const RepackLayout r = repack_layout(p);
    return r.a_bytes + r.b_bytes;
  }
  const SplitLayout s = split_layout(p);
  return (s.a_copy ? 2 : 1) * s.a_bytes + (s.b_copy ? 2 : 1) * s.b_bytes;
}

// Work area of one product: re-laid operands (float32 hi/lo parts, repacked float16), then,
// 256-byte aligned, the partial matrices of a cut contraction.
size_t tc_scratch_bytes(const GemmProblem& p, int sm_count) {
  const size_t ops = operand_scratch_bytes(p);
  const TcPlan plan = plan_tc(p, sm_count, true, read_tunables());
  return plan.ws_bytes ? ((ops + 255) & ~(size_t)255) + plan.ws_bytes : ops;
}

PlanSummary tc_describe_plan(const GemmProblem& p, int sm_count) {
  const TcPlan plan = plan_tc(p, sm_count, true, read_tunables());
  static const int kRows[SHAPE_COUNT] = {0, 256, 256, 128, 128, 256, 256};
  static const int kCols[SHAPE_COUNT] = {0, 512, 256, 256, 128, 128, 64};
  PlanSummary r;
  r.tile_m = kRows[plan.shape]; r.tile_n = kCols[plan.shape];
  r.ctas = r.tile_m / BM;
  r.slabs = plan.slabs; r.parts = plan.splits;
  const int BK = p.dtype == HC_F32 ? 32 : 64;
  const int kslots = (int)(((p.K + BK - 1) / BK + plan.slabs - 1) / plan.slabs);
  r.slots_per_part = plan.splits > 1 ? plan.kb_per_split : kslots;
  r.tiles = ((p.M + r.tile_m - 1) / r.tile_m) * ((p.N + r.tile_n - 1) / r.tile_n) * p.batch * plan.splits;
  r.ws_bytes = plan.ws_bytes;
  return r;
}

// ---- a product, prepared once and issued many times ------------------------------------------
// Planning a product (tile shape, cut, tensor maps: four driver calls) costs the host several
// microseconds, which is as long as the kernel of a small product runs.  A training loop issues
// the same products - same buffers, same shapes - step after step, so the context keeps the
// prepared launches of the products it has seen most recently and a repeat costs one lookup.
namespace {

struct TcPrepared {
  int pre = 0;                       // pre-pass: 0 none, 1 repack float16 operands, 2 split float32 operands
  RepackJob rja, rjb;
  SplitJob sja, sjb;
  int pre_blocks_a = 0, pre_blocks_b = 0;
  CUtensorMap maps[4];
  OutMaps outs;
  TcParams tp;
  TcLaunchFn fn = nullptr;
  bool cut = false;                  // second kernel sums the parts of a cut contraction
  bool reduce_half = false, reduce_fused = false;
  ReduceJob job;
  int reduce_blocks = 0;
  size_t scratch_used = 0;           // bytes of the work area this product touches
  // Address ranges the main kernel reads (operands, bias) and this device's range it writes.
  uintptr_t in_lo[3] = {0, 0, 0}, in_hi[3] = {0, 0, 0};
  uintptr_t out_lo = 0, out_hi = 0;
  bool trackable = false;            // one kernel, no pre-pass, no second kernel: the ranges say it all
};

// What the tensor-core kernel most recently launched on a stream wrote.  Consulted only for
// streams the library owns (nobody else enqueues kernels there), where it decides whether the
// next kernel's operand loads may run ahead of the wait for its predecessor.  A launch that was captured
// into a graph is a predecessor to launches of the same capture only: it has not run, and what is
// launched next on the stream follows what was launched before the capture.
struct StreamTrack {
  cudaStream_t stream = nullptr;
  bool used = false, known = false;
  unsigned long long capture = 0;   // 0: launched, else the capture's id
  uintptr_t lo = 0, hi = 0;
  uint64_t stamp = 0;
};
std::mutex g_track_mu;
StreamTrack g_track[16];
uint64_t g_track_clock = 0;

StreamTrack* track_entry(cudaStream_t stream, bool create) {
  StreamTrack* victim = &g_track[0];
  for (auto& t : g_track) {
    if (t.used && t.stream == stream) return &t;
    if (!t.used ? victim->used : (victim->used && t.stamp < victim->stamp)) victim = &t;
  }
  if (!create) return nullptr;
  *victim = StreamTrack();
  victim->stream = stream;
  victim->used = true;
  return victim;
}


struct TcKey {
  int dtype, a_mn, b_mn, no_split, n_extra, may_split;
  int64_t batch, M, N, K, lda, ldb, ldc, sA, sB, sC, plan_M, plan_N;
  const void *A, *B, *C, *bias, *scratch, *status;
  const void *aux, *pre;
  int fused, act, grad, unused;
  const void* extra[kMaxOut - 1];
};

TcKey make_key(const GemmProblem& p, const void* scratch, const void* status, void* const* extra_out, int n_extra) {
  TcKey k;
  memset(&k, 0, sizeof k);
  k.dtype = (int)p.dtype; k.a_mn = p.a_mn_major; k.b_mn = p.b_mn_major; k.no_split = p.no_split ? 1 : 0;
  k.n_extra = n_extra; k.may_split = n_extra == 0;
  k.batch = p.batch; k.M = p.M; k.N = p.N; k.K = p.K; k.lda = p.lda; k.ldb = p.ldb; k.ldc = p.ldc;
  k.sA = p.strideA; k.sB = p.strideB; k.sC = p.strideC; k.plan_M = p.plan_M; k.plan_N = p.plan_N;
  k.A = p.A; k.B = p.B; k.C = p.C; k.bias = p.bias; k.scratch = scratch; k.status = status;
  if (p.fused) {
    k.fused = 1; k.bias = p.fe.bias; k.act = p.fe.act; k.grad = p.fe.grad; k.aux = p.fe.aux; k.pre = p.fe.pre;
  }
  for (int i = 0; i < n_extra && i < kMaxOut - 1; i++) k.extra[i] = extra_out[i];
  return k;
}

}  // namespace

struct TcCache {
  static constexpr int kEntries = 32;
  struct Entry {
    bool used = false;
    uint64_t stamp = 0;
    TcKey key;
    TcPrepared prep;
  };
  Entry e[kEntries];
  uint64_t clock = 0;
};

TcCache* tc_cache_create() { return new (std::nothrow) TcCache(); }
void tc_cache_destroy(TcCache* c) { delete c; }
void tc_cache_clear(TcCache* c) {
  if (c) for (auto& x : c->e) x.used = false;
}

namespace {

// Everything about a product that does not depend on the stream: pre-pass jobs, tensor maps,
// kernel parameters, which kernel.  `*scratch_needed` receives the work-area bytes the product
// needs; when the area given is smaller, nothing else is filled in and cudaErrorInvalidValue
// comes back, so that the caller can grow the area and ask again.
cudaError_t prepare_tc(const GemmProblem& p, unsigned int* status_word, void* scratch, size_t scratch_bytes,
                       int sm_count, void* const* extra_out, int n_extra, TcPrepared* out, size_t* scratch_needed) {
  TcPrepared& pp = *out;
  const bool f32 = p.dtype == HC_F32;
  const int eb = f32 ? 4 : 2;
  const int BK = 128 / eb;
  const Tunables tun = read_tunables();
  const TcPlan plan = plan_tc(p, sm_count, n_extra == 0, tun);
  const size_t ops_bytes = operand_scratch_bytes(p);
  const size_t need = plan.ws_bytes ? ((ops_bytes + 255) & ~(size_t)255) + plan.ws_bytes : ops_bytes;
  if (scratch_needed) *scratch_needed = need;
  if (need > 0 && (!scratch || scratch_bytes < need)) return cudaErrorInvalidValue;
  pp.scratch_used = need;

  const void *a_hi = p.A, *a_lo = p.A, *b_hi = p.B, *b_lo = p.B;
  int64_t lda = p.lda, ldb = p.ldb, sa = p.strideA, sb = p.strideB;
  int64_t lda_lo = 0, ldb_lo = 0, sa_lo = 0, sb_lo = 0;   // float32: layout of the lo arrays
  pp.pre = 0;
  if (!f32) {
    const RepackLayout r = repack_layout(p);
    if (r.a || r.b) {
      __half* ra = (__half*)scratch;
      __half* rb = (__half*)((char*)scratch + r.a_bytes);
      pp.rja = RepackJob{(const __half*)p.A, ra, r.a_rows, r.a_width, p.lda, r.a_ld, p.strideA, r.a_mat, r.a ? p.batch : 0};
      pp.rjb = RepackJob{(const __half*)p.B, rb, r.b_rows, r.b_width, p.ldb, r.b_ld, p.strideB, r.b_mat, r.b ? p.batch : 0};
      auto blocks = [&](const RepackJob& j) {
        const int64_t work = j.batch * j.rows * j.width;
        int64_t b = (work + 255) / 256;
        return (int)(b > 148 * 8 ? 148 * 8 : b);   // zero blocks for an operand that stays in place
      };
      pp.pre_blocks_a = blocks(pp.rja); pp.pre_blocks_b = blocks(pp.rjb);
      pp.pre = 1;
      if (r.a) { a_hi = a_lo = ra; lda = r.a_ld; sa = r.a_mat; }
      if (r.b) { b_hi = b_lo = rb; ldb = r.b_ld; sb = r.b_mat; }
    }
  } else {
    const SplitLayout s = split_layout(p);
    // Work area: [A lo][A copy, if needed][B lo][B copy, if needed]
    char* at = (char*)scratch;
    float* al = (float*)at; at += s.a_bytes;
    float* ah = nullptr;
    if (s.a_copy) { ah = (float*)at; at += s.a_bytes; }
    float* bl = (float*)at; at += s.b_bytes;
    float* bh = nullptr;
    if (s.b_copy) { bh = (float*)at; at += s.b_bytes; }
    auto vec_ok4 = [](const void* src, int64_t width, int64_t ld, int64_t stride, int64_t batch) {
      return (int)(width % 4 == 0 && ld % 4 == 0 && ((uintptr_t)src & 15) == 0 && (batch == 1 || stride % 4 == 0));
    };
    pp.sja = SplitJob{(const float*)p.A, ah, al, s.a_rows, s.a_width, p.lda, s.a_ld, p.strideA, s.a_mat, p.batch,
                      vec_ok4(p.A, s.a_width, p.lda, p.strideA, p.batch)};
    pp.sjb = SplitJob{(const float*)p.B, bh, bl, s.b_rows, s.b_width, p.ldb, s.b_ld, p.strideB, s.b_mat, p.batch,
                      vec_ok4(p.B, s.b_width, p.ldb, p.strideB, p.batch)};
    auto blocks = [&](const SplitJob& j) {
      const int64_t work = j.batch * j.rows * (j.vec4 ? j.width / 4 : j.width);
      int64_t b = (work + 255) / 256;
      return (int)(b > 148 * 8 ? 148 * 8 : (b < 1 ? 1 : b));
    };
    pp.pre_blocks_a = blocks(pp.sja); pp.pre_blocks_b = blocks(pp.sjb);
    pp.pre = 2;
    a_lo = al; b_lo = bl;
    lda_lo = s.a_ld; ldb_lo = s.b_ld; sa_lo = s.a_mat; sb_lo = s.b_mat;
    if (s.a_copy) { a_hi = ah; lda = s.a_ld; sa = s.a_mat; }
    if (s.b_copy) { b_hi = bh; ldb = s.b_ld; sb = s.b_mat; }
  }

  const int dbg = debug_flags();
  const int kslabs = (int)((p.K + BK - 1) / BK);
  const int shape = plan.shape;
  const int bn = (shape == SHAPE_C1_128 || shape == SHAPE_PAIR_128) ? 128 : shape == SHAPE_PAIR_64 ? 64 : 256;
  const int cta = (shape == SHAPE_C1_256 || shape == SHAPE_C1_128) ? 1 : 2;
  const int b_box = bn / cta;
  // A fused product of few rows copies those rows only: 128-row boxes of rows that are mostly not there cost the copies of the
  // others their time (16384 x 4096 float16 weights, 4 rows: 46 us, 26 with 8-row boxes).
  int a_box = BM;
  if (p.fused && !p.a_mn_major && cta == 1 && p.M <= 64) a_box = p.M <= 8 ? 8 : p.M <= 16 ? 16 : p.M <= 32 ? 32 : 64;
  memset(pp.maps, 0, sizeof pp.maps);
  memset(&pp.outs, 0, sizeof pp.outs);
  if (!make_operand_map(&pp.maps[0], a_hi, eb, p.a_mn_major, p.M, p.K, lda, sa, p.batch, a_box) ||
      !make_operand_map(&pp.maps[2], b_hi, eb, p.b_mn_major, p.N, p.K, ldb, sb, p.batch, b_box))
    return cudaErrorNotSupported;
  if (f32) {
    if (!make_operand_map(&pp.maps[1], a_lo, eb, p.a_mn_major, p.M, p.K, lda_lo, sa_lo, p.batch, a_box) ||
        !make_operand_map(&pp.maps[3], b_lo, eb, p.b_mn_major, p.N, p.K, ldb_lo, sb_lo, p.batch, b_box))
      return cudaErrorNotSupported;
  } else {
    pp.maps[1] = pp.maps[0];   // float16 has no lo parts; the kernel never reads these two
    pp.maps[3] = pp.maps[2];
  }

  TcParams& tp = pp.tp;
  tp.M = p.M; tp.N = p.N;
  // Short contractions are bound by draining results, not by the MMA: they get more epilogue
  // warps (eight up to 8 slabs, sixteen up to 2: each warp's drain is a serial chain of tensor-
  // memory load, conversion, proxy fence and TMA store, and more chains in flight hide more of
  // it - measured +8 % at K = 128, nothing at K = 256, -3 % at K = 512) and fewer operand stages.
  const bool short_k = kslabs <= tun.short_k;
  // Pipeline slots of the small float16 shapes hold two k slabs; the fused 128x128 tile, whose staging ring leaves room for
  // only two such slots, has five of one.
  const int slabs = (p.fused && plan.splits == 1 && !f32 && shape == SHAPE_C1_128) ? 1 : plan.slabs;
  tp.num_k_blocks = (kslabs + slabs - 1) / slabs;
  const bool cut = plan.splits > 1;
  tp.splits = plan.splits;
  tp.kb_per_split = cut ? plan.kb_per_split : tp.num_k_blocks;
  // float32: a window bounds the number of truncating tensor-core accumulations that feed one
  // correctly rounded float32 add in the epilogue.
  const bool windowed = f32 && !(dbg & 2);
  tp.chunk_kb = windowed ? window_slabs() : tp.num_k_blocks;
  if (tp.chunk_kb > tp.num_k_blocks) tp.chunk_kb = tp.num_k_blocks;
  const bool wide = shape == SHAPE_WIDE;
  const int tile_n = wide ? 2 * bn : bn;
  tp.tile_rows = BM * cta;
  tp.tiles_m = (int)((p.M + tp.tile_rows - 1) / tp.tile_rows);
  tp.tiles_n = (int)((p.N + tile_n - 1) / tile_n);
  tp.total_tiles = (int64_t)tp.tiles_m * tp.tiles_n * p.batch * plan.splits;
  // Tile rows that share a sweep over the columns.  A wave of CTA pairs then touches g tile rows
  // of A and (pairs / g) tile columns of B; the bytes are least near g = sqrt(pairs x tile_n / tile_m):
  // 8 for 256x256 pairs, 12-16 for 256x512 (measured at 16384^3: 6.51 ms with 8, 6.35 with 16).
  tp.group_m = tun.group_m > 0 ? tun.group_m : wide ? 16 : 16 / cta;
  tp.a_mn_major = p.a_mn_major; tp.b_mn_major = p.b_mn_major;
  tp.status = status_word;
  tp.skip_input_wait = 0;
  // Where the tiles go: the result itself, or - for a cut contraction - float32 partial matrices
  // in the work area (part z of matrix m at index m * parts + z), which a second kernel sums.
  void* out_base = p.C;
  int out_bytes = eb;
  int64_t out_ld = p.ldc, out_stride = p.strideC, out_mats = p.batch;
  tp.bias = p.bias;
  tp.a_box_rows = a_box;
  tp.fe = p.fe;
  // 16-byte accesses to the tensors laid out like the result
  tp.fe.vec = ((((uintptr_t)p.fe.aux | (uintptr_t)p.fe.pre) & 15) == 0 && (p.ldc * eb) % 16 == 0) ? 1 : 0;
  if (p.fused && !cut && tp.fe.vec) {
    // maps 1 and 2 of the results' array: the kept pre-activation and the auxiliary tensor
    if (p.fe.pre && !make_output_map(&pp.outs.m[1], p.fe.pre, eb, p.N, p.M, p.ldc, p.strideC, p.batch)) return cudaErrorNotSupported;
    if (p.fe.aux && !make_output_map(&pp.outs.m[2], const_cast<void*>(p.fe.aux), eb, p.N, p.M, p.ldc, p.strideC, p.batch)) return cudaErrorNotSupported;
  }
  if (cut) {
    const size_t off = (ops_bytes + 255) & ~(size_t)255;
    out_base = (char*)scratch + off;
    out_bytes = 4;
    out_ld = plan.ws_ld; out_stride = p.M * plan.ws_ld; out_mats = p.batch * plan.splits;
    tp.bias = nullptr;
  }
  tp.C = out_base; tp.ldc = out_ld; tp.strideC = out_stride;
  tp.vec_ok = (((uintptr_t)out_base & 15) == 0 && (out_ld * out_bytes) % 16 == 0 && (out_stride * out_bytes) % 16 == 0) ? 1 : 0;
  // Results leave through TMA stores when the result can be described to TMA (16-byte aligned
  // base and pitches); otherwise from registers.
  tp.tma_store = 0;
  tp.n_out = 1;
  if (tp.vec_ok && !(dbg & 128) && p.M < (1ll << 31) && p.N < (1ll << 31) && out_ld * out_bytes < (1ll << 40) &&
      make_output_map(&pp.outs.m[0], out_base, out_bytes, p.N, p.M, out_ld, out_stride, out_mats))
    tp.tma_store = 1;
  if (n_extra > 0) {
    // Extra destinations only exist on the TMA-store path.
    if (!tp.tma_store || cut) return cudaErrorNotSupported;
    for (int i = 0; i < n_extra; i++) {
      if (((uintptr_t)extra_out[i] & 15) != 0 ||
          !make_output_map(&pp.outs.m[1 + i], extra_out[i], eb, p.N, p.M, p.ldc, p.strideC, p.batch))
        return cudaErrorNotSupported;
    }
    tp.n_out = 1 + n_extra;
  }

  {
    auto span = [&](const void* base, int64_t rows_, int64_t ld, int64_t stride, int64_t batch, int idx) {
      const int64_t per = rows_ * ld;
      const int64_t elems = (batch - 1) * (stride > per ? stride : per) + per;
      pp.in_lo[idx] = (uintptr_t)base;
      pp.in_hi[idx] = (uintptr_t)base + (uintptr_t)(elems * eb);
    };
    span(p.A, p.a_mn_major ? p.K : p.M, p.lda, p.strideA, p.batch, 0);
    span(p.B, p.b_mn_major ? p.K : p.N, p.ldb, p.strideB, p.batch, 1);
    pp.in_lo[2] = (uintptr_t)p.bias;
    pp.in_hi[2] = p.bias ? (uintptr_t)p.bias + (uintptr_t)(p.N * eb) : 0;
    const int64_t per_c = p.M * p.ldc;
    pp.out_lo = (uintptr_t)p.C;
    pp.out_hi = (uintptr_t)p.C + (uintptr_t)(((p.batch - 1) * (p.strideC > per_c ? p.strideC : per_c) + per_c) * eb);
    // (a kept pre-activation is a second range it writes)
    pp.trackable = (pp.pre == 0 && !cut && !p.fe.pre);
  }

  TcLaunchFn fn = nullptr;
  if (p.fused && !cut) {
    if (f32 && !windowed) return cudaErrorInvalidValue;   // the fused epilogue is not built for the no-window debug mode
    fn = fused_kernel(f32, shape, kslabs, p.fe);
    if (!fn) return cudaErrorInvalidValue;
  } else if (!f32 && cut) {
    if (shape == SHAPE_PAIR_128) fn = TcConfig<2, 128, 4, 4, false, 2, 1, 2, true>::launch;
    else if (shape == SHAPE_PAIR_64) fn = TcConfig<2, 64, 4, 4, false, 2, 1, 2, true>::launch;
    else if (shape == SHAPE_PAIR) fn = TcConfig<2, 256, 6, 4, false, 2, 1, 1, true>::launch;
    else if (shape == SHAPE_C1_128) fn = TcConfig<2, 128, 3, 4, false, 1, 1, 2, true>::launch;
    else return cudaErrorInvalidValue;
  } else if (!f32) {
    if (wide && tun.wide_epi8) fn = TcConfig<2, 256, 4, 8, false, 2, 2>::launch;
    else if (wide) fn = TcConfig<2, 256, 4, 4, false, 2, 2>::launch;
    else if (shape == SHAPE_PAIR_128) fn = TcConfig<2, 128, 4, 4, false, 2, 1, 2>::launch;
    else if (shape == SHAPE_PAIR_64) fn = TcConfig<2, 64, 4, 4, false, 2, 1, 2>::launch;
    else if (cta == 2 && short_k && kslabs <= 2) fn = TcConfig<2, 256, 4, 16, false, 2>::launch;
    else if (cta == 2 && short_k) fn = TcConfig<2, 256, 4, 8, false, 2>::launch;
    else if (cta == 2) fn = TcConfig<2, 256, 6, 4, false, 2>::launch;
    else if (bn == 256) fn = TcConfig<2, 256, 4, 4, false, 1>::launch;
    else fn = TcConfig<2, 128, 3, 4, false, 1, 1, 2>::launch;
  } else if (windowed) {
    if (shape == SHAPE_PAIR_128) fn = TcConfig<4, 128, 3, 4, true, 2>::launch;
    else if (shape == SHAPE_PAIR_64) fn = TcConfig<4, 64, 4, 4, true, 2>::launch;
    else if (cta == 2) fn = TcConfig<4, 256, 3, 8, true, 2>::launch;
    else if (bn == 256) fn = TcConfig<4, 256, 2, 8, true, 1>::launch;
    else fn = TcConfig<4, 128, 3, 4, true, 1>::launch;
  } else {
#ifdef HC_DIAGNOSTICS
    if (cta == 2) fn = TcConfig<4, 256, 3, 4, false, 2>::launch;
    else if (bn == 256) fn = TcConfig<4, 256, 2, 4, false, 1>::launch;
    else fn = TcConfig<4, 128, 3, 4, false, 1>::launch;
#else
    return cudaErrorInvalidValue;   // float32 always runs windowed in the shipped library
#endif
  }
  pp.fn = fn;
  pp.cut = cut;
  if (cut) {
    // Sum the parts in ascending order, add the bias, round once, store the result.
    ReduceJob& job = pp.job;
    job.ws = (const float*)out_base; job.C = p.C; job.bias = p.bias;
    job.M = p.M; job.N = p.N; job.ws_ld = plan.ws_ld; job.batch = p.batch; job.parts = plan.splits;
    job.ldc = p.ldc; job.strideC = p.strideC;
    job.fe = p.fe;
    const int out_align = f32 ? 15 : 7;   // four results per thread: 16 bytes of float32, 8 of float16
    job.vec_ok = (((uintptr_t)p.C & out_align) == 0 && p.ldc % 4 == 0 && p.strideC % 4 == 0) ? 1 : 0;
    const int64_t work = p.batch * p.M * (plan.ws_ld / 4);
    int64_t blocks = (work + 255) / 256;
    if (blocks > 148 * 8) blocks = 148 * 8;
    pp.reduce_blocks = (int)blocks;
    pp.reduce_half = !f32;
    pp.reduce_fused = p.fused;
  }
  return cudaSuccess;
}

cudaError_t issue_tc(const TcPrepared& pp, int sm_count, cudaStream_t stream, LaunchRecord* rec, bool private_stream) {
  if (rec) { *rec = LaunchRecord(); rec->kernel = HC_KERNEL_TENSOR; rec->scratch_bytes = pp.scratch_used; }
  if (pp.pre == 1) {
    int blocks_a = pp.pre_blocks_a;
    void* args[3] = {(void*)&pp.rja, (void*)&pp.rjb, (void*)&blocks_a};
    cudaError_t e = launch_elementwise((const void*)repack_f16_kernel, args, pp.pre_blocks_a + pp.pre_blocks_b, stream);
    if (e != cudaSuccess) return e;
    if (rec) rec->launches += 1;
  } else if (pp.pre == 2) {
    int blocks_a = pp.pre_blocks_a;
    void* args[3] = {(void*)&pp.sja, (void*)&pp.sjb, (void*)&blocks_a};
    cudaError_t e = launch_elementwise((const void*)split_tf32_kernel, args, pp.pre_blocks_a + pp.pre_blocks_b, stream);
    if (e != cudaSuccess) return e;
    if (rec) rec->launches += 1;
  }
  if (rec) rec->tiles = pp.tp.total_tiles;
  // May the operand loads run ahead of the wait for the previous kernel?  Only on a stream no one
  // else launches kernels on, only against a predecessor whose written range is known, and only
  // when that range and this product's operands are disjoint.  (Anything else enqueued on the
  // stream in between - copies, ordinary kernels, event waits - completes before this kernel
  // starts at all.)
  bool skip = false;
  if (private_stream && overlap_launches()) {
    cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
    unsigned long long capture = 0;
    const bool told = cudaStreamGetCaptureInfo(stream, &status, &capture) == cudaSuccess;
    if (!told) cudaGetLastError();
    if (status == cudaStreamCaptureStatusNone) capture = 0;
    std::lock_guard<std::mutex> lock(g_track_mu);
    StreamTrack* t = track_entry(stream, true);
    if (t->known && told && t->capture == capture && pp.trackable) {
      skip = true;
      for (int i = 0; i < 3; i++)
        if (pp.in_hi[i] > pp.in_lo[i] && pp.in_lo[i] < t->hi && t->lo < pp.in_hi[i]) skip = false;
    }
    t->known = pp.trackable && told;
    t->capture = capture;
    t->lo = pp.out_lo;
    t->hi = pp.out_hi;
    t->stamp = ++g_track_clock;
  }
  // cudaLaunchKernelEx reports this launch's own failure; the thread's sticky-less "last error"
  // may hold another library's earlier error and is not this launch's to report.
  cudaError_t ge;
  if (skip) {
    TcParams tp = pp.tp;
    tp.skip_input_wait = 1;
    ge = pp.fn(pp.maps, pp.outs, tp, sm_count, stream, rec);
  } else {
    ge = pp.fn(pp.maps, pp.outs, pp.tp, sm_count, stream, rec);
  }
  if (ge != cudaSuccess || !pp.cut) return ge;
  void* args[1] = {(void*)&pp.job};
  const void* sum = pp.reduce_fused ? (pp.reduce_half ? (const void*)splitk_reduce_kernel<true, true>
                                                      : (const void*)splitk_reduce_kernel<false, true>)
                                    : (pp.reduce_half ? (const void*)splitk_reduce_kernel<true>
                                                      : (const void*)splitk_reduce_kernel<false>);
  cudaError_t re = launch_elementwise(sum, args, pp.reduce_blocks, stream);
  if (re != cudaSuccess) return re;
  if (rec) rec->launches += 1;
  return cudaSuccess;
}

}  // namespace

void tc_forget_predecessor(cudaStream_t stream) {
  std::lock_guard<std::mutex> lock(g_track_mu);
  StreamTrack* t = track_entry(stream, false);
  if (t) t->known = false;
}

cudaError_t launch_tc(const GemmProblem& p, cudaStream_t stream, unsigned int* status_word, void* scratch,
                      size_t scratch_bytes, int sm_count, LaunchRecord* rec, void* const* extra_out, int n_extra,
                      TcCache* cache, size_t* scratch_needed, bool private_stream) {
  if (scratch_needed) *scratch_needed = 0;
  if (!tc_supported(p)) return cudaErrorNotSupported;
  if (n_extra < 0 || n_extra > kMaxOut - 1 || (n_extra > 0 && !extra_out)) return cudaErrorInvalidValue;
  if (cache && kPlanCacheEnabled) {
    const TcKey key = make_key(p, scratch, status_word, extra_out, n_extra);
    TcCache::Entry* victim = &cache->e[0];
    for (auto& x : cache->e) {
      if (x.used && memcmp(&x.key, &key, sizeof key) == 0) {
        x.stamp = ++cache->clock;
        return issue_tc(x.prep, sm_count, stream, rec, private_stream);
      }
      if (!x.used ? victim->used : (victim->used && x.stamp < victim->stamp)) victim = &x;
    }
    victim->used = false;
    cudaError_t e = prepare_tc(p, status_word, scratch, scratch_bytes, sm_count, extra_out, n_extra, &victim->prep,
                               scratch_needed);
    if (e != cudaSuccess) return e;
    victim->key = key;
    victim->stamp = ++cache->clock;
    victim->used = true;
    return issue_tc(victim->prep, sm_count, stream, rec, private_stream);
  }
  TcPrepared prep;
  cudaError_t e = prepare_tc(p, status_word, scratch, scratch_bytes, sm_count, extra_out, n_extra, &prep, scratch_needed);
  if (e != cudaSuccess) return e;
  return issue_tc(prep, sm_count, stream, rec, private_stream);
}

}  // namespace hc

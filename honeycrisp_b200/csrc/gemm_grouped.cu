// Products grouped by expert: ragged groups of rows, one weight matrix a group, all in one launch of the
// tensor-core kernel (tc_kernel.cuh, kGrouped).
//
//   forward          out[r] = a[r] op(b[g])        for offsets[g] <= r < offsets[g + 1]
//   weight gradient  out[g] = sum over those r of a[r]^T b[r]
//
// The offsets stay on the device: group_setup_kernel turns them into a table of tiles, which the persistent CTAs of
// the product walk, so the host neither waits for the router nor launches once a group, and a captured graph
// follows new offsets.  Groups of few rows take CUDA-core forms where those read or write less (gemm_skinny.cu).  Offsets that leave [0, total_rows] or run backwards are clamped there, so that no table can
// send a copy out of range.
#include "tc_kernel.cuh"

namespace hc {
namespace {

// One CTA.  start/end of every group, clamped and ascending, and the tiles in front of it (forward: tiles_n for
// every tile_rows rows; weight gradient: tiles_per_group each).
__global__ void __launch_bounds__(1024) group_setup_kernel(const int64_t* offsets, int groups, int64_t total_rows, int tile_rows,
                                                           int tiles_n, int tiles_per_group, int* start, int* end, int* first_tile) {
  __shared__ int warp_max[32], warp_sum[32];
  pdl_wait();
  pdl_release();   // the kernel behind sets itself up meanwhile, and waits for this one before it reads the table
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  int reached = 0, tiles = 0;   // over the groups of earlier rounds: largest end, number of tiles
  for (int g0 = 0; g0 < groups; g0 += 1024) {
    const int g = g0 + (int)threadIdx.x;
    const bool live = g < groups;
    auto clamped = [&](int64_t v) { return (int)(v < 0 ? 0 : v > total_rows ? total_rows : v); };
    const int s_raw = live ? clamped(offsets[g]) : 0, e_raw = live ? clamped(offsets[g + 1]) : 0;
    // running maximum of the ends of all groups up to this one
    int top = max(s_raw, e_raw);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, top, o);
      if (lane >= o) top = max(top, v);
    }
    if (lane == 31) warp_max[warp] = top;
    __syncthreads();
    int below = reached;
    for (int w = 0; w < warp; w++) below = max(below, warp_max[w]);
    const int prev = __shfl_up_sync(0xffffffffu, top, 1);
    const int before = lane == 0 ? below : max(below, prev);
    const int s = max(s_raw, before), e = max(e_raw, s);
    int n_tiles = 0;
    if (live) {
      start[g] = s;
      end[g] = e;
      n_tiles = tiles_per_group > 0 ? tiles_per_group : (e - s + tile_rows - 1) / tile_rows * tiles_n;
    }
    int sum = n_tiles;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += v;
    }
    if (lane == 31) warp_sum[warp] = sum;
    __syncthreads();
    int ahead = tiles;
    for (int w = 0; w < warp; w++) ahead += warp_sum[w];
    if (live) first_tile[g] = ahead + sum - n_tiles;
    for (int w = 0; w < 32; w++) { tiles += warp_sum[w]; reached = max(reached, warp_max[w]); }
    __syncthreads();
  }
  if (threadIdx.x == 0) first_tile[groups] = tiles;
}

// The weight gradient's last slab of every group: the rows behind the whole slabs, followed by zeros up to kSlab rows, so
// that the tensor core sums nothing of the neighbour's.  float32 operands as their two halves.
struct TailJob {
  const void* src;
  void *hi, *lo;
  int64_t width, ld_src, ld_dst;
};
template <typename T, int kSlab>
__global__ void __launch_bounds__(256) group_tail_kernel(const TailJob ja, const TailJob jb, const int* start, const int* end) {
  pdl_wait();
  pdl_release();
  const TailJob& j = blockIdx.z == 0 ? ja : jb;
  const int g = blockIdx.x;
  const int s = start[g], n = end[g] - s, rem = n % kSlab;
  if (rem == 0) return;
  const int64_t first = (int64_t)s + n - rem;
  for (int64_t c = (int64_t)blockIdx.y * 256 + threadIdx.x; c < j.width; c += (int64_t)gridDim.y * 256) {
#pragma unroll 8
    for (int r = 0; r < kSlab; r++) {
      const T v = r < rem ? ((const T*)j.src)[(first + r) * j.ld_src + c] : (T)0.0f;
      const int64_t at = ((int64_t)g * kSlab + r) * j.ld_dst + c;
      ((T*)j.hi)[at] = v;
      if constexpr (sizeof(T) == 4) ((float*)j.lo)[at] = split_lo(v);
    }
  }
}

// Rows of the groups set to zero: the product over an empty contraction.
template <typename T>
__global__ void __launch_bounds__(256) group_zero_kernel(const int* start, const int* end, T* out, int64_t cols) {
  pdl_wait();
  const int g = blockIdx.x;
  const int64_t n = (int64_t)(end[g] - start[g]) * cols;
  for (int64_t i = (int64_t)blockIdx.y * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.y * 256)
    out[(int64_t)start[g] * cols + i] = (T)0.0f;
}

size_t round256(size_t n) { return (n + 255) & ~(size_t)255; }

// Where an operand lies for TMA: in place, or in a copy whose rows are 16-byte multiples; float32 operands have their lo half
// beside it.  `mats` matrices of `rows` x `width`.
struct Operand {
  const void* src;
  int64_t mats, rows, width;
  bool copy;
  int64_t ld;                       // of the copy and of the lo half
  size_t copy_bytes, lo_bytes;
  const void* hi = nullptr;
  void* lo = nullptr;
  int64_t hi_ld = 0, hi_stride = 0;
};
Operand describe(const void* src, int64_t mats, int64_t rows, int64_t width, int eb) {
  Operand o;
  o.src = src; o.mats = mats; o.rows = rows; o.width = width;
  o.copy = !operand_ok(src, eb, width, rows * width, mats, rows, width);
  const int64_t unit = 16 / eb;
  o.ld = (width + unit - 1) / unit * unit;
  const size_t bytes = round256((size_t)(mats * rows * o.ld) * eb);
  o.copy_bytes = o.copy ? bytes : 0;
  o.lo_bytes = eb == 4 ? bytes : 0;
  return o;
}
void place(Operand* o, char** at) {
  o->hi = o->src; o->hi_ld = o->width; o->hi_stride = o->rows * o->width;
  if (o->copy) { o->hi = *at; o->hi_ld = o->ld; o->hi_stride = o->rows * o->ld; *at += o->copy_bytes; }
  if (o->lo_bytes) { o->lo = *at; *at += o->lo_bytes; }
}
int blocks_for(int64_t work) {
  const int64_t b = (work + 255) / 256;
  return (int)(b > 148 * 8 ? 148 * 8 : b < 1 ? 1 : b);
}

// Copies and lo halves of both operands, one launch; none where both lie ready.
cudaError_t launch_operands(const Operand& a, const Operand& b, int eb, cudaStream_t stream, LaunchRecord* rec) {
  if (eb == 2) {
    if (!a.copy && !b.copy) return cudaSuccess;
    auto job = [](const Operand& o) {
      return RepackJob{(const __half*)o.src, (__half*)o.hi, o.rows, o.width, o.width, o.ld, o.rows * o.width, o.rows * o.ld, o.copy ? o.mats : 0};
    };
    RepackJob ja = job(a), jb = job(b);
    int blocks_a = a.copy ? blocks_for(a.mats * a.rows * a.width) : 0;
    const int blocks_b = b.copy ? blocks_for(b.mats * b.rows * b.width) : 0;
    void* args[] = {(void*)&ja, (void*)&jb, (void*)&blocks_a};
    rec->launches++;
    return launch_elementwise((const void*)repack_f16_kernel, args, blocks_a + blocks_b, stream);
  }
  auto job = [](const Operand& o) {
    const bool vec = o.width % 4 == 0 && ((uintptr_t)o.src & 15) == 0;
    return SplitJob{(const float*)o.src, o.copy ? (float*)o.hi : nullptr, (float*)o.lo, o.rows, o.width, o.width, o.ld, o.rows * o.width,
                    o.rows * o.ld, o.mats, vec ? 1 : 0};
  };
  SplitJob ja = job(a), jb = job(b);
  int blocks_a = blocks_for(a.mats * a.rows * (ja.vec4 ? a.width / 4 : a.width));
  const int blocks_b = blocks_for(b.mats * b.rows * (jb.vec4 ? b.width / 4 : b.width));
  void* args[] = {(void*)&ja, (void*)&jb, (void*)&blocks_a};
  rec->launches++;
  return launch_elementwise((const void*)split_tf32_kernel, args, blocks_a + blocks_b, stream);
}

// Tile shape by the planner's measured clocks for 64 (float32: 32) of the contraction, for groups of equal size: the
// offsets are not known here.
int choose_shape(const GroupedProblem& p, int sm_count, int64_t m, int64_t n, int64_t k_slabs) {
  const bool f32 = p.dtype == HC_F32;
  struct Cand { int shape, rows, cols, slots; double clk; };
  const Cand cands[] = {{SHAPE_PAIR, 256, 256, sm_count / 2, f32 ? 1700.0 : 600.0},
                        {SHAPE_PAIR_128, 256, 128, sm_count / 2, 340.0},
                        {SHAPE_C1_128, 128, 128, sm_count, f32 ? 1130.0 : 410.0}};
  int best = SHAPE_C1_128;
  double best_cost = -1.0;
  for (const Cand& c : cands) {
    if (f32 && c.shape == SHAPE_PAIR_128) continue;
    const int64_t tiles = p.groups * ((m + c.rows - 1) / c.rows) * ((n + c.cols - 1) / c.cols);
    const int64_t waves = (tiles + c.slots - 1) / c.slots;
    const double cost = (double)waves * ((double)k_slabs * c.clk + 300.0);
    if (best_cost < 0 || cost < best_cost) { best_cost = cost; best = c.shape; }
  }
  return best;
}

// Short contractions are bound by draining results: more epilogue warps, as for the plain products (weight gradients of 64
// groups of 64 rows, 512 x 2048: 47 us with four warps, 37 with sixteen).
TcLaunchFn grouped_kernel(bool f32, int shape, int64_t k_slabs) {
  if (f32)
    return shape == SHAPE_PAIR ? TcConfig<4, 256, 3, 8, true, 2, 1, 1, false, kGrouped>::launch
                               : TcConfig<4, 128, 3, 4, true, 1, 1, 1, false, kGrouped>::launch;
  switch (shape) {
    case SHAPE_PAIR:
      if (k_slabs <= 2) return TcConfig<2, 256, 4, 16, false, 2, 1, 1, false, kGrouped>::launch;
      if (k_slabs <= 8) return TcConfig<2, 256, 4, 8, false, 2, 1, 1, false, kGrouped>::launch;
      return TcConfig<2, 256, 6, 4, false, 2, 1, 1, false, kGrouped>::launch;
    case SHAPE_PAIR_128: return TcConfig<2, 128, 8, 4, false, 2, 1, 1, false, kGrouped>::launch;
    default: return TcConfig<2, 128, 6, 4, false, 1, 1, 1, false, kGrouped>::launch;
  }
}

}  // namespace

cudaError_t launch_grouped(const GroupedProblem& p, cudaStream_t stream, unsigned int* status_word, void* scratch,
                           size_t scratch_bytes, int sm_count, LaunchRecord* rec, size_t* scratch_needed) {
  const bool f32 = p.dtype == HC_F32, wg = p.weight_grad;
  const int eb = f32 ? 4 : 2, BK = 128 / eb;
  *rec = LaunchRecord();
  rec->kernel = HC_KERNEL_TENSOR;
  auto setup = [&](int* start, int tile_rows, int tiles_n, int64_t per_group) {
    const int64_t* offsets = p.offsets;
    int groups = (int)p.groups, per = (int)per_group;
    int64_t total = p.total_rows;
    int *end = start + groups, *first_tile = end + groups;
    void* args[] = {(void*)&offsets, (void*)&groups, (void*)&total, (void*)&tile_rows, (void*)&tiles_n, (void*)&per, (void*)&start, (void*)&end, (void*)&first_tile};
    rec->launches++;
    return launch_behind((const void*)group_setup_kernel, args, dim3(1), dim3(1024), 0, stream);
  };
  if (few_preferred(p)) {
    const size_t need = round256((size_t)(3 * p.groups + 1) * sizeof(int));
    *scratch_needed = need;
    if (!scratch || scratch_bytes < need) return cudaErrorInvalidValue;
    const int strips = few_strips(p);
    const int64_t tiles = (p.total_rows / 8 + p.groups) * strips;   // forward: at most
    if (tiles >= (1ll << 31) || p.total_rows >= (1ll << 31) - 256) return cudaErrorNotSupported;
    int* start = (int*)scratch;
    cudaError_t e = setup(start, 8, strips, wg ? 1 : 0);
    if (e != cudaSuccess) return e;
    const GroupTiles t = {start, start + p.groups, start + 2 * p.groups, (int)p.groups};
    rec->kernel = HC_KERNEL_SIMT;
    rec->tile_m = 8; rec->tiles = tiles; rec->scratch_bytes = need;
    rec->launches++;
    return launch_few(p, t, tiles, stream);
  }
  // Result rows and columns of a group, and the contracted length: the group's rows for the weight gradient.
  const int64_t m = wg ? p.rows : p.total_rows, n = p.cols;
  // Tile coordinates are 32-bit, and a tile may start within the last one of them.
  constexpr int64_t kMost = (1ll << 31) - 256;
  if (m >= kMost || n >= kMost || p.inner >= kMost) return cudaErrorNotSupported;
  const int64_t mean_rows = (p.total_rows + p.groups - 1) / p.groups;
  Operand a = wg ? describe(p.a, 1, p.total_rows, p.rows, eb) : describe(p.a, 1, p.total_rows, p.inner, eb);
  Operand b = wg ? describe(p.b, 1, p.total_rows, p.cols, eb)
                 : p.trans_b ? describe(p.b, p.groups, p.cols, p.inner, eb) : describe(p.b, p.groups, p.inner, p.cols, eb);
  // Work area: the group table, copies and lo halves, the padded last slabs.
  const size_t table = round256((size_t)(3 * p.groups + 1) * sizeof(int));
  const int64_t tail_rows = p.groups * BK;
  const size_t tail_a = wg ? round256((size_t)(tail_rows * a.ld) * eb) : 0, tail_b = wg ? round256((size_t)(tail_rows * b.ld) * eb) : 0;
  const size_t need = table + a.copy_bytes + a.lo_bytes + b.copy_bytes + b.lo_bytes + (f32 ? 2 : 1) * (tail_a + tail_b);
  *scratch_needed = need;
  if (!scratch || scratch_bytes < need) return cudaErrorInvalidValue;
  rec->scratch_bytes = need;
  char* at = (char*)scratch;
  int* start = (int*)at;
  int *end = start + p.groups, *first_tile = end + p.groups;
  at += table;
  const bool empty = !wg && p.inner == 0;
  if (!empty) { place(&a, &at); place(&b, &at); }
  void* tails[4] = {nullptr, nullptr, nullptr, nullptr};   // A hi, A lo, B hi, B lo
  if (wg) {
    tails[0] = at; at += tail_a;
    if (f32) { tails[1] = at; at += tail_a; }
    tails[2] = at; at += tail_b;
    if (f32) { tails[3] = at; at += tail_b; }
  }

  const int64_t k_slabs = ((wg ? mean_rows : p.inner) + BK - 1) / BK;
  const int shape = choose_shape(p, sm_count, wg ? m : mean_rows, n, k_slabs);
  const int cta = shape == SHAPE_C1_128 ? 1 : 2, bn = shape == SHAPE_PAIR ? 256 : 128;
  TcParams tp = {};
  tp.tile_rows = BM * cta;
  tp.tiles_n = (int)((n + bn - 1) / bn);
  tp.tiles_m = wg ? (int)((m + tp.tile_rows - 1) / tp.tile_rows) : 1;
  const int64_t per_group = wg ? (int64_t)tp.tiles_m * tp.tiles_n : 0;
  tp.total_tiles = wg ? per_group * p.groups : (p.total_rows / tp.tile_rows + p.groups) * tp.tiles_n;   // forward: at most
  if (tp.total_tiles >= (1ll << 31)) return cudaErrorNotSupported;

  cudaError_t e = empty ? cudaSuccess : launch_operands(a, b, eb, stream, rec);
  if (e != cudaSuccess) return e;
  e = setup(start, tp.tile_rows, tp.tiles_n, per_group);
  if (e != cudaSuccess) return e;
  if (empty) {
    void* out = p.out;
    int64_t cols = p.cols;
    void* args[] = {(void*)&start, (void*)&end, (void*)&out, (void*)&cols};
    rec->launches++;
    return launch_behind(f32 ? (const void*)group_zero_kernel<float> : (const void*)group_zero_kernel<__half>, args,
                         dim3((unsigned)p.groups, 16), dim3(256), 0, stream);
  }
  if (wg) {
    TailJob ja = {p.a, tails[0], tails[1], p.rows, p.rows, a.ld}, jb = {p.b, tails[2], tails[3], p.cols, p.cols, b.ld};
    const int64_t widest = p.rows > p.cols ? p.rows : p.cols;
    int64_t strips = (widest + 255) / 256;
    if (strips > 64) strips = 64;
    void* args[] = {(void*)&ja, (void*)&jb, (void*)&start, (void*)&end};
    e = launch_behind(f32 ? (const void*)group_tail_kernel<float, 32> : (const void*)group_tail_kernel<__half, 64>, args,
                      dim3((unsigned)p.groups, (unsigned)strips, 2), dim3(256), 0, stream);
    if (e != cudaSuccess) return e;
    rec->launches++;
  }

  CUtensorMap maps[4];
  OutMaps outs;
  memset(maps, 0, sizeof maps);
  memset(&outs, 0, sizeof outs);
  const int a_mn = wg ? 1 : 0, b_mn = wg || !p.trans_b ? 1 : 0;
  auto operand = [&](CUtensorMap* map, const void* base, const Operand& o, int64_t ld, int64_t stride, bool mn, int box) {
    return make_operand_map(map, base, eb, mn, mn ? o.width : o.rows, mn ? o.rows : o.width, ld, stride, o.mats, box);
  };
  if (!operand(&maps[0], a.hi, a, a.hi_ld, a.hi_stride, a_mn, BM) || !operand(&maps[2], b.hi, b, b.hi_ld, b.hi_stride, b_mn, bn / cta))
    return cudaErrorNotSupported;
  maps[1] = maps[0]; maps[3] = maps[2];
  if (f32 && (!operand(&maps[1], a.lo, a, a.ld, a.rows * a.ld, a_mn, BM) || !operand(&maps[3], b.lo, b, b.ld, b.rows * b.ld, b_mn, bn / cta)))
    return cudaErrorNotSupported;
  if (!wg && (!operand(&outs.m[5], a.hi, a, a.hi_ld, a.hi_stride, false, kShortBox) ||
              (f32 && !operand(&outs.m[6], a.lo, a, a.ld, a.rows * a.ld, false, kShortBox))))
    return cudaErrorNotSupported;
  if (wg)
    for (int i = 0; i < 4; i++) {
      if (!tails[i]) continue;
      const Operand& o = i < 2 ? a : b;
      if (!make_operand_map(&outs.m[1 + i], tails[i], eb, true, o.width, tail_rows, o.ld, tail_rows * o.ld, 1, BM)) return cudaErrorNotSupported;
    }
  const int64_t out_mats = wg ? p.groups : 1;
  tp.M = m; tp.N = n;
  tp.num_k_blocks = wg ? 1 : (int)((p.inner + BK - 1) / BK);
  tp.splits = 1;
  tp.kb_per_split = tp.num_k_blocks;
  tp.chunk_kb = f32 ? window_slabs() : (1 << 30);
  tp.group_m = 16 / cta;
  tp.a_mn_major = a_mn; tp.b_mn_major = b_mn;
  tp.C = p.out; tp.ldc = n; tp.strideC = m * n;
  tp.status = status_word;
  tp.n_out = 1;
  tp.a_box_rows = BM;
  tp.vec_ok = (((uintptr_t)p.out & 15) == 0 && (n * eb) % 16 == 0 && (out_mats == 1 || (m * n * eb) % 16 == 0)) ? 1 : 0;
  tp.tma_store = tp.vec_ok && n * eb < (1ll << 40) && make_output_map(&outs.m[0], p.out, eb, n, m, n, m * n, out_mats) ? 1 : 0;
  tp.groups = GroupTable{start, end, first_tile, (int)p.groups, wg ? 1 : 0};
  rec->tiles = tp.total_tiles;
  return grouped_kernel(f32, shape, k_slabs)(maps, outs, tp, sm_count, stream, rec);
}

}  // namespace hc

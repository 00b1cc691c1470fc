// C ABI of the operators around a feed-forward block: products with a fused epilogue, the gradient
// through an activation, layer normalisation, products grouped by expert, AdamW.  Declarations in
// include/hc_cuda.h.  Arguments are checked before anything is enqueued.
#include <cmath>
#include <cstring>

#include "common.cuh"

using hc::DeviceGuard;

namespace {

hc_status invalid(hc_ctx* ctx, const char* msg) { return hc::ctx_fail(ctx, HC_ERR_INVALID_ARGUMENT, msg); }

bool known(hc_dtype t) { return t == HC_F16 || t == HC_F32; }
int64_t bytes_of(hc_dtype t) { return t == HC_F16 ? 2 : 4; }
bool misaligned(const void* p, int64_t bytes) { return ((uintptr_t)p & (uintptr_t)(bytes - 1)) != 0; }

// Elements of a dense tensor of up to three axes, in bytes; false when they do not fit.
bool tensor_bytes(int64_t a, int64_t b, int64_t c, int64_t elem, int64_t* out) {
  return !__builtin_mul_overflow(a, b, out) && !__builtin_mul_overflow(*out, c, out) && !__builtin_mul_overflow(*out, elem, out);
}

struct Span { const void* p; int64_t bytes; };
bool overlap(const Span& a, const Span& b) {
  if (!a.p || !b.p || a.bytes <= 0 || b.bytes <= 0) return false;
  const uintptr_t x = (uintptr_t)a.p, y = (uintptr_t)b.p;
  return x < y + (uintptr_t)b.bytes && y < x + (uintptr_t)a.bytes;
}
bool same(const Span& a, const Span& b) { return a.p == b.p && a.bytes == b.bytes; }

hc_status launched(hc_ctx* ctx, cudaError_t e, int launches, const char* what) {
  hc::ctx_count_launches(ctx, launches);
  hc::tc_forget_predecessor(hc::ctx_stream(ctx));
  return e == cudaSuccess ? HC_OK : hc::ctx_cuda_fail(ctx, e, what);
}

}  // namespace

#define HC_ENTER(ctx)                                    \
  if (!(ctx)) return HC_ERR_INVALID_ARGUMENT;            \
  std::lock_guard<std::mutex> lock(hc::ctx_mutex(ctx));  \
  DeviceGuard guard(hc::ctx_device(ctx));                \
  if (!guard.ok) return hc::ctx_fail(ctx, HC_ERR_CUDA, "the context's device cannot be made current")

extern "C" {

hc_status hc_matmul_epilogue(hc_ctx* ctx, hc_dtype dtype, const void* a, int trans_a, const void* b, int trans_b,
                             int64_t rows, int64_t inner, int64_t cols, const hc_epilogue* ep, void* out) {
  HC_ENTER(ctx);
  if (!ep) return invalid(ctx, "null epilogue");
  if (ep->activation < HC_ACT_NONE || ep->activation > HC_ACT_SILU) return invalid(ctx, "unknown activation");
  if (ep->grad_pre && (ep->bias || ep->residual || ep->pre))
    return invalid(ctx, "grad_pre excludes bias, residual and pre");
  hc::GemmProblem p;
  hc_status s = hc::ctx_build_problem(ctx, dtype, 1, a, trans_a, b, trans_b, 0, rows, inner, cols, out, &p);
  if (s != HC_OK) return s;
  const int64_t eb = bytes_of(dtype);
  for (const void* q : {a, b, (const void*)out, ep->bias, ep->residual, (const void*)ep->pre, ep->grad_pre})
    if (misaligned(q, eb)) return invalid(ctx, "a tensor is not aligned to its elements");
  const int64_t n = rows * cols * eb;   // build_problem has checked that it fits
  const Span sa = {a, rows * inner * eb}, sb = {b, inner * cols * eb}, so = {out, n}, sbias = {ep->bias, cols * eb};
  const Span sres = {ep->residual, n}, spre = {ep->pre, n}, sgrad = {ep->grad_pre, n};
  if (overlap(so, sa) || overlap(so, sb) || overlap(so, sbias) || overlap(so, spre) || (overlap(so, sres) && !same(so, sres)) ||
      (overlap(so, sgrad) && !same(so, sgrad)))
    return invalid(ctx, "the result overlaps another tensor");
  if (overlap(spre, sa) || overlap(spre, sb) || overlap(spre, sbias) || overlap(spre, sres))
    return invalid(ctx, "the kept pre-activation overlaps another tensor");
  p.fused = true;
  p.fe.act = ep->activation;
  p.fe.bias = ep->bias;
  p.fe.pre = ep->pre;
  p.fe.grad = ep->grad_pre ? 1 : 0;
  p.fe.aux = ep->grad_pre ? ep->grad_pre : ep->residual;
  return hc::ctx_run_problem(ctx, p, 2 * rows * inner * cols);
}

hc_status hc_activation_grad(hc_ctx* ctx, hc_dtype dtype, int activation, const void* grad, const void* pre, int64_t rows,
                             int64_t cols, void* dpre, float* bias_grad) {
  HC_ENTER(ctx);
  if (!known(dtype)) return hc::ctx_fail(ctx, HC_ERR_NOT_IMPLEMENTED, "activation gradient: only float16 and float32 are implemented");
  if (activation < HC_ACT_NONE || activation > HC_ACT_SILU) return invalid(ctx, "unknown activation");
  if (rows < 0 || cols < 0) return invalid(ctx, "negative dimension");
  const int64_t eb = bytes_of(dtype);
  int64_t n;
  if (!tensor_bytes(rows, cols, 1, 4, &n)) return invalid(ctx, "tensor size overflows int64");
  n = rows * cols * eb;
  if (n > 0 && (!grad || !pre || !dpre)) return invalid(ctx, "null tensor");
  if (misaligned(grad, eb) || misaligned(pre, eb) || misaligned(dpre, eb) || misaligned(bias_grad, 4))
    return invalid(ctx, "a tensor is not aligned to its elements");
  const Span sg = {grad, n}, sp = {pre, n}, sd = {dpre, n}, sb = {bias_grad, cols * 4};
  if ((overlap(sd, sg) && !same(sd, sg)) || (overlap(sd, sp) && !same(sd, sp)) || overlap(sb, sd) || overlap(sb, sg) || overlap(sb, sp))
    return invalid(ctx, "a result overlaps another tensor");
  if (cols == 0 || (rows == 0 && !bias_grad)) return HC_OK;
  void* scratch = nullptr;
  if (bias_grad) {
    hc_status s = hc::ctx_scratch(ctx, hc::activation_grad_scratch(dtype, rows, cols), &scratch);
    if (s != HC_OK) return s;
  }
  int launches = 0;
  cudaError_t e = hc::launch_activation_grad(dtype, activation, grad, pre, rows, cols, dpre, bias_grad, (float*)scratch, &launches,
                                             hc::ctx_stream(ctx));
  return launched(ctx, e, launches, "activation gradient");
}

hc_status hc_layer_norm(hc_ctx* ctx, hc_dtype dtype, hc_dtype param_dtype, const void* x, const void* weight, const void* bias,
                        int64_t rows, int64_t cols, float epsilon, void* out, float* mean, float* rstd) {
  HC_ENTER(ctx);
  if (!known(dtype) || !known(param_dtype))
    return hc::ctx_fail(ctx, HC_ERR_NOT_IMPLEMENTED, "layer norm: only float16 and float32 are implemented");
  if (rows < 0 || cols < 1) return invalid(ctx, "layer norm needs at least one column and no negative dimension");
  if (!(epsilon >= 0.0f)) return invalid(ctx, "epsilon must not be negative");
  const int64_t eb = bytes_of(dtype), pb = bytes_of(param_dtype);
  int64_t n;
  if (!tensor_bytes(rows, cols, 1, 4, &n)) return invalid(ctx, "tensor size overflows int64");
  n = rows * cols * eb;
  if (rows == 0) return HC_OK;
  if (!x || !out) return invalid(ctx, "null tensor");
  if (misaligned(x, eb) || misaligned(out, eb) || misaligned(weight, pb) || misaligned(bias, pb) || misaligned(mean, 4) || misaligned(rstd, 4))
    return invalid(ctx, "a tensor is not aligned to its elements");
  const Span sx = {x, n}, so = {out, n}, sw = {weight, cols * pb}, sb = {bias, cols * pb}, sm = {mean, rows * 4}, sr = {rstd, rows * 4};
  if ((overlap(so, sx) && !same(so, sx)) || overlap(so, sw) || overlap(so, sb) || overlap(so, sm) || overlap(so, sr) || overlap(sm, sx) ||
      overlap(sr, sx) || overlap(sm, sr) || overlap(sm, sw) || overlap(sm, sb) || overlap(sr, sw) || overlap(sr, sb))
    return invalid(ctx, "a result overlaps another tensor");
  cudaError_t e = hc::launch_layer_norm(dtype, param_dtype, x, weight, bias, rows, cols, epsilon, out, mean, rstd, hc::ctx_sm_count(ctx),
                                        hc::ctx_stream(ctx));
  return launched(ctx, e, 1, "layer norm");
}

hc_status hc_layer_norm_grad(hc_ctx* ctx, hc_dtype dtype, hc_dtype param_dtype, const void* grad, const void* x, const void* weight,
                             const float* mean, const float* rstd, int64_t rows, int64_t cols, void* dx, void* weight_grad,
                             void* bias_grad) {
  HC_ENTER(ctx);
  if (!known(dtype) || !known(param_dtype))
    return hc::ctx_fail(ctx, HC_ERR_NOT_IMPLEMENTED, "layer norm: only float16 and float32 are implemented");
  if (rows < 0 || cols < 1) return invalid(ctx, "layer norm needs at least one column and no negative dimension");
  const int64_t eb = bytes_of(dtype), pb = bytes_of(param_dtype);
  int64_t n;
  if (!tensor_bytes(rows, cols, 1, 4, &n)) return invalid(ctx, "tensor size overflows int64");
  n = rows * cols * eb;
  if (rows > 0 && (!grad || !x || !mean || !rstd)) return invalid(ctx, "null tensor");
  if (misaligned(x, eb) || misaligned(grad, eb) || misaligned(dx, eb) || misaligned(weight, pb) || misaligned(weight_grad, pb) ||
      misaligned(bias_grad, pb) || misaligned(mean, 4) || misaligned(rstd, 4))
    return invalid(ctx, "a tensor is not aligned to its elements");
  const Span in[] = {{grad, n}, {x, n}, {weight, cols * pb}, {mean, rows * 4}, {rstd, rows * 4}};
  const Span res[] = {{dx, n}, {weight_grad, cols * pb}, {bias_grad, cols * pb}};
  const bool sums = weight_grad || bias_grad;
  for (int i = 0; i < 3; i++) {
    for (int k = 0; k < 5; k++)
      if (overlap(res[i], in[k]) && !(i == 0 && k < 2 && !sums && same(res[i], in[k])))
        return invalid(ctx, "a result overlaps another tensor");
    for (int k = 0; k < i; k++)
      if (overlap(res[i], res[k])) return invalid(ctx, "two results overlap");
  }
  if (!sums && (!dx || rows == 0)) return HC_OK;
  void* scratch = nullptr;
  if (sums) {
    hc_status s = hc::ctx_scratch(ctx, hc::layer_norm_grad_scratch(dtype, rows, cols, hc::ctx_sm_count(ctx)), &scratch);
    if (s != HC_OK) return s;
  }
  int launches = 0;
  cudaError_t e = hc::launch_layer_norm_grad(dtype, param_dtype, grad, x, weight, mean, rstd, rows, cols, dx, weight_grad, bias_grad,
                                             (float*)scratch, hc::ctx_sm_count(ctx), &launches, hc::ctx_stream(ctx));
  return launched(ctx, e, launches, "layer norm gradient");
}

}  // extern "C"

namespace {
hc_status run_grouped(hc_ctx* ctx, const hc::GroupedProblem& p) {
  const int64_t eb = bytes_of(p.dtype);
  const int64_t width = p.weight_grad ? p.rows : p.inner;
  int64_t na, nb, no;
  if (!tensor_bytes(p.total_rows, width, 1, 4, &na) || !tensor_bytes(p.weight_grad ? 1 : p.groups, p.weight_grad ? p.total_rows : p.inner, p.cols, 4, &nb) ||
      !tensor_bytes(p.weight_grad ? p.groups : 1, p.weight_grad ? p.rows : p.total_rows, p.cols, 4, &no))
    return invalid(ctx, "tensor size overflows int64");
  na = na / 4 * eb; nb = nb / 4 * eb; no = no / 4 * eb;
  if (no == 0) return HC_OK;
  if (!p.offsets || !p.out || (na > 0 && !p.a) || (nb > 0 && !p.b)) return invalid(ctx, "null tensor");
  if (misaligned(p.offsets, 8) || misaligned(p.a, eb) || misaligned(p.b, eb) || misaligned(p.out, eb))
    return invalid(ctx, "a tensor is not aligned to its elements");
  const Span so = {p.out, no};
  if (overlap(so, {p.a, na}) || overlap(so, {p.b, nb}) || overlap(so, {p.offsets, (p.groups + 1) * 8}))
    return invalid(ctx, "the result overlaps another tensor");
  // The table of groups and the tiles' coordinates are 32-bit, and a copy may start up to a tile behind the last row.
  if (p.total_rows >= (1ll << 31) - 256)
    return hc::ctx_fail(ctx, HC_ERR_NOT_IMPLEMENTED, "grouped product of 2^31 - 256 rows or more");
  if (p.weight_grad && p.total_rows == 0) {
    cudaError_t e = cudaMemsetAsync(p.out, 0, (size_t)no, hc::ctx_stream(ctx));
    return launched(ctx, e, 0, "grouped product");
  }
  hc::LaunchRecord rec;
  size_t need = 0;
  void* scratch = nullptr;
  // The first call only asks for the size of the work area.
  cudaError_t e = hc::launch_grouped(p, hc::ctx_stream(ctx), hc::ctx_status_word(ctx), nullptr, 0, hc::ctx_sm_count(ctx), &rec, &need);
  if (e == cudaErrorInvalidValue && need > 0) {
    hc_status s = hc::ctx_scratch(ctx, need, &scratch);
    if (s != HC_OK) return s;
    e = hc::launch_grouped(p, hc::ctx_stream(ctx), hc::ctx_status_word(ctx), scratch, need, hc::ctx_sm_count(ctx), &rec, &need);
  }
  if (e == cudaErrorNotSupported)
    return hc::ctx_fail(ctx, HC_ERR_NOT_IMPLEMENTED, "grouped product too large for the tensor-core kernel's 32-bit tile coordinates");
  hc::ctx_note_launch(ctx, rec, 2 * p.total_rows * width * p.cols);
  return launched(ctx, e, 0, "grouped product");
}
}  // namespace

extern "C" {

hc_status hc_grouped_matmul(hc_ctx* ctx, hc_dtype dtype, int64_t group_count, const int64_t* offsets, const void* a, const void* b,
                            int trans_b, int64_t total_rows, int64_t inner, int64_t cols, void* out) {
  HC_ENTER(ctx);
  if (!known(dtype)) return hc::ctx_fail(ctx, HC_ERR_NOT_IMPLEMENTED, "grouped matmul: only float16 and float32 are implemented");
  if (group_count < 0 || total_rows < 0 || inner < 0 || cols < 0) return invalid(ctx, "negative dimension");
  if (group_count > 65535) return invalid(ctx, "at most 65535 groups");
  if (group_count == 0) return HC_OK;
  const hc::GroupedProblem p = {dtype, false, trans_b != 0, group_count, total_rows, 0, inner, cols, offsets, a, b, out};
  return run_grouped(ctx, p);
}

hc_status hc_grouped_matmul_weight_grad(hc_ctx* ctx, hc_dtype dtype, int64_t group_count, const int64_t* offsets, const void* a,
                                        const void* b, int64_t total_rows, int64_t rows, int64_t cols, void* out) {
  HC_ENTER(ctx);
  if (!known(dtype)) return hc::ctx_fail(ctx, HC_ERR_NOT_IMPLEMENTED, "grouped matmul: only float16 and float32 are implemented");
  if (group_count < 0 || total_rows < 0 || rows < 0 || cols < 0) return invalid(ctx, "negative dimension");
  if (group_count > 65535) return invalid(ctx, "at most 65535 groups");
  if (group_count == 0) return HC_OK;
  const hc::GroupedProblem p = {dtype, true, false, group_count, total_rows, rows, 0, cols, offsets, a, b, out};
  return run_grouped(ctx, p);
}

hc_status hc_adamw(hc_ctx* ctx, const hc_adamw_tensor* tensors, int64_t tensor_count, int64_t step, double lr, double beta1,
                   double beta2, double epsilon, double weight_decay) {
  HC_ENTER(ctx);
  if (tensor_count < 0 || (tensor_count > 0 && !tensors)) return invalid(ctx, "null table of tensors");
  if (step < 1) return invalid(ctx, "the step counts from 1");
  if (!(beta1 >= 0.0 && beta1 < 1.0) || !(beta2 >= 0.0 && beta2 < 1.0)) return invalid(ctx, "beta1 and beta2 lie in [0, 1)");
  if (!(epsilon >= 0.0)) return invalid(ctx, "epsilon must not be negative");
  for (int64_t i = 0; i < tensor_count; i++) {
    const hc_adamw_tensor& t = tensors[i];
    if (!known(t.param_dtype) || !known(t.grad_dtype))
      return hc::ctx_fail(ctx, HC_ERR_NOT_IMPLEMENTED, "AdamW: only float16 and float32 are implemented");
    if (t.count < 0 || t.count > (1ll << 42)) return invalid(ctx, "a tensor's count is negative or too large");
    if (t.count == 0) continue;
    if (!t.param || !t.grad || !t.moment1 || !t.moment2) return invalid(ctx, "null tensor");
    if (misaligned(t.param, bytes_of(t.param_dtype)) || misaligned(t.grad, bytes_of(t.grad_dtype)) || misaligned(t.moment1, 4) ||
        misaligned(t.moment2, 4) || misaligned(t.param_copy, 2))
      return invalid(ctx, "a tensor is not aligned to its elements");
    const Span all[] = {{t.param, t.count * bytes_of(t.param_dtype)}, {t.moment1, t.count * 4}, {t.moment2, t.count * 4},
                        {t.param_copy, t.count * 2}, {t.grad, t.count * bytes_of(t.grad_dtype)}};
    for (int k = 0; k < 4; k++)
      for (int l = k + 1; l < 5; l++)
        if (overlap(all[k], all[l])) return invalid(ctx, "a tensor's buffers overlap");
  }
  hc::AdamWFactors f;
  f.lr = (float)lr;
  f.beta1 = (float)beta1; f.one_minus_beta1 = (float)(1.0 - beta1);
  f.beta2 = (float)beta2; f.one_minus_beta2 = (float)(1.0 - beta2);
  f.epsilon = (float)epsilon;
  f.decay = (float)(1.0 - lr * weight_decay);
  f.inv_c1 = (float)(1.0 / (1.0 - std::pow(beta1, (double)step)));
  f.inv_c2 = (float)(1.0 / (1.0 - std::pow(beta2, (double)step)));
  int launches = 0;
  cudaError_t e = hc::launch_adamw(tensors, tensor_count, f, &launches, hc::ctx_stream(ctx));
  return launched(ctx, e, launches, "AdamW");
}

}  // extern "C"

"""The operators of a feed-forward block's training step and of its serving form, as cases that can be timed.

Four families, each through the entry points of `honeycrisp_b200.CUDABackend`:

  linear   `matmulEpilogue` / `activationGrad`: a product with bias, activation and residual in its epilogue, the
           product that carries a gradient through an activation, and the gradient of an activation with the bias's
  norm     `layerNorm` / `layerNormGrad`: layer normalisation, forward and backward with the parameters' gradients
  experts  `groupedMatmul` / `groupedMatmulWeightGrad`: products grouped by expert, with ragged groups of rows
  adamw    `adamW`: one AdamW step over many tensors

`run` computes a case in elementary torch operations, or, where `own` is true, with the framework's calls.
"""
import math
import random

import torch

own = False

DTYPES = {"float16": torch.float16, "float32": torch.float32}


def listed():
    return [
        # Serving: the up projection of a feed-forward block for a batch of four sequences, one new token each.
        dict(name="linear_decode", op="linear", direction="forward", dtype="float16", rows=4, inner=4096, cols=16384,
             trans_b=False, activation="gelu", bias=True, residual=False, pre=False),
        # Training: the up projection of 16384 tokens; the pre-activation is kept for the backward pass.
        dict(name="linear_up_train", op="linear", direction="forward", dtype="float16", rows=16384, inner=4096, cols=16384,
             trans_b=False, activation="gelu", bias=True, residual=False, pre=True),
        # The down projection, whose result is added to the residual stream; weights stored [out, in].
        dict(name="linear_down_residual", op="linear", direction="forward", dtype="float16", rows=2048, inner=16384, cols=4096,
             trans_b=True, activation="none", bias=True, residual=True, pre=False),
        # Backward of the down projection carried through the activation behind it: (dY . W^T) * act'(pre).
        dict(name="linear_grad_in", op="linear", direction="grad_in", dtype="float16", rows=4096, inner=4096, cols=16384,
             trans_b=True, activation="gelu_tanh", bias=False, residual=False, pre=False),
        # A small float32 layer of odd sizes: nothing is a multiple of a tile or of 16 bytes.
        dict(name="linear_f32_odd", op="linear", direction="forward", dtype="float32", rows=1001, inner=1023, cols=2049,
             trans_b=False, activation="silu", bias=True, residual=True, pre=False),
        # A training step's normalisation of 16384 tokens: forward, then backward with the parameters' gradients.
        dict(name="norm_train", op="norm", direction="train", dtype="float16", rows=16384, cols=4096, affine=True),
        # Serving: one normalisation of a few rows, where the launch is what counts.
        dict(name="norm_decode_f32", op="norm", direction="forward", dtype="float32", rows=4, cols=4099, affine=True),
        # 16384 tokens routed to eight experts, unevenly; one expert gets none.
        dict(name="experts_train", op="experts", direction="forward", dtype="float16", groups=8, rows=16384, tail=0, inner=4096,
             cols=4096, empty=1, skew=1.0),
        # The experts' weight gradients of the same step: the ragged length is the contracted one.
        dict(name="experts_weight_grad", op="experts", direction="grad_weight", dtype="float16", groups=8, rows=16384, tail=0,
             inner=2048, cols=4096, empty=1, skew=1.0),
        # Serving: 128 routed tokens over 64 experts, two rows each on average, and padding rows behind the last.
        dict(name="experts_decode", op="experts", direction="forward", dtype="float16", groups=64, rows=128, tail=9, inner=1024,
             cols=4096, empty=5, skew=0.5),
        # float32 master weights of eight blocks, float16 gradients, a float16 copy of the new weights for the next step.
        dict(name="adamw_blocks", op="adamw", dtype="float32", grad="float16", copy=True, layers=8, width=1024, hidden=8192,
             packed=False),
        # Many small float32 tensors of odd sizes, back to back in one buffer: most of them start off a 16-byte boundary.
        dict(name="adamw_small", op="adamw", dtype="float32", grad="float32", copy=False, layers=12, width=63, hidden=257,
             packed=True),
    ]


def _size(rng, low, high):
    """A length between low and high, even over the logarithm, half of them rounded to a multiple of eight."""
    n = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    return max(low, min(high, (n + 7) // 8 * 8 if n >= 16 and rng.random() < 0.5 else n))


def draw(rng):
    op = rng.choice(["linear", "linear", "norm", "experts", "experts", "adamw"])
    dtype = rng.choice(["float16", "float16", "float32"])
    if op == "linear":
        direction = rng.choice(["forward", "forward", "grad_in", "act_grad"])
        rows, inner, cols = _size(rng, 1, 16384), _size(rng, 8, 16384), _size(rng, 8, 16384)
        while rows * inner * cols > (1 << 38):
            inner = max(8, inner // 2)
        return dict(op=op, direction=direction, dtype=dtype, rows=rows, inner=inner, cols=cols,
                    trans_b=rng.random() < 0.5, activation=rng.choice(["none", "relu", "gelu", "gelu_tanh", "silu"]),
                    bias=rng.random() < 0.7, residual=rng.random() < 0.5, pre=rng.random() < 0.4)
    if op == "norm":
        cols = _size(rng, 1, 32768)
        rows = _size(rng, 1, max(1, min(65536, (1 << 26) // cols)))
        return dict(op=op, direction=rng.choice(["forward", "train"]), dtype=dtype, rows=rows, cols=cols,
                    affine=rng.random() < 0.8)
    if op == "experts":
        groups = _size(rng, 1, 128)
        rows, inner, cols = _size(rng, 1, 16384), _size(rng, 8, 8192), _size(rng, 8, 8192)
        while groups * inner * cols > (1 << 28) or rows * inner * cols > (1 << 37):
            inner, cols = max(8, inner * 2 // 3), max(8, cols * 2 // 3)
        return dict(op=op, direction=rng.choice(["forward", "grad_in", "grad_weight"]), dtype=dtype, groups=groups, rows=rows,
                    tail=rng.choice([0, 0, 1, 37]), inner=inner, cols=cols, empty=rng.randint(0, groups // 4),
                    skew=rng.choice([0.0, 0.5, 1.0, 3.0]))
    width, hidden, layers = _size(rng, 8, 4096), _size(rng, 8, 8192), rng.randint(1, 24)
    while layers * width * hidden > (1 << 26):
        layers, hidden = max(1, layers // 2), max(8, hidden * 2 // 3)
    half = dtype == "float16"
    return dict(op=op, dtype=dtype, grad="float16" if half else rng.choice(["float16", "float32"]),
                copy=not half and rng.random() < 0.5, layers=layers, width=width, hidden=hidden, packed=rng.random() < 0.5)


# ---- what a case's program holds before the call ------------------------------------------------------------------

def _normal(gen, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)


def _uniform(gen, shape, dtype, inner):
    """Weights as a Linear layer draws them: uniform within sqrt(3 / inner)."""
    return ((torch.rand(shape, generator=gen, device="cuda") * 2 - 1) * math.sqrt(3.0 / inner)).to(dtype)


def _group_ends(case, seed):
    """Offsets of the groups' rows: `groups` + 1 of them, the last one `rows`; `empty` groups have no row."""
    rng = random.Random(seed * 7919 + 17)
    share = [(rng.random() + 1e-3) ** case["skew"] for _ in range(case["groups"])]
    for g in rng.sample(range(case["groups"]), case["empty"]):
        share[g] = 0.0
    total, at, ends = sum(share) or 1.0, 0.0, [0]
    for s in share:
        at += s
        ends.append(int(round(case["rows"] * at / total)))
    ends[-1] = case["rows"]
    return ends


def _adamw_counts(case):
    w, h = case["width"], case["hidden"]
    return [w * h, h, h * w, w, w, w] * case["layers"]


def _adamw_starts(case):
    step = 1 if case["packed"] else 64
    starts, at = [], 0
    for n in _adamw_counts(case):
        starts.append(at)
        at += -(-n // step) * step
    return starts, at


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    t = DTYPES[case["dtype"]]
    s = {"case": case, "dtype": t}
    if case["op"] == "linear":
        rows, inner, cols, direction = case["rows"], case["inner"], case["cols"], case["direction"]
        empty = lambda: torch.empty(rows, cols, dtype=t, device="cuda")  # noqa: E731
        s["out"] = empty()
        if direction == "act_grad":
            s["grad"] = _normal(gen, (rows, cols), t, 0.1)
            s["pre_in"] = _normal(gen, (rows, cols), t, 1.5)
            s["bias_grad"] = torch.empty(cols, dtype=torch.float32, device="cuda")
            return s
        s["a"] = _normal(gen, (rows, inner), t)
        s["b"] = _uniform(gen, (cols, inner) if case["trans_b"] else (inner, cols), t, inner)
        if direction == "grad_in":
            s["pre_in"] = _normal(gen, (rows, cols), t, 1.5)
            return s
        s["bias"] = _normal(gen, (cols,), t, 0.3) if case["bias"] else None
        s["residual"] = _normal(gen, (rows, cols), t) if case["residual"] else None
        s["pre"] = empty() if case["pre"] else None
    elif case["op"] == "norm":
        rows, cols = case["rows"], case["cols"]
        # A residual stream: every column has an offset and a scale of its own, a few of them large.
        scale = torch.exp(0.5 * torch.randn(cols, generator=gen, device="cuda"))
        s["x"] = ((torch.randn(rows, cols, generator=gen, device="cuda") + 0.5 * torch.randn(cols, generator=gen, device="cuda")) * scale).to(t)
        s["weight"] = 1 + 0.2 * torch.randn(cols, generator=gen, device="cuda") if case["affine"] else None
        s["bias"] = 0.2 * torch.randn(cols, generator=gen, device="cuda") if case["affine"] else None
        s["out"] = torch.empty_like(s["x"])
        if case["direction"] == "train":
            s["grad"] = _normal(gen, (rows, cols), t, 0.1)
            s["mean"], s["rstd"] = (torch.empty(rows, dtype=torch.float32, device="cuda") for _ in range(2))
            s["dx"] = torch.empty_like(s["x"])
            s["dweight"], s["dbias"] = (torch.empty(cols, dtype=torch.float32, device="cuda") if case["affine"] else None for _ in range(2))
    elif case["op"] == "experts":
        rows, inner, cols, groups = case["rows"] + case["tail"], case["inner"], case["cols"], case["groups"]
        s["ends"] = _group_ends(case, seed)
        s["offsets"] = torch.tensor(s["ends"], dtype=torch.int64).cuda()
        s["a"] = _normal(gen, (rows, inner), t)
        if case["direction"] == "grad_weight":
            s["b"] = _normal(gen, (rows, cols), t, 0.1)
            s["out"] = torch.empty(groups, inner, cols, dtype=t, device="cuda")
        else:
            shape = (groups, cols, inner) if case["direction"] == "grad_in" else (groups, inner, cols)
            s["b"] = _uniform(gen, shape, t, inner)
            s["out"] = torch.full((rows, cols), 0.25, dtype=t, device="cuda")  # rows behind the last group stay
    else:
        starts, total = _adamw_starts(case)
        s["param"] = _normal(gen, (total,), t, 0.05)
        s["grad"] = _normal(gen, (total,), DTYPES[case["grad"]], 1e-2)
        s["m"] = _normal(gen, (total,), torch.float32, 1e-2)
        s["v"] = _normal(gen, (total,), torch.float32, 1e-2) ** 2
        s["copy"] = torch.zeros(total, dtype=torch.float16, device="cuda") if case["copy"] else None
        s["parts"] = [slice(b, b + n) for b, n in zip(starts, _adamw_counts(case))]
        s["hyper"] = dict(step=10, learningRate=1e-3, beta1=0.9, beta2=0.999, epsilon=1e-8, weightDecay=0.01)
        if own:
            # The optimiser's table of tensors, laid out once for all steps.
            s["plan"] = _backend().adamWPlan([dict(param=s["param"][p], grad=s["grad"][p], moment1=s["m"][p], moment2=s["v"][p],
                                                   copy=s["copy"][p] if case["copy"] else None) for p in s["parts"]])
    return s


# ---- the plain forms ----------------------------------------------------------------------------------------------

_C = math.sqrt(2.0 / math.pi)


def _activation(z, name):
    if name == "relu":
        return torch.where(z < 0, torch.zeros_like(z), z)
    if name == "gelu":
        return 0.5 * z * (1 + torch.erf(z / math.sqrt(2.0)))
    if name == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(_C * (z + 0.044715 * z * z * z)))
    if name == "silu":
        return z / (1 + torch.exp(-z))
    return z


def _activation_slope(z, name):
    if name == "relu":
        return (z > 0).to(z.dtype)
    if name == "gelu":
        return 0.5 * (1 + torch.erf(z / math.sqrt(2.0))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    if name == "gelu_tanh":
        th = torch.tanh(_C * (z + 0.044715 * z * z * z))
        return 0.5 * (1 + th) + 0.5 * z * (1 - th * th) * _C * (1 + 3 * 0.044715 * z * z)
    if name == "silu":
        sg = 1 / (1 + torch.exp(-z))
        return sg * (1 + z * (1 - sg))
    return torch.ones_like(z)


def _plain_linear(s, case):
    t = s["dtype"]
    if case["direction"] == "act_grad":
        d = s["grad"].float() * _activation_slope(s["pre_in"].float(), case["activation"])
        return {"out": d.to(t), "bias_grad": d.sum(0)}
    b = s["b"].float()
    z = s["a"].float() @ (b.t() if case["trans_b"] else b)
    if case["direction"] == "grad_in":
        return {"out": (z * _activation_slope(s["pre_in"].float(), case["activation"])).to(t)}
    if s["bias"] is not None:
        z = z + s["bias"].float()
    y = _activation(z, case["activation"])
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return {"out": y.to(t), **({"pre": z.to(t)} if case["pre"] else {})}


EPSILON = 1e-5


def _plain_norm(s, case):
    t, x = s["dtype"], s["x"].float()
    mean = x.mean(1, keepdim=True)
    d = x - mean
    rstd = 1 / torch.sqrt((d * d).mean(1, keepdim=True) + EPSILON)
    h = d * rstd
    y = h * s["weight"] + s["bias"] if case["affine"] else h
    if case["direction"] == "forward":
        return {"out": y.to(t)}
    g = s["grad"].float()
    gw = g * s["weight"] if case["affine"] else g
    dx = rstd * (gw - gw.mean(1, keepdim=True) - h * (gw * h).mean(1, keepdim=True))
    r = {"out": y.to(t), "mean": mean[:, 0], "rstd": rstd[:, 0], "dx": dx.to(t)}
    return {**r, "dweight": (g * h).sum(0), "dbias": g.sum(0)} if case["affine"] else r


def _plain_experts(s, case):
    out, a, b, ends = s["out"], s["a"], s["b"], s["ends"]
    for g in range(case["groups"]):
        rows = slice(ends[g], ends[g + 1])
        if case["direction"] == "grad_weight":
            out[g] = a[rows].float().t() @ b[rows].float()
        else:
            w = b[g].float()
            out[rows] = (a[rows].float() @ (w.t() if case["direction"] == "grad_in" else w)).to(out.dtype)
    return {"out": out}


def _plain_adamw(s, case):
    h = s["hyper"]
    c1, c2 = 1 - h["beta1"] ** h["step"], 1 - h["beta2"] ** h["step"]
    for p in s["parts"]:
        g, m, v, w = s["grad"][p].float(), s["m"][p], s["v"][p], s["param"][p].float()
        m.copy_(h["beta1"] * m + (1 - h["beta1"]) * g)
        v.copy_(h["beta2"] * v + (1 - h["beta2"]) * g * g)
        w = w * (1 - h["learningRate"] * h["weightDecay"]) - h["learningRate"] * (m / c1) / (torch.sqrt(v / c2) + h["epsilon"])
        s["param"][p].copy_(w)
        if case["copy"]:
            s["copy"][p].copy_(w)
    return {k: s[k] for k in ("param", "m", "v", "copy") if s[k] is not None}


# ---- the framework's calls ----------------------------------------------------------------------------------------

_the_backend = None


def _backend():
    """The program's backend, on torch's default stream (the legacy stream, whose handle is 1)."""
    global _the_backend
    if _the_backend is None:
        from honeycrisp_b200 import CUDABackend
        _the_backend = CUDABackend(torch.cuda.current_device())
        _the_backend.useStream(1)
    return _the_backend


def _own(s, case):
    be, t = _backend(), case["dtype"]
    if case["op"] == "linear":
        rows, inner, cols = case["rows"], case["inner"], case["cols"]
        if case["direction"] == "act_grad":
            be.activationGrad(s["grad"], s["pre_in"], rows, cols, t, case["activation"], out=s["out"], biasGrad=s["bias_grad"], mark=False)
            return {"out": s["out"], "bias_grad": s["bias_grad"]}
        if case["direction"] == "grad_in":
            be.matmulEpilogue(s["a"], False, s["b"], case["trans_b"], rows, inner, cols, t, activation=case["activation"],
                              gradPre=s["pre_in"], out=s["out"], mark=False)
            return {"out": s["out"]}
        be.matmulEpilogue(s["a"], False, s["b"], case["trans_b"], rows, inner, cols, t, activation=case["activation"],
                          bias=s["bias"], residual=s["residual"], pre=s["pre"], out=s["out"], mark=False)
        return {"out": s["out"], **({"pre": s["pre"]} if case["pre"] else {})}
    if case["op"] == "norm":
        rows, cols = case["rows"], case["cols"]
        if case["direction"] == "forward":
            be.layerNorm(s["x"], s["weight"], s["bias"], rows, cols, t, epsilon=EPSILON, out=s["out"], mark=False)
            return {"out": s["out"]}
        be.layerNorm(s["x"], s["weight"], s["bias"], rows, cols, t, epsilon=EPSILON, out=s["out"], mean=s["mean"], rstd=s["rstd"], mark=False)
        be.layerNormGrad(s["grad"], s["x"], s["weight"], s["mean"], s["rstd"], rows, cols, t, out=s["dx"],
                         weightGrad=s["dweight"], biasGrad=s["dbias"], mark=False)
        return {k: s[k] for k in ("out", "mean", "rstd", "dx", "dweight", "dbias") if s[k] is not None}
    if case["op"] == "experts":
        rows, inner, cols = case["rows"] + case["tail"], case["inner"], case["cols"]
        if case["direction"] == "grad_weight":
            be.groupedMatmulWeightGrad(case["groups"], s["offsets"], s["a"], s["b"], rows, inner, cols, t, out=s["out"], mark=False)
        else:
            be.groupedMatmul(case["groups"], s["offsets"], s["a"], s["b"], case["direction"] == "grad_in", rows, inner, cols, t,
                             out=s["out"], mark=False)
        return {"out": s["out"]}
    be.adamW(s["plan"], mark=False, **s["hyper"])
    return {k: s[k] for k in ("param", "m", "v", "copy") if s[k] is not None}


def run(state):
    case = state["case"]
    if own:
        return _own(state, case)
    return {"linear": _plain_linear, "norm": _plain_norm, "experts": _plain_experts, "adamw": _plain_adamw}[case["op"]](state, case)


# ---- what a pass cannot do without --------------------------------------------------------------------------------

def work(case):
    e = 2 if case["dtype"] == "float16" else 4
    if case["op"] == "linear":
        rows, inner, cols = case["rows"], case["inner"], case["cols"]
        if case["direction"] == "act_grad":
            return {"bytes": 3 * rows * cols * e + 4 * cols, "flops": 2 * rows * cols}
        extra = 1 if case["direction"] == "grad_in" else case["residual"] + case["pre"]
        row = cols * e if case["direction"] == "forward" and case["bias"] else 0
        return {"bytes": (rows * inner + inner * cols + (1 + extra) * rows * cols) * e + row, "flops": 2 * rows * inner * cols}
    if case["op"] == "norm":
        n, params = case["rows"] * case["cols"], 8 * case["cols"] if case["affine"] else 0
        if case["direction"] == "forward":
            return {"bytes": 2 * n * e + params, "flops": 8 * n}
        return {"bytes": 4 * n * e + 2 * params + 8 * case["rows"], "flops": 20 * n}
    if case["op"] == "experts":
        rows, inner, cols, used = case["rows"], case["inner"], case["cols"], min(case["groups"] - case["empty"], case["rows"])
        if case["direction"] == "grad_weight":
            moved = rows * (inner + cols) + case["groups"] * inner * cols
        else:
            moved = rows * (inner + cols) + used * inner * cols
        return {"bytes": moved * e, "flops": 2 * rows * inner * cols}
    n = sum(_adamw_counts(case))
    g = 2 if case["grad"] == "float16" else 4
    return {"bytes": n * (2 * e + g + 16 + (2 if case["copy"] else 0)), "flops": 15 * n}


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------

def _phi(z):
    return torch.special.erfc(-z * 0.7071067811865476) / 2


def _exact_activation(z, name):
    """The activation's value and slope."""
    if name == "relu":
        return z.clamp(min=0), torch.heaviside(z, torch.zeros((), dtype=z.dtype, device=z.device))
    if name == "gelu":
        return z * _phi(z), _phi(z) + z * (-z.square() / 2).exp() * 0.3989422804014327
    if name == "gelu_tanh":
        u = 2 * 0.7978845608028654 * (z + 0.044715 * z ** 3)
        sg = torch.sigmoid(u)
        return z * sg, sg + z * sg * torch.sigmoid(-u) * 2 * 0.7978845608028654 * (1 + 0.134145 * z ** 2)
    if name == "silu":
        sg = torch.sigmoid(z)
        return z * sg, sg + z * sg * torch.sigmoid(-z)
    return z, torch.ones_like(z)


def _exact_linear(s, case):
    d = lambda k: s[k].double()  # noqa: E731
    if case["direction"] == "act_grad":
        r = d("grad") * _exact_activation(d("pre_in"), case["activation"])[1]
        return {"out": r, "bias_grad": r.sum(0)}
    z = torch.einsum("rk,ck->rc" if case["trans_b"] else "rk,kc->rc", d("a"), d("b"))
    if case["direction"] == "grad_in":
        return {"out": z.mul_(_exact_activation(d("pre_in"), case["activation"])[1])}
    z = z if s["bias"] is None else z.add_(d("bias"))
    y = _exact_activation(z, case["activation"])[0]
    y = y if s["residual"] is None else y + d("residual")
    return {"out": y, "pre": z} if case["pre"] else {"out": y}


def _exact_norm(s, case):
    x = s["x"].double()
    var, mean = torch.var_mean(x, dim=1, unbiased=False)
    rstd = (var + EPSILON).rsqrt()
    h = (x - mean[:, None]).mul_(rstd[:, None])
    w = s["weight"].double() if case["affine"] else torch.ones(case["cols"], dtype=torch.float64, device="cuda")
    y = torch.addcmul(s["bias"].double(), h, w) if case["affine"] else h.clone()
    if case["direction"] == "forward":
        return {"out": y}
    g = s["grad"].double()
    n = case["cols"]
    a, b = torch.mv(g, w) / n, torch.mv(g * h, w) / n
    dx = (g * w - a[:, None] - h * b[:, None]) * rstd[:, None]
    r = {"out": y, "mean": mean, "rstd": rstd, "dx": dx}
    if case["affine"]:
        r["dweight"], r["dbias"] = torch.einsum("rc,rc->c", g, h), g.sum(0)
    return r


def _exact_experts(s, case):
    a, b, ends = s["a"], s["b"], s["ends"]
    if case["direction"] == "grad_weight":
        return {"out": torch.stack([torch.einsum("ri,rc->ic", a[i:j].double(), b[i:j].double()) for i, j in zip(ends, ends[1:])])}
    kind = "ri,ci->rc" if case["direction"] == "grad_in" else "ri,ic->rc"
    parts = [torch.einsum(kind, a[i:j].double(), b[g].double()) for g, (i, j) in enumerate(zip(ends, ends[1:]))]
    return {"out": torch.cat(parts + [s["out"][ends[-1]:].double()])}


def _exact_adamw(s, case):
    """The whole buffers at once: what lies between two tensors keeps its values."""
    h = s["hyper"]
    inside = torch.zeros(s["param"].numel(), dtype=torch.bool, device="cuda")
    for p in s["parts"]:
        inside[p] = True
    g, m, v, w = (s[k].double() for k in ("grad", "m", "v", "param"))
    m2, v2 = torch.lerp(g, m, h["beta1"]), torch.lerp(g.square(), v, h["beta2"])
    update = m2 / (1 - h["beta1"] ** h["step"]) / ((v2 / (1 - h["beta2"] ** h["step"])).sqrt() + h["epsilon"])
    w2 = w - h["learningRate"] * (update + h["weightDecay"] * w)
    r = {k: torch.where(inside, new, old) for k, new, old in (("param", w2, w), ("m", m2, m), ("v", v2, v))}
    if case["copy"]:
        r["copy"] = torch.where(inside, w2, s["copy"].double())
    return r


def exact(case, seed):
    s = prepare(case, seed)
    return {"linear": _exact_linear, "norm": _exact_norm, "experts": _exact_experts, "adamw": _exact_adamw}[case["op"]](s, case)

"""The work whose speed is measured for the feed-forward operators: the linear layer
with bias, activation and residual in its epilogue, the gated feed-forward block, and
SwiGLU with its inputs kept in 8 bits for the backward. One pass each (training:
forward + backward; serving: forward), through the framework's entry points (``own``)
or in plain tensor operations.

The sizes are those of the workloads that this repository is built around (a
Qwen3-style text model: hidden 2048, MLP 6144, 4 x 2048 tokens, a ragged batch of 1777
tokens) and of what users of the same entry points bring besides: the linear layers of a
vision tower over image patches, single tokens, short prompts, odd widths, fp32 and
fp16 models.

The definitions, of which both forms are computed:

  linear   z = x W^T + b, y = act(z) + residual, with act one of none, silu, gelu (by the
           error function) and gelu_tanh. Backward: dz = dy act'(z), dx = dz W,
           dW = dz^T x, db = the sum of dz's rows, dresidual = dy.
  mlp      g = x Wg^T, u = x Wu^T, h = silu(g) u, y = h Wd^T + residual. Backward:
           dh = dy Wd, dg = dh u silu'(g), du = dh silu(g), dx = dg Wg + du Wu,
           dWg = dg^T x, dWu = du^T x, dWd = dy^T h, dresidual = dy.
  swiglu   h = silu(g) u, dg = dh u silu'(g), du = dh silu(g).

With checkpoint "fp8" the backward reads z (linear), g and u (mlp, swiglu; h is formed of
them again) as they were held in 8 bits: each row in blocks of 32 elements (the last one
shorter), with e = max(floor(log2 m) - 7, -126) for the largest finite magnitude m of a
block (e = -126 where that is 0), element v as v / 2^e rounded to the nearest number of
e4m3 (3 bits of mantissa, smallest step 2^-9, ties to even), NaN where v is not finite.
"""

import math

import torch

own = False

DEV = "cuda"
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BLOCK = 32


# ------------------------------------------------------------------ the cases

def listed():
    return [
        # an output projection with its residual, one token being decoded: launches,
        # host time and the weight's bytes count
        dict(name="linear_token", kind="linear", tokens=1, ins=2048, outs=2048, act="none",
             bias=False, residual=True, train=False, checkpoint="none", dtype="bf16"),
        # the first linear layer of a vision block over the patches of several images
        dict(name="linear_gelu_patches", kind="linear", tokens=8192, ins=1152, outs=4304,
             act="gelu_tanh", bias=True, residual=False, train=True, checkpoint="none",
             dtype="bf16"),
        # the same over one image, its inner activations kept in 8 bits
        dict(name="linear_gelu_patches_fp8", kind="linear", tokens=2916, ins=1152, outs=4304,
             act="gelu_tanh", bias=True, residual=False, train=True, checkpoint="fp8",
             dtype="bf16"),
        # the second linear layer of a vision block, which adds the block's residual
        dict(name="linear_residual_patches", kind="linear", tokens=8192, ins=4304, outs=1152,
             act="none", bias=True, residual=True, train=True, checkpoint="none", dtype="bf16"),
        # a short batch of a model kept in fp32, odd widths
        dict(name="linear_fp32_odd", kind="linear", tokens=517, ins=1001, outs=777, act="gelu",
             bias=True, residual=True, train=True, checkpoint="none", dtype="fp32"),
        # the feed-forward block of one token being decoded
        dict(name="mlp_token", kind="mlp", tokens=1, hidden=2048, inter=6144, residual=True,
             train=False, checkpoint="none", dtype="bf16"),
        # a full training batch
        dict(name="mlp_train", kind="mlp", tokens=8192, hidden=2048, inter=6144, residual=False,
             train=True, checkpoint="none", dtype="bf16"),
        # a ragged training batch, gate and up kept in 8 bits
        dict(name="mlp_ragged_fp8", kind="mlp", tokens=1777, hidden=2048, inter=6144,
             residual=True, train=True, checkpoint="fp8", dtype="bf16"),
        # a short prompt through a small model kept in fp16
        dict(name="mlp_fp16_short", kind="mlp", tokens=37, hidden=1024, inter=2816, residual=False,
             train=False, checkpoint="none", dtype="fp16"),
        # the activation of a full training batch, its inputs kept in 8 bits
        dict(name="swiglu_fp8", kind="swiglu", rows=8192, cols=6144, checkpoint="fp8",
             dtype="bf16"),
        # a ragged batch of an odd width in fp32
        dict(name="swiglu_fp8_fp32_odd", kind="swiglu", rows=1777, cols=1001, checkpoint="fp8",
             dtype="fp32"),
        # a few tokens in fp16
        dict(name="swiglu_fp8_fp16_short", kind="swiglu", rows=37, cols=6144, checkpoint="fp8",
             dtype="fp16"),
    ]


def _log_int(rng, lo, hi):
    """An integer spread over the logarithm of [lo, hi]."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, lo, hi):
    """A feature size: a multiple of 64, of 8 or any, spread over the logarithm."""
    step = rng.choice([64, 64, 8, 1])
    return step * _log_int(rng, max(1, lo // step), hi // step)


def draw(rng):
    kind = rng.choice(["linear", "linear", "linear", "mlp", "mlp", "swiglu"])
    if kind == "swiglu":
        return dict(kind=kind, rows=_log_int(rng, 1, 8192), cols=_width(rng, 7, 6144),
                    checkpoint="fp8", dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]))
    dtype = rng.choice(["bf16", "bf16", "bf16", "bf16", "fp16", "fp32"])
    train = rng.random() < 0.7
    tokens = _log_int(rng, 1, 8192 if dtype == "bf16" else 1024)
    held = "fp8" if train and dtype == "bf16" and rng.random() < 0.4 else "none"
    if kind == "mlp":
        return dict(kind=kind, tokens=tokens, hidden=_width(rng, 72, 2048),
                    inter=_width(rng, 72, 6144), residual=rng.random() < 0.5, train=train,
                    checkpoint=held, dtype=dtype)
    act = rng.choice(["none", "silu", "gelu", "gelu_tanh"])
    return dict(kind=kind, tokens=tokens, ins=_width(rng, 72, 4352), outs=_width(rng, 72, 4352),
                act=act, bias=rng.random() < 0.7, residual=rng.random() < 0.5, train=train,
                checkpoint="none" if act == "none" else held, dtype=dtype)


def work(case):
    size = torch.empty((), dtype=DTYPES[case["dtype"]]).element_size()
    if case["kind"] == "swiglu":
        n = case["rows"] * case["cols"]
        # gate, up, dh read and h, dgate, dup written; the 8 bits written and read
        held = 2 * (n + case["rows"] * -(-case["cols"] // BLOCK))
        return {"bytes": 6 * n * size + 2 * held, "flops": 20 * n}
    n, train = case["tokens"], case["train"]
    passes = 2 if train else 1
    if case["kind"] == "mlp":
        h, i = case["hidden"], case["inter"]
        weights, inner = 3 * h * i, 2 * n * i
        moved = 2 * n * h + (n * h if case["residual"] else 0) + weights
        flops = 6 * n * h * i
        if train:
            moved += 2 * n * h + weights  # dy, dx; the weights' gradients
    else:
        i, o = case["ins"], case["outs"]
        weights, inner = i * o, n * o if case["act"] != "none" else 0
        moved = n * i + n * o + (n * o if case["residual"] else 0) + weights
        moved += o if case["bias"] else 0
        flops = 2 * n * i * o
        if train:
            moved += n * o + n * i + weights + (o if case["bias"] else 0)
    if train:
        flops *= 3
        moved *= size
        # what the backward needs of the forward, written and read
        moved += passes * (inner * 33 // 32 if case["checkpoint"] == "fp8" else inner * size)
        return {"bytes": moved, "flops": flops}
    return {"bytes": moved * size, "flops": flops}


# ------------------------------------------------------------------ the inputs

class _Rng:
    """Tensors drawn on the GPU from one seed."""

    def __init__(self, seed):
        self.g = torch.Generator(device=DEV).manual_seed(seed)

    def normal(self, shape, dtype, std=1.0):
        t = torch.empty(shape, dtype=torch.float32, device=DEV).normal_(0.0, std, generator=self.g)
        return t.to(dtype)

    def features(self, shape, dtype):
        """Activations whose features differ in size, as those of a model do."""
        scale = torch.exp(self.normal((shape[-1],), torch.float32, 0.5))
        return (self.normal(shape, torch.float32) * scale).to(dtype)


def prepare(case, seed):
    rng, dtype = _Rng(seed), DTYPES[case["dtype"]]
    s = dict(case=case, res=None, bias=None)
    if case["kind"] == "swiglu":
        shape = (case["rows"], case["cols"])
        s["gate"] = rng.features(shape, dtype).requires_grad_()
        s["up"] = rng.features(shape, dtype).requires_grad_()
        s["dy"] = rng.normal(shape, dtype)
        return s
    train = case["train"]
    if case["kind"] == "mlp":
        h, i = case["hidden"], case["inter"]
        s["x"] = rng.normal((case["tokens"], h), dtype)
        s["weights"] = [rng.normal((i, h), dtype, h ** -0.5), rng.normal((i, h), dtype, h ** -0.5),
                        rng.normal((h, i), dtype, i ** -0.5)]
        out = (case["tokens"], h)
    else:
        s["x"] = rng.normal((case["tokens"], case["ins"]), dtype)
        s["weights"] = [rng.normal((case["outs"], case["ins"]), dtype, case["ins"] ** -0.5)]
        out = (case["tokens"], case["outs"])
        s["bias"] = rng.normal(out[1:], dtype, 0.1) if case["bias"] else None
    s["res"] = rng.normal(out, dtype) if case["residual"] else None
    s["dy"] = rng.normal(out, dtype) if train else None
    for t in _inputs(s):
        t.requires_grad_(train)
    return s


def _inputs(s):
    """What gradients are taken of."""
    if s["case"]["kind"] == "swiglu":
        return [s["gate"], s["up"]]
    return [t for t in (s["x"], *s["weights"], s["bias"], s["res"]) if t is not None]


# ------------------------------------------------------------- the plain forms

def _held(v, checkpoint):
    """v [rows, cols] in 32 bits as the backward reads it."""
    if checkpoint != "fp8":
        return v
    rows, cols = v.shape
    n = -(-cols // BLOCK)
    b = torch.nn.functional.pad(v, (0, n * BLOCK - cols)).view(rows, n, BLOCK)
    finite = torch.isfinite(b)
    m = torch.where(finite, b.abs(), torch.zeros_like(b)).amax(-1, keepdim=True)
    e = torch.where(m > 0, torch.frexp(m).exponent - 8, -126).clamp_min(-126)  # m = f 2^k, f >= 1/2
    scale = torch.exp2(e.float())
    q = torch.where(finite, b / scale, torch.full_like(b, math.nan))
    q = q.to(torch.float8_e4m3fn).float() * scale
    return q.view(rows, n * BLOCK)[:, :cols]


def _act(z, act):
    """act(z) and act'(z)."""
    if act == "none":
        return z, torch.ones_like(z)
    if act == "silu":
        s = 1.0 / (1.0 + torch.exp(-z))
        return z * s, s * (1.0 + z * (1.0 - s))
    if act == "gelu":
        c = 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5)))
        return z * c, c + z * torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)
    r = math.sqrt(2.0 / math.pi)
    t = torch.tanh(r * (z + 0.044715 * z * z * z))
    return 0.5 * z * (1.0 + t), \
        0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * r * (1.0 + 3 * 0.044715 * z * z)


def _plain_swiglu(s):
    g, u, dh = (s[k].detach().float() for k in ("gate", "up", "dy"))
    h = _act(g, "silu")[0] * u
    g, u = _held(g, "fp8"), _held(u, "fp8")
    a, d = _act(g, "silu")
    return [h, dh * u * d, dh * a]


def _plain_linear(s):
    case, x, w = s["case"], s["x"].detach().float(), s["weights"][0].detach().float()
    z = x @ w.t()
    if s["bias"] is not None:
        z = z + s["bias"].detach().float()
    y = _act(z, case["act"])[0]
    if s["res"] is not None:
        y = y + s["res"].detach().float()
    if not case["train"]:
        return [y]
    dy = s["dy"].float()
    dz = dy
    if case["act"] != "none":
        dz = dy * _act(_held(z, case["checkpoint"]), case["act"])[1]
    out = [y, dz @ w, dz.t() @ x]
    if s["bias"] is not None:
        out.append(dz.sum(0))
    return out if s["res"] is None else [*out, dy]


def _plain_mlp(s):
    case, x = s["case"], s["x"].detach().float()
    wg, wu, wd = (w.detach().float() for w in s["weights"])
    g, u = x @ wg.t(), x @ wu.t()
    y = (_act(g, "silu")[0] * u) @ wd.t()
    if s["res"] is not None:
        y = y + s["res"].detach().float()
    if not case["train"]:
        return [y]
    dy = s["dy"].float()
    g, u = _held(g, case["checkpoint"]), _held(u, case["checkpoint"])
    a, d = _act(g, "silu")
    dh = dy @ wd
    dg, du = dh * u * d, dh * a
    out = [y, dg @ wg + du @ wu, dg.t() @ x, du.t() @ x, dy.t() @ (a * u)]
    return out if s["res"] is None else [*out, dy]


# ------------------------------------------------------------------- one pass

PLAIN = {"linear": _plain_linear, "mlp": _plain_mlp, "swiglu": _plain_swiglu}


def run(s):
    if own:
        return _run_own(s)
    return [t.to(DTYPES[s["case"]["dtype"]]) for t in PLAIN[s["case"]["kind"]](s)]


def _call(s):
    from metal_liger_amd.ops.fused_linear import fused_linear
    from metal_liger_amd.ops.fused_swiglu import fused_swiglu
    from metal_liger_amd.ops.fused_swiglu_mlp import fused_swiglu_mlp
    case = s["case"]
    held = None if case["checkpoint"] == "none" else case["checkpoint"]
    if case["kind"] == "swiglu":
        return fused_swiglu(s["gate"], s["up"], checkpoint=held)
    if case["kind"] == "mlp":
        return fused_swiglu_mlp(s["x"], *s["weights"], residual=s["res"], checkpoint=held)
    act = None if case["act"] == "none" else case["act"]
    return fused_linear(s["x"], s["weights"][0], s["bias"], activation=act, residual=s["res"],
                        checkpoint=held)


def _run_own(s):
    if s["dy"] is None:
        with torch.no_grad():
            return [_call(s)]
    y = _call(s)
    return [y, *torch.autograd.grad(y, _inputs(s), s["dy"])]


# ------------------------------------------------------------------ in 64 bits

def _held64(v):
    """v as 8 bits hold it, rounded by hand."""
    out = torch.empty_like(v)
    for c in range(0, v.shape[1], BLOCK):
        b = v[:, c:c + BLOCK]
        m = torch.nan_to_num(b.abs(), nan=0.0, posinf=0.0).max(1, keepdim=True).values
        e = torch.where(m > 0, torch.floor(torch.log2(m.clamp_min(1e-300))) - 7, -126.0)
        # log2 may round up to a whole number just below one
        e = torch.where((m > 0) & (torch.exp2(e + 7) > m), e - 1, e).clamp_min(-126.0)
        q = b / torch.exp2(e)
        k = torch.floor(torch.log2(q.abs().clamp_min(2.0 ** -6)))
        k = torch.where(torch.exp2(k) > q.abs().clamp_min(2.0 ** -6), k - 1, k)
        step = torch.exp2(k - 3)
        q = torch.round(q / step) * step
        out[:, c:c + BLOCK] = torch.where(torch.isfinite(b), q * torch.exp2(e), math.nan)
    return out


class _Held64(torch.autograd.Function):
    """act(z), whose derivative is taken at z as it was held."""

    @staticmethod
    def forward(ctx, z, act, checkpoint):
        ctx.act = act
        ctx.save_for_backward(_held64(z) if checkpoint == "fp8" else z)
        return act(z)

    @staticmethod
    def backward(ctx, dy):
        with torch.enable_grad():
            z = ctx.saved_tensors[0].detach().requires_grad_()
            return torch.autograd.grad(ctx.act(z), z, dy)[0], None, None


ACT64 = {"none": lambda z: z * 1.0, "silu": lambda z: z * torch.sigmoid(z),
         "gelu": lambda z: z * torch.special.ndtr(z),
         "gelu_tanh": lambda z: z * torch.sigmoid(2 * math.sqrt(2 / math.pi)
                                                  * (z + 0.044715 * z ** 3))}


def _gated64(g, u, checkpoint, dh):
    """(dg, du, h) of the backward."""
    g, u = ((_held64(t) if checkpoint == "fp8" else t).detach().requires_grad_() for t in (g, u))
    h = ACT64["silu"](g) * u
    return [*torch.autograd.grad(h, [g, u], dh), h.detach()]


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "swiglu":
        g, u, dh = (s[k].detach().double() for k in ("gate", "up", "dy"))
        return [ACT64["silu"](g) * u, *_gated64(g, u, "fp8", dh)[:2]]
    double = [t.detach().double().requires_grad_(case["train"]) for t in _inputs(s)]
    x, rest = double[0], double[1:]
    dy = s["dy"].double() if case["train"] else None
    if case["kind"] == "linear":
        z = x @ rest[0].t()
        if case["bias"]:
            z = z + rest[1]
        y = _Held64.apply(z, ACT64[case["act"]], case["checkpoint"])
        if case["residual"]:
            y = y + rest[-1]
        return [y.detach(), *(torch.autograd.grad(y, double, dy) if case["train"] else [])]
    with torch.no_grad():
        wg, wu, wd = rest[:3]
        g, u = x @ wg.t(), x @ wu.t()
        y = (ACT64["silu"](g) * u) @ wd.t()
        if case["residual"]:
            y = y + rest[3]
    if not case["train"]:
        return [y]
    dg, du, h = _gated64(g, u, case["checkpoint"], dy @ wd.detach())
    with torch.no_grad():
        out = [y, dg @ wg + du @ wu, dg.t() @ x, du.t() @ x, dy.t() @ h]
    return [*out, dy] if case["residual"] else out

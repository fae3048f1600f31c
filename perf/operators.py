"""The work whose speed is measured for dropout, the LoRA projections with
dropout on the adapters' input, and the token embedding with its gradient: one
pass each, forward + backward (a frozen embedding: forward), through the
framework's entry points (``own``) or in plain tensor operations.

The sizes are those of the workloads that this repository is built around (a
Qwen3-style text model: hidden 2048, 16 / 8 heads of 128, MLP 6144, vocabulary
151936, rank-16 adapters, 4 x 2048 tokens) and of what users of the same entry
points bring besides: short prompts, ragged batches, odd widths, fp32 models.

The definitions, of which both forms are computed:

  dropout    with T = round(65536 p) and q = T / 65536, element i of x in row-major
             order is kept where its random number of 16 bits is at least T:
             y_i = x_i / (1 - q), else 0 (+ residual_i). The number is the
             (i mod 8)-th 16-bit part, low halves first, of the four words that
             seven rounds of Philox4x32 (Salmon et al., "Parallel random numbers:
             as easy as 1, 2, 3", 2011) make of the counter (i div 8, stream, 0)
             and the 64-bit seed as key. The gradient passes through the same mask.
  lora       y = X W^T + s (drop(X) A^T) B^T, projection j of a block on stream j of
             its seed (q, k, v: 0, 1, 2; gate, up, down: 0, 1, 2).
  embedding  y_n = s W[id_n]; dW[v] = s times the sum of dy_n over the n with id_n = v,
             0 for the row of padding_idx.
"""

import math

import numpy as np
import torch
import torch.nn as nn

own = False

DEV = "cuda"
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
M32 = 0xFFFFFFFF


# ------------------------------------------------------------------ the cases

def listed():
    return [
        # the embedding output of one token, as an adapter's input is dropped in a
        # step of one token: launches and host time count
        dict(name="dropout_token", kind="dropout", rows=1, cols=2048, p=0.1, dtype="bf16",
             residual=False),
        # the hidden states of 4 x 2048 tokens
        dict(name="dropout_bf16", kind="dropout", rows=8192, cols=2048, p=0.1, dtype="bf16",
             residual=False),
        # a ragged batch of an odd width in fp32, added to its residual
        dict(name="dropout_residual_fp32_odd", kind="dropout", rows=3333, cols=1001, p=0.05,
             dtype="fp32", residual=True),
        # the MLP's inner activations, added to a residual
        dict(name="dropout_residual_bf16_wide", kind="dropout", rows=8192, cols=6144, p=0.2,
             dtype="bf16", residual=True),
        # an output projection of a short prompt, PEFT's default rank
        dict(name="lora_dropout_linear_short", kind="linear", tokens=37, hidden=1024, out=1024,
             rank=8, p=0.1, dtype="bf16"),
        # the q, k, v projections of a full training batch
        dict(name="lora_dropout_qkv", kind="qkv", tokens=8192, hidden=2048, q_out=2048, kv_out=1024,
             rank=16, p=0.05, dtype="bf16"),
        # the MLP block of a ragged batch, a larger rank
        dict(name="lora_dropout_mlp_ragged", kind="mlp", tokens=1777, hidden=2048, inter=6144,
             rank=32, p=0.1, dtype="bf16"),
        # an output projection of a model kept in fp32
        dict(name="lora_dropout_linear_fp32", kind="linear", tokens=1000, hidden=2048, out=2048,
             rank=16, p=0.05, dtype="fp32"),
        # the frozen embedding of a LoRA run, a tiny model and a short prompt
        dict(name="embedding_frozen_tiny", kind="embedding", train=False, tokens=16, vocab=512,
             hidden=128, scale=math.sqrt(128), same=0.0, pad=False, dtype="bf16"),
        # the trained embedding of the text model, 4 x 2048 tokens of text
        dict(name="embedding_train", kind="embedding", train=True, tokens=8192, vocab=151936,
             hidden=2048, scale=1.0, same=0.0, pad=False, dtype="bf16"),
        # image and text: most positions hold the image's token
        dict(name="embedding_image", kind="embedding", train=True, tokens=16384, vocab=151936,
             hidden=2048, scale=1.0, same=0.7, pad=False, dtype="bf16"),
        # an odd vocabulary and width in fp32, scaled, padded batch
        dict(name="embedding_fp32_odd", kind="embedding", train=True, tokens=3001, vocab=64007,
             hidden=1001, scale=math.sqrt(1001), same=0.3, pad=True, dtype="fp32"),
    ]


def _log_int(rng, lo, hi):
    """An integer spread over the logarithm of [lo, hi]."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, lo, hi, step=64):
    """A feature size: a multiple of `step`, spread over the logarithm."""
    return step * _log_int(rng, max(1, lo // step), hi // step)


def draw(rng):
    kind = rng.choice(["dropout", "dropout", "linear", "qkv", "mlp", "embedding", "embedding"])
    p = round(rng.uniform(0.01, 0.5), 3)
    if kind == "dropout":
        cols = _width(rng, 64, 6144) if rng.random() < 0.6 else _log_int(rng, 7, 6144)
        return dict(kind=kind, rows=_log_int(rng, 1, 8192), cols=cols, p=p,
                    dtype=rng.choice(["bf16", "bf16", "fp16"]), residual=rng.random() < 0.5)
    if kind == "embedding":
        train = rng.random() < 0.6  # the tables that are trained are those of whole models
        low = 1024 if train else 7
        hidden = _width(rng, max(low, 64), 2048) if rng.random() < 0.6 else _log_int(rng, low, 2048)
        return dict(kind=kind, train=train, tokens=_log_int(rng, 1, 16384),
                    vocab=_log_int(rng, 32000 if train else 100, 151936), hidden=hidden, scale=rng.choice([1.0, math.sqrt(hidden)]),
                    same=rng.choice([0.0, 0.3, 0.7, 1.0]), pad=rng.random() < 0.3,
                    dtype=rng.choice(["bf16", "bf16", "fp16"]))
    tokens = _log_int(rng, 1, 8192)
    if kind == "qkv":
        kv = _width(rng, 128, 1024)
        return dict(kind=kind, tokens=tokens, hidden=_width(rng, 256, 2048),
                    q_out=kv * rng.choice([1, 2]), kv_out=kv, rank=rng.choice([4, 8, 16, 32, 64]),
                    p=p, dtype="bf16")
    if kind == "mlp":
        return dict(kind=kind, tokens=min(tokens, 2048), hidden=_width(rng, 256, 2048),
                    inter=_width(rng, 512, 6144), rank=rng.choice([4, 8, 16, 32, 64]), p=p,
                    dtype="bf16")
    dtype = rng.choice(["fp32", "bf16"])
    step = 64 if rng.random() < 0.75 else 1
    return dict(kind=kind, tokens=tokens if dtype == "bf16" else min(tokens, 2048),
                hidden=_width(rng, 72, 2048, step), out=_width(rng, 72, 2048, step),
                rank=rng.choice([4, 8, 12, 16, 32]), p=p, dtype=dtype)


def _projections(case):
    """(name, in features, out features) of a LoRA block's projections."""
    h = case["hidden"]
    if case["kind"] == "qkv":
        return [("q_proj", h, case["q_out"]), ("k_proj", h, case["kv_out"]),
                ("v_proj", h, case["kv_out"])]
    if case["kind"] == "mlp":
        return [("gate_proj", h, case["inter"]), ("up_proj", h, case["inter"]),
                ("down_proj", case["inter"], h)]
    return [("o_proj", h, case["out"])]


def work(case):
    size = torch.empty((), dtype=DTYPES[case["dtype"]]).element_size()
    if case["kind"] == "dropout":
        n = case["rows"] * case["cols"]
        return {"bytes": n * size * (5 if case["residual"] else 4), "flops": 2 * n}
    if case["kind"] == "embedding":
        n, v, h = case["tokens"], case["vocab"], case["hidden"]
        rows = min(n, v)  # rows of the table that the tokens can name
        moved, flops = (rows * h + n * h) * size + 8 * n, n * h
        if case["train"]:
            moved, flops = moved + (n * h + v * h) * size + 8 * n, 2 * flops
        return {"bytes": moved, "flops": flops}
    n, r = case["tokens"], case["rank"]
    moved = flops = 0
    for _, i, o in _projections(case):
        moved += i * o + 2 * r * (i + o)  # W once; A, B and their gradients
        flops += 4 * n * i * o + 6 * n * r * (i + o)
    if case["kind"] == "mlp":  # x, y, dy, dx; gate, up and h stay inside
        moved += 4 * n * case["hidden"]
    else:
        moved += 2 * n * case["hidden"] + 2 * n * sum(o for _, _, o in _projections(case))
    return {"bytes": moved * size, "flops": flops}


# ------------------------------------------------------------------ the inputs

class _Rng:
    """Tensors drawn on the GPU from one seed."""

    def __init__(self, seed):
        self.g = torch.Generator(device=DEV).manual_seed(seed)

    def normal(self, shape, dtype, std=1.0):
        t = torch.empty(shape, dtype=torch.float32, device=DEV).normal_(0.0, std, generator=self.g)
        return t.to(dtype)

    def uniform(self, shape, dtype, bound):
        t = torch.empty(shape, dtype=torch.float32, device=DEV)
        return t.uniform_(-bound, bound, generator=self.g).to(dtype)

    def seed(self):
        """A dropout seed, on the GPU as a captured step needs it."""
        return torch.randint(0, 2 ** 62, (1,), generator=self.g, device=DEV)

    def tokens(self, n, vocab):
        """Ids as text has them: the logarithm of the rank evenly spread."""
        u = torch.rand((n,), generator=self.g, device=DEV, dtype=torch.float64)
        return (torch.exp(u * math.log(vocab)).long() - 1).clamp_(0, vocab - 1)

    def positions(self, n, share):
        return torch.rand((n,), generator=self.g, device=DEV) < share


class _LoraLinear(nn.Module):
    """A frozen linear layer with one adapter, laid out as PEFT lays it out:
    A uniform as nn.Linear's default, B as after some training, alpha = 2 r."""

    def __init__(self, rng, in_f, out_f, rank, p, dtype):
        super().__init__()
        self.base_layer = nn.Module()
        self.base_layer.weight = nn.Parameter(rng.normal((out_f, in_f), dtype, 0.02), False)
        a, b = nn.Module(), nn.Module()
        a.weight = nn.Parameter(rng.uniform((rank, in_f), dtype, in_f ** -0.5))
        b.weight = nn.Parameter(rng.normal((out_f, rank), dtype, 0.02))
        self.lora_A, self.lora_B = nn.ModuleDict({"default": a}), nn.ModuleDict({"default": b})
        self.lora_dropout = nn.ModuleDict({"default": nn.Dropout(p)})
        self.scaling = {"default": 2.0}

    def parts(self):
        return (self.base_layer.weight, self.lora_A["default"].weight,
                self.lora_B["default"].weight, self.scaling["default"],
                self.lora_dropout["default"].p)


def _adapters(block):
    return [t for m in block.children() for t in m.parts()[1:3]]


def prepare(case, seed):
    rng, dtype = _Rng(seed), DTYPES[case["dtype"]]
    s = dict(case=case)
    if case["kind"] == "dropout":
        shape = (case["rows"], case["cols"])
        s["x"] = rng.normal(shape, dtype).requires_grad_()
        s["res"] = rng.normal(shape, dtype).requires_grad_() if case["residual"] else None
        s["dy"] = rng.normal(shape, dtype)
        s["seed"] = rng.seed()
    elif case["kind"] == "embedding":
        n, v, h = case["tokens"], case["vocab"], case["hidden"]
        s["weight"] = rng.normal((v, h), dtype, 0.02).requires_grad_(case["train"])
        ids = rng.tokens(n, v)
        s["ids"] = torch.where(rng.positions(n, case["same"]), v // 2, ids)
        s["pad"] = None
        if case["pad"]:  # the end of a padded batch
            s["pad"] = v - 1
            s["ids"][n - n // 8:] = v - 1
        s["dy"] = rng.normal((n, h), dtype) if case["train"] else None
    else:
        s["block"] = nn.Module()
        for name, i, o in _projections(case):
            setattr(s["block"], name, _LoraLinear(rng, i, o, case["rank"], case["p"], dtype))
        s["x"] = rng.normal((case["tokens"], case["hidden"]), dtype).requires_grad_()
        outs = [o for _, _, o in _projections(case)]
        s["dy"] = [rng.normal((case["tokens"], o), dtype)
                   for o in (outs[-1:] if case["kind"] == "mlp" else outs)]
        s["seed"] = rng.seed()
    return s


# ------------------------------------------------------------- the plain forms

def _threshold(p):
    return min(65536, int(math.floor(p * 65536 + 0.5)))


def _drop_scale(p):
    t = _threshold(p)
    return 65536.0 / (65536 - t) if t < 65536 else 0.0


def _factors(x, p, seed, stream):
    """1 / (1 - q) where x's elements are kept and 0 where not, in 32 bits."""
    n = x.numel()
    i = torch.arange((n + 7) // 8, device=x.device)
    a, b, c, d = i & M32, i >> 32, torch.full_like(i, stream), torch.zeros_like(i)
    k, m = seed & M32, (seed >> 32) & M32
    for _ in range(7):
        u, v = a * 0xD2511F53, c * 0xCD9E8D57  # of 64 bits, which wrap as unsigned ones do
        a, b, c, d = ((v >> 32) & M32) ^ b ^ k, v & M32, ((u >> 32) & M32) ^ d ^ m, u & M32
        k, m = (k + 0x9E3779B9) & M32, (m + 0xBB67AE85) & M32
    w = torch.stack((a, b, c, d), 1)
    u16 = torch.stack((w & 0xFFFF, w >> 16), 2).view(-1)[:n]
    return ((u16 >= _threshold(p)).float() * _drop_scale(p)).view(x.shape)


def _plain_dropout(s):
    x, res, dy = s["x"].detach(), s["res"], s["dy"]
    f = _factors(x, s["case"]["p"], s["seed"], 0)
    y, dx = x.float() * f, (dy.float() * f).to(x.dtype)
    if res is None:
        return [y.to(x.dtype), dx]
    return [(y + res.detach().float()).to(x.dtype), dx, dy]


def _plain_embedding(s):
    w, ids, dy = s["weight"].detach(), s["ids"], s["dy"]
    scale = s["case"]["scale"]
    y = (w[ids].float() * scale).to(w.dtype)
    if dy is None:
        return [y]
    dw = torch.zeros(w.shape, dtype=torch.float32, device=w.device)
    dw.index_add_(0, ids, dy.float())
    if s["pad"] is not None:
        dw[s["pad"]] = 0.0
    return [y, (dw * scale).to(w.dtype)]


def _plain_lora(linear, x, seed, stream):
    """The output, and what the gradient needs of it; x and all else in 32 bits."""
    w, a, b, scale, p = linear.parts()
    f = _factors(x, p, seed, stream)
    w, a, b = w.float(), a.detach().float(), b.detach().float()
    xa = (x * f) @ a.t()
    return x @ w.t() + scale * (xa @ b.t()), (x, f, w, a, b, scale, xa)


def _plain_lora_grad(saved, dy):
    x, f, w, a, b, scale, xa = saved
    q = scale * (dy @ b)
    return dy @ w + (q @ a) * f, q.t() @ (x * f), scale * (dy.t() @ xa)


def _plain_qkv(s):
    x, dys = s["x"].detach().float(), [t.float() for t in s["dy"]]
    outs, saved = zip(*(_plain_lora(m, x, s["seed"], j)
                        for j, m in enumerate(s["block"].children())))
    grads = [_plain_lora_grad(k, dy) for k, dy in zip(saved, dys)]
    return [*outs, sum(g[0] for g in grads), *(t for g in grads for t in g[1:])]


def _plain_mlp(s):
    x, dy = s["x"].detach().float(), s["dy"][0].float()
    gate_proj, up_proj, down_proj = s["block"].children()
    gate, saved_g = _plain_lora(gate_proj, x, s["seed"], 0)
    up, saved_u = _plain_lora(up_proj, x, s["seed"], 1)
    sig = 1.0 / (1.0 + torch.exp(-gate))
    y, saved_d = _plain_lora(down_proj, gate * sig * up, s["seed"], 2)
    dh, *grads_d = _plain_lora_grad(saved_d, dy)
    dx_u, *grads_u = _plain_lora_grad(saved_u, dh * gate * sig)
    dx_g, *grads_g = _plain_lora_grad(saved_g, dh * up * sig * (1.0 + gate * (1.0 - sig)))
    return [y, dx_g + dx_u, *grads_g, *grads_u, *grads_d]


# ------------------------------------------------------------------- one pass

def run(s):
    kind = s["case"]["kind"]
    if own:
        return _run_own(s, kind)
    if kind == "dropout":
        return _plain_dropout(s)
    if kind == "embedding":
        return _plain_embedding(s)
    out = _plain_mlp(s) if kind == "mlp" else _plain_qkv(s)
    return [t.to(s["x"].dtype) for t in out]


def _run_own(s, kind):
    from metal_liger_amd.ops.fused_dropout import fused_dropout
    from metal_liger_amd.ops.fused_embedding import fused_embedding
    from metal_liger_amd.ops.fused_lora import (apply_fused_lora_linear, apply_fused_lora_mlp,
                                                apply_fused_lora_qkv)
    grad = torch.autograd.grad
    if kind == "dropout":
        y = fused_dropout(s["x"], s["case"]["p"], residual=s["res"], seed=s["seed"])
        return [y, *grad(y, [s["x"]] if s["res"] is None else [s["x"], s["res"]], s["dy"])]
    if kind == "embedding":
        y = fused_embedding(s["ids"], s["weight"], scale=s["case"]["scale"], padding_idx=s["pad"])
        return [y, *grad(y, [s["weight"]], s["dy"])] if s["case"]["train"] else [y]
    block, x = s["block"], s["x"]
    if kind == "qkv":
        outs = list(apply_fused_lora_qkv(block, x, lora_dropout=True, seed=s["seed"]))
    elif kind == "mlp":
        outs = [apply_fused_lora_mlp(block, x, lora_dropout=True, seed=s["seed"])]
    else:
        outs = [apply_fused_lora_linear(block.o_proj, x, lora_dropout=True, seed=s["seed"])]
    return [*outs, *grad(outs, [x, *_adapters(block)], s["dy"])]


# ------------------------------------------------------------------ in 64 bits

def _mask64(shape, p, seed, stream):
    """Dropout's factors in 64 bits, from numpy's unsigned integers."""
    n = int(np.prod(shape))
    mask = np.uint64(M32)
    blocks = np.arange((n + 7) // 8, dtype=np.uint64)
    ctr = [blocks & mask, blocks >> np.uint64(32), np.full_like(blocks, stream),
           np.zeros_like(blocks)]
    key = [int(seed) & M32, (int(seed) >> 32) & M32]
    for _ in range(7):
        lo_a, lo_c = ctr[0] * np.uint64(0xD2511F53), ctr[2] * np.uint64(0xCD9E8D57)
        ctr = [(lo_c >> np.uint64(32)) ^ ctr[1] ^ np.uint64(key[0]), lo_c & mask,
               (lo_a >> np.uint64(32)) ^ ctr[3] ^ np.uint64(key[1]), lo_a & mask]
        key = [(key[0] + 0x9E3779B9) & M32, (key[1] + 0xBB67AE85) & M32]
    numbers = np.stack(ctr, 1).astype("<u4").view("<u2").reshape(-1)[:n]
    limit = min(65536, int(math.floor(p * 65536 + 0.5)))
    rate = limit / 65536
    factors = np.where(numbers >= limit, 1.0 / (1.0 - rate) if rate < 1 else 0.0, 0.0)
    return torch.from_numpy(factors.reshape(shape)).to(DEV)


def _lora64(linear, x, seed, stream, leaves):
    w, a, b, scale, p = linear.parts()
    a, b = (t.detach().double().requires_grad_() for t in (a, b))
    leaves += [a, b]
    dropped = x * _mask64(tuple(x.shape), p, seed, stream)
    return x @ w.double().t() + scale * (dropped @ a.t()) @ b.t()


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "dropout":
        f = _mask64((case["rows"], case["cols"]), case["p"], s["seed"].item(), 0)
        y, dx = s["x"].detach().double() * f, s["dy"].double() * f
        if not case["residual"]:
            return [y, dx]
        return [y + s["res"].detach().double(), dx, s["dy"].double()]
    if case["kind"] == "embedding":
        w = s["weight"].detach().double().mul_(case["scale"])
        y = w[s["ids"]]
        if not case["train"]:
            return [y]
        dw = w.zero_()
        keep = s["ids"] != (-1 if s["pad"] is None else s["pad"])
        dw.index_put_((s["ids"][keep],), s["dy"][keep].double(), accumulate=True)
        return [y, dw.mul_(case["scale"])]
    x, leaves, key = s["x"].detach().double().requires_grad_(), [], s["seed"].item()
    if case["kind"] == "mlp":
        gate_proj, up_proj, down_proj = s["block"].children()
        gate, up = _lora64(gate_proj, x, key, 0, leaves), _lora64(up_proj, x, key, 1, leaves)
        outs = [_lora64(down_proj, gate * torch.sigmoid(gate) * up, key, 2, leaves)]
    else:
        outs = [_lora64(m, x, key, j, leaves) for j, m in enumerate(s["block"].children())]
    grads = torch.autograd.grad(outs, [x, *leaves], [t.double() for t in s["dy"]])
    return [*(o.detach() for o in outs), *grads]

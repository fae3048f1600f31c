"""The feed-forward operators in 64 bits on the CPU: tensors held in 8 bits, the linear
layer with activation and residual, the gated block, and their gradients by formula.
(Parity unpinned: the reference has none of them.)"""

import math

import torch

BLOCK = 32


def held_exponents(v):
    """e of each block of 32 along the last dimension: max(floor(log2 m) - 7, -126) for
    the largest finite magnitude m, -126 where that is 0. [..., ceil(n / 32)] integers."""
    v = v.double()
    n = v.shape[-1]
    pad = torch.nn.functional.pad(v, (0, -n % BLOCK))
    m = pad.unflatten(-1, (-1, BLOCK)).abs()
    m = torch.where(torch.isfinite(m), m, torch.zeros_like(m)).amax(-1)
    k = torch.frexp(m).exponent.long() - 1          # floor(log2 m)
    return torch.where(m > 0, k - 7, torch.full_like(k, -126)).clamp_min(-126)


def held_bytes(v):
    """(bytes, scale bytes) as the kernels write them, for finite or other v."""
    v, e = v.double(), held_exponents(v)
    s = torch.ldexp(torch.ones((), dtype=torch.float64), e).repeat_interleave(BLOCK, -1)
    q = v / s[..., :v.shape[-1]]
    a = torch.nan_to_num(q.abs(), nan=0.0, posinf=0.0)
    k = (torch.frexp(a).exponent.long() - 1).clamp_min(-6)   # octave, subnormal below 2^-6
    step = torch.ldexp(torch.ones((), dtype=torch.float64), k - 3)
    r = torch.round(a / step)                                # ties to even
    up = r == 16                                             # rounded into the next octave
    k, r = torch.where(up, k + 1, k), torch.where(up, torch.full_like(r, 8.0), r)
    normal = r >= 8
    code = torch.where(normal, (k + 7) * 8 + (r.long() - 8), r.long())
    code = torch.where(torch.isfinite(v), code, torch.full_like(code, 0x7F))
    code = code + 128 * (torch.signbit(v) & torch.isfinite(v)).long()
    return code.to(torch.uint8), (e + 127).to(torch.uint8)


def held_values(codes, scales):
    """What the bytes (or fp16 elements) stand for, in 64 bits."""
    if codes.dtype == torch.float16:
        s = torch.ldexp(torch.ones((), dtype=torch.float64), scales.long() - 127)
        return codes.double() * s.repeat_interleave(BLOCK, -1)[..., :codes.shape[-1]]
    c = codes.long()
    mag, sign = c & 0x7F, 1.0 - 2.0 * (c >> 7).double()
    k, f = mag >> 3, (mag & 7).double()
    one = torch.ones((), dtype=torch.float64)
    val = torch.where(k > 0, torch.ldexp(1 + f / 8, k - 7), f / 8 * torch.ldexp(one, k * 0 - 6))
    val = torch.where(mag == 0x7F, torch.full_like(val, math.nan), val)
    s = torch.ldexp(one, scales.long() - 127).repeat_interleave(BLOCK, -1)
    return sign * val * s[..., :c.shape[-1]]


def act(z, name):
    if name is None:
        return z
    if name == "silu":
        return z * torch.sigmoid(z)
    if name == "gelu":
        return z * torch.special.ndtr(z)
    return z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))


def act_grad(z, name):
    if name is None:
        return torch.ones_like(z)
    if name == "silu":
        s = torch.sigmoid(z)
        return s * (1 + z * (1 - s))
    if name == "gelu":
        return torch.special.ndtr(z) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    c = 2 * math.sqrt(2 / math.pi)
    s = torch.sigmoid(c * (z + 0.044715 * z ** 3))
    return s + z * s * (1 - s) * c * (1 + 3 * 0.044715 * z ** 2)


# The largest |act'| and |act''| of the three activations: 1.1290 (gelu, gelu_tanh) and
# 2 phi(0) = 0.7979 (gelu; gelu_tanh 0.7979, silu 0.5).
ACT_GRAD_MAX, ACT_GRAD2_MAX = 1.13, 0.8

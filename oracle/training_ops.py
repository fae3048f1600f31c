"""CPU restatements, in 64 bits, of the operators that the reference leaves to
torch and this library fuses: dropout from a counter-based generator, LoRA
projections with dropout on the adapters' input, and the token embedding with its
gradient. What the HIP path is tested against.
"""

import numpy as np
import torch

_M32 = np.uint64(0xFFFFFFFF)


def philox4x32(counter, key, rounds):
    """Philox4x32 (Salmon et al., 2011) of counters [n, 4] under the key (k0, k1):
    uint32 words [n, 4]."""
    a, b, c, d = (np.asarray(counter, dtype=np.uint64)[:, i] for i in range(4))
    k0, k1 = key
    for _ in range(rounds):
        u, v = a * np.uint64(0xD2511F53), c * np.uint64(0xCD9E8D57)
        a, b, c, d = ((v >> np.uint64(32)) ^ b ^ np.uint64(k0), v & _M32,
                      (u >> np.uint64(32)) ^ d ^ np.uint64(k1), u & _M32)
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return np.stack([a, b, c, d], 1).astype(np.uint32)


def dropout_threshold(p):
    return int(np.floor(p * 65536 + 0.5))


def dropout_factors(shape, p, seed, stream=0, first=0):
    """65536 / (65536 - T) where an element is kept and 0 where it is dropped, for
    elements first .. of a tensor in row-major order."""
    n = int(np.prod(shape))
    low, high = first // 8, (first + n + 7) // 8
    blocks = np.arange(low, high, dtype=np.uint64)
    counter = np.stack([blocks & _M32, blocks >> np.uint64(32), np.full_like(blocks, stream),
                        np.zeros_like(blocks)], 1)
    seed %= 1 << 64
    words = philox4x32(counter, (seed & 0xFFFFFFFF, seed >> 32), 7)
    numbers = words.astype("<u4").view("<u2").reshape(-1)[first - 8 * low:][:n].astype(np.int64)
    t = dropout_threshold(p)
    f = np.where(numbers >= t, 65536 / (65536 - t) if t < 65536 else 0.0, 0.0)
    return torch.from_numpy(f.reshape(shape))


def lora_dropout(x, params, dys, factors):
    """Outputs and gradients of projections y_i = x W^T + s (f_i x A^T) B^T: params
    [(W, A, B, s)], dys their outputs' gradients, factors f_i (dropout_factors).
    Returns (outs, dx, [(dA, dB)])."""
    x = x.double()
    outs, dx, grads = [], torch.zeros_like(x), []
    for (w, a, b, s), dy, f in zip(params, dys, factors):
        w, a, b, dy = w.double(), a.double(), b.double(), dy.double()
        xd = x * f
        xa, q = xd @ a.t(), s * (dy @ b)
        outs.append(x @ w.t() + s * (xa @ b.t()))
        dx += dy @ w + f * (q @ a)
        grads.append((q.t() @ xd, s * (dy.t() @ xa)))
    return outs, dx, grads


def embedding_grad(ids, dy, vocab, scale=1.0, padding_idx=None):
    """The gradient [vocab, hidden] of scale * table[ids]; ids outside are skipped."""
    ids, dy = ids.reshape(-1), dy.reshape(-1, dy.shape[-1]).double()
    dw = torch.zeros(vocab, dy.shape[-1], dtype=torch.float64)
    keep = (ids >= 0) & (ids < vocab)
    if padding_idx is not None:
        keep &= ids != padding_idx % vocab
    return dw.index_add_(0, ids[keep].long(), dy[keep]).mul_(scale)

"""Fused token embedding on MI355X: the lookup with its scaling, and the gradient
of the table (no counterpart in the reference, whose models keep nn.Embedding).

The gradient sums the tokens' rows in fp32 in an order that the ids and their number
alone decide, so that it is bit-reproducible, and rounds once. Both directions can be
differentiated again; forward mode and torch.func's transforms are refused.
"""

from __future__ import annotations

import torch
import torch.nn as nn

from metal_liger_amd import _custom_ops as cops


class _FusedEmbeddingFunction(torch.autograd.Function):
    """scale * weight[ids]; saves the ids alone."""

    @staticmethod
    def forward(ctx, ids, weight, scale: float, padding_idx: int):
        ctx.save_for_backward(ids)
        ctx.scale, ctx.padding_idx = scale, padding_idx
        ctx.vocab, ctx.dtype = weight.shape[0], weight.dtype
        return cops.embedding_fwd(ids, weight, scale)

    @staticmethod
    def backward(ctx, dy):
        ids, = ctx.saved_tensors
        if dy.dtype != ctx.dtype:
            dy = dy.to(ctx.dtype)
        args = (ids, dy, ctx.vocab, ctx.padding_idx, ctx.scale)
        grad = _EmbeddingGradFunction.apply if torch.is_grad_enabled() else cops.embedding_bwd
        return None, grad(*args), None, None


class _EmbeddingGradFunction(torch.autograd.Function):
    """The table's gradient, itself differentiable (create_graph): linear in dy, whose
    gradient is the lookup of the table that arrives, zero where an id gives none."""

    @staticmethod
    def forward(ctx, ids, dy, vocab: int, padding_idx: int, scale: float):
        ctx.save_for_backward(ids)
        ctx.vocab, ctx.padding_idx, ctx.scale = vocab, padding_idx, scale
        return cops.embedding_bwd(ids, dy, vocab, padding_idx, scale)

    @staticmethod
    def backward(ctx, ddw):
        ids, = ctx.saved_tensors
        keep = (ids >= 0) & (ids < ctx.vocab) & (ids != ctx.padding_idx)
        y = _FusedEmbeddingFunction.apply(ids, ddw, ctx.scale, ctx.padding_idx)
        ddy = torch.where(keep.unsqueeze(-1), y, torch.zeros((), dtype=y.dtype, device=y.device))
        return None, ddy, None, None, None


def fused_embedding(ids: torch.Tensor, weight: torch.Tensor, scale: float = 1.0,
                    padding_idx: int | None = None) -> torch.Tensor:
    """scale * weight[ids]: ids int64 or int32 of any shape, weight [vocab, hidden]
    of fp32, bf16 or fp16; returns [*ids.shape, hidden] in weight's dtype.

    padding_idx (negative: counted from the end): the row that gets no gradient.
    An id outside the table gives a row of NaN and no gradient (nn.Embedding ends
    the process there).
    """
    vocab = weight.shape[0]
    if padding_idx is None:
        padding_idx = -1
    elif not -vocab <= padding_idx < vocab:
        raise ValueError(f"embedding: padding_idx {padding_idx} outside a table of {vocab} rows")
    else:
        padding_idx %= vocab
    return _FusedEmbeddingFunction.apply(ids, weight, float(scale), padding_idx)


def _fusable(module: nn.Module) -> bool:
    """An nn.Embedding as it is (a subclass may compute something else), without
    the options that the fused op does not have."""
    return (type(module) is nn.Embedding and module.max_norm is None and not module.sparse
            and not module.scale_grad_by_freq)


class MetalLigerEmbedding(nn.Module):
    """Drop-in for an nn.Embedding, whose parameter it shares (state_dict keys and
    tied weights are unchanged); `scale` multiplies the output."""

    def __init__(self, original: nn.Embedding, scale: float = 1.0):
        super().__init__()
        if not _fusable(original):
            raise ValueError("MetalLigerEmbedding: a plain nn.Embedding without max_norm, sparse "
                             f"or scale_grad_by_freq is needed (got {original})")
        self.weight = original.weight
        self.num_embeddings, self.embedding_dim = original.weight.shape
        self.padding_idx, self.scale = original.padding_idx, scale

    def forward(self, input: torch.Tensor) -> torch.Tensor:
        return fused_embedding(input, self.weight, self.scale, self.padding_idx)

    def extra_repr(self) -> str:
        return f"{self.num_embeddings}, {self.embedding_dim}, scale={self.scale}"


class _FusedEmbeddingForward:
    """Forward of a routed nn.Embedding: its own while the table is frozen. (A lookup
    alone gains nothing here: up to 8192 tokens it takes 13 us on the host, nn.Embedding
    7-12; 16384 x 2048 in bf16 21 us both; 65536 x 2048, 80 and 93.)"""

    def __init__(self, module: nn.Embedding):
        self.module = module

    def __call__(self, input):
        if not self.module.weight.requires_grad:
            return nn.Embedding.forward(self.module, input)
        return fused_embedding(input, self.module.weight, padding_idx=self.module.padding_idx)


def patch_embedding(model: nn.Module) -> int:
    """Routes the model's token embeddings (plain nn.Embedding modules called
    ``embed_tokens``, or inside a wrapper of that name as PEFT's modules_to_save
    makes one) through the fused op and returns how many were routed. Only the
    instances' ``forward`` changes, and what it does only while the table is trained;
    modules already routed are left as they are."""
    routed = 0
    for name, module in model.named_modules():
        if "embed_tokens" not in name.split(".") or not _fusable(module):
            continue
        if getattr(module, "_metal_liger_fused_embedding", False):
            continue
        module.forward = _FusedEmbeddingForward(module)
        module._metal_liger_fused_embedding = True
        routed += 1
    return routed

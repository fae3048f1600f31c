"""Dropout, LoRA dropout and the embedding without a GPU: sizes that a launch cannot
hold, and what the drop-in modules and the patcher leave as torch has it."""

import pytest
import torch
import torch.nn as nn


def test_lora_dropout_refuses_more_tokens_than_a_launch_holds():
    from metal_liger_amd import _hip
    L = _hip.lib()
    p = 4096  # (never read: the call is refused on the host)
    for tokens in (-1, (1 << 28) - 31, 1 << 28, (1 << 31) - 1):
        rc = L.ml_lora_dropout_xa(1, p, tokens, 64, 64, p, 16, _hip.geom([100]), p, 0, p, 16, None)
        assert rc == 1 and b"token count" in L.ml_last_error(), (tokens, L.ml_last_error())
        one = _hip.ptrs([p])
        rc = L.ml_lora_dropout_bwd(1, p, tokens, 64, one, _hip.geom([64]), one, p, one,
                                   _hip.floats([1.0]), p, 16, _hip.geom([100]), p, 0, p, p, one, 0,
                                   p, 16, None)
        assert rc == 1 and b"token count" in L.ml_last_error(), (tokens, L.ml_last_error())


def test_the_modules_take_their_argument_by_torch_s_name():
    """(On the CPU the call gets as far as the check of the device.)"""
    from metal_liger_amd import MetalLigerDropout, MetalLigerEmbedding
    from metal_liger_amd.ops.fused_embedding import patch_embedding
    root = nn.Module()
    root.embed_tokens = nn.Embedding(8, 4)
    assert patch_embedding(root) == 1
    x, ids = torch.zeros(4), torch.zeros(3, dtype=torch.long)
    for call in (lambda: MetalLigerDropout(0.5)(input=x),
                 lambda: MetalLigerDropout(0.5)(input=x, residual=x),
                 lambda: MetalLigerEmbedding(nn.Embedding(8, 4))(input=ids),
                 lambda: root.embed_tokens(input=ids)):
        with pytest.raises(ValueError, match="ROCm GPU"):
            call()
    assert MetalLigerDropout(0.5).eval()(input=x) is x


def test_a_routed_embedding_is_torch_s_own_while_its_table_is_frozen():
    from metal_liger_amd.ops.fused_embedding import patch_embedding
    root = nn.Module()
    root.embed_tokens = nn.Embedding(8, 4, padding_idx=2).requires_grad_(False)
    assert patch_embedding(root) == 1
    ids = torch.tensor([[1, 2], [7, 1]])
    assert torch.equal(root.embed_tokens(ids), root.embed_tokens.weight[ids])
    root.embed_tokens.requires_grad_(True)               # trained from here on
    with pytest.raises(ValueError, match="ROCm GPU"):
        root.embed_tokens(ids)


def test_a_seed_may_be_missing_only_where_nothing_is_dropped():
    from metal_liger_amd import _hip
    L = _hip.lib()
    assert L.ml_abi_version() >= 13
    assert L.ml_dropout(4096, None, 4096, 0, 0, 1.0, None, 0, 0, None) == 0    # nothing to do
    rc = L.ml_dropout(4096, None, 4096, 8, 1, 1.0, None, 0, 0, None)
    assert rc == 1 and b"null pointer" in L.ml_last_error()
    rc = L.ml_dropout(4096, None, 4096, 8, 0, 1.0, None, 0, 9, None)           # past the pointers
    assert rc == 1 and b"dtype" in L.ml_last_error()

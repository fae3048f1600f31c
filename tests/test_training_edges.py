"""Dropout, LoRA dropout and the embedding without a GPU: sizes that a launch cannot
hold, and what the drop-in modules and the patcher leave as torch has it."""


def test_lora_dropout_refuses_more_tokens_than_a_launch_holds():
    from metal_liger_amd import _hip
    L = _hip.lib()
    p = 4096  # (never read: the call is refused on the host)
    for tokens in (-1, (1 << 28) - 31, 1 << 28, (1 << 31) - 1):
        rc = L.ml_lora_dropout_xa(1, p, tokens, 64, 64, p, 16, _hip.geom([100]), p, 0, p, 16, None)
        assert rc == 1 and b"token count" in L.ml_last_error(), (tokens, L.ml_last_error())

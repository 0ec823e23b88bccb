"""The token mixers' Python calls refuse host tensors before anything is launched."""
import pytest


def _calls(mcv):
    import torch
    half = lambda *s: torch.zeros(*s, dtype=torch.float16)       # noqa: E731
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)          # noqa: E731
    gates = dict(g=torch.zeros(6, 4), beta=torch.zeros(6, 4))
    qkv = dict(q=half(6, 2, 64), k=half(6, 2, 64), v=half(6, 4, 64))
    freq, axis = mcv.rotary_axes_table(32, 1e4, (6, 5, 5), device="cpu")
    where = dict(positions=torch.zeros(3, 6, dtype=torch.int64), freq=freq, axis=axis)
    caches = dict(k_cache=half(5, 16, 2, 64), v_cache=half(5, 16, 2, 64))
    return [
        (mcv.gated_delta_rule, dict(**qkv, **gates, state=torch.zeros(1, 4, 64, 64))),
        (mcv.gated_delta_rule, dict(**qkv, **gates, cu_seqlens=torch.tensor([0, 6], dtype=torch.int32))),
        (mcv.gated_delta_rule_step, dict(**qkv, **gates, state=torch.zeros(6, 4, 64, 64))),
        (mcv.paged_attention_decode, dict(q=half(3, 8, 64), **caches, block_table=i32(3, 4), seq_lens=i32(3))),
        (mcv.rotary_axes, dict(q=qkv["q"], k=qkv["k"], **where)),
        (mcv.rotary_axes_cached, dict(q=qkv["q"], k=qkv["k"], v=half(6, 2, 64), **where, **caches, slots=torch.zeros(6, dtype=torch.int64))),
    ]


@pytest.mark.parametrize("i", range(6))
def test_host_tensors(mcv, i):
    call, args = _calls(mcv)[i]
    with pytest.raises(mcv.McvError, match=f"{call.__name__}: tensors must be on a GPU, got cpu") as refused:
        call(**args)
    assert getattr(refused.value, "status", None) is None        # the library was not called


@pytest.mark.parametrize("i", [4, 5])
def test_host_tensors_of_no_tokens(mcv, i):
    call, args = _calls(mcv)[i]
    for name in ("q", "k", "v", "slots"):
        if name in args:
            args[name] = args[name][:0]
    args["positions"] = args["positions"][:, :0]
    with pytest.raises(mcv.McvError, match="must be on a GPU"):
        call(**args)

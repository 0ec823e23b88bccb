"""CPU tests of what the token mixers refuse: every check stands before the first launch."""
import ctypes

import pytest

P = 1 << 20                                                      # a 16-byte aligned address that no call reads
INVALID, SHAPE, UNSUPPORTED, NO_DEVICE = 1, 2, 4, 5


def _call(mcv, name, args, **change):
    vals = dict(args, **change)
    return getattr(mcv.lib(), name)(*vals.values())


DELTA = dict(q=P, q_row=2048, q_head=128, k=P, k_row=2048, k_head=128, v=P, v_row=4096, v_head=128, g=P, g_row=32, beta=P,
             beta_row=32, state=P, state_out=P, state_index=0, n_states=2, cu=P, B=2, T=100, Hk=16, Hv=32, Dk=128, Dv=128,
             scale=0.1, normalize=1, out=P, ws=0, ws_bytes=0, stream=0)
ATTN = dict(q=P, q_row=2048, q_head=256, k=P, k_page=8192, k_token=512, k_head=256, v=P, v_page=8192, v_token=512, v_head=256,
            pages=100, page_size=16, table=P, table_row=8, width=8, lens=P, max_len=128, B=3, Hq=8, Hkv=2, D=256, scale=0.1,
            out=P, ws=0, ws_bytes=0, stream=0)
ROTARY = dict(q=P, q_row=2048, q_head=256, k=P, k_row=512, k_head=256, pos=P, pos_axis=7, pos_token=1, axes=3, freq=P, axis=P,
              T=7, Hq=8, Hkv=2, D=256, rot=64, q_out=P, qo_row=2048, qo_head=256, k_out=P, ko_row=512, ko_head=256, stream=0)
CACHED = dict(q=P, q_row=2048, q_head=256, k=P, k_row=512, k_head=256, v=P, v_row=512, v_head=256, pos=P, pos_axis=7,
              pos_token=1, axes=3, freq=P, axis=P, T=7, Hq=8, Hkv=2, D=256, rot=64, q_out=P, qo_row=2048, qo_head=256, kc=P,
              kc_page=8192, kc_token=512, kc_head=256, vc=P, vc_page=8192, vc_token=512, vc_head=256, pages=4, page_size=16,
              slots=P, stream=0)

REFUSED = [
    ("mcv_delta_rule", DELTA, [
        (INVALID, dict(q=0)), (INVALID, dict(k=0)), (INVALID, dict(v=0)), (INVALID, dict(g=0)), (INVALID, dict(beta=0)),
        (INVALID, dict(state_out=0)), (INVALID, dict(out=0)),
        (SHAPE, dict(B=0)), (SHAPE, dict(B=-1)), (SHAPE, dict(T=-1)), (SHAPE, dict(Hk=0)), (SHAPE, dict(Hv=0)),
        (SHAPE, dict(Hv=24)), (SHAPE, dict(Dk=96)), (SHAPE, dict(Dv=24)), (SHAPE, dict(Dv=0)), (SHAPE, dict(Dv=272)),
        (SHAPE, dict(n_states=1)), (SHAPE, dict(n_states=0, state_index=P)), (SHAPE, dict(cu=0, B=3, n_states=3)),
        (SHAPE, dict(q_row=-8)), (SHAPE, dict(g_row=-1)),
        (UNSUPPORTED, dict(q=P + 2)), (UNSUPPORTED, dict(k_row=2044)), (UNSUPPORTED, dict(v_head=4)),
        (UNSUPPORTED, dict(state=P + 4)), (UNSUPPORTED, dict(out=P + 8))]),
    ("mcv_paged_attention", ATTN, [
        (INVALID, dict(q=0)), (INVALID, dict(k=0)), (INVALID, dict(v=0)), (INVALID, dict(table=0)), (INVALID, dict(lens=0)),
        (INVALID, dict(out=0)),
        (SHAPE, dict(B=0)), (SHAPE, dict(Hq=9)), (SHAPE, dict(Hkv=0)), (SHAPE, dict(D=96)), (SHAPE, dict(page_size=0)),
        (SHAPE, dict(page_size=24)), (SHAPE, dict(pages=0)), (SHAPE, dict(pages=2 ** 31)), (SHAPE, dict(width=0)),
        (SHAPE, dict(max_len=-1)), (SHAPE, dict(k_token=-512)), (SHAPE, dict(table_row=-1)), (SHAPE, dict(B=2 ** 30)),
        (UNSUPPORTED, dict(q=P + 2)), (UNSUPPORTED, dict(k_token=516)), (UNSUPPORTED, dict(v=P + 8)),
        (UNSUPPORTED, dict(out=P + 2))]),
    ("mcv_rotary_axes", ROTARY, [
        (INVALID, dict(q=0)), (INVALID, dict(k=0)), (INVALID, dict(pos=0)), (INVALID, dict(freq=0)), (INVALID, dict(axis=0)),
        (INVALID, dict(q_out=0)), (INVALID, dict(k_out=0)),
        (SHAPE, dict(T=0)), (SHAPE, dict(Hq=0)), (SHAPE, dict(Hkv=-1)), (SHAPE, dict(D=100)), (SHAPE, dict(D=520, rot=2)),
        (SHAPE, dict(rot=0)), (SHAPE, dict(rot=63)), (SHAPE, dict(rot=258)), (SHAPE, dict(axes=0)), (SHAPE, dict(pos_axis=-1)),
        (UNSUPPORTED, dict(q=P + 2)), (UNSUPPORTED, dict(ko_row=500)), (UNSUPPORTED, dict(q_out=P + 8))]),
    ("mcv_rotary_axes_cached", CACHED, [
        (INVALID, dict(v=0)), (INVALID, dict(kc=0)), (INVALID, dict(vc=0)), (INVALID, dict(slots=0)),
        (SHAPE, dict(pages=0)), (SHAPE, dict(page_size=0)), (SHAPE, dict(rot=3)), (SHAPE, dict(vc_page=-8)),
        (UNSUPPORTED, dict(vc_token=12)), (UNSUPPORTED, dict(kc=P + 2))]),
]


@pytest.mark.parametrize("name,args,status,change", [(n, a, s, c) for n, a, cs in REFUSED for s, c in cs])
def test_refused_before_any_launch(mcv, name, args, status, change):
    assert _call(mcv, name, args, **change) == status
    assert mcv.lib().mcv_last_error().decode().startswith(name[4:])


@pytest.mark.parametrize("name,args", [(n, a) for n, a, _ in REFUSED])
def test_what_is_not_refused_needs_a_device(mcv, name, args):
    import torch
    if torch.cuda.is_available():
        pytest.skip("would launch on addresses that are not memory")
    assert _call(mcv, name, args) == NO_DEVICE


def test_python_refusals(mcv):
    """The Python entry points look at types, shapes and layouts before the library is called."""
    import torch
    T, Hk, Hv, D = 6, 2, 4, 64
    half = lambda *s: torch.zeros(*s, dtype=torch.float16)       # noqa: E731
    ok = dict(q=half(T, Hk, D), k=half(T, Hk, D), v=half(T, Hv, D), g=torch.zeros(T, Hv), beta=torch.zeros(T, Hv),
              state=torch.zeros(1, Hv, D, D))
    for bad in (dict(q=torch.zeros(T, Hk, D)), dict(k=half(T, Hk, 2 * D)), dict(k=half(T + 1, Hk, D)), dict(v=half(T, Hv * D)),
                dict(v=half(T - 1, Hv, D)), dict(g=torch.zeros(T, Hk)), dict(beta=torch.zeros(T, Hv).half()),
                dict(g=torch.zeros(Hv, T).t()), dict(state=torch.zeros(2, Hv, D, D)), dict(state=torch.zeros(1, Hv, D, D).double()),
                dict(state=torch.zeros(1, Hv, D, D).transpose(2, 3)), dict(v=half(T, Hv, 2 * D)[..., ::2]),
                dict(out=half(T, Hv, D + 16)), dict(cu_seqlens=torch.zeros(2)), dict(cu_seqlens=torch.zeros(1, dtype=torch.int32)),
                dict(state_index=torch.zeros(1, dtype=torch.int64)), dict(state=None, state_index=torch.zeros(1, dtype=torch.int32))):
        with pytest.raises(mcv.McvError, match="gated_delta_rule"):
            mcv.gated_delta_rule(**{**ok, **bad})
    with pytest.raises(mcv.McvError, match="gated_delta_rule_step"):
        mcv.gated_delta_rule_step(**ok)                          # one state for six sequences
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)          # noqa: E731
    ok = dict(q=half(3, 8, D), k_cache=half(5, 16, 2, D), v_cache=half(5, 16, 2, D), block_table=i32(3, 4), seq_lens=i32(3))
    for bad in (dict(q=half(3, 8, 2 * D)), dict(q=half(3, 8 * D)), dict(k_cache=half(5, 16, 2 * D)), dict(v_cache=half(4, 16, 2, D)),
                dict(v_cache=torch.zeros(5, 16, 2, D)), dict(block_table=i32(2, 4)), dict(block_table=i32(4, 3).t()),
                dict(block_table=torch.zeros(3, 4, dtype=torch.int64)), dict(seq_lens=i32(4)), dict(seq_lens=torch.zeros(3)),
                dict(out=half(3, 8, 2 * D))):
        with pytest.raises(mcv.McvError, match="paged_attention_decode"):
            mcv.paged_attention_decode(**{**ok, **bad})
    freq, axis = mcv.rotary_axes_table(32, 1e4, (6, 5, 5), device="cpu")
    ok = dict(q=half(T, 4, D), k=half(T, 2, D), positions=torch.zeros(3, T, dtype=torch.int64), freq=freq, axis=axis)
    for bad in (dict(q=half(T + 1, 4, D)), dict(k=half(T, 2, 32)), dict(positions=torch.zeros(3, T)),
                dict(positions=torch.zeros(T, dtype=torch.int64)), dict(positions=torch.zeros(3, T + 1, dtype=torch.int64)),
                dict(freq=freq.float()), dict(axis=axis[:-1]), dict(q_out=half(T, 4, 32)), dict(k_out=half(T, 4, D)),
                dict(q=half(T, 4, 2 * D)[..., ::2])):
        with pytest.raises(mcv.McvError, match="rotary_axes"):
            mcv.rotary_axes(**{**ok, **bad})
    ok.update(v=half(T, 2, D), k_cache=half(5, 16, 2, D), v_cache=half(5, 16, 2, D), slots=torch.zeros(T, dtype=torch.int64))
    for bad in (dict(v=half(T, 2, 32)), dict(slots=i32(T)), dict(slots=torch.zeros(T + 1, dtype=torch.int64)),
                dict(k_cache=half(5, 16, 4, D)), dict(v_cache=half(5, 16, 2 * D))):
        with pytest.raises(mcv.McvError, match="rotary_axes_cached"):
            mcv.rotary_axes_cached(**{**ok, **bad})


def test_rotary_axes_table(mcv):
    freq, axis = mcv.rotary_axes_table(64, 1e7, (11, 11, 10), device="cpu")
    assert axis.tolist() == [0, 1, 2] * 10 + [0, 1]
    assert freq[0] == 1 and abs(freq[16].item() - 1e7 ** -0.5) < 1e-18
    assert mcv.rotary_axes_table(16, 1e4, (4, 2, 2), False, device="cpu")[1].tolist() == [0, 0, 0, 0, 1, 1, 2, 2]
    for rot, sections in ((64, (11, 11, 11)), (63, (31,)), (8, (5, -1)), (8, (0, 4))):
        with pytest.raises(mcv.McvError, match="rotary_axes_table"):
            mcv.rotary_axes_table(rot, 1e4, sections, device="cpu")

"""CPU tests of what the chunked attention, the page calls and the residual norm refuse: every check stands before the first launch."""
import pytest

P = 1 << 20                                                      # a 16-byte aligned address that no call reads
Q, R = P + (1 << 30), P + (1 << 31)                              # and two far from it
INVALID, SHAPE, UNSUPPORTED, NO_DEVICE = 1, 2, 4, 5

CHUNK = dict(q=P, q_row=2048, q_head=256, k=P, k_page=8192, k_token=512, k_head=256, v=P, v_page=8192, v_token=512, v_head=256,
             pages=100, page_size=16, table=P, table_row=8, width=8, lens=P, max_len=128, cu=P, B=3, T=40, Hq=8, Hkv=2, D=256, scale=0.1,
             out=P, ws=0, ws_bytes=0, stream=0)
APPEND = dict(table=P, table_row=8, width=8, lens=Q, cu=P, B=3, T=40, page_size=16, free=P, capacity=100, count=P, slots=P, positions=P,
              lens_out=R, count_out=P, stream=0)
TRUNCATE = dict(table=P, table_row=8, width=8, lens=Q, keep=P, B=3, page_size=16, free=P, capacity=100, count=P, lens_out=R, count_out=P, stream=0)
ADD = dict(x=P, x_row=1024, residual=Q, r_row=1024, gamma=P, M=100, H=1024, eps=1e-6, sum=R, sum_row=1024, out=P + (1 << 29), stream=0)
ADD8 = dict(x=P, x_row=1024, residual=Q, r_row=1024, gamma=P, M=100, H=1024, eps=1e-6, sum=R, sum_row=1024, normed=0, xq=P, s32=P, s16=0, stream=0)

REFUSED = [
    ("mcv_paged_attention_chunk", CHUNK, [
        (INVALID, dict(q=0)), (INVALID, dict(k=0)), (INVALID, dict(v=0)), (INVALID, dict(table=0)), (INVALID, dict(lens=0)), (INVALID, dict(out=0)),
        (SHAPE, dict(B=0)), (SHAPE, dict(T=0)), (SHAPE, dict(T=-1)), (SHAPE, dict(Hq=9)), (SHAPE, dict(Hkv=0)), (SHAPE, dict(D=96)),
        (SHAPE, dict(page_size=0)), (SHAPE, dict(page_size=24)), (SHAPE, dict(pages=0)), (SHAPE, dict(pages=2 ** 31)), (SHAPE, dict(width=0)),
        (SHAPE, dict(max_len=-1)), (SHAPE, dict(k_token=-512)), (SHAPE, dict(table_row=-1)), (SHAPE, dict(T=2 ** 29)), (SHAPE, dict(B=2 ** 30)),
        (SHAPE, dict(cu=0)),                                     # 40 rows of 3
        (UNSUPPORTED, dict(q=P + 2)), (UNSUPPORTED, dict(k_token=516)), (UNSUPPORTED, dict(v=P + 8)), (UNSUPPORTED, dict(out=P + 2)),
        (UNSUPPORTED, dict(v_token=2 ** 26))]),
    ("mcv_paged_append", APPEND, [
        (INVALID, dict(table=0)), (INVALID, dict(lens=0)), (INVALID, dict(lens_out=0)), (INVALID, dict(slots=0)), (INVALID, dict(positions=0)),
        (INVALID, dict(count=0)), (INVALID, dict(count_out=0)), (INVALID, dict(lens_out=Q + 4)), (INVALID, dict(lens_out=P + 12)),
        (SHAPE, dict(B=0)), (SHAPE, dict(B=2 ** 29)), (SHAPE, dict(T=-1)), (SHAPE, dict(T=2 ** 31)), (SHAPE, dict(cu=0)), (SHAPE, dict(page_size=0)),
        (SHAPE, dict(page_size=2 ** 21)), (SHAPE, dict(width=0)), (SHAPE, dict(table_row=-1)), (SHAPE, dict(table_row=7)), (SHAPE, dict(table_row=0)),
        (SHAPE, dict(capacity=-1)), (SHAPE, dict(capacity=2 ** 31))]),
    ("mcv_paged_truncate", TRUNCATE, [
        (INVALID, dict(table=0)), (INVALID, dict(lens=0)), (INVALID, dict(lens_out=0)), (INVALID, dict(free=0)), (INVALID, dict(count=0)),
        (INVALID, dict(count_out=0)), (INVALID, dict(lens_out=Q + 8)), (INVALID, dict(lens_out=P - 4)),
        (SHAPE, dict(B=0)), (SHAPE, dict(page_size=-16)), (SHAPE, dict(width=2 ** 31)), (SHAPE, dict(table_row=-1))]),
    ("mcv_rms_norm_add", ADD, [
        (INVALID, dict(x=0)), (INVALID, dict(residual=0)), (INVALID, dict(gamma=0)), (INVALID, dict(sum=0)), (INVALID, dict(out=0)),
        (INVALID, dict(sum=P + 2)), (INVALID, dict(sum=Q, sum_row=2048)), (INVALID, dict(out=R)), (INVALID, dict(out=P, x_row=2048)),
        (INVALID, dict(out=Q + 64)), (INVALID, dict(x_row=0, sum=P)),
        (SHAPE, dict(M=0)), (SHAPE, dict(H=0)), (SHAPE, dict(M=2 ** 31)), (SHAPE, dict(eps=-1.0)), (SHAPE, dict(eps=float("nan"))),
        (SHAPE, dict(x_row=-1)), (SHAPE, dict(sum_row=1000))]),
    ("mcv_rms_norm_add_w8a8_quantize", ADD8, [
        (INVALID, dict(x=0)), (INVALID, dict(residual=0)), (INVALID, dict(gamma=0)), (INVALID, dict(sum=0)), (INVALID, dict(xq=0)),
        (INVALID, dict(s32=0)), (INVALID, dict(sum=P + 2)), (INVALID, dict(normed=R)), (SHAPE, dict(M=-1)), (SHAPE, dict(sum_row=0))]),
]


def _call(mcv, name, args, **change):
    return getattr(mcv.lib(), name)(*dict(args, **change).values())


@pytest.mark.parametrize("name,args,status,change", [(n, a, s, c) for n, a, cs in REFUSED for s, c in cs])
def test_refused_before_any_launch(mcv, name, args, status, change):
    assert _call(mcv, name, args, **change) == status
    assert mcv.lib().mcv_last_error().decode().startswith(name[4:])


@pytest.mark.parametrize("name,args,change", [(n, a, {}) for n, a, _ in REFUSED] + [
    ("mcv_paged_append", APPEND, dict(lens_out=Q)), ("mcv_paged_append", APPEND, dict(free=0, count=0, count_out=0, table_row=0)),
    ("mcv_paged_append", APPEND, dict(T=0, slots=0, positions=0)), ("mcv_paged_append", APPEND, dict(B=1, T=9, cu=0, table_row=0)),
    ("mcv_paged_truncate", TRUNCATE, dict(lens_out=P)), ("mcv_paged_truncate", TRUNCATE, dict(keep=0, lens_out=Q)),
    ("mcv_rms_norm_add", ADD, dict(sum=P)), ("mcv_rms_norm_add", ADD, dict(sum=Q)), ("mcv_rms_norm_add", ADD, dict(out=P)),
    ("mcv_rms_norm_add", ADD, dict(x_row=0, r_row=0)), ("mcv_rms_norm_add", ADD, dict(M=1, sum_row=0)),
    ("mcv_rms_norm_add", ADD, dict(x_row=2048, sum_row=2048, sum=P + 2048)), ("mcv_rms_norm_add", ADD, dict(x_row=2048, sum_row=2048, x=R + 2048))])
def test_what_is_not_refused_needs_a_device(mcv, name, args, change):
    import torch
    if torch.cuda.is_available():
        pytest.skip("would launch on addresses that are not memory")
    assert _call(mcv, name, args, **change) == NO_DEVICE


def _python_calls():
    import torch
    half = lambda *s: torch.zeros(*s, dtype=torch.float16)       # noqa: E731
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)          # noqa: E731
    i64 = lambda *s: torch.zeros(*s, dtype=torch.int64)          # noqa: E731
    T, D, H = 6, 64, 32
    return {
        "paged_attention_chunk": (
            dict(q=half(T, 8, D), k_cache=half(5, 16, 2, D), v_cache=half(5, 16, 2, D), block_table=i32(2, 4), seq_lens=i32(2), cu_seqlens=i32(3)),
            [dict(q=half(T, 8, 2 * D)), dict(q=half(T, 8 * D)), dict(q=torch.zeros(T, 8, D)), dict(q=half(T, 8, 2 * D)[..., ::2]),
             dict(k_cache=half(5, 16, 2 * D)), dict(v_cache=half(4, 16, 2, D)), dict(v_cache=torch.zeros(5, 16, 2, D)), dict(block_table=i32(3, 4)),
             dict(block_table=i32(4, 2).t()), dict(block_table=i64(2, 4)), dict(seq_lens=i64(2)), dict(seq_lens=i32(2, 1)), dict(seq_lens=i32(4)[::2]),
             dict(cu_seqlens=i32(2)), dict(cu_seqlens=i64(3)), dict(cu_seqlens=None, seq_lens=i32(4), block_table=i32(4, 4)),
             dict(out=half(T, 8, 2 * D)), dict(out=half(T, 16, D)[:, ::2]), dict(q=[1])]),
        "paged_append": (
            dict(block_table=i32(2, 4), seq_lens=i32(2), cu_seqlens=i32(3), page_size=16, tokens=T, free_pages=i32(9), free_count=i32(1)),
            [dict(block_table=i32(3, 4)), dict(block_table=i64(2, 4)), dict(seq_lens=i64(2)), dict(cu_seqlens=i32(2)), dict(cu_seqlens=None, tokens=5),
             dict(tokens=-1), dict(free_pages=None), dict(free_count=None), dict(free_count=i32(2)), dict(free_pages=i64(9)), dict(free_pages=i32(18)[::2]),
             dict(seq_lens_out=i32(3)), dict(free_count_out=i64(1)), dict(slots=i64(5)), dict(slots=i32(T)), dict(positions=i64(T, 1))]),
        "paged_truncate": (
            dict(block_table=i32(2, 4), seq_lens=i32(2), keep=i32(2), page_size=16, free_pages=i32(9), free_count=i32(1)),
            [dict(block_table=i32(2, 4).float()), dict(seq_lens=i32(3)), dict(keep=i32(3)), dict(keep=i64(2)), dict(free_pages=None), dict(free_count=i32(3)),
             dict(seq_lens_out=i64(2)), dict(free_count_out=i32(2))]),
        "rms_norm_add": (
            dict(x=half(T, H), residual=half(T, H), gamma=half(H), eps=1e-6),
            [dict(x=half(T * H)), dict(x=torch.zeros(T, H)), dict(x=half(H, T).t()), dict(residual=half(T, H + 8)), dict(residual=half(1, H)),
             dict(gamma=half(H + 1)), dict(gamma=torch.zeros(H)), dict(out=half(T, 2 * H)[:, :H]), dict(residual_out=half(T, 2 * H)[:, ::2])]),
        "rms_norm_add_w8a8_quantize": (
            dict(x=half(T, H), residual=half(T, H), gamma=half(H), eps=1e-6),
            [dict(x=half(T, H, 1)), dict(normed=half(T, 2 * H)[:, :H]), dict(x_scale_f16=half(T + 1)), dict(x_scale_f16=torch.zeros(T)),
             dict(residual_out=torch.zeros(T, H))]),
    }


@pytest.mark.parametrize("name", list(_python_calls()))
def test_python_refusals(mcv, name):
    """Types, shapes and layouts are looked at before the library is called, and host tensors after them."""
    args, bad = _python_calls()[name]
    call = getattr(mcv, name)
    with pytest.raises(mcv.McvError, match=f"{name}: tensors must be on a GPU, got cpu") as refused:
        call(**args)
    assert getattr(refused.value, "status", None) is None
    for change in bad:
        with pytest.raises(mcv.McvError, match=f"^{name}: (?!tensors must)"):
            call(**{**args, **change})
    with pytest.raises(TypeError):
        call(**{**args, **({"eps": "x"} if "eps" in args else {"page_size": 1.5} if "page_size" in args else {"max_seq_len": "x"})})


def test_workspace_bytes(mcv):
    size = mcv.lib().mcv_paged_attention_chunk_workspace_bytes
    assert size(1, 100, 8, 2, 256, 256) == 0                     # nothing to cut
    most = size(8, 5000, 8, 2, 256, 1 << 20)
    assert 0 < most <= 192 << 20
    for T, length in ((1, 300), (24, 5000), (31, 1 << 20), (32, 4096), (5000, 300)):
        assert 0 < size(8, T, 8, 2, 256, length) <= most
    for bad in ((0, 5, 8, 2, 256, 999), (1, 0, 8, 2, 256, 999), (1, 5, 8, 3, 256, 999), (1, 5, 8, 2, 0, 999), (1, 5, 8, 2, 256, -1), (1, 2 ** 30, 8, 2, 256, 999)):
        assert size(*bad) == 0


def test_python_keeps_enough_for_every_call(mcv):
    size = mcv.lib().mcv_paged_attention_chunk_workspace_bytes
    for D in (64, 128, 256):
        for Hq, Hkv in ((8, 2), (1, 1), (500, 1)):
            for T in (1, 3, 128, 100000):
                for length in (0, 256, 257, 2048, 1 << 30, 1 << 40):
                    assert size(1, T, Hq, Hkv, D, length) <= mcv.mixers.CHUNK_WORKSPACE_BYTES

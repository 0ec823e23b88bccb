"""CPU tests of calls of paged_attention_chunk whose `out` lies on q's rows, of those whose rows only lie around it, and of
positions that are none."""
import pytest

from test_chunk_host import CHUNK, INVALID, NO_DEVICE, P, _call

T, HQ, D = 40, 8, 256                                            # CHUNK's
ROWS = 2 * T * HQ * D                                            # bytes of out


def _overlap(q, row, head, out, t=T, hq=HQ, d=D):
    """Byte for byte."""
    q_at = {q + 2 * (i * row + h * head + 8 * e) for i in range(t) for h in range(hq) for e in range(d // 8)}
    return any(out <= a < out + 2 * t * hq * d for a in q_at)


PLACES = [
    # q_row, q_head, out - q
    (2048, 256, 16), (2048, 256, -16), (2048, 256, ROWS - 16), (2048, 256, 16 - ROWS), (2048, 256, 4096), (4096, 256, 0), (2048, 0, 0), (0, 256, 0),
    (0, 0, 496), (4096, 512, 2 * 4096), (256, 10240, 0), (2304, 256, -ROWS + 16), (81920 + 64, 256, 4096), (256, 40 * 256 + 81920, 2 * 40 * 256),
    # apart, or in the gaps
    (2048, 256, ROWS), (2048, 256, -ROWS), (2304, 256, -ROWS), (0, 256, 4096), (0, 0, 512), (0, 0, -ROWS), (90000, 256, 4096), (90000, 256, 4096 + 32),
    (256, 40 * 256 + 81920, 512 * 40), (81920 + 2048, 256, 4096),
]


@pytest.mark.parametrize("row,head,off", PLACES)
def test_out_on_q(mcv, row, head, off):
    import torch
    q, out = P + (1 << 28), P + (1 << 28) + off
    got = lambda: _call(mcv, "mcv_paged_attention_chunk", CHUNK, q=q, q_row=row, q_head=head, out=out)      # noqa: E731
    if _overlap(q, row, head, out):
        assert got() == INVALID
        assert mcv.lib().mcv_last_error().decode() == "paged_attention_chunk: out overlaps q without being it"
    elif not torch.cuda.is_available():                          # (would launch on addresses that are not memory)
        assert got() == NO_DEVICE


@pytest.mark.parametrize("change", [dict(), dict(T=1, cu=P, q_row=0), dict(T=1, q_row=999 * 8, B=1, cu=0), dict(Hq=2, Hkv=2, q_row=512, q_head=256),
                                    dict(Hq=1, Hkv=1, q_row=256, q_head=0)])
def test_out_is_q(mcv, change):
    import torch
    if torch.cuda.is_available():
        pytest.skip("would launch on addresses that are not memory")
    assert _call(mcv, "mcv_paged_attention_chunk", CHUNK, **change) == NO_DEVICE


def test_positions_of_another_shape(mcv):
    import torch
    half, i32, i64 = (lambda *s, t=t: torch.zeros(*s, dtype=t) for t in (torch.float16, torch.int32, torch.int64))
    args = dict(q=half(6, 8, 64), k_cache=half(5, 16, 2, 64), v_cache=half(5, 16, 2, 64), block_table=i32(2, 4), seq_lens=i32(2), cu_seqlens=i32(3))
    for bad in (i32(6), i64(5), i64(6, 1), i64(12)[::2]):
        with pytest.raises(mcv.McvError, match=r"^paged_attention_chunk: positions must be contiguous int64 \[6\]"):
            mcv.paged_attention_chunk(**args, positions=bad)
    with pytest.raises(mcv.McvError, match="tensors must be on a GPU"):
        mcv.paged_attention_chunk(**args, positions=i64(6))

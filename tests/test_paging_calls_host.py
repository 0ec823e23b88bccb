"""CPU tests of calls of paged_append and paged_truncate that would not do what they say, and are refused before any launch."""
import pytest


def _args():
    import torch
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)          # noqa: E731
    return dict(block_table=i32(2, 4), seq_lens=i32(2), cu_seqlens=i32(3), page_size=16, tokens=6, free_pages=i32(9), free_count=i32(1))


def test_offsets_of_a_batch_of_unknown_rows(mcv):
    """Offsets are clamped to the rows that there are: with neither `tokens` nor `slots` they would be to one a sequence."""
    import torch
    args = dict(_args(), tokens=None)
    with pytest.raises(mcv.McvError, match="^paged_append: cu_seqlens needs tokens"):
        mcv.paged_append(**args)
    for rows in (dict(tokens=6), dict(slots=torch.zeros(6, dtype=torch.int64)), dict(cu_seqlens=None)):
        with pytest.raises(mcv.McvError, match="tensors must be on a GPU"):      # (all that is left to refuse here)
            mcv.paged_append(**{**args, **rows})


def test_a_count_that_nothing_would_write(mcv):
    """Without free_pages there are no pages to count, and free_count_out would be left as it was."""
    args = _args()
    args = dict(args, free_count_out=args["free_count"].clone(), free_pages=None, free_count=None)
    with pytest.raises(mcv.McvError, match="^paged_append: free_count_out without free_pages"):
        mcv.paged_append(**args)
    from test_chunk_host import APPEND, INVALID, P, _call
    assert _call(mcv, "mcv_paged_append", APPEND, free=0, count=0, count_out=P) == INVALID
    assert mcv.lib().mcv_last_error().decode() == "paged_append: free_count_out without free_pages"

"""The workspace that paged attention asks for covers every shorter bound on the lengths."""
import pytest


@pytest.mark.parametrize("B,Hq,Hkv,D", [(1, 8, 2, 256), (40, 2, 1, 64), (33, 16, 1, 128), (700, 32, 8, 128)])
def test_bytes_grow_with_the_bound(mcv, B, Hq, Hkv, D):
    need = [mcv.lib().mcv_paged_attention_workspace_bytes(B, Hq, Hkv, D, n) for n in (0, 1, 128, 129, 5000, 10 ** 6, 2 ** 30, 2 ** 40, 2 ** 62)]
    assert need == sorted(need) and need[0] == 0 and need[-1] > 0


@pytest.mark.parametrize("B,T,long", [(1, 9, 0), (1, 10, 1), (2, 19, 0), (2, 20, 1), (8, 39, 0), (8, 40, 1), (16, 47, 0), (16, 48, 1), (41, 41, 0),
                                      (41, 72, 0), (41, 73, 1), (41, 103, 1), (700, 731, 0), (700, 732, 1)])
def test_batches_that_may_hold_a_prompt(mcv, B, T, long):
    """One sequence may have all tokens but one of each other: past some 32 the chunked form is ready for it."""
    assert (mcv.lib().mcv_delta_rule_workspace_bytes(B, T, 16, 16, 128, 128) > 0) == bool(long)

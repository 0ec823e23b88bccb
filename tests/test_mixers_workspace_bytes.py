"""The workspace that paged attention asks for covers every shorter bound on the lengths."""
import pytest


@pytest.mark.parametrize("B,Hq,Hkv,D", [(1, 8, 2, 256), (40, 2, 1, 64), (33, 16, 1, 128), (700, 32, 8, 128)])
def test_bytes_grow_with_the_bound(mcv, B, Hq, Hkv, D):
    need = [mcv.lib().mcv_paged_attention_workspace_bytes(B, Hq, Hkv, D, n) for n in (0, 1, 128, 129, 5000, 10 ** 6, 2 ** 30, 2 ** 40, 2 ** 62)]
    assert need == sorted(need) and need[0] == 0 and need[-1] > 0

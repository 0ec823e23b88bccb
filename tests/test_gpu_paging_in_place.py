"""GPU tests of paged_append and paged_truncate in place where the state has a launch of its own and every wave of its workgroup
has sequences: lengths and count must come from what the call found, whichever wave is last."""
import pytest

from test_gpu_mixers import _gen, _torch
from test_gpu_paging import _Pool, _cu, _ints, _same

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B,n,lacking", [(200, 30, 0), (200, 30, 7), (700, 9, 0), (700, 9, 100), (1000, 20, 1), (1000, 20, 900), (1500, 5, 40)])
def test_the_last_pages(mcv, cuda, B, n, lacking):
    """More than 2048 tokens, and pages that just suffice or run out inside the last sequences: all that had room keep it."""
    torch = _torch()
    page = 16
    per = -(-n // page)
    for turn in range(8):
        pool = _Pool(turn, B, 2 * per + 1, page, B * per)
        pool.count -= lacking
        table, lens, free, count = pool.on(cuda)
        slots, positions, same = mcv.paged_append(table, lens, None, page, tokens=B * n, free_pages=free, free_count=count)
        assert same is lens
        want = pool.append([n] * B, B * n)
        assert slots.tolist() == want[0] and positions.tolist() == want[1], turn
        assert pool.count == -lacking
        _same(pool, table, lens, free, count, turn)
        assert sum(pool.lens) == sum(s >= 0 for s in want[0])
        pool.count = max(pool.count, 0)                          # a count below zero is none
        keep = (torch.rand(B, generator=_gen(turn)) * (n + 1)).int().tolist()
        mcv.paged_truncate(table, lens, _ints(keep, cuda), page, free, count)
        pool.truncate(keep)
        _same(pool, table, lens, free, count, turn)


def test_growing_shares_in_place(mcv, cuda):
    """Ragged sequences, the later ones longer, over a pool whose last page goes to the last sequence."""
    B, page = 600, 16
    n = [1 + 40 * i // B for i in range(B)]
    pool = _Pool(3, B, 4, page, sum(-(-m // page) for m in n))
    table, lens, free, count = pool.on(cuda)
    slots, _, _ = mcv.paged_append(table, lens, _cu(n, cuda), page, tokens=sum(n), free_pages=free, free_count=count)
    assert slots.tolist() == pool.append(n, sum(n))[0] and count.item() == 0
    _same(pool, table, lens, free, count)

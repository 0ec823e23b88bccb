"""GPU tests of values that are not finite in the caches of paged_attention_chunk: an element of V makes of a row that sees its
token, in its d, what a sum with it is (an infinity, or NaN where a NaN or both infinities are seen), and every other value has
the bits that it has with a zero in the element's place.  Scores here are a few units at most, so that no weight is zero."""
import math

import pytest

from test_gpu_chunk_attention import _case
from test_gpu_mixers import _gen, _torch

pytestmark = pytest.mark.gpu

SHAPES = [
    # new, held, Hq, Hkv, D, page: in one part, in up to four, in more
    ([70, 5], [0, 30], 8, 2, 64, 16),
    ([300], [90], 16, 16, 64, 32),
    ([3, 40], [6000, 900], 8, 2, 64, 32),
    ([130, 1, 0, 33], [0, 200, 9, 64], 32, 8, 128, 16),
    ([700], [900], 12, 1, 128, 128),
    ([9, 9, 1], [4000, 4000, 10], 8, 2, 128, 32),
    ([60], [100], 8, 2, 256, 16),
    ([1100], [0], 8, 2, 256, 16),
    ([24], [1100], 8, 2, 256, 16),
    ([5, 5, 5], [9000, 10, 2000], 8, 2, 256, 32),
]


def _spoil(seed, table, v, n, held, page, many):
    """(token, head, d, value) of each sequence: anywhere in the cache, and among its new tokens."""
    torch = _torch()
    gen, marks = _gen(seed), []
    v = v.clone()
    for b, (m, h) in enumerate(zip(n, held)):
        own = []
        for i in range(many if m else 0):
            t = int(torch.randint(h, h + m, (1,), generator=gen)) if i % 2 else int(torch.randint(0, h + m, (1,), generator=gen))
            head, d = (int(torch.randint(0, s, (1,), generator=gen)) for s in v.shape[2:])
            value = (math.inf, -math.inf, math.nan)[i % 3]
            d = own[-1][2] if own and i % 5 == 4 else d          # two in one column
            own.append((t, head, d, value))
            v[table[b, t // page], t % page, head, d] = value
        marks.append(own)
    return v, marks


def _kinds(q, marks, v, table, n, held, Hkv, page):
    """What is not finite in the output (0 where it is)."""
    torch = _torch()
    T, Hq, D = q.shape
    up, down = (torch.zeros(T, Hq, D, dtype=torch.bool) for _ in range(2))
    first = 0
    for b, own in enumerate(marks):
        for t, head, d, _ in own:
            value = v[table[b, t // page], t % page, head, d].item()       # (the last of two marks in one place)
            rows = slice(first + max(0, t - held[b]), first + n[b])
            heads = slice(head * Hq // Hkv, (head + 1) * Hq // Hkv)
            if value != -math.inf:
                up[rows, heads, d] = True
            if value != math.inf:
                down[rows, heads, d] = True
        first += n[b]
    zero = torch.zeros(T, Hq, D)
    return zero.masked_fill(up, math.inf).masked_fill(down, -math.inf).masked_fill(up & down, math.nan)


@pytest.mark.parametrize("n,held,Hq,Hkv,D,page", SHAPES)
@pytest.mark.parametrize("many", [1, 2, 40])
def test_values(mcv, cuda, n, held, Hq, Hkv, D, page, many):
    torch = _torch()
    q, k, v, table, lens, cu, _ = _case(D + many, n, held, Hq, Hkv, D, page, sharp=0.3)
    bad, marks = _spoil(many, table, v, n, held, page, many)
    a = [x.to(cuda) for x in (q, k, torch.where(bad.isfinite(), v, torch.where(v.isfinite(), 0, v)), table, lens, cu)]
    clean = mcv.paged_attention_chunk(*a).cpu()
    assert clean.isfinite().all()
    a[2] = bad.to(cuda)
    want = _kinds(q, marks, bad, table, n, held, Hkv, page)
    for _ in range(2):
        got = mcv.paged_attention_chunk(*a).cpu()
        assert torch.equal(got.isnan(), want.isnan())
        assert torch.equal(got == math.inf, want == math.inf) and torch.equal(got == -math.inf, want == -math.inf)
        assert torch.equal(got[want == 0], clean[want == 0])
    a[2] = v.to(cuda)                            # the workspace's counters are as they were
    assert mcv.paged_attention_chunk(*a).isfinite().all()


def test_keys_and_values_together(mcv, cuda):
    """A NaN key makes all of the rows that see it NaN, beside values that are not finite before and after it."""
    torch = _torch()
    n, held, page = [90, 20], [40, 3000], 16
    q, k, v, table, lens, cu, _ = _case(3, n, held, 8, 2, 128, page, sharp=0.3)
    k[table[0, 100 // page], 100 % page, 0, 3] = math.nan
    v[table[0, 20 // page], 20 % page, 0, 7] = math.inf
    v[table[0, 110 // page], 110 % page, 0, 9] = -math.inf
    v[table[1, 5 // page], 5 % page, 1, 127] = math.nan
    got = mcv.paged_attention_chunk(*(x.to(cuda) for x in (q, k, v, table, lens, cu))).cpu()
    assert got[60:90, :4].isnan().all() and got[:90, 4:].isfinite().all()
    assert (got[:60, :4, 7] == math.inf).all() and got[90:, :4].isfinite().all() and got[90:, 4:, 127].isnan().all()
    got[:60, :4, 7], got[90:, 4:, 127] = 0, 0
    assert got[:60].isfinite().all() and got[90:].isfinite().all()


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("n,held", [([40], [30]), ([300], [90]), ([700], [0]), ([3, 4], [3000, 5])])
@pytest.mark.parametrize("value", [math.inf, math.nan])
def test_a_key_in_any_part(mcv, cuda, D, n, held, value):
    """A score that is infinite or NaN makes its row NaN in all its d, in whichever part of the cache the key lies, and its
    head's later rows; the other cache head's and earlier rows keep their bits."""
    torch = _torch()
    q, k, v, table, lens, cu, _ = _case(6, n, held, 8, 2, D, 16, sharp=0.1)
    q = q.abs() + 0.01
    a = [x.to(cuda) for x in (q, k, v, table, lens, cu)]
    clean = mcv.paged_attention_chunk(*a).cpu()
    for at in (0, (n[0] + held[0]) // 2, n[0] + held[0] - 2):
        bad = k.clone()
        bad[table[0, at // 16], at % 16, 1, 3] = value
        a[1] = bad.to(cuda)
        got = mcv.paged_attention_chunk(*a).cpu()
        first = max(0, at - held[0])
        assert got[first:n[0], 4:].isnan().all()
        got[first:n[0], 4:] = clean[first:n[0], 4:]
        assert (got == clean).all()


def test_rows_of_no_weight(mcv, cuda):
    """All scores -inf: zeros, whatever V holds; a query that is not finite: its own rows only."""
    torch = _torch()
    for n, held in (([40], [30]), ([3], [3000])):
        q, k, v, table, lens, cu, _ = _case(4, n, held, 4, 2, 64, 16, sharp=0.3)
        a = [x.to(cuda) for x in (q.abs() + 0.01, torch.full_like(k, -math.inf), torch.full_like(v, math.inf), table, lens, cu)]
        assert (mcv.paged_attention_chunk(*a) == 0).all()
        q[n[0] // 2, 1, 5] = math.nan
        got = mcv.paged_attention_chunk(*(x.to(cuda) for x in (q, k, v, table, lens, cu)))
        assert got[n[0] // 2, 1].isnan().all()
        got[n[0] // 2, 1] = 0
        assert got.isfinite().all()


def test_one_sequence_of_many(mcv, cuda):
    """An infinity in one of 90 sequences' caches: the others keep their bits."""
    torch = _torch()
    n, held = [1 + i % 4 for i in range(90)], [(37 * i) % 800 for i in range(90)]
    q, k, v, table, lens, cu, _ = _case(5, n, held, 8, 2, 128, 16, sharp=0.3)
    a = [x.to(cuda) for x in (q, k, v, table, lens, cu)]
    clean = mcv.paged_attention_chunk(*a)
    a[2][table[50, 0].item(), 3, 0, 11] = math.inf
    got = mcv.paged_attention_chunk(*a)
    mine = slice(sum(n[:50]), sum(n[:51]))
    assert (got[mine, :4, 11] == math.inf).all()
    got[mine, :4, 11] = clean[mine, :4, 11]
    assert (got == clean).all()


@pytest.mark.parametrize("D,Hq,Hkv", [(64, 8, 2), (128, 8, 2), (256, 8, 2)])
@pytest.mark.parametrize("n,held", [(64, 40000), (2000, 0)])
def test_time_does_not_grow_with_the_cache(mcv, cuda, D, Hq, Hkv, n, held):
    """An infinity that every row sees costs a second pass over the cache's part that holds it, not one a row."""
    torch = _torch()
    pages = (n + held + 15) // 16
    k, v = (torch.randn(pages, 16, Hkv, D, device=cuda).half() for _ in range(2))
    q = (0.3 * torch.randn(n, Hq, D, device=cuda)).half()
    table, lens = torch.arange(pages, device=cuda).int()[None], torch.tensor([n + held], device=cuda).int()

    def once():
        begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        begin.record()
        out = mcv.paged_attention_chunk(q, k, v, table, lens)
        end.record()
        torch.cuda.synchronize()
        return begin.elapsed_time(end), out

    once()
    usual = sorted(once()[0] for _ in range(5))[2]
    v[0, 5, 0, 3] = math.inf
    got = sorted(once()[0] for _ in range(5))[2]
    assert (once()[1][5 - min(5, held):, :Hq // Hkv, 3] == math.inf).all()
    assert got < 5 * usual + 0.1, (got, usual)

"""GPU tests of paged_attention_chunk with positions: new tokens that are not the last of their sequence's length, as after an
append without room for all of them.  Against the definition in 64 bits with test_gpu_chunk_attention's tolerance: token i of a
sequence sees its first min(place + i + 1, length) tokens."""
import math

import pytest

from test_gpu_chunk_attention import _case, _close, _cu
from test_gpu_mixers import _gen, _torch

pytestmark = pytest.mark.gpu


def _ref(q, kv, n, lens, base, scale):
    torch = _torch()
    T, Hq, D = q.shape
    out, size = (torch.zeros(T, Hq, D, dtype=torch.float64) for _ in range(2))
    first = 0
    for b, (k, v) in enumerate(kv):
        L = lens[b]
        k, v = k[:L].double(), v[:L].double()
        hidden = torch.arange(L) > torch.arange(base[b], base[b] + n[b])[:, None]
        for h in range(Hq if n[b] and L else 0):
            kh, vh = k[:, h * k.shape[1] // Hq], v[:, h * v.shape[1] // Hq]
            w = torch.softmax((q[first:first + n[b], h].double() @ kh.t() * scale).masked_fill(hidden, -math.inf), 1)
            out[first:first + n[b], h] = w @ vh
            size[first:first + n[b], h] = w @ vh.abs()
        first += n[b]
    return out, size


def _positions(n, base, rows, cuda):
    torch = _torch()
    at = [torch.arange(b, b + m) for m, b in zip(n, base)]
    return torch.cat((*at, torch.zeros(rows - sum(n), dtype=torch.int64))).to(cuda)


CASES = [
    # new, tokens held before, tokens of them that have no room, Hq, Hkv, D, page
    ([5], [30], [3], 8, 2, 256, 16),
    ([24], [1100], [20], 8, 2, 256, 16),
    ([1100], [0], [300], 8, 2, 256, 16),
    ([300, 40, 7], [0, 100, 64], [299, 0, 7], 8, 2, 64, 16),
    ([70, 33], [900, 31], [70, 33], 32, 8, 128, 32),
    ([9, 0, 4, 1], [4000, 50, 0, 20], [1, 0, 4, 1], 8, 2, 128, 32),
    ([1] * 5, [15, 16, 64, 3000, 1], [1, 0, 1, 1, 0], 16, 16, 64, 16),
    ([130], [126], [1], 12, 1, 128, 128),
    ([3 + i % 7 for i in range(90)], [11 * i for i in range(90)], [i % 4 for i in range(90)], 4, 2, 64, 16),
]


@pytest.mark.parametrize("n,held,short,Hq,Hkv,D,page", CASES)
def test_without_room_for_all(mcv, cuda, n, held, short, Hq, Hkv, D, page):
    torch = _torch()
    q, k, v, table, lens, cu, kv = _case(len(n) + D, n, held, Hq, Hkv, D, page)
    cut = [m - s for m, s in zip(lens.tolist(), short)]
    a = [x.to(cuda) for x in (q, k, v, table, torch.tensor(cut, dtype=torch.int32), cu)]
    got = mcv.paged_attention_chunk(*a, positions=_positions(n, held, len(q), cuda))
    _close(got, _ref(q, kv, n, cut, held, D ** -0.5))
    assert (mcv.paged_attention_chunk(*a, positions=_positions(n, held, len(q), cuda)) == got).all()


@pytest.mark.parametrize("n,held,short,Hq,Hkv,D,page", CASES)
def test_with_room_for_all(mcv, cuda, n, held, short, Hq, Hkv, D, page):
    """The bits of the call without positions."""
    q, k, v, table, lens, cu, _ = _case(len(n) + D, n, held, Hq, Hkv, D, page)
    a = [x.to(cuda) for x in (q, k, v, table, lens, cu)]
    assert (mcv.paged_attention_chunk(*a, positions=_positions(n, held, len(q), cuda)) == mcv.paged_attention_chunk(*a)).all()


def test_before_the_last_tokens(mcv, cuda):
    """Places inside a longer sequence, with rows of no sequence around, equal shares, and places that are out of range."""
    torch = _torch()
    n, held = [20, 20, 20], [300, 40, 0]
    q, k, v, table, lens, cu, kv = _case(5, n, held, 8, 2, 128, 16)
    base = [100, 3, 0]
    a = [x.to(cuda) for x in (q, k, v, table, lens)]
    want = _ref(q, kv, n, lens.tolist(), base, 128 ** -0.5)
    _close(mcv.paged_attention_chunk(*a, cu.to(cuda), positions=_positions(n, base, 60, cuda)), want)
    _close(mcv.paged_attention_chunk(*a, positions=_positions(n, base, 60, cuda)), want)
    wide = torch.cat((q[:4], q, q[:3]))
    out = torch.full_like(wide, 7.0).to(cuda)
    at = torch.cat((torch.full((4,), -1), _positions(n, base, 60, "cpu"), torch.full((3,), -1)))
    mcv.paged_attention_chunk(wide.to(cuda), *a[1:], (cu + 4).to(cuda), positions=at.to(cuda), out=out)
    _close(out[4:-3], want)
    assert (out[:4] == 7).all() and (out[-3:] == 7).all()
    far = _positions(n, base, 60, "cpu")
    far[0], far[20], far[40] = 2 ** 40, -5, -2 ** 62             # all of the sequence; from its first token on
    _close(mcv.paged_attention_chunk(*a, positions=far.to(cuda)), _ref(q, kv, n, lens.tolist(), [320, 0, 0], 128 ** -0.5))


@pytest.mark.parametrize("pages,width", [(9, 8), (40, 3)])
def test_after_an_append_that_fell_short(mcv, cuda, pages, width):
    """Too few pages, or full table rows: the tokens that had room attend as if the others had not been there."""
    torch = _torch()
    page, Hq, Hkv, D = 16, 8, 2, 64
    n, before = [5, 60, 20, 30], [30, 10, 40, 0]
    free = torch.randperm(pages, generator=_gen(3)).int().to(cuda)
    count = torch.tensor([pages], dtype=torch.int32, device=cuda)
    table = torch.full((4, width), -1, dtype=torch.int32, device=cuda)
    lens = torch.zeros(4, dtype=torch.int32, device=cuda)
    kc, vc = (torch.zeros(pages, page, Hkv, D, dtype=torch.float16, device=cuda) for _ in range(2))
    kv = [[torch.zeros(0, Hkv, D).half()] * 2 for _ in n]
    for m in (before, n):
        T = sum(m)
        cu = _cu(m).to(cuda)
        base = lens.tolist()
        slots, places, _ = mcv.paged_append(table, lens, cu, page, tokens=T, free_pages=free, free_count=count)
        q, k, v = (torch.randn(T, h, D, generator=_gen(T + i)).half() for i, h in enumerate((Hq, Hkv, Hkv)))
        live = slots.cpu() >= 0
        for cache, new in ((kc, k), (vc, v)):
            cache.view(-1, Hkv, D)[slots[slots >= 0]] = new[live].to(cuda)
        for b in range(4):
            rows = slice(int(cu[b]), int(cu[b + 1]))
            kv[b] = [torch.cat((old, new[rows][live[rows]])) for old, new in zip(kv[b], (k, v))]
        assert lens.tolist() == [len(x) for x, _ in kv]
        got = mcv.paged_attention_chunk(q.to(cuda), kc, vc, table, lens, cu, positions=places)
        _close(got, _ref(q, kv, m, lens.tolist(), base, D ** -0.5))
    assert not live.all()

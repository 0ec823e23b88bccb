"""GPU tests of the attention of chunks of new tokens (paged_attention_chunk) against its definition in 64 bits.

Tolerances.  A rounding to fp16 is off by at most H = 2^-11 of the value: one of the output, one of each softmax weight,
counted against the sum of the magnitudes that the weights enter.  The rounded weights are what the softmax's sum adds up, so
that they sum to one: with weights w (1 + d), |d| <= H, the quotient sum w (1 + d) v / sum w (1 + d) is off from o = sum w v /
sum w by sum w d (v - o) / sum w (1 + d), at most H (sum w |v| / sum w + |o|) to first order.  Scores, the softmax's sums and the products' sums are in
32 bits: a score, a sum of D products in blocks, moves its weight by 2^-17 at the sizes used here; weights below
2^-14 in fp16, which begin 2^-29 below the row's largest, are off by up to 2^-40 of it each."""
import math

import pytest

from test_gpu_mixers import _attn_case, _gen, _torch

pytestmark = pytest.mark.gpu

H = 2.0 ** -11


def _case(seed, n, held, Hq, Hkv, D, page, sharp=2.0, width=None):
    """q [sum n, Hq, D] with caches, table and lengths, and the tokens' k and v of each sequence."""
    torch = _torch()
    lens = [a + b for a, b in zip(n, held)]
    _, k, v, table, length, kv = _attn_case(seed, lens, Hq, Hkv, D, page, width)
    q = (sharp * torch.randn(sum(n), Hq, D, generator=_gen(seed + 1))).half()
    return q, k, v, table, length, _cu(n), kv


def _cu(n):
    torch = _torch()
    return torch.tensor([0, *torch.tensor(n).cumsum(0).tolist()], dtype=torch.int32)


def _ref(q, kv, n, lens, scale, live=None):
    """out and the magnitudes its sums run over; lens: lengths as the call has them."""
    torch = _torch()
    T, Hq, D = q.shape
    out, size = torch.zeros(T, Hq, D, dtype=torch.float64), torch.zeros(T, Hq, D, dtype=torch.float64)
    first = 0
    for b, (k, v) in enumerate(kv):
        L = lens[b]
        k, v = k[:L].double(), v[:L].double()
        place = torch.arange(L - n[b], L)[:, None]
        hidden = torch.arange(L) > place
        if live is not None:
            hidden = hidden | ~live[b][:L]
            v = torch.where(live[b][:L, None, None], v, 0)
            k = torch.where(live[b][:L, None, None], k, 0)
        for h in range(Hq if n[b] and L else 0):
            kh, vh = k[:, h * k.shape[1] // Hq], v[:, h * v.shape[1] // Hq]
            s = (q[first:first + n[b], h].double() @ kh.t() * scale).masked_fill(hidden, -math.inf)
            w = torch.exp(s - s.amax(1, keepdim=True).clamp_min(-1e300))
            w = w / w.sum(1, keepdim=True).clamp_min(1e-300)
            out[first:first + n[b], h] = w @ vh
            size[first:first + n[b], h] = w @ vh.abs()
        first += n[b]
    return out, size


def _close(got, ref):
    want, size = ref
    err = (got.cpu().double() - want).abs()
    bound = 2 * H * want.abs() + (H + 2.0 ** -17) * size + 2.0 ** -24          # |o| of the weights' and of the output's rounding
    assert (err <= bound).all(), ((err - bound).max(), err.argmax())
    # the two roundings' spread: each uniform in its half step (0.42 H rms), independent over weights
    spread = 1.5 * 0.6 * H * want.norm() + 2.0 ** -25 * want.numel() ** 0.5
    assert err.norm() <= spread, err.norm() / spread


CASES = [
    # new, held, Hq, Hkv, D, page
    ([1], [0], 1, 1, 64, 16),
    ([1], [1], 8, 2, 256, 16),
    ([2], [0], 8, 2, 256, 16),
    ([24], [1100], 8, 2, 256, 16),
    ([31], [2], 8, 2, 256, 16),
    ([32], [0], 8, 2, 256, 32),
    ([33], [64], 8, 2, 256, 64),
    ([64], [63], 16, 16, 64, 16),
    ([65], [191], 16, 16, 64, 48),
    ([129], [0], 32, 8, 128, 16),
    ([300], [0], 8, 2, 256, 16),
    ([1100], [0], 8, 2, 256, 16),
    ([700], [900], 12, 1, 128, 128),
    ([77], [3000], 7, 1, 64, 32),
    ([5], [4097], 40, 1, 128, 16),
    ([3], [500], 130, 1, 64, 16),
    ([1, 0, 5, 40, 0, 1, 128], [10, 20, 0, 700, 0, 3000, 0], 8, 2, 256, 32),
    ([0, 0, 17], [100, 0, 1], 32, 8, 128, 16),
    ([1] * 9, [0, 1, 15, 16, 62, 63, 64, 65, 2000], 32, 8, 128, 16),
    ([200, 300, 1], [0, 50, 1000], 6, 3, 128, 16),
    ([4], [20000], 8, 2, 256, 64),
    ([70], [9000], 4, 2, 128, 32),
]


@pytest.mark.parametrize("n,held,Hq,Hkv,D,page", CASES)
def test_chunk(mcv, cuda, n, held, Hq, Hkv, D, page):
    q, k, v, table, lens, cu, kv = _case(len(n) + D, n, held, Hq, Hkv, D, page)
    a = [x.to(cuda) for x in (q, k, v, table, lens, cu)]
    got = mcv.paged_attention_chunk(*a)
    _close(got, _ref(q, kv, n, lens.tolist(), D ** -0.5))
    assert (mcv.paged_attention_chunk(*a) == got).all()          # the same bits: joined in one order
    tight = mcv.paged_attention_chunk(*a, scale=0.05, max_seq_len=int(lens.max()), out=got)
    assert tight is got
    _close(got, _ref(q, kv, n, lens.tolist(), 0.05))


@pytest.mark.parametrize("B,new,longest,Hq,Hkv,D,page", [(150, 12, 900, 4, 2, 64, 16), (65, 3, 3000, 8, 1, 128, 32), (300, 1, 40, 6, 3, 256, 16),
                                                         (64, 40, 700, 20, 1, 128, 16), (129, 9, 130, 16, 8, 64, 16)])
def test_many_sequences(mcv, cuda, B, new, longest, Hq, Hkv, D, page):
    """More sequences than lanes of a wave, some of none: cut in parts, whole, and both together."""
    torch = _torch()
    held = (torch.rand(B, generator=_gen(B)) ** 3 * (longest + 1)).int()
    held[0], held[B // 2], held[-1] = 0, longest, longest - 1
    n = (torch.rand(B, generator=_gen(B + 1)) * (new + 1)).int()
    n[0], n[B // 2], n[-1] = new, new, 0
    q, k, v, table, lens, cu, kv = _case(B + D, n.tolist(), held.tolist(), Hq, Hkv, D, page)
    got = mcv.paged_attention_chunk(*(x.to(cuda) for x in (q, k, v, table, lens, cu)))
    _close(got, _ref(q, kv, n.tolist(), lens.tolist(), D ** -0.5))


def test_equal_chunks_without_cu(mcv, cuda):
    q, k, v, table, lens, cu, kv = _case(2, [5] * 7, [9, 0, 100, 33, 64, 1, 700], 8, 2, 128, 16)
    a = [x.to(cuda) for x in (q, k, v, table, lens)]
    got = mcv.paged_attention_chunk(*a)
    assert (got == mcv.paged_attention_chunk(*a, cu.to(cuda))).all()
    _close(got, _ref(q, kv, [5] * 7, lens.tolist(), 128 ** -0.5))


def test_one_token_each_is_the_decoding_call(mcv, cuda):
    q, k, v, table, lens, _, kv = _case(3, [1] * 5, [3, 900, 0, 64, 31], 8, 2, 256, 16)
    a = [x.to(cuda) for x in (q, k, v, table, lens)]
    ref = _ref(q, kv, [1] * 5, lens.tolist(), 1 / 16)
    _close(mcv.paged_attention_chunk(*a), ref)
    _close(mcv.paged_attention_decode(*a), ref)


def test_rows_of_no_sequence_stay(mcv, cuda):
    """Rows before the first sequence, behind the last one and of a batch whose offsets are out of range."""
    torch = _torch()
    n, held = [40, 3], [0, 70]
    q, k, v, table, lens, cu, kv = _case(4, n, held, 8, 2, 128, 16)
    wide = torch.randn(60, 8, 128, generator=_gen(1)).half()
    wide[7:50] = q
    out = torch.full((60, 8, 128), 7.0, dtype=torch.float16, device=cuda)
    a = [x.to(cuda) for x in (wide, k, v, table, lens)]
    mcv.paged_attention_chunk(*a, (cu + 7).to(cuda), out=out)
    assert (out[:7] == 7).all() and (out[50:] == 7).all()
    _close(out[7:50], _ref(q, kv, n, lens.tolist(), 128 ** -0.5))
    out.fill_(7)
    mcv.paged_attention_chunk(*a, torch.tensor([-5, 7, 10 ** 9], dtype=torch.int32, device=cuda), out=out)      # 0, 7, 60
    # of 53 new rows the second sequence's 73 tokens are enough; the first's 40 are for 7
    want = _ref(wide, kv, [7, 53], lens.tolist(), 128 ** -0.5)
    _close(out, want)
    out.fill_(7)
    mcv.paged_attention_chunk(*a, torch.tensor([30, 20, 10], dtype=torch.int32, device=cuda), out=out)          # descending: no rows
    assert (out == 7).all()


def test_rows_before_the_first_token(mcv, cuda):
    """A length shorter than the new tokens: the first rows see nothing and are zero."""
    n, held = [50, 6, 200], [0, 0, 0]
    q, k, v, table, lens, cu, kv = _case(5, n, held, 8, 2, 64, 16)
    lens[0], lens[1], lens[2] = 20, 0, 199
    got = mcv.paged_attention_chunk(*(x.to(cuda) for x in (q, k, v, table, lens, cu)))
    _close(got, _ref(q, kv, n, lens.tolist(), 0.125))
    assert (got[:30] == 0).all() and (got[50:57] == 0).all() and (got[30] != 0).any() and (got[57] != 0).any()


def test_lengths_out_of_range(mcv, cuda):
    torch = _torch()
    n, held = [8, 8, 8], [56, 56, 56]
    q, k, v, table, lens, cu, kv = _case(6, n, held, 4, 1, 64, 16)
    a = [x.to(cuda) for x in (q, k, v, table, torch.tensor([10 ** 9, -5, 50], dtype=torch.int32), cu)]
    _close(mcv.paged_attention_chunk(*a), _ref(q, kv, n, [64, 0, 50], 0.125))
    _close(mcv.paged_attention_chunk(*a, max_seq_len=33), _ref(q, kv, n, [33, 0, 33], 0.125))
    assert (mcv.paged_attention_chunk(*a, max_seq_len=0) == 0).all()
    assert (mcv.paged_attention_chunk(*a, max_seq_len=2 ** 40) == mcv.paged_attention_chunk(*a)).all()


@pytest.mark.parametrize("D,page", [(64, 16), (128, 32), (256, 16)])
def test_absent_pages(mcv, cuda, D, page):
    """Page numbers outside the cache are left out, wherever they stand; rows that see none are zero."""
    torch = _torch()
    n, held = [90, 40, 33], [600, 0, 0]
    q, k, v, table, lens, cu, kv = _case(7, n, held, 8, 2, D, page)
    live = [torch.ones(m, dtype=torch.bool) for m in lens.tolist()]
    for b, i, bad in [(0, 0, -1), (0, 5, k.shape[0]), (0, 620 // page, 2 ** 31 - 1), (1, 0, -2 ** 31)] + [(2, i, -1 - i) for i in range(-(-33 // page))]:
        table[b, i] = bad
        live[b][i * page:(i + 1) * page] = False
    got = mcv.paged_attention_chunk(*(x.to(cuda) for x in (q, k, v, table, lens, cu)))
    _close(got, _ref(q, kv, n, lens.tolist(), D ** -0.5, live))
    assert (got[130:] == 0).all() and (got[90:90 + page] == 0).all()


def test_orders(mcv, cuda):
    """Caches in another order, k and v in one pool, q as columns of a wider row, one table for all sequences."""
    torch = _torch()
    n, held = [30, 4, 64], [40, 196, 64]
    q, k, v, table, lens, cu, kv = _case(8, n, held, 8, 4, 64, 32)
    want = _ref(q, kv, n, lens.tolist(), 0.125)
    wide = torch.zeros(98, 8, 2, 64).half()
    wide[:, :, 0] = q
    both = torch.stack((k, v), 1).permute(0, 1, 3, 2, 4).contiguous().to(cuda)         # [pages, 2, Hkv, page, D]
    got = mcv.paged_attention_chunk(wide.to(cuda)[:, :, 0], both[:, 0].permute(0, 2, 1, 3), both[:, 1].permute(0, 2, 1, 3),
                                    table.to(cuda), lens.to(cuda), cu.to(cuda))
    _close(got, want)
    # a common beginning, continued differently: two sequences over one row of pages
    got = mcv.paged_attention_chunk(*(x.to(cuda) for x in (q[34:], k, v)), table[2:].to(cuda).expand(2, -1),
                                    torch.tensor([100, 128], dtype=torch.int32, device=cuda), torch.tensor([0, 36, 64], dtype=torch.int32, device=cuda))
    _close(got, _ref(q[34:], [kv[2], kv[2]], [36, 28], [100, 128], 0.125))


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("n,held", [([70], [0]), ([3], [2000]), ([40, 20], [30, 900])])
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
def test_not_finite_values_reach_those_that_see_them(mcv, cuda, D, n, held, value):
    """One V of the last sequence's middle new token: rows before it are as if it were not there."""
    torch = _torch()
    q, k, v, table, lens, cu, kv = _case(9, n, held, 8, 2, D, 16)
    at = held[-1] + n[-1] // 2
    page, place = table[-1, at // 16].item(), at % 16
    a = [x.to(cuda) for x in (q, k, v, table, lens, cu)]
    clean = mcv.paged_attention_chunk(*a)
    v[page, place, 1, 5] = value
    a[2] = v.to(cuda)
    got = mcv.paged_attention_chunk(*a)
    sees = torch.zeros(sum(n), dtype=torch.bool)
    sees[sum(n) - n[-1] + n[-1] // 2:] = True
    hit = got[sees.to(cuda)][:, 4:, 5].cpu()                     # the second cache head's query heads
    assert torch.isnan(hit).all() if math.isnan(value) else (hit == value).all()
    got[sees.to(cuda), 4:, 5] = 0
    assert torch.isfinite(got).all()
    # the rows that were done over are other sums of the same values
    ref = _ref(q, kv, n, lens.tolist(), D ** -0.5)
    got[sees.to(cuda), 4:, 5] = clean[sees.to(cuda), 4:, 5]
    _close(got, ref)


def test_not_finite_keys(mcv, cuda):
    """A NaN key reaches the rows that see it; a score of -inf weighs nothing, wherever it stands."""
    torch = _torch()
    n, held = [70], [100]
    q, k, v, table, lens, cu, kv = _case(10, n, held, 8, 2, 64, 16)
    q = q.abs() + 0.01
    bad = k.clone()
    bad[table[0, 130 // 16], 130 % 16, 0, 3] = math.nan
    got = mcv.paged_attention_chunk(*(x.to(cuda) for x in (q, bad, v, table, lens, cu)))
    assert torch.isnan(got[30:, :4]).all() and torch.isfinite(got[:30]).all() and torch.isfinite(got[:, 4:]).all()
    live = [torch.ones(170, dtype=torch.bool)]
    for t in (0, 5, 64, 65, 120, 150, *range(96, 112)):
        bad = bad if t else k.clone()
        bad[table[0, t // 16], t % 16] = -math.inf
        live[0][t] = False
    got = mcv.paged_attention_chunk(*(x.to(cuda) for x in (q, bad, v, table, lens, cu)))
    _close(got, _ref(q, kv, n, [170], 0.125, live))


def test_one_token_far_above_the_others(mcv, cuda):
    """Its v is zero, so that what is left is the others' small weights, down to 2^-24 of the largest."""
    torch = _torch()
    for far in (10.0, 16.0):
        q, k, v, table, lens, cu, kv = _case(11, [40], [4096], 4, 1, 64, 16, sharp=0.0)
        q[..., 0] = 1.0
        for t, (kk, vv) in [(7, kv[0])]:
            k[..., 0], kk[..., 0] = 0.0, 0.0
            k[table[0, 0], 7, 0, 0] = kk[t, 0, 0] = far
            v[table[0, 0], 7] = vv[t] = 0.0
        got = mcv.paged_attention_chunk(*(x.to(cuda) for x in (q, k, v, table, lens, cu)), scale=1.0)
        want, size = _ref(q, kv, [40], [4136], 1.0)
        err = (got.cpu().double() - want).abs()
        assert (err <= 2 * H * want.abs() + (H + 2.0 ** -17) * size + 2.0 ** -24).all()


def test_large_scores(mcv, cuda):
    """Scores of some thousands, growing and falling along the cache: no overflow, and every rise of the maximum counted."""
    torch = _torch()
    for rising in (1.0, -1.0):
        q, k, v, table, lens, cu, kv = _case(12, [70], [500], 8, 2, 128, 16, sharp=0.0)
        q[..., 1] = 1.0
        for t in range(570):
            kv[0][0][t, :, 1] = rising * 8.0 * (t // 3)
            k[table[0, t // 16], t % 16, :, 1] = rising * 8.0 * (t // 3)
        got = mcv.paged_attention_chunk(*(x.to(cuda) for x in (q, k, v, table, lens, cu)), scale=1.0)
        _close(got, _ref(q, kv, [70], [570], 1.0))


def test_far_offsets(mcv, cuda):
    """Pages past 2^32 bytes, and strides that put neighbouring tokens far apart."""
    torch = _torch()
    D, page = 64, 16
    q, k, v, table, lens, cu, kv = _case(13, [20], [100], 2, 1, D, page)
    step = 1 << 25                                               # elements: tokens 64 MiB apart, pages 1 GiB
    flat = torch.zeros(5 * page * step, dtype=torch.float16, device=cuda)
    pages = [0, 4, 2]
    views = [flat.as_strided((5, page, 1, D), (page * step, step, D, 1), off) for off in (0, 4096)]
    for cache, src in zip(views, (k, v)):
        for t in range(48):
            cache[pages[t // page], t % page] = src[table[0, t // page], t % page].to(cuda)
    far = torch.tensor([pages], dtype=torch.int32, device=cuda)
    n = torch.tensor([48], dtype=torch.int32, device=cuda)
    got = mcv.paged_attention_chunk(q.to(cuda), *views, far, n)
    _close(got, _ref(q, kv, [20], [48], D ** -0.5))


def test_nothing_to_do(mcv, cuda):
    torch = _torch()
    half = lambda *s: torch.zeros(*s, dtype=torch.float16, device=cuda)      # noqa: E731
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device=cuda)         # noqa: E731
    cache = half(5, 16, 2, 64)
    assert mcv.paged_attention_chunk(half(0, 8, 64), cache, cache, i32(0, 4), i32(0)).shape == (0, 8, 64)
    assert mcv.paged_attention_chunk(half(0, 8, 64), cache, cache, i32(3, 4), i32(3), i32(4)).shape == (0, 8, 64)
    held = half(6, 8, 64) + 1
    assert mcv.paged_attention_chunk(half(6, 8, 64), cache, cache, i32(3, 4), i32(3), i32(4), out=held) is held and (held == 1).all()
    with pytest.raises(mcv.McvError, match="paged_attention_chunk"):
        mcv.paged_attention_chunk(half(0, 8, 96), half(5, 16, 2, 96), half(5, 16, 2, 96), i32(0, 4), i32(0))


def test_on_another_stream(mcv, cuda):
    torch = _torch()
    side = torch.cuda.Stream()
    a = [x.to(cuda) for x in _case(14, [100, 3], [0, 5000], 8, 2, 128, 32)[:6]]
    torch.cuda.synchronize()
    want = mcv.paged_attention_chunk(*a)
    torch.cuda.synchronize()
    got = mcv.paged_attention_chunk(*a, stream=side)
    side.synchronize()
    assert (got == want).all()


def test_in_a_graph(mcv, cuda):
    """Captured once, replayed with other inputs and lengths in the same buffers, eager calls between."""
    torch = _torch()
    cases = [_case(s, n, held, 8, 2, 128, 32, width=170)[:6] for s, n, held in ((1, [60, 4], [0, 5000]), (2, [1, 63], [77, 300]))]
    pool = max(c[1].shape[0] for c in cases)
    cases = [[x.to(cuda) for x in (c[0], *(torch.cat((t, t.new_zeros(pool - t.shape[0], *t.shape[1:]))) for t in c[1:3]), *c[3:])] for c in cases]
    hold = [x.clone() for x in cases[0]]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = mcv.paged_attention_chunk(*hold)
    for turn in (0, 1, 0, 1):
        want = mcv.paged_attention_chunk(*cases[turn])
        for x, y in zip(hold, cases[turn]):
            x.copy_(y)
        graph.replay()
        torch.cuda.synchronize()
        assert (got == want).all(), turn

"""GPU tests of the token mixers (include/mcv_mixers.h) against their definitions in 64 bits.

Tolerances.  A rounding to fp16 is off by at most 2^-11 of the value (H below), one
to two fp16 parts by 2^-22.  Every output is one rounding of 32-bit arithmetic, plus,
where a product runs on fp16 matrix operands, one rounding per rounded operand,
counted against the sum of the magnitudes that it enters."""
import math

import pytest

pytestmark = pytest.mark.gpu

H = 2.0 ** -11


def _torch():
    import torch
    return torch


def _gen(seed):
    return _torch().Generator().manual_seed(seed)


# ------------------------------------------------------------ gated delta rule --
def _delta_ref(q, k, v, g, beta, state, lens, scale, normalize):
    """out, the magnitudes its sums run over, and the final states, token by token in 64 bits."""
    torch = _torch()
    q, k, v, g, beta = (x.double() for x in (q, k, v, g, beta))
    if normalize:
        q, k = (x / (x.square().sum(-1, keepdim=True) + 1e-6).sqrt() for x in (q, k))
    r = v.shape[1] // k.shape[1]
    q, k = q.repeat_interleave(r, 1), k.repeat_interleave(r, 1)
    out, size, states, t = torch.zeros_like(v), torch.zeros_like(v), [], 0
    for b, n in enumerate(lens):
        S = state[b].double().clone()
        A = S.abs()
        for _ in range(n):
            e = g[t].exp()[:, None, None]
            S, A = e * S, e * A
            u = (v[t] - (S * k[t][..., None]).sum(1)) * beta[t][:, None]
            S = S + k[t][..., None] * u[:, None]
            A = A + k[t].abs()[..., None] * u.abs()[:, None]
            out[t] = scale * (S * q[t][..., None]).sum(1)
            size[t] = scale * (A * q[t].abs()[..., None]).sum(1)
            t += 1
        states.append(S)
    return out, size, torch.stack(states)


def _delta_case(seed, lens, Hk, Hv, Dk, Dv, lean=0.5, rate=1.0):
    torch = _torch()
    gen = _gen(seed)
    T, B = sum(lens), len(lens)
    qkv = torch.randn(T, 2 * Hk * Dk + Hv * Dv, generator=gen)
    qkv[:, Hk * Dk:2 * Hk * Dk] += lean * torch.randn(1, Hk * Dk, generator=gen)
    qkv = qkv.half()
    q = qkv[:, :Hk * Dk].view(T, Hk, Dk)
    k = qkv[:, Hk * Dk:2 * Hk * Dk].view(T, Hk, Dk)
    v = qkv[:, 2 * Hk * Dk:].view(T, Hv, Dv)
    g = -rate * torch.rand(Hv, generator=gen) * torch.nn.functional.softplus(torch.randn(T, Hv, generator=gen) - 2)
    beta = torch.sigmoid(torch.randn(T, Hv, generator=gen))
    state = 0.3 * torch.randn(B, Hv, Dk, Dv, generator=gen)
    return q, k, v, g, beta, state


def _delta_close(out, state, ref, what=""):
    torch = _torch()
    want, size, S = ref
    err = (out.cpu().double() - want).abs()
    # one rounding of out; the rounded state, scores and corrected values of a chunk
    assert (err <= H * want.abs() + 3 * H * size + 2.0 ** -24).all(), (what, (err - H * want.abs() - 3 * H * size).max())
    if want.numel():
        # the four roundings' spread: each uniform in its half step (0.42 H rms), added in quadrature 0.84 H; below
        # 2^-14 fp16's half step is 2^-25 whatever the value
        spread = 1.5 * H * want.norm() + 2.0 ** -25 * want.numel() ** 0.5
        assert err.norm() <= spread, (what, err.norm() / spread)
    # two fp16 parts of each operand, four operands on a path, 32-bit sums
    e = (state.cpu().double() - S).norm() / S.norm().clamp_min(1e-30)
    assert e <= 16 * 2.0 ** -22, (what, e)


def _cu(lens, device):
    torch = _torch()
    return torch.tensor([0, *torch.tensor(lens).cumsum(0).tolist()], dtype=torch.int32, device=device)


DELTA = [
    # lens, Hk, Hv, Dk, Dv
    ([1], 1, 1, 64, 16),
    ([1], 16, 16, 128, 128),
    ([2, 0, 1], 2, 4, 128, 64),
    ([63], 2, 2, 64, 64),
    ([64], 2, 2, 128, 128),
    ([65], 1, 3, 128, 48),
    ([0, 77, 1, 200, 64, 0], 2, 4, 128, 128),
    ([300, 5], 3, 3, 64, 256),
    ([129, 127], 2, 2, 128, 32),
    ([1000], 1, 2, 128, 128),
]


@pytest.mark.parametrize("lens,Hk,Hv,Dk,Dv", DELTA)
@pytest.mark.parametrize("normalize", [True, False])
def test_delta_rule(mcv, cuda, lens, Hk, Hv, Dk, Dv, normalize):
    q, k, v, g, beta, state = _delta_case(sum(lens) + Hv, lens, Hk, Hv, Dk, Dv)
    if not normalize:
        k = k / 8 / Dk ** 0.5 * 4
    scale = 0.7 / Dk ** 0.5
    ref = _delta_ref(q, k, v, g, beta, state, lens, scale, normalize)
    a = [x.to(cuda) for x in (q, k, v, g, beta, state)]
    keep = a[5].clone()
    out, final = mcv.gated_delta_rule(*a, cu_seqlens=_cu(lens, cuda), scale=scale, normalize=normalize)
    assert (a[5] == keep).all()
    _delta_close(out, final, ref)
    out2, same = mcv.gated_delta_rule(*a, cu_seqlens=_cu(lens, cuda), scale=scale, normalize=normalize, state_out=a[5])
    assert same is a[5] and (same == final).all() and (out2 == out).all()          # in place, and the same bits


@pytest.mark.parametrize("B,Hk,Hv,Dk,Dv", [(1, 16, 16, 128, 128), (3, 2, 4, 64, 64), (37, 4, 4, 128, 128), (300, 2, 4, 128, 16)])
def test_delta_step(mcv, cuda, B, Hk, Hv, Dk, Dv):
    q, k, v, g, beta, state = _delta_case(B, [1] * B, Hk, Hv, Dk, Dv)
    ref = _delta_ref(q, k, v, g, beta, state, [1] * B, Dk ** -0.5, True)
    a = [x.to(cuda) for x in (q, k, v, g, beta, state)]
    out, final = mcv.gated_delta_rule_step(*a, normalize=True)
    assert final is a[5]
    _delta_close(out, final, ref)


def test_delta_step_of_a_pool(mcv, cuda):
    """Sequences at rows of a pool in any order, one of them absent."""
    torch = _torch()
    B, pool = 5, 9
    q, k, v, g, beta, state = _delta_case(5, [1] * B, 2, 2, 128, 64)
    index = torch.tensor([7, 0, -1, 8, 9], dtype=torch.int32)
    states = torch.randn(pool, 2, 128, 64, generator=_gen(1))
    for b, i in enumerate(index.tolist()):
        if 0 <= i < pool:
            states[i] = state[b]
    ref = _delta_ref(q, k, v, g, beta, state, [1] * B, 128 ** -0.5, True)
    a = [x.to(cuda) for x in (q, k, v, g, beta)]
    dev = states.to(cuda)
    out, final = mcv.gated_delta_rule_step(*a, dev, normalize=True, state_index=index.to(cuda))
    assert final is dev
    on = [0, 1, 3]
    got = dev[index[on].long().to(cuda)]
    _delta_close(out[on], got, tuple(x[on] for x in ref))
    assert (out[[2, 4]] == 0).all()
    rest = [i for i in range(pool) if i not in index[on].tolist()]
    assert (dev.cpu()[rest] == states[rest]).all()


@pytest.mark.parametrize("B,longest", [(64, 90), (65, 70), (130, 40), (700, 30)])
def test_delta_many_sequences(mcv, cuda, B, longest):
    """More sequences than lanes of a wave, some empty, with tokens before the first and behind the last."""
    torch = _torch()
    lens = (torch.rand(B, generator=_gen(B)) * (longest + 1)).int().tolist()
    lens[0], lens[B // 2], lens[-1] = longest, 0, 65
    q, k, v, g, beta, state = _delta_case(B, [3, *lens, 5], 1, 2, 64, 32)
    rows = slice(3, 3 + sum(lens))
    ref = _delta_ref(*(x[rows] for x in (q, k, v, g, beta)), state[1:-1], lens, 0.125, True)
    cu = 3 + _cu(lens, cuda)
    a = [x.to(cuda) for x in (q, k, v, g, beta)]
    out = torch.full(v.shape, 7.0, dtype=torch.float16, device=cuda)
    _, final = mcv.gated_delta_rule(*a, state[1:-1].to(cuda), cu_seqlens=cu, scale=0.125, normalize=True, out=out)
    _delta_close(out[rows], final, ref)
    assert (out[:3] == 7).all() and (out[rows.stop:] == 7).all()


@pytest.mark.parametrize("lens", [[1] * 20 + [90] + [1] * 20, [0, 3, 9, 10, 11, 64, 65, 200, 2, 1] * 2, [1, 1, 30], [0] * 17 + [300],
                                  [5, 0, 0, 0, 0, 0, 80], [2] * 30, [6] * 30, [1] * 16 + [63]])
def test_delta_short_and_long_together(mcv, cuda, lens):
    """Sequences of one token beside whole prompts, on either side of every rule's border; a pool with one state absent."""
    torch = _torch()
    B = len(lens)
    q, k, v, g, beta, state = _delta_case(B + sum(lens), lens, 2, 4, 128, 64)
    a = [x.to(cuda) for x in (q, k, v, g, beta, state)]
    ref = _delta_ref(q, k, v, g, beta, state, lens, 0.1, True)
    out, final = mcv.gated_delta_rule(*a, cu_seqlens=_cu(lens, cuda), scale=0.1, normalize=True)
    _delta_close(out, final, ref)
    index = torch.arange(B - 1, -1, -1, dtype=torch.int32)
    index[B // 2] = -1
    pool = state.flip(0).contiguous().to(cuda)
    out2, same = mcv.gated_delta_rule(*a[:5], pool, cu_seqlens=_cu(lens, cuda), scale=0.1, normalize=True, state_index=index.to(cuda))
    on = [b for b in range(B) if b != B // 2]
    rows = torch.repeat_interleave(torch.arange(B), torch.tensor(lens)).to(cuda)
    assert same is pool and (pool.flip(0)[on] == final[on]).all() and (pool.flip(0)[B // 2].cpu() == state[B // 2]).all()
    assert (out2[rows != B // 2] == out[rows != B // 2]).all() and (out2[rows == B // 2] == 0).all()


def test_delta_in_several_passes(mcv, cuda):
    """So many heads that the workspace holds a few chunks at a time: sequences across its passes, and between them."""
    lens = [300, 0, 900, 40, 260]
    q, k, v, g, beta, state = _delta_case(12, lens, 256, 256, 64, 16)
    assert mcv.lib().mcv_delta_rule_workspace_bytes(5, 1500, 256, 256, 64, 16) < mcv.lib().mcv_delta_rule_workspace_bytes(1, 64, 256, 256, 64, 16) * 14
    ref = _delta_ref(q, k, v, g, beta, state, lens, 0.125, True)
    out, final = mcv.gated_delta_rule(*(x.to(cuda) for x in (q, k, v, g, beta, state)), cu_seqlens=_cu(lens, cuda), scale=0.125,
                                      normalize=True)
    _delta_close(out, final, ref)


def test_delta_pool_over_sequences(mcv, cuda):
    """Whole sequences at rows of a pool, one absent (its outputs zero), one without tokens; then into another pool."""
    torch = _torch()
    lens, index, pool = [70, 33, 0, 150], [5, 8, 2, 0], 8
    q, k, v, g, beta, state = _delta_case(13, lens, 2, 2, 128, 64)
    states = torch.randn(pool, 2, 128, 64, generator=_gen(2))
    for b, i in enumerate(index):
        if i < pool:
            states[i] = state[b]
    ref = _delta_ref(q, k, v, g, beta, state, lens, 128 ** -0.5, True)
    a = [x.to(cuda) for x in (q, k, v, g, beta)]
    where = dict(cu_seqlens=_cu(lens, cuda), state_index=torch.tensor(index, dtype=torch.int32, device=cuda), normalize=True)
    other = torch.full_like(states, 3.0).to(cuda)
    dev = states.to(cuda)
    out, final = mcv.gated_delta_rule(*a, dev, state_out=other, **where)
    assert final is other and (dev.cpu() == states).all()
    out2, same = mcv.gated_delta_rule(*a, dev, **where)
    assert same is dev and (out2 == out).all()
    on = [0, 2, 3]
    rows = torch.tensor([i for b, n in enumerate(lens) for i in [b] * n])
    rows_on = rows != 1
    for got in (other, dev):
        _delta_close(out[rows_on.to(cuda)], got[[index[b] for b in on]], (ref[0][rows_on], ref[1][rows_on], ref[2][on]))
    assert (out[(rows == 1).to(cuda)] == 0).all()
    rest = [i for i in range(pool) if i not in index]
    assert (dev.cpu()[rest] == states[rest]).all() and (other[rest] == 3).all()


def test_delta_no_tokens(mcv, cuda):
    torch = _torch()
    q, k, v, g, beta, state = (x.to(cuda) for x in _delta_case(14, [0, 0], 2, 2, 64, 32))
    out, final = mcv.gated_delta_rule(q, k, v, g, beta, state, cu_seqlens=torch.zeros(3, dtype=torch.int32, device=cuda))
    assert out.shape == (0, 2, 32) and (final == state).all()


@pytest.mark.parametrize("n", [1, 40, 333])
def test_delta_continues(mcv, cuda, n):
    """A sequence cut anywhere and continued from its state, against the whole."""
    q, k, v, g, beta, state = _delta_case(n, [400], 2, 2, 128, 128)
    a = [x.to(cuda) for x in (q, k, v, g, beta)]
    s0 = state.to(cuda)
    ref = _delta_ref(q, k, v, g, beta, state, [400], 128 ** -0.5, True)
    o1, s1 = mcv.gated_delta_rule(*(x[:n] for x in a), s0, normalize=True)
    o2, s2 = mcv.gated_delta_rule(*(x[n:] for x in a), s1, normalize=True)
    _delta_close(_torch().cat((o1, o2)), s2, ref)


@pytest.mark.parametrize("lens", [[1], [5, 3], [200], [64, 130]])
def test_delta_extremes(mcv, cuda, lens):
    """No state, keys all alike, zero keys and queries, a decay that forgets all, beta 0 and 1."""
    torch = _torch()
    q, k, v, g, beta, _ = _delta_case(11, lens, 2, 2, 128, 64, lean=3.0)
    k[: sum(lens) // 3, 0] = k[:1, 0]
    k[sum(lens) // 2, 1] = 0
    q[sum(lens) // 2, 0] = 0
    g[sum(lens) // 2:, 0] *= 200
    g[sum(lens) // 3, 1] = -math.inf
    beta[::3] = 1
    beta[1::3] = 0
    zero = torch.zeros(len(lens), 2, 128, 64)
    ref = _delta_ref(q, k, v, g, beta, zero, lens, 128 ** -0.5, True)
    out, final = mcv.gated_delta_rule(*(x.to(cuda) for x in (q, k, v, g, beta)), cu_seqlens=_cu(lens, cuda), normalize=True)
    _delta_close(out, final, ref)


@pytest.mark.parametrize("size", [2.0 ** -10, 1.0, 400.0])
def test_delta_sizes_of_values(mcv, cuda, size):
    """Values and states far from one, and keys of any length when they are normalised."""
    q, k, v, g, beta, state = _delta_case(3, [150, 9], 1, 2, 128, 64)
    v, state, k, q = v * size, state * size, k * size, q * 3
    ref = _delta_ref(q, k, v, g, beta, state, [150, 9], 128 ** -0.5, True)
    out, final = mcv.gated_delta_rule(*(x.to(cuda) for x in (q, k, v, g, beta, state)), cu_seqlens=_cu([150, 9], cuda),
                                      normalize=True)
    _delta_close(out, final, ref)


# ------------------------------------------------------------- paged attention --
def _attn_case(seed, lens, Hq, Hkv, D, page, width=None, sharp=2.0):
    torch = _torch()
    gen = _gen(seed)
    B = len(lens)
    need = [-(-n // page) for n in lens]
    width = max(need + [1]) if width is None else width
    pool = sum(need) + 2
    order = torch.randperm(pool, generator=gen).int()
    table = torch.full((B, width), -7, dtype=torch.int32)
    k = torch.full((pool, page, Hkv, D), math.nan).half()
    v = torch.full((pool, page, Hkv, D), math.inf).half()
    at, kv = 0, []
    for b, n in enumerate(lens):
        own = order[at:at + need[b]]
        at += need[b]
        table[b, :need[b]] = own
        kk, vv = (torch.randn(n, Hkv, D, generator=gen).half() for _ in range(2))
        for i, p in enumerate(own.tolist()):
            m = min(page, n - i * page)
            k[p, :m], v[p, :m] = kk[i * page:i * page + m], vv[i * page:i * page + m]
        kv.append((kk, vv))
    q = (sharp * torch.randn(B, Hq, D, generator=gen)).half()
    return q, k, v, table, torch.tensor(lens, dtype=torch.int32), kv


def _attn_ref(q, kv, Hkv, scale, live=None):
    """out and the magnitudes its sum runs over."""
    torch = _torch()
    B, Hq, D = q.shape
    out, size = torch.zeros(B, Hq, D, dtype=torch.float64), torch.zeros(B, Hq, D, dtype=torch.float64)
    for b, (k, v) in enumerate(kv):
        on = slice(None) if live is None else live[b]
        k, v = k.double()[on], v.double()[on]
        if len(k) == 0:
            continue
        for h in range(Hq):
            w = torch.softmax(k[:, h // (Hq // Hkv)] @ q[b, h].double() * scale, 0)
            out[b, h] = w @ v[:, h // (Hq // Hkv)]
            size[b, h] = w @ v[:, h // (Hq // Hkv)].abs()
    return out, size


def _attn_close(got, ref):
    want, size = ref
    err = (got.cpu().double() - want).abs()
    # one rounding of out, one of each softmax weight, 32-bit scores (exp of a score off by 2^-18)
    assert (err <= H * want.abs() + (H + 2.0 ** -17) * size + 2.0 ** -24).all(), (err - H * want.abs() - H * size).max()


ATTN = [
    # lens, Hq, Hkv, D, page
    ([1], 1, 1, 64, 16),
    ([17], 8, 2, 256, 16),
    ([1100], 8, 2, 256, 16),
    ([0, 1, 15, 16, 31, 32, 33, 700], 8, 2, 256, 32),
    ([5, 300, 0, 64], 32, 8, 128, 16),
    ([2500, 7], 12, 1, 128, 48),
    ([333], 16, 16, 64, 64),
    ([4097, 129], 40, 2, 64, 128),
    ([20000], 8, 2, 256, 64),
]


@pytest.mark.parametrize("lens,Hq,Hkv,D,page", ATTN)
def test_paged_attention(mcv, cuda, lens, Hq, Hkv, D, page):
    q, k, v, table, n, kv = _attn_case(len(lens) + D, lens, Hq, Hkv, D, page)
    a = [x.to(cuda) for x in (q, k, v, table, n)]
    got = mcv.paged_attention_decode(*a)
    _attn_close(got, _attn_ref(q, kv, Hkv, D ** -0.5))
    again = mcv.paged_attention_decode(*a)
    assert (again == got).all()                                  # the same bits: joined in one order
    tight = mcv.paged_attention_decode(*a, scale=0.05, max_seq_len=max(lens), out=got)
    assert tight is got
    _attn_close(got, _attn_ref(q, kv, Hkv, 0.05))


@pytest.mark.parametrize("B,longest,Hq,Hkv,D,page", [(150, 900, 4, 2, 64, 16), (65, 3000, 8, 1, 128, 32), (300, 40, 6, 3, 256, 16),
                                                     (64, 700, 20, 1, 128, 16), (129, 130, 16, 8, 64, 16)])
def test_paged_attention_many_sequences(mcv, cuda, B, longest, Hq, Hkv, D, page):
    """More sequences than lanes of a wave, from none to the longest: cut in parts, whole, and both together."""
    torch = _torch()
    lens = (torch.rand(B, generator=_gen(B)) ** 3 * (longest + 1)).int()
    lens[0], lens[B // 2], lens[-1] = 0, longest, longest - 1
    q, k, v, table, n, kv = _attn_case(B + D, lens.tolist(), Hq, Hkv, D, page)
    got = mcv.paged_attention_decode(*(x.to(cuda) for x in (q, k, v, table, n)))
    _attn_close(got, _attn_ref(q, kv, Hkv, D ** -0.5))


def test_paged_attention_absent_pages(mcv, cuda):
    """Page numbers outside the cache are left out, wherever they stand; a row of none gives zeros."""
    torch = _torch()
    page, lens = 16, [600, 40, 33]
    q, k, v, table, n, kv = _attn_case(3, lens, 8, 2, 128, page)
    live = [torch.ones(m, dtype=torch.bool) for m in lens]
    for b, i, bad in [(0, 0, -1), (0, 5, k.shape[0]), (0, 37, 2 ** 31 - 1), (1, 2, -2 ** 31), (2, 0, -1), (2, 1, -1), (2, 2, 10 ** 6)]:
        table[b, i] = bad
        live[b][i * page:(i + 1) * page] = False
    got = mcv.paged_attention_decode(*(x.to(cuda) for x in (q, k, v, table, n)))
    _attn_close(got, _attn_ref(q, kv, 2, 128 ** -0.5, live))
    assert (got[2] == 0).all()


def test_paged_attention_lengths_out_of_range(mcv, cuda):
    """Lengths past the table or max_seq_len are cut, negative ones are none."""
    torch = _torch()
    q, k, v, table, _, kv = _attn_case(4, [64, 64, 64, 64], 4, 1, 64, 16)
    n = torch.tensor([10 ** 9, -5, 64, 50], dtype=torch.int32)
    a = [x.to(cuda) for x in (q, k, v, table, n)]
    cut = lambda m: [(x[:min(m, max(0, i))], y[:min(m, max(0, i))]) for (x, y), i in zip(kv, n.tolist())]  # noqa: E731
    _attn_close(mcv.paged_attention_decode(*a), _attn_ref(q, cut(64), 1, 64 ** -0.5))
    _attn_close(mcv.paged_attention_decode(*a, max_seq_len=33), _attn_ref(q, cut(33), 1, 64 ** -0.5))
    assert (mcv.paged_attention_decode(*a, max_seq_len=0) == 0).all()


def test_paged_attention_orders(mcv, cuda):
    """Caches in another order, k and v in one pool, q as columns of a wider row, one table for all rows."""
    torch = _torch()
    lens = [70, 200, 128]
    q, k, v, table, n, kv = _attn_case(5, lens, 8, 4, 64, 32)
    want = _attn_ref(q, kv, 4, 0.125)
    wide = torch.zeros(3, 8, 2, 64).half()
    wide[:, :, 0] = q
    both = torch.stack((k, v), 1).permute(0, 1, 3, 2, 4).contiguous().to(cuda)         # [pages, 2, Hkv, page, D]
    got = mcv.paged_attention_decode(wide.to(cuda)[:, :, 0], both[:, 0].permute(0, 2, 1, 3), both[:, 1].permute(0, 2, 1, 3),
                                     table.to(cuda), n.to(cuda))
    _attn_close(got, want)
    # every token of a prompt as a row of its own, over the sequence's one table
    rows = torch.arange(1, 129, dtype=torch.int32)
    qs = torch.randn(128, 8, 64, generator=_gen(8)).half()
    got = mcv.paged_attention_decode(qs.to(cuda), k.to(cuda), v.to(cuda), table[2:].to(cuda).expand(128, -1), rows.to(cuda))
    _attn_close(got, _attn_ref(qs, [(kv[2][0][:i], kv[2][1][:i]) for i in rows.tolist()], 4, 0.125))


def test_paged_attention_infinite_scores(mcv, cuda):
    """Keys of -inf (a score of -inf) weigh nothing, also where a whole tile or row has them; very large scores do not overflow."""
    torch = _torch()
    q, k, v, table, n, kv = _attn_case(6, [200, 48], 4, 1, 64, 16)
    q = q.abs() + 0.1
    live = [torch.ones(200, dtype=torch.bool), torch.zeros(48, dtype=torch.bool)]
    live[0][:70] = False
    for b, (kk, _) in enumerate(kv):
        for t in (~live[b]).nonzero()[:, 0].tolist():
            k[table[b, t // 16], t % 16] = -math.inf
    got = mcv.paged_attention_decode(*(x.to(cuda) for x in (q, k, v, table, n)))
    _attn_close(got[:1], tuple(x[:1] for x in _attn_ref(q[:1], kv[:1], 1, 0.125, live[:1])))
    assert (got[1] == 0).all()                                   # as a row whose mask leaves nothing
    q, k, v, table, n, kv = _attn_case(7, [300], 4, 1, 64, 16, sharp=500.0)
    got = mcv.paged_attention_decode(*(x.to(cuda) for x in (q, k, v, table, n)))
    want, size = _attn_ref(q, kv, 1, 0.125)
    # scores near 10^4: 32 bits are off by 2^-10, exp of that
    assert ((got.cpu().double() - want).abs() <= H * want.abs() + (H + 2.0 ** -8) * size + 2.0 ** -24).all()


def test_paged_attention_far_offsets(mcv, cuda):
    """Pages whose elements lie past 2^31 and 2^32 from the start of the cache."""
    torch = _torch()
    page, Hkv, D = 64, 2, 256
    pages = 2 ** 32 // (page * Hkv * D) + 8
    k = torch.zeros(pages, page, Hkv, D, dtype=torch.float16, device=cuda)
    q, ks, vs, table, n, kv = _attn_case(9, [150], 8, Hkv, D, page)
    far = torch.tensor([pages - 1, pages // 2 + 1, 3], dtype=torch.int32)
    v = torch.zeros_like(k)
    for i, p in enumerate(far.tolist()):
        k[p], v[p] = ks[table[0, i]].to(cuda), vs[table[0, i]].to(cuda)
    got = mcv.paged_attention_decode(q.to(cuda), k, v, far[None].to(cuda), n.to(cuda))
    _attn_close(got, _attn_ref(q, kv, Hkv, D ** -0.5))


# ------------------------------------------------------------- rotary positions --
def _rotary_ref(x, pos, freq, axis):
    torch = _torch()
    half = freq.numel()
    angle = pos[axis.long().clamp(0, pos.shape[0] - 1)].t().double() * freq
    c, s = angle.cos()[:, None], angle.sin()[:, None]
    a, b, r = x[..., :half].double(), x[..., half:2 * half].double(), x[..., 2 * half:].double()
    size = torch.cat(((a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs(), 0 * r), -1)
    return torch.cat((a * c - b * s, b * c + a * s, r), -1), size


def _rotary_close(got, ref):
    want, size = ref
    err = (got.cpu().double() - want).abs()
    # one rounding; cosine, sine, two products and a sum in 32 bits
    assert (err <= H * want.abs() + 2.0 ** -21 * size + 2.0 ** -25).all(), err.max()


@pytest.mark.parametrize("T,Hq,Hkv,D,rot,sections,mixed", [
    (1, 8, 2, 256, 64, (11, 11, 10), True),
    (5, 16, 4, 128, 128, (24, 20, 20), False),
    (333, 3, 1, 64, 64, (12, 10, 10), True),
    (40, 2, 5, 72, 18, (3, 6), False),
    (7, 1, 1, 8, 2, (1,), False),
    (1000, 8, 2, 256, 64, (11, 11, 10), True),
    (9, 4, 4, 512, 512, (64, 64, 64, 64), True),
])
def test_rotary_axes(mcv, cuda, T, Hq, Hkv, D, rot, sections, mixed):
    torch = _torch()
    gen = _gen(T + D)
    freq, axis = mcv.rotary_axes_table(rot, 1e6, sections, mixed, device="cpu")
    assert [axis.tolist().count(a) for a in range(len(sections))] == list(sections)
    pos = torch.randint(0, 10 ** 7, (len(sections), T), generator=gen)
    qkv = torch.randn(T, (Hq + 2 * Hkv) * D, generator=gen).half()
    q, k = qkv[:, :Hq * D].view(T, Hq, D), qkv[:, Hq * D:(Hq + Hkv) * D].view(T, Hkv, D)
    dev = qkv.to(cuda)
    a = (dev[:, :Hq * D].view(T, Hq, D), dev[:, Hq * D:(Hq + Hkv) * D].view(T, Hkv, D))
    where = (pos.to(cuda), freq.to(cuda), axis.to(cuda))
    qo, ko = mcv.rotary_axes(*a, *where)
    _rotary_close(qo, _rotary_ref(q, pos, freq, axis))
    _rotary_close(ko, _rotary_ref(k, pos, freq, axis))
    rest = dev[:, (Hq + Hkv) * D:].clone()
    assert mcv.rotary_axes(*a, *where, q_out=a[0], k_out=a[1])[0] is a[0]          # in place
    assert (a[0] == qo).all() and (a[1] == ko).all() and (dev[:, (Hq + Hkv) * D:] == rest).all()


def test_rotary_axes_one_row_of_positions(mcv, cuda):
    """Text: one row of positions for all axes, and axes outside the rows there are."""
    torch = _torch()
    freq, axis = mcv.rotary_axes_table(64, 1e7, (11, 11, 10), device="cpu")
    axis[0], axis[1] = -3, 9
    q = torch.randn(6, 4, 64, generator=_gen(2)).half()
    pos = torch.arange(100000, 100006)[None]
    qo, _ = mcv.rotary_axes(q.to(cuda), q.to(cuda), pos.to(cuda).expand(3, -1), freq.to(cuda), axis.to(cuda))
    _rotary_close(qo, _rotary_ref(q, pos, freq, axis))


@pytest.mark.parametrize("T,Hq,Hkv,D,rot,page", [(1, 8, 2, 256, 64, 16), (77, 4, 2, 128, 128, 32), (300, 2, 1, 64, 36, 5)])
def test_rotary_axes_cached(mcv, cuda, T, Hq, Hkv, D, rot, page):
    torch = _torch()
    gen = _gen(T)
    half = rot // 2
    freq, axis = mcv.rotary_axes_table(rot, 1e4, (half - 2 * (half // 3), half // 3, half // 3), device="cpu")
    pos = torch.randint(0, 5000, (3, T), generator=gen)
    qkv = torch.randn(T, (Hq + 2 * Hkv) * D, generator=gen).half()
    q, k, v = (t.view(T, -1, D) for t in qkv.split((Hq * D, Hkv * D, Hkv * D), 1))
    pages = -(-T // page) + 2
    slots = torch.randperm(pages * page, generator=gen)[:T]
    if T > 4:
        slots[1], slots[3] = -1, pages * page
    old = torch.randn(2, pages, Hkv, page, D, generator=gen).half()
    dev = old.to(cuda)
    kc, vc = dev[0].transpose(1, 2), dev[1].transpose(1, 2)
    d = qkv.to(cuda)
    args = [t.view(T, -1, D) for t in d.split((Hq * D, Hkv * D, Hkv * D), 1)]
    qo = mcv.rotary_axes_cached(*args, pos.to(cuda), freq.to(cuda), axis.to(cuda), kc, vc, slots.to(cuda))
    _rotary_close(qo, _rotary_ref(q, pos, freq, axis))
    ok = (slots >= 0) & (slots < pages * page)
    flat = [t.cpu().reshape(pages * page, Hkv, D) for t in (kc, vc)]
    want = _rotary_ref(k, pos, freq, axis)
    _rotary_close(flat[0][slots[ok]], tuple(x[ok] for x in want))
    assert (flat[1][slots[ok]] == v[ok]).all()
    rest = torch.ones(pages * page, dtype=torch.bool)
    rest[slots[ok]] = False
    before = [t.transpose(1, 2).reshape(pages * page, Hkv, D) for t in old]
    assert all((x[rest] == y[rest]).all() for x, y in zip(flat, before))


# -------------------------------------------------------------- streams, graphs --
def test_mixers_on_another_stream(mcv, cuda):
    torch = _torch()
    side = torch.cuda.Stream()
    q, k, v, g, beta, state = (x.to(cuda) for x in _delta_case(1, [300], 2, 2, 128, 128))
    aq, ak, av, table, n = (x.to(cuda) for x in _attn_case(1, [5000], 8, 2, 128, 32)[:5])
    torch.cuda.synchronize()
    want = (*mcv.gated_delta_rule(q, k, v, g, beta, state, normalize=True), mcv.paged_attention_decode(aq, ak, av, table, n))
    torch.cuda.synchronize()
    got = (*mcv.gated_delta_rule(q, k, v, g, beta, state, normalize=True, stream=side),
           mcv.paged_attention_decode(aq, ak, av, table, n, stream=side))
    side.synchronize()
    assert all((x == y).all() for x, y in zip(got, want))


def test_mixers_in_a_graph(mcv, cuda):
    """Captured once, replayed with other inputs in the same buffers, eager calls between."""
    torch = _torch()
    cases = [[x.to(cuda) for x in _delta_case(s, [200, 1], 2, 2, 128, 128)] for s in (1, 2)]
    cu = _cu([200, 1], cuda)
    attn = [[x.to(cuda) for x in _attn_case(s, [n, 40], 8, 2, 128, 32, width=160)[:5]] for s, n in ((1, 5000), (2, 77))]
    pool = max(a[1].shape[0] for a in attn)
    attn = [[a[0], *(torch.cat((t, t.new_zeros(pool - t.shape[0], *t.shape[1:]))) for t in a[1:3]), *a[3:]] for a in attn]
    hold, ahold = [x.clone() for x in cases[0]], [x.clone() for x in attn[0]]
    step = lambda c, a: (*mcv.gated_delta_rule(*c, cu_seqlens=cu, normalize=True), mcv.paged_attention_decode(*a))  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(hold, ahold)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = step(hold, ahold)
    for turn in (0, 1, 0, 1):
        want = step(cases[turn], attn[turn])
        for x, y in zip(hold + ahold, cases[turn] + attn[turn]):
            x.copy_(y)
        graph.replay()
        torch.cuda.synchronize()
        assert all((x == y).all() for x, y in zip(got, want)), turn


def test_mixers_share_a_workspace_with_the_gemm(mcv, cuda):
    """On one stream all of them use one buffer, whose counters each leaves zero."""
    torch = _torch()
    c = [x.to(cuda) for x in _delta_case(1, [500], 1, 1, 64, 64)]
    a = [x.to(cuda) for x in _attn_case(1, [900, 3], 8, 2, 64, 16)[:5]]
    w = mcv.W4A16QuantizedWeight.from_awq(*mcv.quantize_int4(torch.randn(3584, 1024, generator=_gen(1)).half().view(torch.int16).numpy()))
    x = torch.randn(70, 3584, generator=_gen(2)).half().to(cuda)
    first = None
    for _ in range(3):
        got = (mcv.matmul_w4a16(x, w), *mcv.gated_delta_rule(*c, normalize=True), mcv.paged_attention_decode(*a))
        first = first or [t.clone() for t in got]
        assert all((t == u).all() for t, u in zip(got, first))
    for ws in mcv._GEMM_WS.values():
        assert (ws[:4096] == 0).all()

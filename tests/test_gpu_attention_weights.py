"""One-token paged attention where most weights are far below the largest: the sum over
the values and the sum of the weights have to agree however far.

Tolerance.  Weights are held in two fp16 parts below 2^15 (off by 2^-21 of each, or by 2^-39
of the largest) and summed in 32 bits, scores are 32 bits of values below 64
(exp of them off by 2^-19): 2^-17 of the magnitudes of the sum, and one rounding of the output."""
import math

import pytest

from test_gpu_mixers import H, _attn_case, _attn_ref

pytestmark = pytest.mark.gpu


def _close(got, ref):
    want, size = ref
    err = (got.cpu().double() - want).abs()
    room = H * want.abs() + 2.0 ** -17 * size + 2.0 ** -24
    assert (err <= room).all(), (err / room).max()


def _sink(q, k, v, table, kv, b, at, page, value):
    """Token `at` of sequence b has nearly all the weight: scores of 10 to 24 (one a head) where the others have 0."""
    Hq, D = q.shape[1:]
    group = Hq // k.shape[2]
    kk, vv = kv[b]
    kk.zero_()
    kk[at, :, 0] = 8.0
    vv.copy_(1 + vv.float() / 8)
    vv[at] = value
    q[b].zero_()
    for h in range(Hq):
        q[b, h, 0] = (10 + 14 * (h % group) / max(group - 1, 1)) / 8 * math.sqrt(D)
    for i, p in enumerate(table[b, :-(-len(kk) // page)].tolist()):
        n = min(page, len(kk) - i * page)
        k[p, :n], v[p, :n] = kk[i * page:i * page + n], vv[i * page:i * page + n]


@pytest.mark.parametrize("lens,Hq,Hkv,D,page", [([32], 8, 1, 64, 16), ([32], 8, 2, 256, 16), ([2000], 16, 2, 128, 16),
                                                ([4096, 77, 1, 600], 12, 2, 64, 32), ([30000], 8, 2, 256, 64), ([40000, 9], 15, 1, 128, 64)])
@pytest.mark.parametrize("value", [0.0, 0.02, -3.0])
@pytest.mark.parametrize("place", ["first", "middle", "last"])
def test_one_token_far_above_the_others(mcv, cuda, lens, Hq, Hkv, D, page, value, place):
    q, k, v, table, n, kv = _attn_case(sum(lens) + D, lens, Hq, Hkv, D, page)
    for b, m in enumerate(lens):
        _sink(q, k, v, table, kv, b, {"first": 0, "middle": m // 2, "last": m - 1}[place], page, value)
    got = mcv.paged_attention_decode(*(x.to(cuda) for x in (q, k, v, table, n)))
    _close(got, _attn_ref(q, kv, Hkv, D ** -0.5))


@pytest.mark.parametrize("lens,Hq,Hkv,D,page", [([1], 1, 1, 64, 16), ([1100], 8, 2, 256, 16), ([0, 31, 33, 700, 2], 8, 2, 256, 32),
                                                ([2500, 7], 12, 1, 128, 48), ([20000], 16, 16, 64, 64)])
def test_weights_are_not_rounded_to_16_bits(mcv, cuda, lens, Hq, Hkv, D, page):
    q, k, v, table, n, kv = _attn_case(len(lens) + Hq, lens, Hq, Hkv, D, page, sharp=1.0)
    got = mcv.paged_attention_decode(*(x.to(cuda) for x in (q, k, v, table, n)))
    _close(got, _attn_ref(q, kv, Hkv, D ** -0.5))


def test_largest_values(mcv, cuda):
    """Values and counts at which sums pass fp16's range long before the average does."""
    q, k, v, table, n, kv = _attn_case(5, [9000, 64], 8, 2, 128, 64, sharp=0.1)
    for b, (_, vv) in enumerate(kv):
        vv.copy_(60000 * (1 if b else -1) + 1000 * vv.float().clamp(-5, 5))
        for i, p in enumerate(table[b, :-(-len(vv) // 64)].tolist()):
            m = min(64, len(vv) - i * 64)
            v[p, :m] = vv[i * 64:i * 64 + m]
    got = mcv.paged_attention_decode(*(x.to(cuda) for x in (q, k, v, table, n)))
    _close(got, _attn_ref(q, kv, 2, 128 ** -0.5))


@pytest.mark.parametrize("lens,D", [([40], 64), ([3000, 5], 256), ([900, 33, 64], 128)])
def test_infinite_values(mcv, cuda, lens, D):
    """An infinite value makes its column of the output infinite, two of different signs or a NaN make it NaN."""
    q, k, v, table, n, kv = _attn_case(sum(lens), lens, 8, 2, D, 32, sharp=1.0)
    for b, (m, (_, vv)) in enumerate(zip(lens, kv)):
        vv[m // 2, 0, 3], vv[m - 1, 0, 9], vv[0, 1, 20] = math.inf, -math.inf, math.nan
        vv[0, 1, 40], vv[m // 3, 1, 40] = math.inf, -math.inf
        vv[0, 0, 33] = vv[m - 1, 0, 33] = math.inf
        for i, p in enumerate(table[b, :-(-m // 32)].tolist()):
            rows = min(32, m - i * 32)
            v[p, :rows] = vv[i * 32:i * 32 + rows]
    got = mcv.paged_attention_decode(*(x.to(cuda) for x in (q, k, v, table, n))).cpu().double()
    want, size = _attn_ref(q, kv, 2, D ** -0.5)
    off = ~want.isfinite()
    assert off.any() and (got[off].isnan() == want[off].isnan()).all()
    inf = want.isinf()
    assert inf.any() and (got[inf] == want[inf]).all()
    want[off], size[off], got[off] = 0, 0, 0
    _close(got, (want, size))

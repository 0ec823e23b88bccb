"""GPU tests of paged_attention_chunk where scores are so large that neighbouring 32-bit numbers are whole units apart.  Scores
here are such numbers to the bit, and the scale is ln 2, whose product with log2 e is one in 32 bits: the softmax's weights are
powers of two and known exactly, and test_gpu_chunk_attention's tolerance holds with nothing for the scores."""
import math

import pytest

from test_gpu_chunk_attention import H, _case, _ref
from test_gpu_mixers import _torch

pytestmark = pytest.mark.gpu


def _scores(q, k, table, kv, page, far, sign, steps):
    """q . k of token t becomes sign 2^far + steps[t] 2^(far - 23)."""
    torch = _torch()
    side = 2.0 ** (far // 2)
    q[...], k[...] = 0.0, 0.0
    q[..., 0], q[..., 1] = sign * side, max(1.0, 2.0 ** (far - 23))
    for b, (kk, _) in enumerate(kv):
        kk[...] = 0.0
        kk[..., 0] = side
        kk[..., 1] = steps[:len(kk), None].to(kk.dtype)
        for t in range(0, len(kk), page):
            rows = kk[t:t + page]
            k[table[b, t // page], :len(rows)] = rows


STEPS = {
    "rising": lambda t: t // 100,
    "falling": lambda t: 40 - t // 100,
    "many below a few": lambda t: 4 * (t > 2000),
    "a few below many": lambda t: 6 * (t < 900) + 4 * (t % 64 == 63),
}


@pytest.mark.parametrize("n,held,D", [([40], [2200], 64), ([700], [1600], 128), ([9], [2100], 256), ([64], [0], 256)])
@pytest.mark.parametrize("far", [22, 24, 26, 28, 30])
@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("steps", list(STEPS))
def test_far_scores(mcv, cuda, n, held, D, far, sign, steps):
    torch = _torch()
    q, k, v, table, lens, cu, kv = _case(far, n, held, 4, 2, D, 16)
    _scores(q, k, table, kv, 16, far, sign, STEPS[steps](torch.arange(sum(n) + sum(held))).int())
    got = mcv.paged_attention_chunk(*(x.to(cuda) for x in (q, k, v, table, lens, cu)), scale=math.log(2))
    want, size = _ref(q, kv, n, lens.tolist(), math.log(2))
    err = (got.cpu().double() - want).abs()
    bound = 2 * H * want.abs() + (H + 2.0 ** -17) * size + 2.0 ** -24
    assert (err <= bound).all(), ((err - bound).max(), err.max())


@pytest.mark.parametrize("far", [3e4, 6e4])
def test_as_large_as_they_come(mcv, cuda, far):
    """Every element of q and k near fp16's end: scores that no two tokens share leave each row its best token's v."""
    torch = _torch()
    q, k, v, table, lens, cu, kv = _case(7, [30], [600], 8, 2, 256, 16)
    q[...] = far
    t = torch.arange(630)
    for kk, _ in kv:
        kk[...] = (far / 2 * (1 + ((7 * t) % 630) / 630))[:, None, None].half()
        for i in range(0, 630, 16):
            rows = kk[i:i + 16]
            k[table[0, i // 16], :len(rows)] = rows
    got = mcv.paged_attention_chunk(*(x.to(cuda) for x in (q, k, v, table, lens, cu))).cpu()
    for row in range(30):
        seen = kv[0][0][:601 + row, 0, 0].float()
        best = seen == seen.max()
        want = kv[0][1][:601 + row][best].double().mean(0)       # (of equal keys the mean)
        for h in range(8):
            assert ((got[row, h].double() - want[h // 4]).abs() <= 3 * H * want[h // 4].abs() + H * kv[0][1].abs().max()).all()

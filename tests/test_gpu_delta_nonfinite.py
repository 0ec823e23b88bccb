"""The gated delta rule with an infinity or NaN in its inputs: what it reaches by the
definition (the token's own outputs and all later ones of its columns) is not finite,
everything else is as if it were not there, whichever form the length picks."""
import math

import pytest

from test_gpu_mixers import H, _cu, _delta_case, _delta_ref, _torch

pytestmark = pytest.mark.gpu


def _check(mcv, cuda, inputs, lens, scale, normalize, state_too=True):
    torch = _torch()
    ref, size, S = _delta_ref(*inputs, lens, scale, normalize)
    out, final = mcv.gated_delta_rule(*(x.to(cuda) for x in inputs), cu_seqlens=_cu(lens, cuda), scale=scale, normalize=normalize)
    out, final = out.cpu().double(), final.cpu().double()
    on = ref.isfinite()
    assert 0 < on.sum() < on.numel()                             # the case has both
    assert (out.isfinite() == on).all(), (out.isfinite() != on).nonzero()[:4]
    # as in test_gpu_mixers: one rounding of out, and the two-part operands' 2^-21 counted at three roundings
    assert ((out - ref).abs()[on] <= (H * ref.abs() + 3 * H * size + 2.0 ** -24)[on]).all()
    if state_too:
        on = S.isfinite()
        assert (final.isfinite() == on).all(), (final.isfinite() != on).nonzero()[:4]
        where = on.all(-2)                                       # whole columns of a state
        a, b = final.transpose(-1, -2)[where], S.transpose(-1, -2)[where]
        assert (a - b).norm() <= 16 * 2.0 ** -22 * b.norm()


BAD = [math.inf, -math.inf, math.nan]


@pytest.mark.parametrize("n,at", [(n, at) for n in (9, 64, 65, 200) for at in (0, 5, 31, 47, 63, 70, 129) if at < n])
@pytest.mark.parametrize("bad", BAD)
def test_in_v(mcv, cuda, n, at, bad):
    q, k, v, g, beta, state = _delta_case(n + at, [n, 40], 2, 4, 128, 64)
    v[at, 1, 3], v[at, 2, 50] = bad, 1.0
    _check(mcv, cuda, (q, k, v, g, beta, state), [n, 40], 0.1, True)


@pytest.mark.parametrize("what", ["k", "g", "beta"])
@pytest.mark.parametrize("at", [0, 20, 31, 63, 100, 149])
@pytest.mark.parametrize("normalize", [True, False])
def test_in_k_and_the_gates(mcv, cuda, what, at, normalize):
    """From that token on the whole head has none left."""
    q, k, v, g, beta, state = _delta_case(at, [150, 12], 2, 4, 128, 32)
    if not normalize:
        k = k / 32
    {"k": k, "g": g, "beta": beta}[what][at, 1] = math.nan
    _check(mcv, cuda, (q, k, v, g, beta, state), [150, 12], 0.1, normalize)


@pytest.mark.parametrize("at", [3, 40, 64, 90])
def test_infinite_k(mcv, cuda, at):
    q, k, v, g, beta, state = _delta_case(at, [100], 1, 2, 64, 32)
    k[at, 0, 7] = math.inf
    _check(mcv, cuda, (q, k, v, g, beta, state), [100], 0.1, True)


@pytest.mark.parametrize("at,bad", [(3, math.inf), (40, math.nan), (77, -math.inf)])
@pytest.mark.parametrize("normalize", [True, False])
def test_in_q(mcv, cuda, at, bad, normalize):
    """Only that token's own outputs."""
    q, k, v, g, beta, state = _delta_case(at, [100], 2, 2, 64, 32)
    if not normalize:
        k = k / 32
    q[at, 1, 7] = bad
    _check(mcv, cuda, (q, k, v, g, beta, state), [100], 0.1, normalize)


@pytest.mark.parametrize("bad", BAD)
def test_in_the_state(mcv, cuda, bad):
    q, k, v, g, beta, state = _delta_case(8, [100, 70], 2, 2, 128, 64)
    state[0, 1, 100, 17] = bad
    state[1, 0, 2, 63] = bad
    _check(mcv, cuda, (q, k, v, g, beta, state), [100, 70], 0.1, True)


@pytest.mark.parametrize("size", [2.0 ** -12, 30000.0])
def test_scale_of_the_others(mcv, cuda, size):
    """An infinite value or state takes no bits from the other columns, nor from the tokens before it."""
    q, k, v, g, beta, state = _delta_case(9, [150], 2, 2, 128, 32)
    v, state = v * size / 4, state * size
    v[140, 0, 1] = math.inf
    state[0, 1, 9, 9] = math.inf
    _check(mcv, cuda, (q, k, v, g, beta, state), [150], 0.1, True)

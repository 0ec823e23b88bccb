"""Batches of short sequences with one longer, around the sizes where both forms of the gated delta rule are launched."""
import pytest

from test_gpu_mixers import _cu, _delta_case, _delta_close, _delta_ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lens", [[1] * 40 + [32], [1] * 40 + [33], [1] * 20 + [63] + [1] * 20, [1] * 7 + [33], [40] + [1] * 7, [2] * 9 + [30], [0] * 10 + [50],
                                  [1] * 15 + [63], [4] * 8 + [9], [5] * 8, [1, 1, 1, 32], [1, 1, 1, 33], [2] * 41, [9] * 5, [12, 3, 11, 8, 10]])
def test_one_longer(mcv, cuda, lens):
    q, k, v, g, beta, state = _delta_case(sum(lens), lens, 2, 4, 128, 64)
    ref = _delta_ref(q, k, v, g, beta, state, lens, 0.1, True)
    out, final = mcv.gated_delta_rule(*(x.to(cuda) for x in (q, k, v, g, beta, state)), cu_seqlens=_cu(lens, cuda), scale=0.1, normalize=True)
    _delta_close(out, final, ref)

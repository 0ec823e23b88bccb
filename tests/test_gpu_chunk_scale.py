"""GPU tests of paged_attention_chunk's scale: none, negative, and so small that 32 bits do not hold it."""
import pytest

from test_gpu_chunk_attention import _case, _close, _ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,held", [([70, 1, 9], [0, 0, 90]), ([24], [1100]), ([3], [3000])])
@pytest.mark.parametrize("scale", [0.0, 1e-30, 1e-42, 1e-46, -1e-60, 5e-324, -0.125])
def test_scales(mcv, cuda, n, held, scale):
    q, k, v, table, lens, cu, kv = _case(1, n, held, 8, 2, 128, 16)
    got = mcv.paged_attention_chunk(*(x.to(cuda) for x in (q, k, v, table, lens, cu)), scale=scale)
    _close(got, _ref(q, kv, n, lens.tolist(), scale))

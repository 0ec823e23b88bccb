"""GPU tests of paged_attention_chunk with its output in the place of q: the bits of a call with an output of its own."""
import math

import pytest

from test_gpu_chunk_nonfinite import SHAPES, _case
from test_gpu_mixers import _torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,held,Hq,Hkv,D,page", SHAPES + [([1] * 70 + [3], [5 * i for i in range(71)], 8, 2, 128, 16)])
@pytest.mark.parametrize("odd", [False, True])
def test_in_place(mcv, cuda, n, held, Hq, Hkv, D, page, odd):
    torch = _torch()
    q, k, v, table, lens, cu, _ = _case(2, n, held, Hq, Hkv, D, page, sharp=0.5)
    if odd:                                      # the rows that see it are made with a second pass over q
        b = next(i for i, m in enumerate(n) if m)
        v[table[b, 0], 0, Hkv - 1, D - 1] = math.inf
    q = torch.cat((q, q[:3]))                    # and rows of no sequence, which stay
    a = [x.to(cuda) for x in (q, k, v, table, lens, cu)]
    want = mcv.paged_attention_chunk(*a, out=a[0].clone())
    for _ in range(3):
        own = a[0].clone()
        assert mcv.paged_attention_chunk(own, *a[1:], out=own) is own
        assert torch.equal(own.view(torch.int16), want.view(torch.int16))
    assert torch.equal(want[-3:], a[0][-3:])
    part = a[0].clone()
    with pytest.raises(mcv.McvError, match="out overlaps q"):
        mcv.paged_attention_chunk(part[:-1], *a[1:], out=part[1:])

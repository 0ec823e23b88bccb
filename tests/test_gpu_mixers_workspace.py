"""The token mixers' workspaces: whose they are, how many there are, and that calls allocate nothing else."""
import pytest

from test_gpu_mixers import _attn_case, _cu, _delta_case, _torch

pytestmark = pytest.mark.gpu


def _delta(cuda, lens, Hk=2, Hv=2, Dk=64, Dv=64):
    a = [x.to(cuda) for x in _delta_case(sum(lens), lens, Hk, Hv, Dk, Dv)]
    return dict(zip(("q", "k", "v", "g", "beta", "state"), a), cu_seqlens=_cu(lens, cuda), normalize=True)


def _spans(buffers):
    return [(b.data_ptr(), b.data_ptr() + b.numel()) for b in buffers]


def test_the_delta_rule_has_its_own(mcv, cuda):
    """Its second launch reads what its first wrote: no call of another kind on the stream may use the same buffer."""
    before = dict(mcv._GEMM_WS)
    mcv.gated_delta_rule(**_delta(cuda, [300]))
    assert mcv._GEMM_WS.keys() == before.keys()
    mcv.paged_attention_decode(*(x.to(cuda) for x in _attn_case(1, [5000], 8, 2, 128, 32)[:5]))
    own, others = _spans(mcv.mixers._DELTA_WS.values()), _spans(mcv._GEMM_WS.values())
    assert own and others and all(a[1] <= b[0] or b[1] <= a[0] for a in own for b in others)


def test_two_sizes_a_stream(mcv, cuda):
    torch = _torch()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for n in (20, 64, 200, 700, 1500, 3000, 6000):
            mcv.gated_delta_rule(**_delta(cuda, [n], 8, 8, 128, 16))
        held = [ws.numel() for (_, stream, _), ws in mcv.mixers._DELTA_WS.items() if stream == side.cuda_stream]
    side.synchronize()
    assert len(held) == 2 and sum(held) <= 208 << 20

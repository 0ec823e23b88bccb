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


def test_attention_has_two_sizes_a_stream(mcv, cuda):
    torch = _torch()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for lens, Hq, Hkv, D in (([300], 2, 2, 64), ([3000], 8, 2, 128), ([20000], 4, 2, 256), ([20000, 7, 0], 16, 1, 256), ([900] * 60, 12, 2, 128)):
            mcv.paged_attention_decode(*(x.to(cuda) for x in _attn_case(1, lens, Hq, Hkv, D, 32)[:5]))
        held = [ws.numel() for (_, stream, _), ws in mcv._GEMM_WS.items() if stream == side.cuda_stream]
    side.synchronize()
    assert len(held) <= 2 and sum(held) <= 24 << 20


def test_calls_allocate_nothing(mcv, cuda):
    """Given their outputs, and once a stream has its workspaces."""
    torch = _torch()
    half = lambda *s: torch.zeros(*s, dtype=torch.float16, device=cuda)      # noqa: E731
    delta = [(c, half(*c["v"].shape), torch.empty_like(c["state"])) for c in (_delta(cuda, lens) for lens in ([3], [300], [1] * 20, [1] * 20 + [400]))]
    step = {n: x for n, x in _delta(cuda, [1] * 5).items() if n != "cu_seqlens"}
    attn = [[x.to(cuda) for x in _attn_case(1, lens, 8, 2, 128, 32)[:5]] for lens in ([9], [700, 0], [20000], [500] * 40)]
    attn = [(a, torch.empty_like(a[0])) for a in attn]
    freq, axis = mcv.rotary_axes_table(64, 1e6, (12, 10, 10))
    pos = torch.arange(3 * 50, device=cuda).view(3, 50)
    q, k, v, qo, ko = half(50, 8, 128), half(50, 2, 128), half(50, 2, 128), half(50, 8, 128), half(50, 2, 128)
    kc, vc, slots = half(5, 16, 2, 128), half(5, 16, 2, 128), torch.arange(50, device=cuda)
    step_out = half(*step["v"].shape)

    def once():
        for c, out, state in delta:
            mcv.gated_delta_rule(**c, out=out, state_out=state)
        mcv.gated_delta_rule_step(**step, out=step_out)
        for a, out in attn:
            mcv.paged_attention_decode(*a, out=out)
        mcv.rotary_axes(q, k, pos, freq, axis, q_out=qo, k_out=ko)
        mcv.rotary_axes_cached(q, k, v, pos, freq, axis, kc, vc, slots, q_out=qo)

    once()
    torch.cuda.synchronize()
    asked = lambda: torch.cuda.memory_stats()["allocation.all.allocated"]    # noqa: E731
    before = asked()
    for _ in range(3):
        once()
    assert asked() == before
    torch.cuda.synchronize()


def test_outputs_of_another_stream(mcv, cuda):
    """What a call on another stream allocates is that stream's: freed at once, the current stream does not get it."""
    torch = _torch()
    side = torch.cuda.Stream()
    delta, step = _delta(cuda, [300]), {n: x for n, x in _delta(cuda, [1] * 5).items() if n != "cu_seqlens"}
    attn = [x.to(cuda) for x in _attn_case(1, [5000], 8, 2, 128, 32)[:5]]
    q, k = torch.randn(50, 8, 128, device=cuda).half(), torch.randn(50, 2, 128, device=cuda).half()
    freq, axis = mcv.rotary_axes_table(64, 1e6, (12, 10, 10))
    pos = torch.arange(3 * 50, device=cuda).view(3, 50)
    cache = [torch.zeros(5, 16, 2, 128, device=cuda).half() for _ in range(2)]
    slots, state_out = torch.arange(50, device=cuda), torch.empty_like(step["state"])
    calls = [
        lambda **on: mcv.gated_delta_rule(**delta, **on),
        lambda **on: mcv.gated_delta_rule_step(**step, state_out=state_out, **on)[:1],
        lambda **on: (mcv.paged_attention_decode(*attn, **on),),
        lambda **on: mcv.rotary_axes(q, k, pos, freq, axis, **on),
        lambda **on: (mcv.rotary_axes_cached(q, k, k, pos, freq, axis, *cache, slots, **on),),
    ]
    for call in calls:
        want = call()
        torch.cuda.synchronize()
        got = call(stream=side)
        side.synchronize()
        assert all((x == y).all() for x, y in zip(got, want))
        where, shapes = {t.data_ptr() for t in got}, [(t.shape, t.dtype) for t in got]
        del got
        fresh = [torch.empty(shape, dtype=dtype, device=cuda) for shape, dtype in shapes for _ in range(4)]
        assert not where & {t.data_ptr() for t in fresh}
        same = call(stream=torch.cuda.current_stream())
        assert all((x == y).all() for x, y in zip(same, want))
    assert torch.cuda.current_stream() != side

"""Token mixers at lengths that take other kernels: four tokens a workgroup of rotary
positions, and attention whose parts are joined in more than one round."""
import pytest

from test_gpu_mixers import _attn_case, _attn_close, _attn_ref, _gen, _rotary_close, _rotary_ref, _torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [4096, 4097, 4098, 4099])
@pytest.mark.parametrize("Hq,Hkv,D,rot", [(8, 2, 256, 64), (3, 1, 64, 64), (2, 2, 128, 32), (1, 1, 16, 16)])
def test_rotary_long(mcv, cuda, T, Hq, Hkv, D, rot):
    torch = _torch()
    gen = _gen(T + D)
    third = rot // 6
    freq, axis = mcv.rotary_axes_table(rot, 1e6, (rot // 2 - 2 * third, third, third), device="cpu")
    pos = torch.randint(0, 10 ** 6, (3, T), generator=gen)
    qkv = torch.randn(T, (Hq + 2 * Hkv) * D, generator=gen).half()
    q, k, v = (t.view(T, -1, D) for t in qkv.split((Hq * D, Hkv * D, Hkv * D), 1))
    where = (pos.to(cuda), freq.to(cuda), axis.to(cuda))
    want = [_rotary_ref(x, pos, freq, axis) for x in (q, k)]
    dev = [t.view(T, -1, D) for t in qkv.to(cuda).split((Hq * D, Hkv * D, Hkv * D), 1)]
    plain = mcv.rotary_axes(*dev[:2], *where)
    for got, ref in zip(plain, want):
        _rotary_close(got, ref)
    page = 16
    pages = -(-T // page) + 2
    slots = torch.randperm(pages * page, generator=gen)[:T]
    slots[1], slots[T - 1], slots[T // 2], slots[T - 3] = -1, pages * page, 2 ** 40, -2 ** 40
    old = torch.randn(2, pages, page, Hkv, D, generator=gen).half()
    kc, vc = old.to(cuda)
    got = mcv.rotary_axes_cached(*dev, *where, kc, vc, slots.to(cuda))
    assert (got == plain[0]).all()
    flat_k, flat_v = (t.cpu().reshape(-1, Hkv, D) for t in (kc, vc))
    ok = (slots >= 0) & (slots < pages * page)
    assert (flat_k[slots[ok]] == plain[1].cpu()[ok]).all() and (flat_v[slots[ok]] == v[ok]).all()
    rest = torch.ones(pages * page, dtype=torch.bool)
    rest[slots[ok]] = False
    assert all((x[rest] == y.reshape(-1, Hkv, D)[rest]).all() for x, y in zip((flat_k, flat_v), old))
    value = dev[2].clone()
    mcv.rotary_axes(*dev[:2], *where, q_out=dev[0], k_out=dev[1])              # in place
    assert (dev[0] == plain[0]).all() and (dev[1] == plain[1]).all() and (dev[2] == value).all()


@pytest.mark.parametrize("long,others,Hq,Hkv,D", [(200000, 39, 2, 1, 64), (70001, 20, 4, 2, 128), (150000, 65, 3, 1, 64)])
def test_attention_joined_in_rounds(mcv, cuda, long, others, Hq, Hkv, D):
    """More than 256 parts of one sequence among many that are short or empty."""
    lens = [i % 3 * 20 for i in range(others)]
    lens.insert(others // 2, long)
    q, k, v, table, n, kv = _attn_case(long, lens, Hq, Hkv, D, 64)
    a = [x.to(cuda) for x in (q, k, v, table, n)]
    got = mcv.paged_attention_decode(*a)
    _attn_close(got, _attn_ref(q, kv, Hkv, D ** -0.5))
    assert (mcv.paged_attention_decode(*a) == got).all()

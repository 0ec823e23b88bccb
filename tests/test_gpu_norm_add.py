"""GPU tests of the residual addition and norm (rms_norm_add, rms_norm_add_w8a8_quantize): to the bit what torch's fp16 addition
and the framework's norms of the sum give, and against the definition in 64 bits."""
import math

import pytest

from test_gpu_mixers import _gen, _torch

pytestmark = pytest.mark.gpu

SHAPES = [(1, 1), (1, 8), (3, 64), (2, 255), (5, 256), (7, 257), (1, 1000), (4, 1001), (1, 1024), (33, 1024), (600, 1024), (2, 1032), (9, 2048), (3, 2050),
          (1100, 3592), (2, 4096), (3, 4097), (2, 8192), (1, 8200), (2, 9001), (1, 20000), (5000, 72)]


def _rows(seed, M, H, dev):
    torch = _torch()
    gen = _gen(seed)
    x = (0.5 * torch.randn(M, H, generator=gen)).half()
    r = (2.0 * torch.randn(M, H, generator=gen) * torch.where(torch.rand(H, generator=gen) < 0.02, 20.0, 1.0)).half()
    g = (1.0 + 0.2 * torch.randn(H, generator=gen)).half()
    return x.to(dev), r.to(dev), g.to(dev)


def _equal(a, b):
    torch = _torch()
    kind = {1: torch.int8, 2: torch.int16, 4: torch.int32}[a.element_size()]
    return a.shape == b.shape and torch.equal(a.contiguous().view(kind), b.contiguous().view(kind))


@pytest.mark.parametrize("M,H", SHAPES)
def test_as_the_separate_calls(mcv, cuda, M, H):
    torch = _torch()
    x, r, g = _rows(M + H, M, H, cuda)
    keep = x.clone(), r.clone()
    total = x + r
    out, res = mcv.rms_norm_add(x, r, g, 1e-6)
    assert _equal(res, total) and _equal(out, mcv.rms_norm(total, g, 1e-6)) and _equal(x, keep[0]) and _equal(r, keep[1])
    scale16 = torch.empty(M, dtype=torch.float16, device=cuda)
    want = mcv.rms_norm_w8a8_quantize(total, g, 1e-6, x_scale_f16=torch.empty_like(scale16))
    got = mcv.rms_norm_add_w8a8_quantize(x, r, g, 1e-6, x_scale_f16=scale16)
    assert got[3] is scale16 and all(_equal(a, b) for a, b in zip(got, (*want, total)))
    none, q, s, no16, res = mcv.rms_norm_add_w8a8_quantize(x, r, g, 1e-6, want_normed=False)
    assert none is None and no16 is None and _equal(q, want[1]) and _equal(s, want[2]) and _equal(res, total)
    # the definition: the sum exact and rounded once; the norm two roundings of 32-bit products and one to fp16
    z = (x.double() + r.double())
    assert _equal(res, z.half())
    z = z.half().double()
    y = z / (z.square().mean(-1, keepdim=True) + 1e-6).sqrt() * g.double()
    # 32 bits: two products, the root and its reciprocal, and the mean of H squares, H / 256 + 11 additions deep
    rel = 2.0 ** -11 + (6 + (H / 256 + 12) / 2) * 2.0 ** -24
    assert ((out.double() - y).abs() <= rel * y.abs() + 2.0 ** -25).all()


@pytest.mark.parametrize("M,H", [(3, 100), (5, 1024), (200, 1024), (2, 2056), (3, 9000)])
def test_in_place(mcv, cuda, M, H):
    x, r, g = _rows(M, M, H, cuda)
    out, total = mcv.rms_norm_add(x, r, g, 1e-5)
    a, b = x.clone(), r.clone()
    got = mcv.rms_norm_add(a, b, g, 1e-5, residual_out=b)
    assert got[1] is b and _equal(b, total) and _equal(got[0], out) and _equal(a, x)
    a, b = x.clone(), r.clone()
    got = mcv.rms_norm_add(a, b, g, 1e-5, out=b, residual_out=a)          # the sum in x's place, the norm in the residual's
    assert got[0] is b and got[1] is a and _equal(a, total) and _equal(b, out)
    want = mcv.rms_norm_add_w8a8_quantize(x, r, g, 1e-5)
    a, b = x.clone(), r.clone()
    got = mcv.rms_norm_add_w8a8_quantize(a, b, g, 1e-5, normed=a, residual_out=b)
    assert got[0] is a and got[4] is b and all(_equal(p, q) for p, q in zip(got[:3], want[:3])) and _equal(b, total)


@pytest.mark.parametrize("M,H", [(3, 72), (40, 1024), (7, 1000), (2, 9000)])
@pytest.mark.parametrize("first", [0, 1, 8])
def test_rows_of_wider_rows(mcv, cuda, M, H, first):
    """Columns of one projection's output, of any alignment; a residual row for all; sums beside what they are of."""
    torch = _torch()
    x, r, g = _rows(M + 1, M, H, cuda)
    out, total = mcv.rms_norm_add(x, r, g, 1e-6)
    wide = torch.full((M, 3 * H + 16), 9.0, dtype=torch.float16, device=cuda)
    wide[:, first:first + H], wide[:, first + H:first + 2 * H] = x, r
    xs, rs, ss = (wide[:, first + i * H:first + (i + 1) * H] for i in range(3))
    got = mcv.rms_norm_add(xs, rs, g, 1e-6, residual_out=ss)
    assert got[1] is ss and _equal(ss, total) and _equal(got[0], out) and _equal(xs, x) and _equal(rs, r)
    assert (wide[:, :first] == 9).all() and (wide[:, first + 3 * H:] == 9).all()
    one = r[:1].expand(M, -1)
    got = mcv.rms_norm_add(x, one, g, 1e-6)
    assert _equal(got[1], x + one) and _equal(got[0], mcv.rms_norm(x + one, g, 1e-6))


def test_not_finite(mcv, cuda):
    """An overflowing sum, an infinity or a NaN does to its row what it does to the separate calls', and to no other row."""
    torch = _torch()
    x, r, g = _rows(5, 6, 512, cuda)
    x[1, 3], r[1, 3] = 60000.0, 60000.0
    x[2, 0] = math.inf
    r[3, 511] = math.nan
    x[4], r[4] = 0.0, 0.0
    total = x + r
    out, res = mcv.rms_norm_add(x, r, g, 1e-6)
    want = mcv.rms_norm(total, g, 1e-6)
    assert torch.equal(res.isnan(), total.isnan()) and torch.equal(res.nan_to_num(), total.nan_to_num())
    assert torch.equal(out.isnan(), want.isnan()) and torch.equal(out.nan_to_num(), want.nan_to_num())
    assert torch.isfinite(out[[0, 4, 5]]).all() and (out[4] == 0).all()


def test_of_no_rows(mcv, cuda):
    torch = _torch()
    x, g = torch.zeros(0, 64, dtype=torch.float16, device=cuda), torch.ones(64, dtype=torch.float16, device=cuda)
    out, res = mcv.rms_norm_add(x, x, g, 1e-6)
    assert out.shape == res.shape == (0, 64)
    out, q, s, _, res = mcv.rms_norm_add_w8a8_quantize(x, x, g, 1e-6)
    assert q.shape == (0, 64) and s.shape == (0,)


def test_in_a_graph_and_on_another_stream(mcv, cuda):
    torch = _torch()
    x, r, g = _rows(8, 20, 1024, cuda)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out, _ = mcv.rms_norm_add(x, r, g, 1e-6, residual_out=r)
        normed, q, s, _, _ = mcv.rms_norm_add_w8a8_quantize(x, r, g, 1e-6)
    for turn in range(3):
        want, total = mcv.rms_norm_add(x, r, g, 1e-6)
        more = mcv.rms_norm_add_w8a8_quantize(x, total, g, 1e-6)
        graph.replay()
        torch.cuda.synchronize()
        assert _equal(out, want) and _equal(r, total) and all(_equal(a, b) for a, b in zip((normed, q, s), more[:3])), turn
    torch.cuda.synchronize()
    want = mcv.rms_norm_add(x, r, g, 1e-6)
    torch.cuda.synchronize()
    got = mcv.rms_norm_add(x, r, g, 1e-6, stream=side)
    side.synchronize()
    assert _equal(got[0], want[0]) and _equal(got[1], want[1])

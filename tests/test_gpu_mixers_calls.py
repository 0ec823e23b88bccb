"""What the token mixers' Python calls take: bounds, empty batches, layouts."""
import pytest

from test_gpu_mixers import _attn_case, _delta_case, _torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bound", [2 ** 30, 2 ** 40, 10 ** 6])
def test_any_bound_past_the_table_is_the_tables(mcv, cuda, bound):
    """A bound on the lengths that the table cannot reach changes nothing, the split of long caches included."""
    a = [x.to(cuda) for x in _attn_case(3, [30000] + [50] * 39, 2, 1, 64, 64)[:5]]
    assert (mcv.paged_attention_decode(*a, max_seq_len=bound) == mcv.paged_attention_decode(*a)).all()


def test_batches_of_none(mcv, cuda):
    torch = _torch()
    half = lambda *s: torch.zeros(*s, dtype=torch.float16, device=cuda)      # noqa: E731
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device=cuda)         # noqa: E731
    f32 = lambda *s: torch.zeros(*s, device=cuda)                            # noqa: E731
    out = mcv.paged_attention_decode(half(0, 8, 64), half(5, 16, 2, 64), half(5, 16, 2, 64), i32(0, 4), i32(0))
    assert out.shape == (0, 8, 64)
    held = half(0, 8, 64)
    assert mcv.paged_attention_decode(half(0, 8, 64), half(5, 16, 2, 64), half(5, 16, 2, 64), i32(0, 4), i32(0), out=held) is held
    state = f32(0, 4, 64, 32)
    out, new = mcv.gated_delta_rule_step(half(0, 2, 64), half(0, 2, 64), half(0, 4, 32), f32(0, 4), f32(0, 4), state)
    assert out.shape == (0, 4, 32) and new is state
    pool = torch.randn(3, 4, 64, 32, device=cuda)
    keep = pool.clone()
    out, new = mcv.gated_delta_rule_step(half(0, 2, 64), half(0, 2, 64), half(0, 4, 32), f32(0, 4), f32(0, 4), pool, state_index=i32(0))
    assert out.shape == (0, 4, 32) and new is pool and (pool == keep).all()
    with pytest.raises(mcv.McvError, match="gated_delta_rule_step"):         # none, and still of the wrong shape
        mcv.gated_delta_rule_step(half(0, 2, 64), half(0, 2, 64), half(0, 4, 32), f32(0, 4), f32(0, 4), f32(0, 4, 64, 64))
    with pytest.raises(mcv.McvError, match="paged_attention"):
        mcv.paged_attention_decode(half(0, 8, 64), half(5, 16, 3, 64), half(5, 16, 3, 64), i32(0, 4), i32(0))
    with pytest.raises(mcv.McvError, match="gated_delta_rule"):
        mcv.gated_delta_rule_step(half(0, 2, 96), half(0, 2, 96), half(0, 4, 32), f32(0, 4), f32(0, 4), f32(0, 4, 96, 32))


def _odd(t, dim):
    """The same values, the stride of a dimension of size 1 one that no access uses."""
    assert t.shape[dim] == 1
    strides = list(t.stride())
    strides[dim] = 3
    return t.as_strided(t.shape, strides)


def _same_bits(x, y):
    """(The rule with keys that are not normalised ends in NaN.)"""
    as_ints = {2: _torch().int16, 4: _torch().int32}[x.element_size()]
    return (x.view(as_ints) == y.view(as_ints)).all()


def test_strides_of_single_rows_and_heads(mcv, cuda):
    """A dimension of size 1 may have any stride."""
    q, k, v, g, beta, state = (x.to(cuda).contiguous() for x in _delta_case(1, [1], 1, 1, 64, 32))
    want = mcv.gated_delta_rule(q, k, v, g, beta, state)
    got = mcv.gated_delta_rule(*(_odd(_odd(x, 0), 1) for x in (q, k, v, g, beta)), state)
    assert all(_same_bits(x, y) for x, y in zip(got, want))
    q, k, v, g, beta, state = (x.to(cuda).contiguous() for x in _delta_case(1, [20], 1, 1, 64, 32))
    want = mcv.gated_delta_rule(q, k, v, g, beta, state)
    got = mcv.gated_delta_rule(*(_odd(x, 1) for x in (q, k, v, g, beta)), state)
    assert all(_same_bits(x, y) for x, y in zip(got, want))
    q, k, v, table, n = (x.to(cuda) for x in _attn_case(1, [70], 1, 1, 64, 16)[:5])
    want = mcv.paged_attention_decode(q, k, v, table, n)
    assert _same_bits(mcv.paged_attention_decode(_odd(_odd(q, 0), 1), _odd(k, 2), _odd(v, 2), _odd(table, 0), n), want)
    torch = _torch()
    freq, axis = mcv.rotary_axes_table(32, 1e4, (6, 5, 5), device=cuda)
    pos = torch.tensor([[5], [3], [9]], device=cuda)
    x, y = (torch.randn(1, 1, 64, device=cuda).half() for _ in range(2))
    want = mcv.rotary_axes(x, y, pos, freq, axis)
    odd = [torch.empty(1, 1, 64, dtype=torch.float16, device=cuda) for _ in range(2)]
    got = mcv.rotary_axes(_odd(_odd(x, 0), 1), _odd(_odd(y, 0), 1), _odd(pos, 1), freq, axis, q_out=_odd(_odd(odd[0], 0), 1), k_out=_odd(odd[1], 0))
    assert all(_same_bits(a, b) for a, b in zip(got, want))

"""What the token mixers' Python calls take: bounds, empty batches, layouts."""
import pytest

from test_gpu_mixers import _attn_case, _torch

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

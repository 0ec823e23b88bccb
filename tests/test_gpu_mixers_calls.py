"""What the token mixers' Python calls take: bounds, empty batches, layouts."""
import pytest

from test_gpu_mixers import _attn_case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bound", [2 ** 30, 2 ** 40, 10 ** 6])
def test_any_bound_past_the_table_is_the_tables(mcv, cuda, bound):
    """A bound on the lengths that the table cannot reach changes nothing, the split of long caches included."""
    a = [x.to(cuda) for x in _attn_case(3, [30000] + [50] * 39, 2, 1, 64, 64)[:5]]
    assert (mcv.paged_attention_decode(*a, max_seq_len=bound) == mcv.paged_attention_decode(*a)).all()

"""Arguments that a call would not heed are refused, on the CPU: nothing is computed before."""
import pytest

from conftest import seeded
from tensorax_b200 import Tensor
from tensorax_b200.nn import GroupedQueryAttention


@pytest.mark.parametrize("more", [{"align": "end"}, {"sinks": 4}, {"align": "end", "sinks": 4, "causal": True}])
def test_alignment_and_sinks_belong_to_a_window(more):
    layer = GroupedQueryAttention(4, 2)
    q, k, v = (Tensor(seeded(i, 1, h, 8, 64).tolist()) for i, h in enumerate((4, 2, 2)))
    with pytest.raises(ValueError, match="window"):
        layer.forward_bhsd(q, k, v, **more)

"""Many rows over a cache whose keys are cut over a cluster: the last CTA's share is a few nodes that do not see each other."""
import numpy as np
import pytest

import tensorax_b200 as ts
from conftest import seeded
from tensorax_b200 import _C
from tensorax_b200.nn import QuantizedKVCache

pytestmark = pytest.mark.gpu

LEAVES = [1, 2, 3, 7, 9]


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("leaves", LEAVES)
@pytest.mark.parametrize("heads, full", [(2, 1024), (1, 1024), (2, 896), (6, 256)])
def test_the_only_key_of_a_share_is_not_finite(heads, full, leaves, d, fmt):
    """The last node's key, or value, is not finite: only that node sees it, and of the CTA's keys it sees that alone."""
    T, page, keys = 64, 16, full + leaves
    table = np.random.default_rng(5).permutation(68)[None].astype(np.int32)
    for of_k in (0, 1):
        kv = [seeded(1 + i, 1, 1, 68 * page, d) for i in range(2)]
        kv[of_k][0, 0, keys - 1, 9] = np.nan if of_k else np.inf
        cache = QuantizedKVCache(68, 1, d, page, fmt)
        cache.write(*(ts.Tensor._wrap(_C.from_numpy(x)) for x in kv), table)
        words = np.array([[(2 << t) - 1 if t < T - leaves else (1 << (T - leaves)) - 1 | 1 << t for t in range(T)]], dtype=np.uint64)
        q = seeded(7, 1, heads, T, d).astype(np.float16)
        got = cache.attend(ts.Tensor._wrap(_C.from_numpy(q)), table, [keys], tree=words).numpy()
        assert np.isnan(got[0, :, T - 1]).all() and np.isfinite(got[0, :, : T - 1]).all()

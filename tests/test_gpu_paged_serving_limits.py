"""The serving calls at the limits of what a batch may hold: tokens cut off by a bound or by the pages held.  Models, tolerances
and helpers are those of test_gpu_paged_serving."""
import numpy as np
import pytest

from tests.gpu_util import ctx, fa
from tests.test_gpu_paged_serving import TreeCase

pytestmark = pytest.mark.gpu


# ---- tokens that a bound or the pages held cut off, inside a tile that holds live tokens only -------

CLIPPED = [  # live tokens, drafted tokens, and the tokens that are left of each sequence: by max_context, or by the pages held
    ([140], [5], 80, None), ([140], [5], 70, None), ([140], [5], None, [6]), ([140], [5], None, [0]), ([140], [70], 80, None), ([140], [70], None, [5]),
    ([150, 1000, 30], [5, 3, 2], 500, None), ([150, 1000, 30], [40, 33, 2], 500, None), ([700, 200, 90], [3, 70, 1], None, [20, 1, 0]),
    ([6000], [3], 4010, None), ([6000], [40], 4010, None), ([9000, 700], [2, 5], None, [301, 2])]


@pytest.mark.parametrize("dtype,Hq,Hkv,D", [(fa.BF16, 4, 1, 64), (fa.BF16, 8, 2, 128), (fa.F32, 4, 2, 64)])
@pytest.mark.parametrize("lens,nodes,most,held", CLIPPED, ids=str)
def test_live_tokens_that_are_cut_off_do_not_count(dtype, Hq, Hkv, D, lens, nodes, most, held):
    """Products of 64 and of 128 rows, items of one CTA and of many parts."""
    t = TreeCase(sum(lens) + D, dtype, Hq, Hkv, D, 16, lens, nodes)
    left = [most] * len(lens)
    if held is not None:
        left = [n * t.page for n in held]
        t.held = np.array(held, np.int32)
    got = t.run(ctx(), max_context=most, status=35)
    t.check(got, t.exact(drop=[(s, n, a + b) for s, (n, a, b) in enumerate(zip(left, lens, nodes)) if n < a + b]))

"""Attention over a paged cache at the ends of the fp32 range: queries, keys and scales each far from one whose scores are
ordinary numbers.  The plain form and the bars are test_gpu_paged's."""
import numpy as np
import pytest

from test_gpu_paged import Tree, dev

pytestmark = pytest.mark.gpu

ROWS = [1, 3, 8, 60]                                    # of 7 heads a KV head: blocks of 16, 32, 64 and 128 rows
HEADS = [(14, 2, 32), (14, 2, 64), (14, 2, 128)]


def put(t, q=None, k=None, v=None):
    """Changed queries, keys and values (arrays of t's shapes) to the device."""
    if q is not None:
        t.q = q.astype(np.float32)
        t.keep["q"] = dev(t.gpu, t.q)
        t.a.q = t.keep["q"].ptr
    for c, x in enumerate((k, v)):
        if x is not None:
            t.c.buf[c] = x.astype(np.float32)
            t.c.put("kv"[c], t.c.buf[c])


@pytest.mark.parametrize("v", [0, 100])
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("heads", HEADS, ids=str)
def test_products_past_fp32_under_a_small_scale(gpu, heads, rows, v):
    """q.K past 2^128, with the scale some tens; v: values of 2^v beside them."""
    t = Tree(gpu, [(200, rows), (40, 2)], *heads, 16, False, kind="tree", scale=2.0**-126, seed=7)
    put(t, t.q * np.float32(2.0**28), t.c.buf[0] * np.float32(2.0**100), t.c.buf[1] * np.float32(2.0**v))
    t.check()

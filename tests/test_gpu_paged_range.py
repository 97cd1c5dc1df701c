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


@pytest.mark.parametrize("sign", [0, -1])
@pytest.mark.parametrize("at", [40, 60, 75, 90, 100, 110, 120])
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("heads", HEADS, ids=str)
def test_small_queries_beside_large_keys(gpu, heads, rows, at, sign):
    """Scores of ordinary size from keys of 2^at and queries of 2^-at; sign -1: every score below zero."""
    t = Tree(gpu, [(200, rows), (40, 2)], *heads, 16, False, kind="tree", seed=at)
    q, k = t.q * np.float32(2.0**-at), t.c.buf[0] * np.float32(2.0**at)
    put(t, -abs(q), abs(k)) if sign else put(t, q, k)
    t.check()


@pytest.mark.parametrize("up", [-1, 1])
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("heads", HEADS, ids=str)
def test_queries_far_smaller_than_keys_are_large(gpu, heads, rows, up):
    """Queries of 2^-112 and keys of 2^100, as they are and with a few keys among them whose scores count."""
    t = Tree(gpu, [(200, rows), (40, 2)], *heads, 16, False, kind="tree", seed=3)
    k = t.c.buf[0] * np.float32(2.0**100)
    if up > 0:
        k[::3] *= np.float32(2.0**12)
    put(t, t.q * np.float32(2.0**-112), k)
    t.check()


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("heads", HEADS, ids=str)
def test_large_queries_and_scale_beside_small_keys(gpu, heads, rows):
    """One value of 2^127 a query, a scale of 2^12, keys of a few 2^-140: scores of a few halves."""
    t = Tree(gpu, [(200, rows), (40, 2)], *heads, 16, False, kind="tree", scale=4096.0, seed=5)
    rng = np.random.default_rng(6)
    q = np.zeros(t.q.shape, np.float32)
    q[..., 5] = np.float32(2.0**127) * rng.choice([-1, 1], q.shape[:2])
    k = np.where(np.isnan(t.c.buf[0]), np.nan, rng.integers(-8, 9, t.c.buf[0].shape) * 2.0**-140)
    put(t, q, k)
    t.check()


@pytest.mark.parametrize("v", [0, 100])
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("heads", HEADS, ids=str)
def test_products_past_fp32_under_a_small_scale(gpu, heads, rows, v):
    """q.K past 2^128, with the scale some tens; v: values of 2^v beside them."""
    t = Tree(gpu, [(200, rows), (40, 2)], *heads, 16, False, kind="tree", scale=2.0**-126, seed=7)
    put(t, t.q * np.float32(2.0**28), t.c.buf[0] * np.float32(2.0**100), t.c.buf[1] * np.float32(2.0**v))
    t.check()


@pytest.mark.parametrize("rows", ROWS)
def test_scale_of_zero_and_the_largest_keys(gpu, rows):
    """The average of the values where the scale is 0, with keys and queries near the largest fp32 number."""
    t = Tree(gpu, [(200, rows), (40, 2)], 14, 2, 64, 16, False, kind="tree", scale=0.0, seed=8)
    put(t, np.sign(t.q) * np.float32(3e38), np.sign(t.c.buf[0]) * np.float32(3e38))
    t.check()


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("rows", ROWS)
def test_smallest_queries(gpu, rows, half):
    """Queries of the smallest fp32 numbers and of zeros beside ordinary keys: the average of what a row sees."""
    t = Tree(gpu, [(200, rows), (40, 2)], 14, 2, 64, 16, half, kind="tree", seed=9)
    q = t.q * np.float32(2.0**-140)
    q[::2] = 0
    put(t, q)
    t.check()


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("scale", [1.3 * 2.0**-132, 1.3 * 2.0**-142])
@pytest.mark.parametrize("rows", ROWS)
def test_subnormal_scale(gpu, rows, scale, half):
    """A scale below fp32's normal range beside queries and keys that make up for it."""
    scale = float(np.float32(scale))
    t = Tree(gpu, [(200, rows), (40, 2)], 14, 2, 64, 16, half, kind="tree", scale=scale, seed=10)
    up = int(np.round(-np.log2(scale))) - 3
    if half:
        put(t, t.q * np.float32(2.0**min(up, 124)))
        t.c.buf[0] = (t.c.buf[0] * np.float16(2.0**(up - min(up, 124)) / 16)).astype(np.float16)
        t.c.put("k", t.c.buf[0])
    else:
        put(t, t.q * np.float32(2.0**(up // 2)), t.c.buf[0] * np.float32(2.0**(up - up // 2)))
    t.check()

"""Attention over a shared prefix at the ends of fp32: values whose sizes differ from group to group of keys by more than
any one power of two covers, in every form of the kernel.

Bars as in test_gpu_score, from the same sums, without their absolute part: relative to sum p |v| of the row
and dim, and one subnormal step (2^-149) for each key and each of the few operations on the result."""
import numpy as np
import pytest

from test_gpu_score import U, Attn, cut_case, renew

pytestmark = pytest.mark.gpu

HD_HEADS = {32: (6, 2, 32), 64: (14, 2, 64), 128: (8, 2, 128)}
# few: at most 32 rows and heads a KV head share a block; step: more, each sequence at most 32; rows: more a sequence; cut:
# the prefix cut ahead.
FORMS = ["few", "step", "rows", "cut_step", "cut_rows"]
SHORT, MANY = [(2, 3), (1, 70)], [(2, 3)] * 9 + [(1, 70), (3, 33)]
LONG = [(41, 3), (2, 140), (70, 0)]


def case(gpu, form, HD, P=330, **kw):
    heads = HD_HEADS[HD]
    if form == "few":
        return Attn(gpu, SHORT, P, *heads, **kw)
    if form == "step":
        rows = -(-33 * heads[1] // heads[0])
        return Attn(gpu, MANY, P, *heads, behind=max(0, rows - 25), **kw)
    if form == "rows":
        return Attn(gpu, LONG, P, *heads, **kw)
    return cut_case(gpu, SHORT if form == "cut_step" else LONG, P + 700, *heads, **kw)


def sized(t, sizes, width):
    """Rows of t in groups of `width` keys, scaled by the sizes in turn."""
    t *= np.resize(np.repeat(np.asarray(sizes, np.float32), width), len(t))[:, None, None]


def exact(c):
    """(out, bar) in 64 bits of the rows that belong to a sequence."""
    G = c.NH // c.NKV
    out, bar = {}, {}
    for b in range(c.a.B):
        q0, q1 = int(c.q_start[b]), int(c.q_start[b + 1])
        first, n = int(c.kv_start[b]), int(c.kv_len[b])
        for r in range(q0, q1):
            seen = min(max(n - (q1 - q0) + (r - q0) + 1, 0), n)
            K = np.concatenate([c.kp, c.ks[first:first + seen]]).astype(np.float64).repeat(G, 1)
            W = np.concatenate([c.vp, c.vs[first:first + seen]]).astype(np.float64).repeat(G, 1)
            q = c.q[r].astype(np.float64)
            s = np.einsum("hd,khd->hk", q, K) * c.scale
            ds = c.HD * U * np.einsum("hd,khd->hk", abs(q), abs(K)) * c.scale
            p = np.exp(s - s.max(1, keepdims=True))
            p /= p.sum(1, keepdims=True)
            out[r] = np.einsum("hk,khd->hd", p, W)
            tol = p * (2 * ds + 2 * (p * ds).sum(1, keepdims=True) + (2 * len(K) + 16) * U)
            bar[r] = np.einsum("hk,khd->hd", tol, abs(W)) + (len(K) + 8) * 2.0**-149
    return out, bar


def compare(c):
    got = c.out()
    want, bar = exact(c)
    for r in want:
        bad = ~(np.abs(got[r] - want[r]) <= bar[r])
        assert not bad.any(), (r, np.argwhere(bad)[0].tolist(), got[r][bad][:3], want[r][bad][:3])
    rest = np.ones(c.R, bool)
    rest[list(want)] = False
    assert np.all(got[rest] == -77.0)


SIZES = [(1e-33, 1.0), (1.0, 1e-33), (1e20, 1e-20), (1e-20, 1e20), (1e7, 1e-34), (1e-34, 1e7), (1e-33,), (1e30, 1e-30, 1.0),
         (1e-37, 1e18, 1e-10), (2e13, 2e-16), (2e-16, 2e13)]


@pytest.mark.parametrize("sizes", SIZES, ids=str)
@pytest.mark.parametrize("HD", [32, 64, 128])
@pytest.mark.parametrize("form", FORMS)
def test_attn_values_of_very_different_size(gpu, form, HD, sizes):
    """Whole groups of keys with values of one size beside groups of another, scores alike: every key keeps its weight."""
    print("sizes", form, HD, sizes, flush=True)
    c = case(gpu, form, HD, seed=HD)
    sized(c.vp, sizes, 128 if len(sizes) == 3 else 32)
    for s, n in zip(c.kv_start, c.kv_len):
        sized(c.vs[s:s + n], sizes, 32)
    renew(gpu, c, "vp", "vs")
    c.call()
    gpu.synchronize()
    compare(c)


@pytest.mark.parametrize("sizes", [(2e13, 2e-16), (2e-16, 1.0, 2e13)], ids=str)
@pytest.mark.parametrize("HD", [32, 64, 128])
@pytest.mark.parametrize("form", FORMS)
def test_attn_values_of_very_different_size_far_scores(gpu, form, HD, sizes):
    """... and scores some hundred binary orders apart, so that small values outweigh large ones in some rows."""
    print("sizes", form, HD, sizes, flush=True)
    c = case(gpu, form, HD, seed=HD + 1, scale=2.0)
    sized(c.vp, sizes, 32)
    renew(gpu, c, "vp")
    c.call()
    gpu.synchronize()
    compare(c)


@pytest.mark.parametrize("HD", [32, 64, 128])
@pytest.mark.parametrize("form", FORMS)
def test_attn_values_at_the_top_of_fp32(gpu, form, HD):
    """Averages of values near fp32's largest are finite, whatever their sum."""
    c = case(gpu, form, HD, seed=HD + 2)
    c.vp[:] = np.where(c.vp > -1.5, np.float32(3e38), np.float32(-1e38))
    c.vs[:] = np.where(np.isnan(c.vs), c.vs, np.float32(2.9e38))
    c.vp[5:150] = 1.0                                          # beside values of an ordinary size
    renew(gpu, c, "vp", "vs")
    c.call()
    gpu.synchronize()
    compare(c)


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("x", [-0.328125, -0.015625, -0.21875])
def test_logprobs_sum_of_many_equal_values(gpu, x, half):
    """Rows of 819200 logits of one value after 8192 larger ones, which every lane sees: rounding errors of one sign.  Bar: an exponential is off by
    3.5 u; a lane adds a tile of 32 in 10 roundings and V / 8192 tiles, then lanes, waves and chunks join in 27: so much of the
    sum, and in its logarithm; the logarithm and the two differences round by 3 u of at most 14; an entropy has a weighted sum of
    the same roundings, times |x|, besides."""
    V, rows = 819200, 513                                      # a row in one piece
    row = np.full(V, x, np.float16 if half else np.float32)
    row[:8192] = 0.0
    size = row.dtype.itemsize
    dx = gpu.DeviceArray(rows * V, np.uint16 if half else np.float32)
    one = gpu.DeviceArray.from_host(row.view(np.uint16) if half else row)
    for r in range(rows):
        gpu.call("sgpu_memcpy_dtod_async", dx.ptr + r * V * size, one.ptr, V * size, None)
    tok = gpu.DeviceArray.from_host(np.tile(np.array([[12, 8200, V - 1]], np.int32), (rows, 1)))
    lp, ent = gpu.DeviceArray((rows, 3)), gpu.DeviceArray(rows)
    need = gpu.lib().sgpu_logprobs_workspace(rows, V, 0)
    ws = gpu.DeviceArray(need, np.uint8)
    gpu.call("sgpu_logprobs_h" if half else "sgpu_logprobs", dx.ptr, V, rows, V, tok.ptr, 3, lp.ptr, ent.ptr, 0, None, None, ws.ptr, need, None)
    gpu.synchronize()
    got, h = lp.to_host(), ent.to_host()
    n = V - 8192
    z = 8192 + n * np.exp(x)
    want = np.array([0.0, x, x]) - np.log(z)
    bar = (V / 8192 + 41 + 3 * 14) * U
    assert np.all(np.abs(got - want) <= bar), (np.abs(got - want).max() / U, bar / U)
    H = np.log(z) - n * np.exp(x) * x / z
    assert np.all(np.abs(h - H) <= bar + 2 * abs(x) * bar), (np.abs(h - H).max() / U, bar / U)
    assert np.all(got == got[0]) and np.all(h == h[0])
    dx.close()

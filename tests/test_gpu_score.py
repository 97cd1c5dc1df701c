"""The operators over several continuations of one prompt (rotary rows, log probabilities, attention
over a shared prefix) against plain implementations in 64 bits.

Bars, from the arithmetic (u = 2^-24, half an fp32 step):
  rope      cos and sin are off by at most 3.6 u (reduction 0.6, series 1, table factor 1, and the
            series' own remainder below 0.1), each product and the sum round once more: 6 u (|a| + |b|);
            an fp16 result rounds once, 2^-11 |y| (2^-25 below its normal range)
  logprobs  every exponential is off by (2 |y| + 2) u where it matters (2^-y |y| is below 1), a lane adds
            V / 256 + 64 of them one by one: relative (V / 256 + 70) u of the sum, so as much in its
            logarithm; the difference to the maximum and the result round once: 2 u of each
  attention a score is a sum of HD products: HD u sum |q k| scale; a weight is off by twice that and 4 u, a
            sum over n keys adds n u, in the output each relative to sum p |v|
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0**-24


def dev(gpu, a):
    return gpu.DeviceArray.from_host(np.ascontiguousarray(a))


# ---- rotary rows ----
def rope64(x, pos, turns, rot, nb, mscale):
    y = x.astype(np.float64).copy()
    bar = np.zeros(x.shape)
    ang = 2 * np.pi * np.mod(pos.astype(np.float64)[:, None] * turns, 1.0)
    c, s = np.cos(ang)[:, None] * mscale, np.sin(ang)[:, None] * mscale
    h = rot // 2
    i0, i1 = (np.arange(0, rot, 2), np.arange(1, rot, 2)) if nb else (np.arange(h), np.arange(h, rot))
    a, b = x[..., i0].astype(np.float64), x[..., i1].astype(np.float64)
    y[..., i0], y[..., i1] = a * c - b * s, a * s + b * c
    bar[..., i0] = bar[..., i1] = 6 * U * (abs(a) + abs(b)) * mscale
    return y, bar


ROPE = [
    # T, H, HD, rot, neighbours, fp16, offset of x in floats, offset of y in values
    (1, 16, 64, 64, 0, False, 0, 0), (1, 1, 2, 2, 1, False, 0, 0), (3, 14, 64, 64, 0, False, 0, 0),
    (5, 3, 80, 40, 0, False, 0, 0), (5, 3, 80, 40, 1, True, 0, 0), (7, 2, 128, 64, 1, True, 0, 0),
    (7, 2, 128, 64, 1, False, 1, 0), (7, 2, 128, 64, 0, True, 0, 1), (4, 5, 33, 6, 0, False, 0, 0), (4, 5, 33, 6, 1, True, 3, 5),
    (2, 3, 256, 256, 0, False, 0, 0), (2, 3, 256, 256, 1, True, 0, 0), (9, 4, 64, 0, 0, True, 0, 0), (9, 4, 64, 0, 0, False, 0, 0),
    (3001, 2, 32, 32, 0, False, 0, 0), (4100, 1, 16, 8, 1, False, 0, 0), (6, 2, 64, 12, 0, False, 0, 0),
    (2, 40, 128, 128, 0, True, 0, 0)]


@pytest.mark.parametrize("case", ROPE, ids=str)
@pytest.mark.parametrize("where", ["none", "far", "back"])
def test_rope_rows(gpu, case, where):
    T, H, HD, rot, nb, half, xo, yo = case
    rng = np.random.default_rng(T * 7 + HD)
    n = H * HD
    xs, ys = n + (5 if xo else 8), n + (3 if yo else 16)
    x = rng.standard_normal(xo + T * xs).astype(np.float32)
    turns = (1e4 ** (-2.0 * np.arange(max(rot // 2, 1)) / max(rot, 1))) / (2 * np.pi)
    mscale, pos0 = 1.25, {"none": 11, "far": 2000000000, "back": 0}[where]
    pos = {"none": None, "far": rng.integers(0, 100000000, T), "back": -rng.integers(0, 1000000, T)}[where]
    at = pos0 + (np.arange(T) if pos is None else pos)
    dt = np.float16 if half else np.float32
    y = np.full(yo + T * ys, 7.0, dt)
    dx, dy, dt_ = dev(gpu, x), dev(gpu, y), dev(gpu, turns)
    dp = None if pos is None else dev(gpu, pos.astype(np.int32))
    gpu.call("sgpu_rope_rows_h" if half else "sgpu_rope_rows", dx.offset(xo), xs, dy.offset(yo), ys, dp.ptr if dp else None, pos0,
             dt_.ptr, rot, nb, mscale, T, H, HD, None)
    gpu.synchronize()
    got = dy.to_host()
    rows = x[xo:].reshape(T, xs)[:, :n].reshape(T, H, HD)
    want, bar = rope64(rows, at, turns, rot, nb, mscale)
    if half:
        bar = bar + np.maximum(np.abs(want) * 2.0**-11, 2.0**-25) * 1.001
    g = got[yo:].reshape(T, ys)
    assert np.array_equal(g[:, n:], np.full((T, ys - n), 7.0, dt)) and np.all(got[:yo] == 7.0)       # what lies between rows
    assert np.all(np.abs(g[:, :n].reshape(T, H, HD).astype(np.float64) - want) <= bar + 1e-300)
    if rot < HD and not half:
        assert np.array_equal(g[:, :n].reshape(T, H, HD)[..., rot:], rows[..., rot:])                # passes through
    assert np.array_equal(dx.to_host(), x)


@pytest.mark.parametrize("nb", [0, 1])
def test_rope_rows_in_place_and_back(gpu, nb):
    """In place, the values past rot bit for bit; turned back by the negated positions."""
    rng = np.random.default_rng(3)
    T, H, HD, rot = 37, 6, 64, 32
    x = rng.standard_normal((T, H * HD + 4)).astype(np.float32)
    x[:, H * HD:] = np.nan
    turns, _ = gpu.rope_turns(rot, 1e4, gpu.ROPE_YARN, 4.0, 2048.0, 32.0, 1.0)
    pos = rng.integers(0, 50000, T).astype(np.int32)
    dx, dt, dp, dn = dev(gpu, x), dev(gpu, turns), dev(gpu, pos), dev(gpu, -pos)
    gpu.call("sgpu_rope_rows", dx.ptr, H * HD + 4, dx.ptr, H * HD + 4, dp.ptr, 0, dt.ptr, rot, nb, 1.0, T, H, HD, None)
    gpu.synchronize()
    got = dx.to_host()
    rows = x[:, :H * HD].reshape(T, H, HD)
    want, bar = rope64(rows, pos, turns, rot, nb, 1.0)
    g = got[:, :H * HD].reshape(T, H, HD)
    assert np.all(np.abs(g - want) <= bar) and np.array_equal(g[..., rot:], rows[..., rot:]) and np.isnan(got[:, H * HD:]).all()
    gpu.call("sgpu_rope_rows", dx.ptr, H * HD + 4, dx.ptr, H * HD + 4, dn.ptr, 0, dt.ptr, rot, nb, 1.0, T, H, HD, None)
    gpu.synchronize()
    back = dx.to_host()[:, :H * HD].reshape(T, H, HD)
    # twice the bar: the pair's length stays, |a| + |b| grows by sqrt 2 at most
    assert np.all(np.abs(back - rows) <= 2.5 * np.maximum(bar, 0) + 0) and np.array_equal(back[..., rot:], rows[..., rot:])


def test_rope_rows_is_the_engines_rope(gpu, og):
    """The table form (sgpu_rope) and the rows form agree on the engines' layout."""
    rng = np.random.default_rng(5)
    T, H, HD, pos0 = 9, 16, 64, 100
    c, s = og.rope_tables(256, HD, 1e6)
    x = rng.standard_normal((T, H, HD)).astype(np.float32)
    dx, dy, dc, ds = dev(gpu, x), dev(gpu, x), dev(gpu, c), dev(gpu, s)
    dt = dev(gpu, gpu.rope_turns(HD, 1e6)[0])
    gpu.call("sgpu_rope", dx.ptr, dc.ptr, ds.ptr, T, H, HD, pos0, None)
    gpu.call("sgpu_rope_rows", dy.ptr, H * HD, dy.ptr, H * HD, None, pos0, dt.ptr, HD, 0, 1.0, T, H, HD, None)
    gpu.synchronize()
    h = HD // 2
    pair = np.abs(x[..., :h]) + np.abs(x[..., h:])
    assert np.all(np.abs(dx.to_host() - dy.to_host()) <= 12 * U * np.concatenate([pair, pair], -1))


# ---- log probabilities ----
def logprobs64(x, tok, k):
    x = x.astype(np.float64)
    m = x.max(1, keepdims=True)
    with np.errstate(all="ignore"):
        z = x - m
        e = np.where(np.isneginf(x), 0.0, np.exp(z))
        Z = e.sum(1, keepdims=True)
        lz = np.log(Z)
        lp = z - lz
        ent = (lz - np.where(e > 0, e * np.where(e > 0, z, 0), 0).sum(1, keepdims=True) / Z)[:, 0]
    none = np.isneginf(m[:, 0])
    lp[none], ent[none] = -np.inf, 0.0
    odd = np.isnan(x).any(1) | np.isposinf(x).any(1)
    lp[odd], ent[odd] = np.nan, np.nan
    V = x.shape[1]
    ids = np.argsort(-x, axis=1, kind="stable")[:, :k]
    top = np.take_along_axis(lp, ids, 1)
    if V < k:
        ids = np.concatenate([ids, np.full((len(x), k - V), -1)], 1)
        top = np.concatenate([top, np.full((len(x), k - V), -np.inf)], 1)
    ids[odd], top[odd] = -1, np.nan
    ok = (tok >= 0) & (tok < V)
    given = np.where(ok, np.take_along_axis(lp, np.where(ok, tok, 0), 1), 0.0)
    return given, ent, top, ids


def run_logprobs(gpu, x, tok, k, ld=None, entropy=True, stream=None, keep=None):
    """x: (rows, V) fp32 or fp16; NaN between the rows where ld > V."""
    rows, V = x.shape
    ld = ld or V
    buf = np.full((rows, ld), np.nan, x.dtype)
    buf[:, :V] = x
    nt = tok.shape[1]
    d = keep if keep is not None else {}
    d["x"] = dev(gpu, buf)
    d["tok"] = dev(gpu, tok.astype(np.int32)) if nt else None
    need = gpu.lib().sgpu_logprobs_workspace(rows, V, k)
    d["ws"] = dev(gpu, np.full(need + 16, 0xA5, np.uint8))
    d["logp"], d["ent"] = dev(gpu, np.full((rows, max(nt, 1)), 5, np.float32)), dev(gpu, np.full(rows, 5, np.float32))
    d["top"], d["ids"] = dev(gpu, np.full((rows, max(k, 1)), 5, np.float32)), dev(gpu, np.full((rows, max(k, 1)), -7, np.int32))
    fn = "sgpu_logprobs_h" if x.dtype == np.float16 else "sgpu_logprobs"

    def call(st=stream):
        gpu.call(fn, d["x"].ptr, ld, rows, V, d["tok"].ptr if nt else None, nt, d["logp"].ptr if nt else None,
                 d["ent"].ptr if entropy else None, k, d["top"].ptr if k else None, d["ids"].ptr if k else None, d["ws"].ptr, need, st)

    def results():
        assert np.all(d["ws"].to_host()[need:] == 0xA5)
        return (d["logp"].to_host()[:, :nt], d["ent"].to_host(), d["top"].to_host()[:, :k], d["ids"].to_host()[:, :k])

    if keep is not None:
        return call, results
    call()
    gpu.synchronize()
    return results()


def check_logprobs(x, tok, k, got):
    V = x.shape[1]
    lp, ent, top, ids = got
    wlp, went, wtop, wids = logprobs64(x, tok, k)
    rel = (V / 256 + 70) * U
    finite = np.where(np.isfinite(x), np.abs(x.astype(np.float64)), 0).max(1) if V else 0

    def near(g, w, extra):
        f = np.isfinite(w)
        assert np.array_equal(np.isfinite(g), f) and np.array_equal(np.isnan(g), np.isnan(w)) and np.array_equal(g[~f & ~np.isnan(w)], w[~f & ~np.isnan(w)])
        with np.errstate(invalid="ignore"):
            bad = f & ~(np.abs(g - np.where(f, w, 0)) <= rel + 4 * U * np.abs(np.where(f, w, 0)) + extra)
        assert not bad.any(), (g[bad][:5], w[bad][:5])

    assert np.array_equal(ids, wids)
    near(lp, wlp, 0)
    near(top, wtop, 0)
    # the entropy is a sum of p |ln p|: its parts carry the exponentials' error
    near(ent, went, rel * np.where(np.isfinite(went), went, 0) * 2)


LOGP = [(1, 151936, 1, 20), (3, 50257, 2, 5), (70, 8192, 1, 1), (2, 8193, 0, 64), (5, 1, 1, 3), (4, 7, 3, 10), (9, 63, 1, 64),
        (6, 64, 1, 64), (2, 65, 1, 64), (33, 1000, 17, 0), (1, 262143, 4, 33), (1030, 2049, 1, 2), (2, 2048, 1, 63)]


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("case", LOGP, ids=str)
def test_logprobs(gpu, case, half):
    rows, V, nt, k = case
    rng = np.random.default_rng(rows + V)
    x = (rng.standard_normal((rows, V)) * 4).astype(np.float16 if half else np.float32)
    tok = rng.integers(0, V, (rows, nt))
    check_logprobs(x, tok, k, run_logprobs(gpu, x, tok, k))
    check_logprobs(x, tok, k, run_logprobs(gpu, x, tok, k, ld=V + 3))


ROWS = {
    "ascending": lambda r, V: np.arange(V) * 0.001,
    "descending": lambda r, V: -np.arange(V) * 0.001,
    "equal": lambda r, V: np.full(V, 2.5),
    "few values": lambda r, V: r.integers(0, 4, V).astype(float),
    "zeros of both signs": lambda r, V: np.where(r.random(V) < 0.5, 0.0, -0.0),
    "around zero": lambda r, V: r.integers(-1, 2, V) * 0.0 + r.integers(-1, 2, V) * 1e-5,
    "masked": lambda r, V: np.where(r.random(V) < 0.9, -np.inf, r.standard_normal(V)),
    "one left": lambda r, V: np.where(np.arange(V) == V // 3, 1.5, -np.inf),
    "nothing left": lambda r, V: np.full(V, -np.inf),
    "lowest": lambda r, V: np.full(V, -65504.0),
    "lowest but one": lambda r, V: np.where(np.arange(V) == V - 1, 3.0, -65504.0),
    "sure": lambda r, V: np.where(np.arange(V) == 5 % V, 60.0, r.standard_normal(V)),
    "far apart": lambda r, V: r.standard_normal(V) * 300,
    "a NaN": lambda r, V: np.where(np.arange(V) == V // 2, np.nan, r.standard_normal(V)),
    "all NaN": lambda r, V: np.full(V, np.nan),
    "an infinity": lambda r, V: np.where(np.arange(V) == V // 2, np.inf, r.standard_normal(V)),
    "negative": lambda r, V: -50 - np.abs(r.standard_normal(V)),
}


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("V,k", [(5, 3), (700, 64), (20011, 20)])
def test_logprobs_of_odd_rows(gpu, V, k, half):
    """All kinds of row side by side, so that a row that goes wrong can harm its neighbours."""
    rng = np.random.default_rng(V)
    x = np.stack([f(rng, V) for f in ROWS.values()]).astype(np.float16 if half else np.float32)
    tok = rng.integers(0, V, (len(x), 4))
    tok[:, 1], tok[:, 2] = -1, V                               # no tokens of the vocabulary
    tok[3] = [np.iinfo(np.int32).min, np.iinfo(np.int32).max, 0, V - 1]
    check_logprobs(x, tok, k, run_logprobs(gpu, x, tok, k, ld=V + 1))


def test_logprobs_lowest_fp32(gpu):
    """Rows masked with the type's lowest value, and logits at its ends."""
    V, low = 9001, np.finfo(np.float32).min
    rng = np.random.default_rng(1)
    x = rng.standard_normal((4, V)).astype(np.float32)
    x[0, ::2] = low
    x[1] = low
    x[2, 10], x[2, 11] = -low, low
    x[3] = np.where(np.arange(V) % 3 == 0, -low, low)
    tok = np.tile(np.array([[0, 10, 11]]), (4, 1))
    lp, ent, top, ids = run_logprobs(gpu, x, tok, 5)
    wlp, went, wtop, wids = logprobs64(x.astype(np.longdouble), tok, 5)
    # a difference of two such numbers leaves fp32: minus infinity
    wlp = np.where(wlp < float(low), -np.inf, wlp)
    assert np.array_equal(ids, wids) and np.allclose(lp, wlp, rtol=4 * U, atol=(V / 256 + 70) * U) and np.allclose(ent, went, atol=1e-4)
    assert np.allclose(top, wtop, rtol=4 * U, atol=(V / 256 + 70) * U)


def test_logprobs_without_entropy_and_unaligned(gpu):
    rng = np.random.default_rng(2)
    x = rng.standard_normal((3, 999)).astype(np.float32)
    tok = rng.integers(0, 999, (3, 1))
    got = run_logprobs(gpu, x, tok, 4, entropy=False)
    assert np.all(got[1] == 5)
    want = logprobs64(x, tok, 4)
    assert np.array_equal(got[3], want[3])


def test_logprobs_streams_and_recorded(gpu):
    """Two streams at once with a workspace each, then a recorded call replayed over new logits."""
    rng = np.random.default_rng(8)
    s1, s2 = gpu.Stream(), gpu.Stream()
    jobs = []
    for s in (s1, s2):
        x = (rng.standard_normal((40, 30011)) * 3).astype(np.float32)
        tok = rng.integers(0, 30011, (40, 1))
        keep = {}
        jobs.append((s, x, tok, keep, *run_logprobs(gpu, x, tok, 7, keep=keep)))
    for _ in range(4):
        for s, _, _, _, call, _ in jobs:
            call(s.h)
    for s, x, tok, _, _, results in jobs:
        s.synchronize()
        check_logprobs(x, tok, 7, results())
    s, x, tok, keep, call, results = jobs[0]
    with gpu.Graph(s) as g:
        call(s.h)
    for i in range(3):
        x = (rng.standard_normal(x.shape) * 3).astype(np.float32)
        gpu.call("sgpu_memcpy_htod", keep["x"].ptr, x.ctypes.data, x.nbytes)
        g.launch()
        s.synchronize()
        check_logprobs(x, tok, 7, results())


# ---- attention over a shared prefix ----
class Attn:
    """One call: seqs = [(query rows, earlier own rows), ...]; values no row may see are NaN."""

    def __init__(self, gpu, seqs, P, NH, NKV, HD, half=False, layout="rows", before=0, behind=0, seed=0, hints=None, scale=None):
        rng = np.random.default_rng(seed)
        self.gpu, self.half, self.P, self.NH, self.NKV, self.HD = gpu, half, P, NH, NKV, HD
        kt = np.float16 if half else np.float32
        nq = [a for a, _ in seqs]
        self.q_start = (before + np.concatenate([[0], np.cumsum(nq)])).astype(np.int32)
        self.R = int(self.q_start[-1]) + behind
        self.kv_len = np.array([a + b for a, b in seqs], np.int32)
        gap = 3
        self.kv_start = np.concatenate([[0], np.cumsum(self.kv_len + gap)[:-1]]).astype(np.int32) if seqs else np.zeros(0, np.int32)
        self.SR = int((self.kv_len + gap).sum()) if seqs else 0
        self.q = rng.standard_normal((self.R, NH, HD)).astype(np.float32) * 1.5
        self.kp, self.vp = (rng.standard_normal((P, NKV, HD)).astype(kt) for _ in range(2))
        own = np.full((2, self.SR, NKV, HD), np.nan, kt)
        for s, n in zip(self.kv_start, self.kv_len):
            own[:, s:s + n] = rng.standard_normal((2, n, NKV, HD))
        self.ks, self.vs = own
        self.scale = scale if scale is not None else HD**-0.5
        a = self.a = gpu.AttnPrefixArgs()
        self.keep = {}

        def put(name, t, stride_of):
            n, h, d = t.shape
            if layout == "heads":                              # head-major, as some caches are
                buf = np.full((h, n + 1, d), np.nan, t.dtype)
                buf[:, :n] = t.transpose(1, 0, 2)
                row, head = d, (n + 1) * d
            else:
                pad = 16 if layout == "padded" else 0
                buf = np.full((n, h * d + pad), np.nan, t.dtype)
                buf[:, :h * d] = t.reshape(n, h * d)
                row, head = h * d + pad, d
            self.keep[name] = dev(gpu, buf)
            setattr(a, name, self.keep[name].ptr if buf.size else None)
            if stride_of:
                setattr(a, stride_of + "_row", row)
                setattr(a, stride_of + "_head", head)

        put("q", self.q, "q")
        put("kp", self.kp, "kp")
        put("vp", self.vp, None)
        put("ks", self.ks, "ks")
        put("vs", self.vs, None)
        self.mark = np.full((self.R, NH, HD), -77.0, np.float32)
        put("out", self.mark, "out")
        for n in ("q_start", "kv_start", "kv_len"):
            self.keep[n] = dev(gpu, getattr(self, n) if len(getattr(self, n)) else np.zeros(1, np.int32))
            setattr(a, n, self.keep[n].ptr)
        a.R, a.B, a.P, a.SR, a.NH, a.NKV, a.HD, a.scale = self.R, len(seqs), P, self.SR, NH, NKV, HD, self.scale
        a.max_q, a.max_kv = hints if hints else (max(nq, default=0), int(self.kv_len.max(initial=0)))
        self.layout = layout
        self.need = gpu.lib().sgpu_attn_prefix_workspace(gpu.byref(a))
        assert self.need > 0
        self.ws = dev(gpu, np.full(self.need + 64, 0xFF, np.uint8))           # NaN everywhere

    def call(self, stream=None):
        self.gpu.call("sgpu_attn_prefix_h" if self.half else "sgpu_attn_prefix", self.gpu.byref(self.a), self.ws.ptr, self.need, stream)

    def out(self):
        assert np.all(self.ws.to_host()[self.need:] == 0xFF)
        o = self.keep["out"].to_host()
        if self.layout == "heads":
            return o[:, :self.R].transpose(1, 0, 2)
        return o[:, :self.NH * self.HD].reshape(self.R, self.NH, self.HD)

    def want(self):
        """(out, bar) in 64 bits, from the ints as the call reads them."""
        R, G = self.R, self.NH // self.NKV
        w, bar = self.mark.astype(np.float64), np.zeros(self.mark.shape)
        for b in range(self.a.B):
            q0, q1 = int(self.q_start[b]), int(self.q_start[b + 1])
            first = min(max(int(self.kv_start[b]), 0), self.SR)
            n = min(max(int(self.kv_len[b]), 0), self.SR - first)
            for r in range(q0, min(q1, R)):
                seen = min(max(n - (q1 - q0) + (r - q0) + 1, 0), n)
                K = np.concatenate([self.kp, self.ks[first:first + seen]]).astype(np.float64)
                W = np.concatenate([self.vp, self.vs[first:first + seen]]).astype(np.float64)
                if len(K) == 0:
                    w[r] = 0.0
                    continue
                Kh, Wh = np.repeat(K, G, 1), np.repeat(W, G, 1)
                q = self.q[r].astype(np.float64)
                s = np.einsum("hd,khd->hk", q, Kh) * self.scale
                ds = self.HD * U * np.einsum("hd,khd->hk", abs(q), abs(Kh)) * abs(self.scale)
                p = np.exp(s - s.max(1, keepdims=True))
                p /= p.sum(1, keepdims=True)
                w[r] = np.einsum("hk,khd->hd", p, Wh)
                mag = np.einsum("hk,khd->hd", p * (2 * ds + 2 * (p * ds).sum(1, keepdims=True) + (2 * len(K) + 16) * U), abs(Wh))
                bar[r] = mag + 1e-30
        return w, bar

    def check(self, stream=None):
        self.call(stream)
        self.gpu.synchronize()
        self.compare()

    def compare(self):
        with np.errstate(invalid="ignore"):
            got, (want, bar) = self.out(), self.want()
            fine = np.isfinite(want)
            assert np.array_equal(np.isfinite(got), fine)
            diff = np.where(fine, np.abs(got - want), 0.0)
            bad = fine & ~(diff <= bar)
        assert not bad.any(), (float(diff.max()), np.argwhere(bad)[:4].tolist())


HEADS = [(14, 2, 64), (12, 12, 64), (8, 2, 128), (6, 2, 32), (1, 1, 64), (40, 1, 128)]
SEQS = {
    "one row": ([(1, 0)], 1),
    "no prefix": ([(5, 0), (1, 7)], 0),
    "decode": ([(1, 3), (1, 0), (1, 40), (1, 129)], 100),
    "no query rows of some": ([(0, 9), (2, 1), (0, 0), (3, 0), (0, 4)], 33),
    "answers": ([(17, 0), (33, 0), (2, 0), (40, 0)], 257),
    "chunk": ([(9, 300), (31, 70)], 64),
    "odd prefix": ([(1, 1)] * 5, 1537),
}


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("heads", HEADS, ids=str)
@pytest.mark.parametrize("name", list(SEQS))
def test_attn_prefix(gpu, name, heads, half):
    seqs, P = SEQS[name]
    Attn(gpu, seqs, P, *heads, half=half, layout=["rows", "padded", "heads"][len(name) % 3], seed=len(name)).check()


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("layout", ["rows", "padded", "heads"])
def test_attn_prefix_layouts_and_rows_of_no_sequence(gpu, layout, half):
    """Rows before the first sequence and behind the last stay as they were."""
    Attn(gpu, [(3, 2), (1, 5)], 70, 14, 2, 64, half=half, layout=layout, before=2, behind=4).check()


def test_attn_prefix_rows_that_see_nothing(gpu):
    """More query rows than keys and no prefix: the first rows are zeros."""
    c = Attn(gpu, [(6, 0), (2, 3)], 0, 6, 2, 32)
    c.kv_len[0] = 4
    c.keep["kv_len"] = dev(gpu, c.kv_len)
    c.a.kv_len = c.keep["kv_len"].ptr
    c.check()
    assert np.all(c.out()[:2] == 0.0) and np.all(np.any(c.out()[2:] != 0, axis=(1, 2)))


def test_attn_prefix_no_own_keys(gpu):
    c = Attn(gpu, [(2, 0), (1, 0)], 333, 14, 2, 64)
    c.kv_len[:] = 0
    c.a.SR, c.SR, c.a.ks, c.a.vs, c.a.kv_start, c.a.kv_len = 0, 0, None, None, None, None
    c.check()


@pytest.mark.parametrize("hints", [(0, 0), (1, 1), (1000, 5000)])
def test_attn_prefix_hints_do_not_matter(gpu, hints):
    Attn(gpu, [(9, 4), (1, 200), (70, 0)], 90, 14, 2, 64, hints=hints).check()


def test_attn_prefix_ints_out_of_range(gpu):
    """Starts and lengths past the buffers are cut to them; nothing outside is read or written."""
    c = Attn(gpu, [(2, 30), (3, 5), (1, 9)], 40, 6, 2, 32)
    c.kv_len[:] = [10**9, -5, 2**31 - 1]
    c.kv_start[:] = [c.SR - 4, 10**9, -3]
    for n in ("ks", "vs"):                                     # what lies between the sequences is seen here
        t = np.nan_to_num(getattr(c, n), nan=0.25)
        setattr(c, n, t)
        c.keep[n] = dev(gpu, t.reshape(c.SR, -1))
        setattr(c.a, n, c.keep[n].ptr)
    for n in ("kv_len", "kv_start"):
        c.keep[n] = dev(gpu, getattr(c, n))
        setattr(c.a, n, c.keep[n].ptr)
    c.check()


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("big", [1e3, 6e4])
def test_attn_prefix_keys_of_very_different_size(gpu, big, half):
    """A key and a value row far larger than the rest, with little weight: the rest keeps its digits."""
    c = Attn(gpu, [(2, 3), (1, 1)], 200, 6, 2, 64, half=half)
    sign = -np.sign(c.q[0].reshape(2, 3, 64).sum(1))
    c.kp[7] = (sign * big / 64).astype(c.kp.dtype)             # scores of the first row far below the others
    c.vp[9] = c.vp[9] * np.asarray(big, c.vp.dtype) / 4
    c.kp[9] = c.kp[7]
    c.vp[20] = 0
    c.kp[21] = 0
    for n in ("kp", "vp"):
        c.keep[n] = dev(gpu, getattr(c, n).reshape(200, -1))
        setattr(c.a, n, c.keep[n].ptr)
    c.check()


@pytest.mark.parametrize("where", ["k", "v"])
def test_attn_prefix_fp32_range(gpu, where):
    """fp32 keys and values keep their exponents: 1e30 beside 1e-30 in different rows and heads."""
    c = Attn(gpu, [(2, 3), (1, 1)], 150, 6, 2, 64, scale=1e-30 if where == "k" else None)
    if where == "k":
        c.kp *= np.float32(1e30)
        c.ks *= np.float32(1e30)
        c.kp[3] *= np.float32(1e-36)
    else:
        c.vp *= (10.0 ** np.linspace(-30, 8, 150)).astype(np.float32)[:, None, None]
        c.vs *= np.float32(1e-10)
    for n in ("kp", "vp", "ks", "vs"):
        c.keep[n] = dev(gpu, getattr(c, n).reshape(len(getattr(c, n)), -1))
        setattr(c.a, n, c.keep[n].ptr)
    c.check()


def test_attn_prefix_large_scores(gpu):
    """Scores in the hundreds: all weight on few keys."""
    Attn(gpu, [(3, 2), (4, 60)], 500, 8, 2, 128, scale=8.0).check()
    Attn(gpu, [(3, 2), (4, 60)], 500, 8, 2, 128, scale=0.0).check()


def test_attn_prefix_non_finite_values(gpu):
    """A NaN that a row sees shows in its heads and dims only; rows and heads that do not see it are untouched."""
    c = Attn(gpu, [(4, 0), (3, 0)], 20, 6, 2, 32)
    first = int(c.kv_start[0])
    c.vs[first + 2, 1, 5] = np.nan                             # rows 2 and 3 of the first sequence, KV head 1
    c.keep["vs"] = dev(gpu, c.vs.reshape(c.SR, -1))
    c.a.vs = c.keep["vs"].ptr
    c.call()
    gpu.synchronize()
    got, bad = c.out(), np.zeros((c.R, 6, 32), bool)
    bad[2:4, 3:, 5] = True
    c.vs[first + 2, 1, 5] = 0.0
    want, bar = c.want()
    assert np.all(np.isnan(got[bad])) and np.all(np.abs(got - want)[~bad & ~_sees(c, first)] <= bar[~bad & ~_sees(c, first)])


def _sees(c, first):
    """Rows and heads whose keys include the poisoned row: their other dims are compared elsewhere."""
    m = np.zeros((c.R, 6, 32), bool)
    m[2:4, 3:] = True
    return m


@pytest.mark.parametrize("half", [False, True])
def test_attn_prefix_long_prefix_far_rows(gpu, half):
    """A prefix cache whose rows lie past 2^32 bytes (wide rows, few of their columns used)."""
    import ctypes as ct

    P, NH, NKV, HD = 2200, 6, 2, 64
    row = 1 << (21 if half else 20)                            # 4 MiB a row, 9.2 GB a tensor
    c = Attn(gpu, [(1, 0), (2, 3)], P, NH, NKV, HD, half=half, seed=4)
    big = [gpu.DeviceArray((P - 1) * row + NKV * HD, np.uint16 if half else np.float32) for _ in range(2)]
    size = 2 if half else 4
    L = gpu.lib()
    for d, src in zip(big, ("kp", "vp")):
        for p in range(P):
            gpu.call("sgpu_memcpy_dtod_async", d.ptr + p * row * size, c.keep[src].ptr + p * NKV * HD * size, NKV * HD * size, None)
    gpu.synchronize()
    assert isinstance(L, ct.CDLL)
    c.a.kp, c.a.vp, c.a.kp_row = big[0].ptr, big[1].ptr, row
    c.check()
    for d in big:
        d.close()


def test_attn_prefix_streams_and_recorded(gpu):
    """Two streams at once; a recorded call replayed while its sequences grow; results equal bit for bit
    those of a call by itself."""
    s1, s2 = gpu.Stream(), gpu.Stream()
    a = Attn(gpu, [(1, 20), (1, 3), (1, 33)], 700, 14, 2, 64, seed=1)
    b = Attn(gpu, [(7, 0), (30, 0)], 333, 8, 2, 128, half=True, seed=2)
    for _ in range(5):
        a.call(s1.h)
        b.call(s2.h)
    s1.synchronize()
    s2.synchronize()
    a.compare()
    b.compare()
    first = a.out().copy()
    a.check()
    assert np.array_equal(first.view(np.uint32), a.out().view(np.uint32))
    with gpu.Graph(s1) as g:
        a.call(s1.h)
    full = a.kv_len.copy()
    for back in (12, 5, 3, 0):
        a.kv_len = np.maximum(full - back, 1).astype(np.int32)
        gpu.call("sgpu_memcpy_htod", a.keep["kv_len"].ptr, a.kv_len.ctypes.data, a.kv_len.nbytes)
        g.launch()
        s1.synchronize()
        a.compare()
        got = a.out().copy()
        a.check()
        assert np.array_equal(got.view(np.uint32), a.out().view(np.uint32))


# Enough row tiles (128 rows and heads of a group) over enough keys that fp32 prefixes are cut to fp16 pieces by a
# kernel of their own first.  Most of the rows belong to no sequence: they count, and stay as they were.
CUT_STEPS = {32: 8192, 64: 8192, 128: 2560}


def cut_case(gpu, seqs, P, NH, NKV, HD, **kw):
    tiles = -(-CUT_STEPS[HD] // (-(-P // 64) * NKV))
    rows = tiles * 128 * NKV // NH + 1
    return Attn(gpu, seqs, P, NH, NKV, HD, before=rows // 3, behind=rows - rows // 3, **kw)


@pytest.mark.parametrize("P", [1037, 2048, 1601])
@pytest.mark.parametrize("seqs", [[(1, 3), (1, 0), (1, 40)], [(17, 0), (0, 5), (33, 0), (2, 30)]], ids=["decode", "answers"])
@pytest.mark.parametrize("heads", [(14, 2, 64), (8, 1, 128), (6, 2, 32), (12, 12, 64), (4, 2, 128)], ids=str)
def test_attn_prefix_cut(gpu, heads, seqs, P):
    cut_case(gpu, seqs, P, *heads, layout=["rows", "padded", "heads"][P % 3], seed=P).check()


def renew(gpu, c, *names):
    for n in names:
        t = getattr(c, n)
        c.keep[n] = dev(gpu, t.reshape(len(t), -1))
        setattr(c.a, n, c.keep[n].ptr)


@pytest.mark.parametrize("heads", [(14, 2, 64), (8, 1, 128), (6, 2, 32)], ids=str)
def test_attn_prefix_cut_odd_keys(gpu, heads):
    """Groups of keys that share no scale, zero values, and values of 1e30 and 1e-30 in different rows."""
    c = cut_case(gpu, [(3, 2), (1, 9)], 1111, *heads, seed=7)
    c.kp[7] *= np.float32(3e-6)
    c.kp[40:72] = 0
    c.vp[100:140] = 0
    c.vp[300] *= np.float32(1e6)
    c.vp[1000:] *= (10.0 ** np.linspace(-30, 8, 111)).astype(np.float32)[:, None, None]
    c.kp[1110] = 0
    renew(gpu, c, "kp", "vp")
    c.check()


@pytest.mark.parametrize("where,value", [("kp", np.nan), ("kp", np.inf), ("vp", np.nan), ("vp", -np.inf)])
def test_attn_prefix_cut_non_finite(gpu, where, value):
    """Every row sees the prefix: the heads (a key) or their dims (a value) are not finite, the others as ever."""
    c = cut_case(gpu, [(2, 2), (1, 0)], 1037, 8, 2, 128, seed=8)
    clean, bar = c.want()
    getattr(c, where)[1036, 1, 5] = value
    renew(gpu, c, where)
    c.call()
    gpu.synchronize()
    got = c.out()
    live = np.zeros(got.shape, bool)
    live[c.q_start[0]:c.q_start[-1], 4:, 5 if where == "vp" else slice(None)] = True
    fine = np.isfinite(got)
    if where == "vp" or np.isnan(value):
        assert not fine[live].any()
    others = ~live if where == "vp" else np.broadcast_to((np.arange(8) < 4)[None, :, None], got.shape)
    assert fine[others].all() and np.all(np.abs(got - clean)[others] <= bar[others])


def test_attn_prefix_cut_streams_and_recorded(gpu):
    s1, s2 = gpu.Stream(), gpu.Stream()
    a = cut_case(gpu, [(1, 20), (1, 3), (1, 33)], 1100, 14, 2, 64, seed=1)
    b = cut_case(gpu, [(7, 0), (30, 0)], 1333, 8, 1, 128, seed=2)
    for _ in range(3):
        a.call(s1.h)
        b.call(s2.h)
    s1.synchronize()
    s2.synchronize()
    a.compare()
    b.compare()
    with gpu.Graph(s1) as g:
        a.call(s1.h)
    full = a.kv_len.copy()
    for back in (12, 5, 0):
        a.kv_len = np.maximum(full - back, 1).astype(np.int32)
        gpu.call("sgpu_memcpy_htod", a.keep["kv_len"].ptr, a.kv_len.ctypes.data, a.kv_len.nbytes)
        g.launch()
        s1.synchronize()
        a.compare()
        got = a.out().copy()
        a.check()
        assert np.array_equal(got.view(np.uint32), a.out().view(np.uint32))


@pytest.mark.parametrize("hints", [(1, 4), (20000, 4)])
def test_attn_prefix_many_sequences(gpu, hints):
    """Also where the hint of a sequence's rows would ask for more blocks than a launch takes: they take turns."""
    Attn(gpu, [(1, i % 4) for i in range(20000)], 9, 2, 1, 32, hints=hints, seed=3).check()


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("V,k", [(24581, 64), (151936, 33), (151936, 64), (50257, 9)])
def test_logprobs_order_of_many_alternatives(gpu, V, k, half):
    """Rows that keep the lists of alternatives busy: values that repeat, rise, fall, or are all the same."""
    rng = np.random.default_rng(V + k)
    i = np.arange(V)
    x = np.stack([np.round(rng.standard_normal(V) * 2) / 2, np.full(V, 1.25), i / V * 8, -i / V * 8, np.where(i >= V - k, 3.0, 0.0),
                  np.where(i % 997 == 5, 2.0 + i / V, rng.standard_normal(V) * 0.1)]).astype(np.float16 if half else np.float32)
    tok = rng.integers(0, V, (len(x), 1))
    check_logprobs(x, tok, k, run_logprobs(gpu, x, tok, k))

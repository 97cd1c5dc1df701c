"""The operators over a paged cache and the adjusted logits against plain implementations in 64 bits.

Bars, from the arithmetic (u = 2^-24, half an fp32 step):
  heads      a normed value rounds three times (1/sqrt, the product with it, the weight's): 3 u; cos and sin are off by at
             most 3.6 u, each product and the sum round once more: 9 u (|a| + |b|) of a rotated pair, 4 u of what passes
             through; an fp16 result rounds once, 2^-11 |y| (2^-25 below its normal range)
  attention  a score is a sum of HD products: HD u sum |q k| scale; a weight is off by twice that and 4 u, a sum over n keys
             adds n u, in the output each relative to sum p |v|
  logits     64 bits, rounded once: half a step of the result's type, and 2^-50 of what was summed
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0**-24


def dev(gpu, a):
    return gpu.DeviceArray.from_host(np.ascontiguousarray(a))


def rounded(want, bar, half):
    return bar + np.maximum(np.abs(want) * 2.0**-11, 2.0**-25) * 1.001 if half else bar


# ---- norms and rotations ----
def heads64(x, w, eps, pos, turns, rot, nb, mscale):
    """(result, bar) of x [T][H][HD]; w [HD] or None."""
    x = x.astype(np.float64)
    if w is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w.astype(np.float64)
    y, bar = x.copy(), 4 * U * abs(x)
    ang = 2 * np.pi * np.mod(np.asarray(pos, np.float64)[:, None] * turns[:rot // 2], 1.0)
    c, s = np.cos(ang)[:, None] * mscale, np.sin(ang)[:, None] * mscale
    h = rot // 2
    i0, i1 = (np.arange(0, rot, 2), np.arange(1, rot, 2)) if nb else (np.arange(h), np.arange(h, rot))
    a, b = x[..., i0], x[..., i1]
    y[..., i0], y[..., i1] = a * c - b * s, a * s + b * c
    bar[..., i0] = bar[..., i1] = 9 * U * (abs(a) + abs(b)) * mscale
    return y, bar


def turns_of(rot, theta=1e4):
    return theta ** (-2.0 * np.arange(max(rot // 2, 1)) / max(rot, 1)) / (2 * np.pi)


QKN = [
    # T, NH, NKV, HD, rot, neighbours, fp16, offset of x in floats, offset of y in values
    (1, 14, 2, 64, 64, 0, False, 0, 0), (1, 1, 0, 2, 2, 1, False, 0, 0), (3, 0, 3, 64, 64, 0, True, 0, 0), (5, 2, 1, 80, 40, 0, False, 0, 0),
    (5, 2, 1, 80, 40, 1, True, 0, 0), (7, 2, 1, 128, 64, 1, True, 0, 0), (7, 2, 1, 128, 64, 1, False, 1, 0), (7, 2, 1, 128, 64, 0, True, 0, 1),
    (4, 3, 2, 33, 6, 0, False, 0, 0), (4, 3, 2, 33, 6, 1, True, 3, 5), (2, 3, 1, 256, 256, 0, False, 0, 0), (2, 3, 1, 512, 256, 1, True, 0, 0),
    (9, 4, 2, 64, 0, 0, True, 0, 0), (3001, 2, 1, 32, 32, 0, False, 0, 0), (4100, 1, 1, 16, 8, 1, False, 0, 0), (6, 2, 1, 64, 12, 0, False, 0, 0),
    (2, 32, 8, 128, 128, 0, True, 0, 0), (3, 2, 1, 520, 64, 0, False, 0, 0), (130, 1, 1, 1, 0, 0, False, 0, 0), (2, 5, 5, 96, 96, 0, False, 0, 0)]


@pytest.mark.parametrize("case", QKN, ids=str)
@pytest.mark.parametrize("where", ["none", "far", "back"])
def test_qk_norm_rope(gpu, case, where):
    T, NH, NKV, HD, rot, nb, half, xo, yo = case
    rng = np.random.default_rng(T * 7 + HD)
    n = (NH + NKV) * HD
    xs, ys = n + (5 if xo else 8), n + (3 if yo else 16)
    x = rng.standard_normal(xo + T * xs).astype(np.float32) * 3
    w = [(1 + 0.3 * rng.standard_normal(HD)).astype(np.float32) for _ in range(2)]
    use = {"none": (0, 1), "far": (0,), "back": (1,)}[where]         # the norm of both, of one
    turns = turns_of(rot)
    pos0 = {"none": 11, "far": 2000000000, "back": 0}[where]
    pos = {"none": None, "far": rng.integers(0, 100000000, T), "back": -rng.integers(0, 1000000, T)}[where]
    d = dev(gpu, x), dev(gpu, turns), [dev(gpu, v) for v in w], dev(gpu, pos.astype(np.int32)) if pos is not None else None
    y = dev(gpu, np.full(yo + T * ys, 777, np.float16 if half else np.float32))
    gpu.call("sgpu_qk_norm_rope_h" if half else "sgpu_qk_norm_rope", d[0].offset(xo), xs, y.offset(yo), ys, d[2][0].ptr if 0 in use else None,
             d[2][1].ptr if 1 in use else None, 1e-6, d[3].ptr if d[3] else None, pos0, d[1].ptr, rot, nb, 1.25, T, NH, NKV, HD, None)
    gpu.synchronize()
    g = y.to_host()
    assert np.all(g[:yo] == 777)
    g = g[yo:].reshape(T, ys)
    assert np.all(g[:, n:] == 777)
    rows = x[xo:].reshape(T, xs)[:, :n].reshape(T, NH + NKV, HD)
    at = pos0 + (pos if pos is not None else np.arange(T))
    for s, k in ((slice(0, NH), 0), (slice(NH, None), 1)):
        want, bar = heads64(rows[:, s], w[k] if k in use else None, 1e-6, at, turns, rot, nb, 1.25)
        got = g[:, :n].reshape(T, NH + NKV, HD)[:, s].astype(np.float64)
        assert np.all(np.abs(got - want) <= rounded(want, bar, half) + 1e-300)


@pytest.mark.parametrize("HD,rot", [(64, 64), (40, 6)])
def test_qk_norm_rope_in_place(gpu, HD, rot):
    rng = np.random.default_rng(3)
    T, NH, NKV = 70, 3, 2
    x = rng.standard_normal((T, (NH + NKV) * HD + 4)).astype(np.float32)
    w = (1 + 0.3 * rng.standard_normal(HD)).astype(np.float32)
    turns, d, dw = turns_of(rot), dev(gpu, x), dev(gpu, w)
    dt = dev(gpu, turns)
    gpu.call("sgpu_qk_norm_rope", d.ptr, x.shape[1], d.ptr, x.shape[1], dw.ptr, dw.ptr, 1e-5, None, 5, dt.ptr, rot, 0, 1.0, T, NH, NKV, HD, None)
    gpu.synchronize()
    got = d.to_host()
    assert np.array_equal(got[:, -4:], x[:, -4:])
    want, bar = heads64(x[:, :-4].reshape(T, -1, HD), w, 1e-5, 5 + np.arange(T), turns, rot, 0, 1.0)
    assert np.all(np.abs(got[:, :-4].reshape(T, -1, HD) - want) <= bar)


@pytest.mark.parametrize("HD", [64, 33])
def test_qk_norm_rope_sizes_of_values(gpu, HD):
    """Heads whose squares leave fp32, heads of zeros and of the smallest values, a NaN that stays in its head."""
    rng = np.random.default_rng(5)
    x = rng.standard_normal((6, 1, HD)).astype(np.float32)
    x[0] *= 1e30
    x[1] *= np.float32(1e-30)
    x[2] = 0
    x[3] = np.float32(1e-42)
    x[5, 0, 7] = np.nan
    w, turns = np.ones(HD, np.float32), turns_of(2)
    d, dw, dt, y = dev(gpu, x), dev(gpu, w), dev(gpu, turns), gpu.DeviceArray(x.shape)
    for eps in (0.0, 1e-6):
        gpu.call("sgpu_qk_norm_rope", d.ptr, HD, y.ptr, HD, dw.ptr, None, eps, None, 0, dt.ptr, 2, 0, 1.0, 6, 1, 0, HD, None)
        gpu.synchronize()
        got = y.to_host()
        with np.errstate(invalid="ignore"):
            want, bar = heads64(x, w, eps, np.arange(6), turns, 2, 0, 1.0)
        ok = [0, 1, 4] if eps == 0 else [0, 1, 2, 3, 4]               # 0 / 0 is not a number
        assert np.all(np.abs(got[ok] - want[ok]) <= bar[ok] + 2.0**-149)
        assert np.isnan(got[5]).all()
        if eps == 0:
            assert np.isnan(got[2]).all()


# ---- the paged cache ----
class Cache:
    """seqs = [(tokens in the cache, new rows), ...]; pages in any order, what no token holds is NaN."""

    def __init__(self, gpu, seqs, NKV, HD, page, half, layout="tokens", before=0, behind=0, seed=0, spare=2):
        rng = self.rng = np.random.default_rng(seed)
        self.gpu, self.seqs, self.NKV, self.HD, self.page, self.half = gpu, seqs, NKV, HD, page, half
        self.len = np.array([a for a, _ in seqs], np.int32)
        nq = [b for _, b in seqs]
        self.q_start = (before + np.concatenate([[0], np.cumsum(nq)])).astype(np.int32)
        self.R = int(self.q_start[-1]) + behind
        need = [-(-(a + b) // page) for a, b in seqs]
        self.pages = sum(need) + spare
        order = rng.permutation(self.pages)
        self.table_pages = max(need + [1]) + 1
        self.table = np.full((len(seqs), self.table_pages), -1, np.int32)
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = order[at:at + n]
            at += n
        kt = np.float16 if half else np.float32
        shape = (self.pages, page, NKV, HD) if layout == "tokens" else (self.pages, NKV, page, HD)
        self.layout = layout
        self.pad = 0 if layout == "tokens" else 16                    # and room behind each page
        self.buf = [np.full((self.pages, page * NKV * HD + self.pad), np.nan, kt) for _ in range(2)]
        self.shape = shape
        for b, (have, n) in enumerate(seqs):
            for t in range(have + n):
                for c in range(2):
                    self.at(c, b, t)[...] = rng.standard_normal((NKV, HD))
        self.keep = {}

    def view(self, c):
        v = self.buf[c][:, :self.page * self.NKV * self.HD].reshape(self.shape)
        return v if self.layout == "tokens" else v.transpose(0, 2, 1, 3)

    def at(self, c, b, t):
        return self.view(c)[self.table[b, t // self.page], t % self.page]

    def fill(self, c):
        """The description's fields, everything on the device."""
        for n, v in (("k", self.buf[0]), ("v", self.buf[1]), ("table", self.table), ("len", self.len), ("q_start", self.q_start)):
            self.keep[n] = dev(self.gpu, v if v.size else np.zeros(1, v.dtype))
            setattr(c, n, self.keep[n].ptr)
        c.page_stride = self.buf[0].shape[1]
        c.kv_row, c.kv_head = (self.NKV * self.HD, self.HD) if self.layout == "tokens" else (self.HD, self.page * self.HD)
        c.pages, c.page, c.table_row, c.table_pages, c.R, c.B = self.pages, self.page, self.table_pages, self.table_pages, self.R, len(self.seqs)

    def put(self, name, value):
        """A changed host array back to its place on the device."""
        self.gpu.call("sgpu_memcpy_htod", self.keep[name].ptr, np.ascontiguousarray(value).ctypes.data, value.nbytes)

    def place(self, b, t):
        """(page, token of it) where a row is written or read; None where there is none."""
        if not 0 <= t < self.table_pages * self.page:
            return None
        p = int(self.table[b, t // self.page])
        return (p, t % self.page) if 0 <= p < self.pages else None


class Append:
    def __init__(self, gpu, seqs, NH, NKV, HD, page, half, rot=None, nb=0, norm=True, depth=None, offset=0, q=True, **kw):
        self.c = c = Cache(gpu, seqs, NKV, HD, page, half, **kw)
        self.gpu, self.half, self.NH, self.nb, self.q = gpu, half, NH, nb, q
        self.rot = HD if rot is None else rot
        rng = np.random.default_rng(c.R + HD)
        n = (NH + 2 * NKV) * HD
        self.row = n + offset
        self.x = rng.standard_normal((c.R, self.row)).astype(np.float32) * 2
        self.w = [(1 + 0.3 * rng.standard_normal(HD)).astype(np.float32) for _ in range(2)] if norm else None
        self.turns = turns_of(self.rot)
        self.pos = depth
        a = self.a = gpu.KvAppendArgs()
        self.keep = dict(x=dev(gpu, self.x), turns=dev(gpu, self.turns), out=dev(gpu, np.full((c.R, NH * HD + 4), -77, np.float32)))
        c.fill(a.c)
        x = self.keep["x"]
        a.q, a.k, a.v = x.offset(0) if q else None, x.offset(NH * HD), x.offset((NH + NKV) * HD)
        a.q_out, a.out_row = self.keep["out"].ptr, NH * HD + 4
        a.q_row = a.k_row = a.v_row = self.row
        a.turns, a.eps, a.mscale, a.rot, a.neighbours, a.NH, a.NKV, a.HD = self.keep["turns"].ptr, 1e-6, 1.0, self.rot, nb, NH, NKV, HD
        if norm:
            self.keep["wq"], self.keep["wk"] = dev(gpu, self.w[0]), dev(gpu, self.w[1])
            a.wq, a.wk = self.keep["wq"].ptr, self.keep["wk"].ptr
        if depth is not None:
            self.keep["pos"] = dev(gpu, np.asarray(depth, np.int32))
            a.pos = self.keep["pos"].ptr

    def call(self, stream=None):
        self.gpu.call("sgpu_kv_append_h" if self.half else "sgpu_kv_append", self.gpu.byref(self.a), stream)

    def want(self):
        """(q, k pages, v pages), each (values, bars), from the ints as the call reads them."""
        c, NH, NKV, HD = self.c, self.NH, self.c.NKV, self.c.HD
        q = np.full((c.R, NH, HD), -77.0), np.zeros((c.R, NH, HD))
        pages = [(c.view(i).astype(np.float64), np.zeros(c.view(i).shape)) for i in range(2)]
        x = self.x[:, :(NH + 2 * NKV) * HD].reshape(c.R, NH + 2 * NKV, HD)
        for b in range(len(c.seqs)):
            for r in range(int(c.q_start[b]), int(c.q_start[b + 1])):
                t = int(c.len[b]) + r - int(c.q_start[b])
                p = [t if self.pos is None else self.pos[r]]
                wq, wk = self.w if self.w else (None, None)
                if self.q:
                    q[0][r], q[1][r] = (v[0] for v in heads64(x[r:r + 1, :NH], wq, 1e-6, p, self.turns, self.rot, self.nb, 1.0))
                to = c.place(b, t)
                if to is None:
                    continue
                k, bar = heads64(x[r:r + 1, NH:NH + NKV], wk, 1e-6, p, self.turns, self.rot, self.nb, 1.0)
                pages[0][0][to], pages[0][1][to] = k[0], rounded(k, bar, self.half)[0]
                v = x[r, NH + NKV:].astype(np.float64)
                pages[1][0][to], pages[1][1][to] = v, rounded(v, np.zeros(v.shape), self.half)
        return q, pages

    def compare(self):
        c = self.c
        (q, qbar), pages = self.want()
        out = self.keep["out"].to_host()
        assert np.all(out[:, -4:] == -77)
        assert np.all(np.abs(out[:, :-4].reshape(q.shape) - q) <= qbar)
        for i, n in enumerate(("k", "v")):
            host = c.keep[n].to_host()
            want, bar = pages[i]
            old = c.buf[i]
            c.buf[i] = host
            got = c.view(i).astype(np.float64)
            c.buf[i] = old
            assert np.array_equal(np.isnan(got), np.isnan(want)) and np.isnan(host[:, c.page * c.NKV * c.HD:]).all()
            assert np.all(np.abs(got - want)[~np.isnan(want)] <= bar[~np.isnan(want)])

    def check(self, stream=None):
        self.call(stream)
        self.gpu.synchronize()
        self.compare()


BATCHES = {
    "one token": [(700, 1)], "first token": [(0, 1)], "decode": [(3, 1), (0, 1), (40, 1), (129, 1)],
    "drafts": [(17, 5), (0, 3), (63, 0), (64, 8), (31, 1)], "prompts": [(0, 70), (100, 33)], "none": [(5, 0), (9, 0)]}


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("heads", [(14, 2, 64), (4, 4, 32), (8, 2, 128), (3, 1, 40), (2, 1, 33), (4, 2, 256)], ids=str)
@pytest.mark.parametrize("name", BATCHES)
def test_kv_append(gpu, name, heads, half):
    for page, layout, norm in ((16, "tokens", True), (1, "heads", False), (100, "heads", True)):
        rot = heads[2] // 4 * 2 if page == 100 else heads[2] // 2 * 2
        Append(gpu, BATCHES[name], *heads, page, half, rot=rot, nb=page == 1, norm=norm, layout=layout, before=2, behind=3).check()


def test_kv_append_positions_offsets_and_no_queries(gpu):
    seqs = [(17, 5), (0, 3), (64, 8)]
    depth = [17, 18, 18, 19, 19, 0, 1, 1, 64, 65, 65, 65, 66, 66, 67, 2000000]
    for offset, q in ((0, True), (1, True), (3, False), (4, False)):
        Append(gpu, seqs, 6, 2, 64, 16, True, depth=depth, offset=offset, q=q).check()
    Append(gpu, seqs, 6, 2, 64, 16, False, rot=0).check()


def test_kv_append_queries_in_place(gpu):
    a = Append(gpu, [(3, 4), (9, 2)], 6, 2, 64, 16, False)
    a.a.q_out, a.a.out_row = a.a.q, a.a.q_row
    a.call()
    gpu.synchronize()
    got = a.keep["x"].to_host()
    (q, bar), _ = a.want()
    assert np.all(np.abs(got[:, :6 * 64].reshape(q.shape) - q) <= bar) and np.array_equal(got[:, 6 * 64:], a.x[:, 6 * 64:])


def test_kv_append_pages_that_are_none(gpu):
    """Page numbers outside the cache, tokens past the table, lengths that make no sense: nothing is written there."""
    for half in (False, True):
        a = Append(gpu, [(17, 5), (0, 30), (64, 8), (5, 1)], 4, 2, 64, 8, half, before=1, behind=1)
        c = a.c
        c.table[1, 1], c.table[1, 3], c.table[2, 8] = c.pages, -5, 2**31 - 1
        c.len[3] = -3
        c.len[0] = c.table_pages * c.page - 2
        c.put("table", c.table)
        c.put("len", c.len)
        before = [x.copy() for x in c.buf]
        # places of the unknown pages are found by place(); the oracle's view starts from the same pages
        a.check()
        assert all(np.array_equal(x, y, equal_nan=True) for x, y in zip(before, c.buf))


def test_kv_append_many_sequences(gpu):
    """More sequences than a wave has lanes, most without rows."""
    seqs = [(b % 7, 1 if b % 5 == 0 else 0) for b in range(700)] + [(3, 2)]
    Append(gpu, seqs, 2, 1, 32, 4, False, before=3, behind=70, norm=False).check()


def test_kv_append_streams_and_recorded(gpu):
    """Two streams at once; a recorded call follows the lengths on the device."""
    s1, s2 = gpu.Stream(), gpu.Stream()
    a = Append(gpu, [(3, 4), (20, 2), (0, 1)], 14, 2, 64, 16, False, seed=1)
    b = Append(gpu, [(7, 30), (0, 9)], 8, 2, 128, 32, True, seed=2)
    for _ in range(4):
        a.call(s1.h)
        b.call(s2.h)
    s1.synchronize()
    s2.synchronize()
    a.compare()
    b.compare()
    a = Append(gpu, [(3, 4), (20, 2), (0, 1)], 14, 2, 64, 16, False, seed=1, spare=5)
    full = a.c.len.copy()
    with gpu.Graph(s1) as g:
        a.call(s1.h)
    for back in (3, 1, 0):
        fresh = Append(gpu, [(3, 4), (20, 2), (0, 1)], 14, 2, 64, 16, False, seed=1, spare=5)
        for n, v in (("k", fresh.c.buf[0]), ("v", fresh.c.buf[1])):
            a.c.put(n, v)
        a.c.len = np.maximum(full - back, 0).astype(np.int32)
        a.c.put("len", a.c.len)
        g.launch()
        s1.synchronize()
        a.compare()


# ---- attention ----
def tree_bits(rng, n, words, kind):
    """Mask words of n drafted rows: a tree's, random ones, or nothing at all."""
    m = np.zeros((n, max(words * 32, n)), bool)
    for i in range(n):
        if kind == "tree":
            if i:
                m[i] = m[rng.integers(max(0, i - 6), i)]
            m[i, i] = True
        elif kind == "random":
            m[i] = rng.random(m.shape[1]) < 0.4                       # bits past the rows, and of later rows, among them
    m = m[:, :words * 32]
    packed = np.packbits(m, axis=1, bitorder="little").reshape(n, words * 4).copy().view(np.uint32)
    return packed.reshape(n, words), m


class Tree:
    def __init__(self, gpu, seqs, NH, NKV, HD, page, half, kind=None, hints=None, scale=None, words=None, seed=0, qlayout="rows", **kw):
        self.c = c = Cache(gpu, seqs, NKV, HD, page, half, seed=seed, **kw)
        self.gpu, self.half, self.NH, self.NKV, self.HD = gpu, half, NH, NKV, HD
        rng = np.random.default_rng(seed + 100)
        self.q = rng.standard_normal((c.R, NH, HD)).astype(np.float32) * 1.5
        nq = [b for _, b in seqs]
        self.scale = scale if scale is not None else HD**-0.5
        a = self.a = gpu.AttnTreeArgs()
        c.fill(a.c)
        self.bits = None
        self.keep = {}
        if kind:
            words = -(-max(max(nq), 1) // 32) if words is None else words
            packed, self.bits = np.zeros((c.R, max(words, 1)), np.uint32), np.zeros((c.R, words * 32), bool)
            for b, n in enumerate(nq):
                r = int(c.q_start[b])
                if words:
                    packed[r:r + n], self.bits[r:r + n] = tree_bits(rng, n, words, kind)
            self.keep["mask"] = dev(gpu, packed)
            a.mask, a.mask_row = self.keep["mask"].ptr, words
        pad = 0 if qlayout == "rows" else 8
        qb = np.full((c.R, NH * HD + pad), np.nan, np.float32)
        qb[:, :NH * HD] = self.q.reshape(c.R, -1)
        self.keep["q"], self.keep["out"] = dev(gpu, qb), dev(gpu, np.full((c.R, NH * HD + pad), -77, np.float32))
        a.q, a.out, a.q_row, a.out_row, a.q_head, a.out_head = self.keep["q"].ptr, self.keep["out"].ptr, NH * HD + pad, NH * HD + pad, HD, HD
        a.NH, a.NKV, a.HD, a.scale = NH, NKV, HD, self.scale
        a.max_q, a.max_kv = hints if hints else (max(nq), max(x + y for x, y in seqs))
        self.need = gpu.lib().sgpu_attn_tree_workspace(gpu.byref(a))
        assert self.need > 0
        self.ws = dev(gpu, np.full(self.need + 64, 0xFF, np.uint8))           # NaN everywhere

    def call(self, stream=None):
        self.gpu.call("sgpu_attn_tree_h" if self.half else "sgpu_attn_tree", self.gpu.byref(self.a), self.ws.ptr, self.need, stream)

    def out(self):
        assert np.all(self.ws.to_host()[self.need:] == 0xFF)
        o = self.keep["out"].to_host()
        assert np.all(o[:, self.NH * self.HD:] == -77)
        return o[:, :self.NH * self.HD].reshape(self.c.R, self.NH, self.HD)

    def keys(self, b, r):
        """The tokens that row r of sequence b sees."""
        c = self.c
        have, i, n = max(int(c.len[b]), 0), r - int(c.q_start[b]), int(c.q_start[b + 1]) - int(c.q_start[b])
        new = [j for j in range(n) if (j <= i if self.bits is None else j < self.bits.shape[1] and self.bits[r, j])]
        return [p for p in (c.place(b, t) for t in list(range(min(have, c.table_pages * c.page))) + [have + j for j in new]) if p]

    def want(self):
        c, G = self.c, self.NH // self.NKV
        w, bar = np.full((c.R, self.NH, self.HD), -77.0), np.zeros((c.R, self.NH, self.HD))
        for b in range(len(c.seqs)):
            for r in range(int(c.q_start[b]), int(c.q_start[b + 1])):
                at = self.keys(b, r)
                if not at:
                    w[r] = 0.0
                    continue
                i = tuple(np.array(at).T)
                K, V = c.view(0)[i].astype(np.float64), c.view(1)[i].astype(np.float64)
                Kh, Vh = np.repeat(K, G, 1), np.repeat(V, G, 1)
                q = self.q[r].astype(np.float64)
                s = np.einsum("hd,khd->hk", q, Kh) * self.scale
                ds = self.HD * U * np.einsum("hd,khd->hk", abs(q), abs(Kh)) * abs(self.scale)
                p = np.exp(s - s.max(1, keepdims=True))
                p /= p.sum(1, keepdims=True)
                w[r] = np.einsum("hk,khd->hd", p, Vh)
                bar[r] = np.einsum("hk,khd->hd", p * (2 * ds + 2 * (p * ds).sum(1, keepdims=True) + (2 * len(K) + 16) * U), abs(Vh)) + 1e-30
        return w, bar

    def compare(self):
        with np.errstate(invalid="ignore", over="ignore"):
            got, (want, bar) = self.out(), self.want()
            fine = np.isfinite(want)
            assert np.array_equal(np.isfinite(got), fine)
            diff = np.where(fine, np.abs(got - want), 0.0)
            bad = fine & ~(diff <= bar)
        assert not bad.any(), (float(diff.max()), np.argwhere(bad)[:4].tolist())

    def check(self, stream=None):
        self.call(stream)
        self.gpu.synchronize()
        self.compare()


HEADS = [(14, 2, 64), (12, 12, 64), (8, 2, 128), (6, 2, 32), (1, 1, 64), (40, 1, 128)]
TREES = {
    "one": [(0, 1)], "step": [(700, 1)], "decode": [(3, 1), (0, 1), (40, 1), (129, 1), (31, 1), (32, 1)],
    "drafts": [(17, 5), (0, 3), (63, 0), (64, 8), (31, 1), (0, 0), (95, 33)], "wide": [(100, 70), (257, 20), (0, 129)]}


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("heads", HEADS, ids=str)
@pytest.mark.parametrize("name", TREES)
def test_attn_tree(gpu, name, heads, half):
    for page, layout, kind in ((16, "tokens", None), (7, "heads", "tree"), (64, "tokens", "random"), (1, "tokens", "tree")):
        Tree(gpu, TREES[name], *heads, page, half, kind=kind, layout=layout, before=2, behind=3, qlayout="padded" if page == 7 else "rows").check()


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("kind", [None, "tree", "random"])
def test_attn_tree_many_rows(gpu, kind, half):
    """More rows a sequence than a block takes at once, keys over several blocks."""
    Tree(gpu, [(500, 200), (33, 90), (1000, 1)], 14, 2, 64, 16, half, kind=kind, before=1, behind=1).check()
    Tree(gpu, [(5, 130), (300, 64)], 4, 4, 128, 32, half, kind=kind).check()


@pytest.mark.parametrize("half", [False, True])
def test_attn_tree_rows_that_see_nothing(gpu, half):
    t = Tree(gpu, [(0, 5), (0, 40), (3, 2)], 4, 2, 64, 16, half, kind="none")
    t.check()
    assert np.all(t.out()[:45] == 0)
    # no word of mask at all; a word less than there are rows
    Tree(gpu, [(0, 5), (40, 3)], 4, 2, 64, 16, half, kind="tree", words=0).check()
    Tree(gpu, [(20, 50), (0, 33)], 4, 2, 64, 16, half, kind="tree", words=1).check()
    Tree(gpu, [(20, 50), (0, 33)], 4, 2, 64, 16, half, kind="tree", words=4).check()


@pytest.mark.parametrize("hints", [(0, 0), (1, 1), (3, 200), (500, 100000), (64, 129)])
def test_attn_tree_hints_do_not_matter(gpu, hints):
    for half in (False, True):
        Tree(gpu, [(700, 1), (10, 40), (0, 3)], 14, 2, 64, 16, half, kind="tree", hints=hints, behind=2).check()


@pytest.mark.parametrize("half", [False, True])
def test_attn_tree_pages_that_are_none(gpu, half):
    """Tokens whose page is not there are not seen; lengths out of range are cut to what the table holds."""
    t = Tree(gpu, [(100, 5), (40, 40), (64, 8), (5, 1), (9, 2)], 14, 2, 64, 8, half, kind="tree")
    c = t.c
    c.table[0, 3], c.table[1, 0], c.table[1, 7], c.table[2, 8] = c.pages, -1, -2**31, 2**31 - 1
    c.table[3, 0] = -7
    c.len[4] = 2**31 - 1
    c.put("table", c.table)
    c.put("len", c.len)
    with np.errstate(invalid="ignore"):
        t.check()
    c.len[4] = -4                                       # counts as none: tokens 0, 1
    c.put("len", c.len)
    c.len[4] = 0
    t.check()


@pytest.mark.parametrize("half", [False, True])
def test_attn_tree_pages_shared_by_sequences(gpu, half):
    """A prompt's whole pages in several tables."""
    t = Tree(gpu, [(48, 4), (40, 3), (50, 1)], 8, 2, 64, 16, half, kind="tree")
    t.c.table[1, :2] = t.c.table[0, :2]
    t.c.table[2, :3] = t.c.table[0, :3]
    t.c.put("table", t.c.table)
    t.check()


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
def test_attn_tree_unseen_values_do_not_matter(gpu, value, half):
    """A drafted token that is not a number reaches the rows that see it, no others."""
    for seqs in ([(50, 12), (9, 3)], [(200, 60), (9, 3)]):
        for c in range(2):
            t = Tree(gpu, seqs, 14, 2, 64, 16, half, kind="tree", seed=4)
            clean, bar = t.want()
            t.c.at(c, 0, seqs[0][0] + 3)[...] = value
            t.c.put("kv"[c], t.c.buf[c])
            t.call()
            gpu.synchronize()
            got = t.out()
            sees = np.zeros(t.c.R, bool)
            sees[:seqs[0][1]] = t.bits[:seqs[0][1], 3]
            assert sees.any() and not sees.all()
            assert np.all(np.abs(got - clean)[~sees] <= bar[~sees])
            if c == 1 or np.isnan(value):
                assert not np.isfinite(got[sees]).any()
            else:                                       # an infinite key: a score of -infinity is no weight
                low = ~np.isnan(got[sees])
                t.bits[:, 3] = False
                less, lessbar = t.want()
                assert np.all(np.abs(got[sees] - less[sees])[low] <= lessbar[sees][low])


@pytest.mark.parametrize("half", [False, True])
def test_attn_tree_values_past_the_end_do_not_matter(gpu, half):
    """Every place that holds no token is NaN (Cache): pages that end inside a tile, whole pages behind the last token."""
    Tree(gpu, [(33, 1), (127, 2), (128, 1), (1, 1)], 14, 2, 64, 50, half, spare=9).check()


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("big", [1e4, 6e4])
@pytest.mark.parametrize("rows", [3, 60])
def test_attn_tree_keys_of_very_different_size(gpu, rows, big, half):
    """A key and a value far larger than the rest, with little weight: the rest keeps its digits."""
    t = Tree(gpu, [(300, rows)], 14, 2, 64, 16, half, kind="tree", seed=7)
    t.c.at(0, 0, 77)[...] = -np.sign(t.q[0, 0]) * 0.5
    for c in range(2):
        t.c.at(c, 0, 9)[...] *= np.asarray(big, np.float32).astype(t.c.buf[c].dtype) / 4
        t.c.put("kv"[c], t.c.buf[c])
    t.check()


@pytest.mark.parametrize("where", [1e30, 1e-30, 1e12, 1e-18, 1e37])
@pytest.mark.parametrize("rows", [3, 60])
def test_attn_tree_fp32_range(gpu, rows, where):
    """Values (and keys beside small queries) of any fp32 size."""
    t = Tree(gpu, [(200, rows), (40, 2)], 14, 2, 64, 16, False, kind="tree", seed=8)
    t.c.buf[1] = (t.c.buf[1] * np.float32(where)).astype(np.float32)
    t.c.put("v", t.c.buf[1])
    t.check()
    t.c.buf[0] = (t.c.buf[0] * np.float32(where)).astype(np.float32)
    t.c.put("k", t.c.buf[0])
    t.q = (t.q / np.float32(where)).astype(np.float32)
    t.keep["q"] = dev(gpu, t.q)
    t.a.q = t.keep["q"].ptr
    t.check()
    if where > 1:                                       # some rows of values that size, among ordinary ones
        t = Tree(gpu, [(200, rows)], 14, 2, 64, 16, False, kind="tree", seed=9)
        t.c.at(1, 0, 20)[...] *= np.float32(where)
        t.c.at(1, 0, 21)[...] /= np.float32(where)
        t.c.at(1, 0, 22)[...] = 0
        t.c.at(0, 0, 23)[...] = 0
        t.c.put("v", t.c.buf[1])
        t.c.put("k", t.c.buf[0])
        t.check()


@pytest.mark.parametrize("half", [False, True])
def test_attn_tree_large_scores(gpu, half):
    Tree(gpu, [(150, 40), (70, 2)], 14, 2, 64, 16, half, kind="tree", scale=6.0).check()
    Tree(gpu, [(150, 40), (70, 2)], 14, 2, 64, 16, half, kind="tree", scale=0.0).check()


def test_attn_tree_long(gpu):
    """Splits of many blocks, ragged: one long sequence among short ones."""
    Tree(gpu, [(9001, 2), (5, 2), (0, 1)], 4, 1, 64, 16, True, kind="tree").check()
    Tree(gpu, [(6001, 1)], 2, 1, 128, 64, False).check()
    Tree(gpu, [(3001, 33)], 7, 1, 64, 16, False, kind="tree").check()


@pytest.mark.parametrize("hints", [(1, 40), (3, 1000)])
def test_attn_tree_many_sequences(gpu, hints):
    seqs = [(b % 50, b % 4) for b in range(600)]
    Tree(gpu, seqs, 2, 1, 32, 8, True, hints=hints, before=1, behind=5).check()


def test_attn_tree_far_pages(gpu):
    """Pages that lie more than 2^32 values apart."""
    stride = (1 << 32) + 64
    big = gpu.DeviceArray(2 * stride + (1 << 22), np.uint8)
    half = 1 << 21
    c = Cache(gpu, [(20, 3)], 1, 64, 16, True, spare=0, seed=3)
    t = Tree(gpu, [(20, 3)], 4, 1, 64, 16, True, kind="tree", spare=0, seed=3)
    n = 16 * 64
    for p in range(2):
        for i, name in enumerate(("k", "v")):
            gpu.call("sgpu_memcpy_htod", big.ptr + i * half + 2 * p * stride, t.c.buf[i][p].ctypes.data, 2 * n)
    t.a.c.k, t.a.c.v, t.a.c.page_stride = big.ptr, big.ptr + half, stride
    assert c.pages == 2
    t.check()
    a = Append(gpu, [(14, 5)], 4, 1, 64, 16, True, spare=0, seed=5)
    for p in range(2):
        for i in range(2):
            gpu.call("sgpu_memcpy_htod", big.ptr + i * half + 2 * p * stride, a.c.buf[i][p].ctypes.data, 2 * n)
    a.a.c.k, a.a.c.v, a.a.c.page_stride = big.ptr, big.ptr + half, stride
    a.call()
    gpu.synchronize()
    for i, name in enumerate(("k", "v")):
        host = np.empty((2, n), np.float16)
        for p in range(2):
            gpu.call("sgpu_memcpy_dtoh", host[p].ctypes.data, big.ptr + i * half + 2 * p * stride, 2 * n)
        a.c.put(name, host)
    a.compare()
    big.close()


def test_attn_tree_streams_and_recorded(gpu):
    """Two streams at once; a recorded call replayed while its sequences grow; results equal bit for bit those of a
    call by itself."""
    s1, s2 = gpu.Stream(), gpu.Stream()
    a = Tree(gpu, [(720, 1), (3, 2), (333, 1)], 14, 2, 64, 16, False, seed=1)
    b = Tree(gpu, [(70, 40), (300, 7)], 8, 2, 128, 32, True, kind="tree", seed=2)
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
    full = a.c.len.copy()
    for back in (300, 5, 3, 0):
        a.c.len = np.maximum(full - back, 0).astype(np.int32)
        a.c.put("len", a.c.len)
        g.launch()
        s1.synchronize()
        a.compare()
        got = a.out().copy()
        a.check()
        assert np.array_equal(got.view(np.uint32), a.out().view(np.uint32))


# ---- logits ----
class Logits:
    def __init__(self, gpu, rows, V, half, hist=(20, 10), bias=3, allow=0.5, seed=0, pad=(0, 0), shared=False, same=False, same_mask=False):
        rng = np.random.default_rng(seed + V)
        self.gpu, self.rows, self.V, self.half, self.same = gpu, rows, V, half, same
        t = np.float16 if half else np.float32
        self.x = np.full((rows, V + pad[0]), 55, t)
        self.x[:, :V] = rng.standard_normal((rows, V)) * 3
        self.pad = pad
        self.rep = (1 + rng.random(rows)).astype(np.float32)
        self.freq, self.pres = rng.standard_normal(rows).astype(np.float32) * 0.5, rng.standard_normal(rows).astype(np.float32)
        n_tok = sum(hist) * rows
        self.tok = rng.integers(-3, V + 3, max(n_tok, 1)).astype(np.int32)           # some outside
        at = np.arange(rows)[:, None] * sum(hist)
        self.span = np.concatenate([np.zeros_like(at) if shared else at, np.full((rows, 1), hist[0]), at + hist[0], np.full((rows, 1), hist[1])], 1).astype(np.int32)
        self.n_tok = n_tok
        self.bias_id = rng.integers(-1, V + 1, (rows, max(bias, 1))).astype(np.int32)  # the same twice, some outside
        self.bias = (rng.standard_normal((rows, max(bias, 1))) * 5).astype(np.float32)
        self.bias_span = np.stack([np.arange(rows) * max(bias, 1), np.full(rows, bias)], 1).astype(np.int32)
        words = -(-V // 32)
        self.allow = rng.integers(0, 2**32, (1 if same_mask else rows, words + 1), dtype=np.uint64).astype(np.uint32)
        if allow != 0.5:
            m = rng.random((self.allow.shape[0], (words + 1) * 32)) < allow
            self.allow = np.packbits(m, axis=1, bitorder="little").view(np.uint32).copy()
        a = self.a = gpu.LogitsArgs()
        d = self.keep = {n: dev(gpu, getattr(self, n)) for n in ("x", "rep", "freq", "pres", "tok", "span", "bias_id", "bias", "bias_span", "allow")}
        d["y"] = dev(gpu, np.full((rows, V + pad[1]), 44, t))
        for n in ("rep", "freq", "pres", "tok", "span", "bias_id", "bias", "bias_span", "allow", "x", "y"):
            setattr(a, n, d[n].ptr)
        a.x_row, a.y_row, a.rows, a.V, a.n_tok, a.n_bias = V + pad[0], V + pad[1], rows, V, n_tok, self.bias.size if bias else 0
        a.allow_row = 0 if same_mask else words + 1
        if same:
            a.y, a.y_row = a.x, a.x_row
        self.same_mask = same_mask

    def call(self, stream=None):
        self.gpu.call("sgpu_logits_adjust_h" if self.half else "sgpu_logits_adjust", self.gpu.byref(self.a), stream)

    def want(self):
        a, V = self.a, self.V
        y = self.x[:, :V].astype(np.float64)
        size = abs(y)
        for r in range(self.rows):
            said = {}
            prompt = set()
            if a.span:
                for k in range(2):
                    f = min(max(int(self.span[r, 2 * k]), 0), self.n_tok)
                    for v in self.tok[f:f + min(max(int(self.span[r, 2 * k + 1]), 0), self.n_tok - f)]:
                        if 0 <= v < V:
                            prompt.add(int(v))
                            if k:
                                said[int(v)] = said.get(int(v), 0) + 1
            with np.errstate(invalid="ignore"):
                for v in prompt:
                    rep = float(self.rep[r]) if a.rep else 1.0
                    y[r, v] = y[r, v] / rep if y[r, v] > 0 else y[r, v] * rep
                for v, n in said.items():
                    f, p = (float(self.freq[r]) if a.freq else 0.0), (float(self.pres[r]) if a.pres else 0.0)
                    y[r, v] = y[r, v] - f * n - p
                    size[r, v] += abs(f) * n + abs(p)
                if a.bias_span and a.n_bias:
                    f = int(self.bias_span[r, 0])
                    last = {int(i): float(b) for i, b in zip(self.bias_id.ravel()[f:f + self.bias_span[r, 1]], self.bias.ravel()[f:f + self.bias_span[r, 1]])}
                    for v, b in last.items():
                        if 0 <= v < V:
                            y[r, v] += b
                            size[r, v] += abs(b)
        if a.allow:
            bits = np.unpackbits(self.allow.view(np.uint8), axis=1, bitorder="little")[:, :V]
            y[np.broadcast_to(bits, y.shape) == 0] = -np.inf
        return y, size

    def compare(self):
        got = self.keep["x" if self.same else "y"].to_host()
        V = self.V
        assert np.all(got[:, V:] == (55 if self.same else 44))
        got = got[:, :V].astype(np.float64)
        want, size = self.want()
        bar = np.abs(want) * 2.0**(-11 if self.half else -24) + 2.0**(-25 if self.half else -150) + size * 2.0**-50
        fine = np.isfinite(want)
        assert np.array_equal(got[~fine], want[~fine], equal_nan=True)
        assert np.all(np.abs(got[fine] - want[fine]) <= bar[fine])

    def check(self, stream=None):
        self.call(stream)
        self.gpu.synchronize()
        self.compare()


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("V", [1, 7, 31, 32, 33, 1000, 8191, 8192, 8193, 50257, 151936])
@pytest.mark.parametrize("rows", [1, 3])
def test_logits_adjust(gpu, rows, V, half):
    for same in (False, True):
        Logits(gpu, rows, V, half, same=same, pad=(3, 5)).check()
    Logits(gpu, rows, V, half, hist=(0, 2000), bias=0, allow=0.01, pad=(1, 0)).check()
    Logits(gpu, rows, V, half, hist=(1500, 0), bias=300, allow=0.99, shared=True, same_mask=True).check()


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("without", ["span", "rep", "freq", "pres", "bias_span", "allow", "all"])
def test_logits_adjust_steps_left_out(gpu, without, half):
    for same in (False, True):
        t = Logits(gpu, 2, 9000, half, same=same, hist=(100, 3000))
        for n in ("span", "rep", "freq", "pres", "bias_span", "allow"):
            if without in (n, "all"):
                setattr(t.a, n, None)
        t.check()


@pytest.mark.parametrize("half", [False, True])
def test_logits_adjust_odd_values(gpu, half):
    """Infinities and NaN, zeros of both signs; spans out of range; a grammar that allows nothing."""
    t = Logits(gpu, 3, 500, half, hist=(200, 300), allow=0.9)
    t.x[:, :400:7], t.x[:, 1:400:7], t.x[:, 2:400:7], t.x[:, 3:400:7] = np.inf, -np.inf, np.nan, -0.0
    t.gpu.call("sgpu_memcpy_htod", t.keep["x"].ptr, t.x.ctypes.data, t.x.nbytes)
    t.span[0] = [-5, 2**31 - 1, 1400, 2**31 - 1]
    t.span[1] = [2**31 - 1, 5, 10, -5]
    t.gpu.call("sgpu_memcpy_htod", t.keep["span"].ptr, t.span.ctypes.data, t.span.nbytes)
    t.allow[2] = 0
    t.gpu.call("sgpu_memcpy_htod", t.keep["allow"].ptr, t.allow.ctypes.data, t.allow.nbytes)
    t.check()
    assert np.all(t.keep["y"].to_host()[2, :500] == -np.inf)


def test_logits_adjust_many_rows_and_unaligned(gpu):
    Logits(gpu, 300, 8200, True, hist=(50, 9)).check()
    t = Logits(gpu, 2, 3000, False)
    big = dev(gpu, np.concatenate([np.zeros(1, np.float32), t.x.ravel()]))
    t.a.x = big.offset(1)
    t.check()


def test_logits_adjust_streams_and_recorded(gpu):
    s1, s2 = gpu.Stream(), gpu.Stream()
    a, b = Logits(gpu, 3, 50257, False, hist=(300, 200)), Logits(gpu, 70, 9000, True, bias=40)
    for _ in range(4):
        a.call(s1.h)
        b.call(s2.h)
    s1.synchronize()
    s2.synchronize()
    a.compare()
    b.compare()
    with gpu.Graph(s1) as g:
        a.call(s1.h)
    for n in (5, 0, 100):                               # the output grows on the device
        a.span[:, 3] = n
        gpu.call("sgpu_memcpy_htod", a.keep["span"].ptr, a.span.ctypes.data, a.span.nbytes)
        g.launch()
        s1.synchronize()
        a.compare()


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("HD,page", [(64, 16), (32, 24), (128, 48)])
def test_attn_tree_more_row_tiles_than_blocks_of_the_device(gpu, HD, page, half):
    """So many sequences and KV heads that each row tile has a block of its own: ragged ones, some without rows or tokens."""
    seqs = [(b * 7 % 90, b % 3) for b in range(270)] + [(0, 1), (0, 0), (210, 1)]
    Tree(gpu, seqs, 8, 4, HD, page, half, before=1, behind=2).check()
    seqs = [(b * 5 % 70, 5 + b % 9) for b in range(130)] + [(0, 12), (9, 0), (150, 40)]
    Tree(gpu, seqs, 32, 8, HD, page, half, kind="tree", behind=1).check()


@pytest.mark.parametrize("half", [False, True])
def test_attn_tree_without_rows_and_alone(gpu, half):
    """No new rows at all; one sequence, whose table's row has no stride; no token with a place."""
    t = Tree(gpu, [(5, 0), (9, 0)], 4, 2, 64, 16, half, before=2, behind=3)
    t.check()
    assert np.all(t.out() == -77)
    t = Tree(gpu, [(77, 3)], 14, 2, 64, 48, half, kind="tree")
    t.a.c.table_row = 0
    t.check()
    a = Append(gpu, [(77, 3)], 14, 2, 64, 48, half)
    a.a.c.table_row = 0
    a.check()
    t = Tree(gpu, [(77, 3)], 14, 2, 64, 48, half, kind="tree")
    t.a.c.pages = 0
    t.call()
    gpu.synchronize()
    assert np.all(t.out() == 0)


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("HD", [32, 64, 128])
@pytest.mark.parametrize("rows", [1, 5, 12, 30])
def test_cache_without_pages(gpu, rows, HD, half):
    """No page, or no entry in the table, and no buffers: nothing is read or written there, rows see nothing."""
    for pages, table_pages in ((0, 3), (3, 0)):
        for seqs in ([(5, rows)], [(5, rows)] * 70):
            t = Tree(gpu, seqs, 14, 2, HD, 16, half, before=1)
            t.a.c.k = t.a.c.v = t.a.c.table = None
            t.a.c.pages, t.a.c.table_pages = pages, table_pages
            t.call()
            a = Append(gpu, seqs, 14, 2, HD, 16, half, before=1)
            a.a.c.k = a.a.c.v = a.a.c.table = None
            a.a.c.pages, a.a.c.table_pages = pages, table_pages
            a.call()
            gpu.synchronize()
            assert np.all(t.out()[1:] == 0) and np.all(t.out()[0] == -77)
            (q, bar), _ = a.want()
            got = a.keep["out"].to_host()[:, :-4].reshape(q.shape)
            assert np.all(np.abs(got - q) <= bar)


@pytest.mark.parametrize("rows", [1, 3, 8, 40])
@pytest.mark.parametrize("HD", [64, 128])
def test_attn_tree_sizes_that_change_from_key_to_key(gpu, HD, rows):
    """Runs of keys of one size and single keys of others, 2^-12 to 2^6 of the ordinary: tiles of one scale, and of many."""
    t = Tree(gpu, [(300, rows), (70, rows)], 14, 2, HD, 16, False, kind="tree", seed=11)
    rng = np.random.default_rng(5)
    for c in range(2):
        for b, (have, n) in enumerate(t.c.seqs):
            for at in range(have + n):
                k = int(rng.integers(-12, 7)) if at % 128 >= 64 else -8 if c and at < 32 else 0
                t.c.at(c, b, at)[...] *= np.float32(2.0**k)
        t.c.put("kv"[c], t.c.buf[c])
    t.check()


@pytest.mark.parametrize("rows", [1, 40])
def test_attn_tree_scale_zero(gpu, rows):
    """The average of the values, whatever the keys' size."""
    t = Tree(gpu, [(100, rows)], 14, 2, 64, 16, False, kind="tree", scale=0.0, seed=12)
    t.c.buf[0] = (t.c.buf[0] * np.float32(2.0**100)).astype(np.float32)
    t.c.put("k", t.c.buf[0])
    t.check()


@pytest.mark.parametrize("B", [3, 100])
def test_attn_tree_starts_that_fall(gpu, B):
    """No batch has them; the call ends, rows' results are open, what lies around them stays (out), the next call is right."""
    t = Tree(gpu, [(30, 3)] * B, 14, 2, 64, 16, False)
    t.c.q_start[1:-1] = np.where(np.arange(B - 1) % 2, 0, t.c.R)
    t.c.put("q_start", t.c.q_start)
    t.call()
    gpu.synchronize()
    t.out()
    t.c.q_start[:] = np.minimum(3 * np.arange(B + 1), t.c.R)
    t.c.put("q_start", t.c.q_start)
    t.check()


def test_attn_tree_recorded_calls_share_a_workspace(gpu):
    """Two recorded calls on one stream with one workspace, in turn, each replay as the call by itself."""
    s = gpu.Stream()
    a = Tree(gpu, [(720, 1), (3, 2), (333, 1)], 14, 2, 64, 16, False, seed=1)
    b = Tree(gpu, [(70, 40), (300, 7)], 8, 2, 128, 32, True, kind="tree", seed=2)
    big = a if a.need > b.need else b
    small = b if big is a else a
    small.ws = big.ws
    small.need, need = big.need, small.need
    graphs = []
    for t in (a, b):
        with gpu.Graph(s) as g:
            t.call(s.h)
        graphs.append(g)
    for _ in range(3):
        for g in graphs:
            g.launch()
        s.synchronize()
        a.compare()
        b.compare()
    small.need = need


def test_logits_adjust_tables_over_many_chunks(gpu):
    """More tokens and biases than stay in registers, a block taking all chunks of its row."""
    for half, same in ((False, False), (True, True)):
        Logits(gpu, 260, 20000, half, hist=(3000, 2500), bias=1500, allow=0.8, same=same).check()


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("heads", HEADS, ids=str)
@pytest.mark.parametrize("name", ["decode", "drafts", "wide"])
def test_attn_tree_one_long_among_short(gpu, name, heads, half):
    """Steps dealt over blocks and joined: a long sequence behind short ones, rows of no sequence around them."""
    for page, layout, kind in ((16, "tokens", "tree"), (24, "heads", None)):
        Tree(gpu, TREES[name] + [(2600, 2)], *heads, page, half, kind=kind, layout=layout, before=2, behind=3).check()


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("B", [64, 65, 700, 4200])
def test_attn_tree_many_sequences_one_long(gpu, B, half):
    """More sequences than a wave, or 64 waves, has lanes, dealt: without rows, without tokens, a long one in the middle and at the end."""
    seqs = [(b * 7 % 40, b % 3) for b in range(B)]
    seqs[B // 2], seqs[-1] = (3500, 2), (2000, 1)
    Tree(gpu, seqs, 2, 1, 32, 64, half, before=1, behind=2).check()


# ---- as they are used together ----
def test_drafted_trees_checked_step_by_step(gpu):
    """Rows of drafted trees appended and attended to, twice, the sequences growing by what was taken in between; then their
    logits adjusted and scored: eagerly, and as one recorded step replayed over the same device ints."""
    NH, NKV, HD, page, V = 14, 2, 64, 16, 3001
    seqs = [(30, 6), (0, 4), (63, 9)]
    rng = np.random.default_rng(12)
    s = gpu.Stream()

    def build():
        ap = Append(gpu, seqs, NH, NKV, HD, page, False, norm=True, seed=6, spare=4)
        at = Tree(gpu, seqs, NH, NKV, HD, page, False, kind="tree", seed=6, spare=4)
        for n in ("k", "v", "table", "len", "q_start"):
            setattr(at.a.c, n, getattr(ap.a.c, n))
        ap.a.out_row = NH * HD
        at.a.q, at.a.q_row = ap.a.q_out, NH * HD
        return ap, at

    ap, at = build()
    lo = Logits(gpu, ap.c.R, V, False, hist=(40, 20), bias=4, allow=0.7)
    tok = rng.integers(0, V, (ap.c.R, 1)).astype(np.int32)
    dt, lp, ent = dev(gpu, tok), gpu.DeviceArray((ap.c.R, 1)), gpu.DeviceArray(ap.c.R)
    need = gpu.lib().sgpu_logprobs_workspace(ap.c.R, V, 0)
    ws = gpu.DeviceArray(need, np.uint8)

    def step(stream):
        ap.call(stream)
        at.call(stream)
        lo.call(stream)
        gpu.call("sgpu_logprobs", lo.a.y, V, ap.c.R, V, dt.ptr, 1, lp.ptr, ent.ptr, 0, None, None, ws.ptr, need, stream)

    def verify():
        (q, qbar), pages = ap.want()
        for i, n in enumerate(("k", "v")):
            host = ap.c.keep[n].to_host()
            want, bar = pages[i]
            got = host.reshape(want.shape)
            assert np.array_equal(np.isnan(got), np.isnan(want)) and np.all(np.abs(got - want)[~np.isnan(want)] <= bar[~np.isnan(want)])
            ap.c.buf[i], at.c.buf[i] = host, host
        got_q = ap.keep["out"].to_host().ravel()[:ap.c.R * NH * HD].reshape(q.shape)
        assert np.all(np.abs(got_q - q) <= qbar)
        at.q, at.c.len, at.c.table = got_q, ap.c.len, ap.c.table
        at.compare()
        lo.compare()
        y = lo.keep["y"].to_host().astype(np.float64)
        with np.errstate(divide="ignore"):
            m = y.max(1, keepdims=True)
            want = (y - m)[np.arange(ap.c.R), tok[:, 0]] - np.log(np.exp(y - m).sum(1))
        got = lp.to_host()[:, 0]
        fine = np.isfinite(want)
        assert np.array_equal(got[~fine], want[~fine]) and np.all(np.abs(got[fine] - want[fine]) <= (V / 256 + 80) * U * (1 + abs(want[fine])))

    step(None)
    gpu.synchronize()
    verify()
    with gpu.Graph(s) as g:
        step(s.h)
    for taken in ([0, 0, 0], [2, 1, 0], [0, 3, 3], [1, 1, 1]):
        ap.c.len = (ap.c.len + np.array(taken)).astype(np.int32)
        ap.c.put("len", ap.c.len)
        g.launch()
        s.synchronize()
        verify()


@pytest.mark.parametrize("half", [False, True])
def test_many_rows_equal_their_parts(gpu, half):
    """Rows past the size from which they are streamed, against calls of a part each, bit for bit: norms and rotations, appending."""
    rng = np.random.default_rng(21)
    NH, NKV, HD, T = 4, 2, 64, 33000
    n, kt = (NH + 2 * NKV) * HD, np.float16 if half else np.float32
    assert T * n > 16 << 20 > T // 3 * n
    x, w = dev(gpu, rng.standard_normal((T, n)).astype(np.float32)), dev(gpu, (1 + 0.3 * rng.standard_normal(HD)).astype(np.float32))
    turns = dev(gpu, turns_of(HD))
    cuts = [0, 11000, 20001, T]
    for nb in (0, 1):
        got = []
        for parts in ([(0, T)], list(zip(cuts, cuts[1:]))):
            y = dev(gpu, np.zeros((T, n), kt))
            for t0, t1 in parts:
                gpu.call("sgpu_qk_norm_rope_h" if half else "sgpu_qk_norm_rope", x.offset(t0 * n), n, y.offset(t0 * n), n, w.ptr, w.ptr, 1e-6, None,
                         t0, turns.ptr, HD, nb, 1.0, t1 - t0, NH, NKV, HD, None)
            gpu.synchronize()
            got.append(y.to_host())
        assert np.array_equal(got[0].view(np.uint8), got[1].view(np.uint8)) and np.all(got[0][:, (NH + NKV) * HD:] == 0)
    got = []
    for parts in ([(0, T)], list(zip(cuts, cuts[1:]))):
        k, v, q = (gpu.DeviceArray((T // 64 + 1, 64, NKV, HD), kt), gpu.DeviceArray((T // 64 + 1, 64, NKV, HD), kt), gpu.DeviceArray((T, NH * HD)))
        for d in (k, v, q):
            d.fill_bytes(0)
        table = dev(gpu, rng.permutation(T // 64 + 1).astype(np.int32) if not got else got[0][3])
        for t0, t1 in parts:
            a = gpu.KvAppendArgs()
            keep = dev(gpu, np.array([t0], np.int32)), dev(gpu, np.array([0, t1 - t0], np.int32))
            a.c.k, a.c.v, a.c.page_stride, a.c.kv_row, a.c.kv_head, a.c.pages, a.c.page = k.ptr, v.ptr, 64 * NKV * HD, NKV * HD, HD, T // 64 + 1, 64
            a.c.table, a.c.table_row, a.c.table_pages, a.c.len, a.c.q_start, a.c.R, a.c.B = table.ptr, T, T // 64 + 1, keep[0].ptr, keep[1].ptr, t1 - t0, 1
            a.q, a.k, a.v = x.offset(t0 * n), x.offset(t0 * n + NH * HD), x.offset(t0 * n + (NH + NKV) * HD)
            a.q_row = a.k_row = a.v_row = n
            a.q_out, a.out_row, a.turns, a.wq, a.wk = q.offset(t0 * NH * HD), NH * HD, turns.ptr, w.ptr, w.ptr
            a.eps, a.mscale, a.rot, a.NH, a.NKV, a.HD = 1e-6, 1.0, HD, NH, NKV, HD
            gpu.call("sgpu_kv_append_h" if half else "sgpu_kv_append", gpu.byref(a), None)
            gpu.synchronize()
        got.append([d.to_host() for d in (k, v, q, table)])
    assert all(np.array_equal(a.view(np.uint8), b.view(np.uint8)) for a, b in zip(*got))

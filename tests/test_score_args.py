"""Arguments of the operators over several continuations of one prompt, without a device: what is
refused is refused before any device work, calls without work succeed, and the rotary tables (a host
function) match their formulas."""
import ctypes as ct
import math

import numpy as np
import pytest

BAD = -1


def args(sg, **kw):
    """A well-formed description at addresses that no call here may reach."""
    a = sg.AttnPrefixArgs()
    base = dict(q=1 << 20, kp=2 << 20, vp=3 << 20, ks=4 << 20, vs=5 << 20, out=6 << 20, q_start=7 << 20, kv_start=8 << 20,
                kv_len=9 << 20, q_row=448, q_head=64, out_row=448, out_head=64, kp_row=64, kp_head=64, ks_row=64, ks_head=64, R=3,
                B=2, P=10, SR=5, NH=7, NKV=1, HD=64, max_q=2, max_kv=3, scale=0.125)
    for k, v in {**base, **kw}.items():
        setattr(a, k, v)
    return a


REFUSED = [dict(R=-1), dict(B=-1), dict(P=-1), dict(SR=-1), dict(NH=0), dict(NKV=0), dict(NH=6, NKV=4), dict(HD=48), dict(HD=0),
           dict(max_q=-1), dict(max_kv=-1), dict(scale=math.nan), dict(scale=math.inf), dict(scale=-0.1), dict(q=None),
           dict(out=None), dict(q_start=None), dict(kp=None), dict(vp=None), dict(ks=None), dict(vs=None), dict(kv_start=None),
           dict(kv_len=None), dict(q=(1 << 20) + 4), dict(kp=(1 << 20) + 8), dict(vs=(1 << 20) + 4), dict(out=(1 << 20) + 4),
           dict(q_start=(1 << 20) + 2), dict(q_row=450), dict(q_head=66), dict(kp_row=66), dict(kp_row=0), dict(ks_row=-64),
           dict(kp_row=(1 << 22) + 64), dict(out_row=0), dict(out_head=2), dict(R=1 << 26)]


@pytest.mark.parametrize("kw", REFUSED, ids=[",".join(f"{k}={v}" for k, v in r.items()) for r in REFUSED])
def test_attn_prefix_refuses(sg, kw):
    L = sg.lib()
    for fn in ("sgpu_attn_prefix", "sgpu_attn_prefix_h"):
        assert getattr(L, fn)(ct.byref(args(sg, **kw)), 16 << 20, 1 << 40, None) == BAD
    assert L.sgpu_attn_prefix_workspace(ct.byref(args(sg, **kw))) == 0


def test_attn_prefix_without_work_and_null(sg):
    L = sg.lib()
    assert L.sgpu_attn_prefix(None, None, 0, None) == BAD
    assert L.sgpu_attn_prefix_workspace(None) == 0
    for kw in (dict(R=0), dict(B=0), dict(R=0, q=None, out=None)):
        assert L.sgpu_attn_prefix(ct.byref(args(sg, **kw)), None, 0, None) == 0
    # fp16 rows: whole 16 bytes are 8 values
    assert L.sgpu_attn_prefix_h(ct.byref(args(sg, kp_row=68)), 16 << 20, 1 << 40, None) == BAD


def test_logprobs_refuses(sg):
    L = sg.lib()
    p = 1 << 20

    def call(fn="sgpu_logprobs", x=p, ld=100, rows=2, V=100, tok=p, nt=1, logp=p, ent=p, k=3, tl=p, ti=p, ws=p, nb=1 << 30):
        return getattr(L, fn)(x, ld, rows, V, tok, nt, logp, ent, k, tl, ti, ws, nb, None)

    for kw in (dict(rows=-1), dict(V=0), dict(V=-5), dict(nt=-1), dict(k=-1), dict(k=65), dict(ld=99), dict(x=None), dict(tok=None),
               dict(logp=None), dict(tl=None), dict(ti=None), dict(ws=None), dict(ws=p + 8), dict(x=p + 2), dict(nb=10),
               dict(rows=1 << 24)):
        assert call(**kw) == BAD, kw
    assert call(fn="sgpu_logprobs_h", x=p + 1) == BAD
    assert call(rows=0, x=None, ws=None) == 0
    assert L.sgpu_logprobs_workspace(2, 100, 3) > 0
    for bad in ((0, 100, 3), (2, 0, 3), (2, 100, 65), (2, 100, -1)):
        assert L.sgpu_logprobs_workspace(*bad) == 0


def test_rope_rows_refuses(sg):
    L = sg.lib()
    p = 1 << 20

    def call(fn="sgpu_rope_rows", x=p, xs=128, y=p, ys=128, pos=p, pos0=0, turns=p, rot=64, nb=0, T=2, H=2, HD=64):
        return getattr(L, fn)(x, xs, y, ys, pos, pos0, turns, rot, nb, 1.0, T, H, HD, None)

    for kw in (dict(T=-1), dict(H=-1), dict(HD=0), dict(rot=-2), dict(rot=3), dict(rot=66), dict(HD=512, rot=258, xs=1024, ys=1024),
               dict(xs=127), dict(ys=127), dict(x=None), dict(y=None), dict(turns=None), dict(x=p + 2), dict(y=2 * p + 2),
               dict(pos=p + 2), dict(turns=p + 4), dict(ys=256)):
        assert call(**kw) == BAD, kw
    assert call(fn="sgpu_rope_rows_h", y=2 * p + 1) == BAD
    assert call(T=0, x=None, y=None) == 0
    assert call(H=0, x=None, y=None) == 0
    assert call(rot=0, turns=None) == 0                    # in place and nothing to rotate


def test_rope_turns_formulas(sg):
    tau = 2 * math.pi
    rot, theta = 64, 1e4
    f = theta ** (-2.0 * np.arange(rot // 2) / rot)
    got, m = sg.rope_turns(rot, theta)
    assert np.allclose(got * tau, f, rtol=1e-14) and m == 1.0
    got, _ = sg.rope_turns(rot, theta, sg.ROPE_LINEAR, 8.0)
    assert np.allclose(got * tau, f / 8, rtol=1e-14)
    got, _ = sg.rope_turns(rot, theta, sg.ROPE_BASE, 8.0)
    assert got[0] * tau == pytest.approx(1.0) and got[-1] * tau == pytest.approx(f[-1] / 8, rel=1e-12)
    got, _ = sg.rope_turns(rot, theta, sg.ROPE_BANDS, 8.0, 8192.0, 1.0, 4.0)
    n = 8192 * f / tau
    assert np.allclose(got[n > 4] * tau, f[n > 4], rtol=1e-14) and np.allclose(got[n < 1] * tau, f[n < 1] / 8, rtol=1e-14)
    mid = (n > 1) & (n < 4)
    w = (n[mid] - 1) / 3
    assert mid.any() and np.allclose(got[mid] * tau, w * f[mid] + (1 - w) * f[mid] / 8, rtol=1e-13)
    got, m = sg.rope_turns(rot, theta, sg.ROPE_YARN, 16.0, 4096.0, 32.0, 1.0)
    at = [rot * math.log(4096 / (b * tau)) / (2 * math.log(theta)) for b in (32, 1)]
    lo, hi = max(math.floor(at[0]), 0), min(math.ceil(at[1]), rot - 1)
    w = 1 - np.clip((np.arange(rot // 2) - lo) / (hi - lo), 0, 1)
    assert np.allclose(got * tau, w * f + (1 - w) * f / 16, rtol=1e-13)
    assert m == pytest.approx(0.1 * math.log(16) + 1, rel=1e-7)
    assert sg.rope_turns(2, theta, sg.ROPE_BASE, 8.0)[0][0] * tau == pytest.approx(1.0)


def test_rope_turns_refuses(sg):
    L = sg.lib()
    out = np.empty(256)
    good = dict(rot=64, scaling=4, theta=1e4, factor=2.0, ctx=4096.0, lo=32.0, hi=1.0)

    def call(**kw):
        v = {**good, **kw}
        c = sg.RopeCfg(*[v[n] for n in ("rot", "scaling", "theta", "factor", "ctx", "lo", "hi")])
        return L.sgpu_rope_turns(ct.byref(c), out.ctypes.data, None)

    assert call() == 0
    for kw in (dict(rot=0), dict(rot=63), dict(rot=258), dict(scaling=-1), dict(scaling=5), dict(theta=1.0), dict(theta=math.nan),
               dict(theta=math.inf), dict(factor=0.5), dict(factor=math.nan), dict(ctx=0.0), dict(lo=1.0, hi=32.0), dict(hi=0.0),
               dict(scaling=3, lo=4.0, hi=4.0), dict(scaling=3, lo=0.0, hi=1.0)):
        assert call(**kw) == BAD, kw
    assert call(scaling=0, factor=0.0) == 0                # unused there
    c = sg.RopeCfg(64, 0, 1e4, 1, 0, 0, 0)
    assert L.sgpu_rope_turns(None, out.ctypes.data, None) == BAD and L.sgpu_rope_turns(ct.byref(c), None, None) == BAD


def test_qwen_score_null_engine(sg):
    assert sg.lib().sgpu_qwen_score(None, None, 1, None, None, 0, None, None, 0, None, None) == sg.SGPU_ERR_INVALID_ARG


def test_attn_prefix_number_of_sequences(sg):
    L = sg.lib()
    many = dict(R=1 << 22, NH=8, NKV=8, q_head=64, q_row=512, out_row=512, kp_row=512, ks_row=512)
    for B, fine in (((1 << 20) - 1, True), (1 << 20, False)):
        for max_q in (1, 1 << 22):                             # a hint asks for no more blocks than a launch takes
            a = args(sg, **many, B=B, max_q=max_q)
            assert (L.sgpu_attn_prefix_workspace(ct.byref(a)) > 0) == fine
            if not fine:
                assert L.sgpu_attn_prefix(ct.byref(a), 16 << 20, 1 << 60, None) == BAD

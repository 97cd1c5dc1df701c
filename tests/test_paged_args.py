"""Arguments of the operators over a paged cache and of the adjusted logits, without a device: what is refused is
refused before any device work, and calls without work succeed."""
import ctypes as ct
import math

import pytest

BAD = -1
P = 1 << 20                                             # addresses that no call here may reach


def cache(sg, c, **kw):
    base = dict(k=P, v=2 * P, page_stride=16 * 128, kv_row=128, kv_head=64, pages=9, page=16, table=3 * P, table_row=4, table_pages=4,
                len=4 * P, q_start=5 * P, R=3, B=2)
    for k, v in {**base, **kw}.items():
        setattr(c, k, v)


def split(sg, kw):
    names = {n for n, _ in sg.PagedKv._fields_}
    return {k: v for k, v in kw.items() if k in names}, {k[1:] if k.startswith("_") else k: v for k, v in kw.items() if k not in names}


def append(sg, **kw):
    a = sg.KvAppendArgs()
    mine, rest = split(sg, kw)
    cache(sg, a.c, **mine)
    base = dict(q=6 * P, k=7 * P, v=8 * P, q_out=9 * P, q_row=448, k_row=128, v_row=128, out_row=448, turns=10 * P, eps=1e-6,
                mscale=1.0, rot=64, NH=7, NKV=2, HD=64)
    for k, v in {**base, **rest}.items():
        setattr(a, k, v)
    return a


CACHE = [dict(R=-1), dict(B=-1), dict(pages=-1), dict(page=0), dict(table_pages=-1), dict(page=1 << 29), dict(len=None),
         dict(q_start=None), dict(len=4 * P + 2), dict(q_start=5 * P + 1), dict(k=None), dict(v=None), dict(table=None),
         dict(table=3 * P + 2), dict(page_stride=0), dict(page_stride=-2048), dict(kv_row=0), dict(kv_head=-64), dict(table_row=3),
         dict(page_stride=1 << 45)]


def ids(cases):
    return [",".join(f"{k}={v}" for k, v in c.items()) for c in cases]


APPEND = CACHE + [dict(_k=None), dict(_v=None), dict(_k=7 * P + 2), dict(k_row=127), dict(v_row=100), dict(q_out=None), dict(q_row=447),
                  dict(out_row=447), dict(q_out=6 * P, out_row=512), dict(NH=-1), dict(NKV=0), dict(HD=0), dict(rot=63), dict(rot=66),
                  dict(rot=-2), dict(turns=None), dict(turns=10 * P + 4), dict(pos=P + 2), dict(eps=-1.0), dict(eps=math.nan),
                  dict(eps=math.inf), dict(wq=P + 1), dict(wk=P + 2), dict(HD=512, rot=258, q_row=1 << 20, k_row=1 << 20),
                  dict(NH=1 << 17, q_row=1 << 30, out_row=1 << 30)]


@pytest.mark.parametrize("kw", APPEND, ids=ids(APPEND))
def test_kv_append_refuses(sg, kw):
    for fn in ("sgpu_kv_append", "sgpu_kv_append_h"):
        assert getattr(sg.lib(), fn)(ct.byref(append(sg, **kw)), None) == BAD


def test_kv_append_without_work(sg):
    L = sg.lib()
    assert L.sgpu_kv_append(None, None) == BAD and L.sgpu_kv_append_h(None, None) == BAD
    for kw in (dict(R=0), dict(B=0), dict(R=0, _k=None, len=None)):
        assert L.sgpu_kv_append(ct.byref(append(sg, **kw)), None) == 0
    assert L.sgpu_kv_append(ct.byref(append(sg, k=P + 2)), None) == BAD            # fp32 pages
    assert L.sgpu_kv_append_h(ct.byref(append(sg, k=P + 1)), None) == BAD


def tree(sg, **kw):
    a = sg.AttnTreeArgs()
    mine, rest = split(sg, kw)
    cache(sg, a.c, **mine)
    base = dict(q=6 * P, out=7 * P, q_row=448, q_head=64, out_row=448, out_head=64, mask=8 * P, mask_row=1, NH=14, NKV=2, HD=64,
                max_q=2, max_kv=60, scale=0.125)
    for k, v in {**base, **rest}.items():
        setattr(a, k, v)
    return a


TREE = CACHE + [dict(NH=0), dict(NKV=0), dict(NH=7), dict(HD=48), dict(HD=256), dict(max_q=-1), dict(max_kv=-1), dict(scale=math.nan),
                dict(scale=math.inf), dict(scale=-0.5), dict(q=None), dict(out=None), dict(q=6 * P + 4), dict(out=7 * P + 8),
                dict(q_row=450), dict(q_row=0), dict(q_head=66), dict(out_row=-448), dict(out_head=2), dict(mask=8 * P + 2),
                dict(mask_row=-1), dict(mask_row=(1 << 26) + 1), dict(k=P + 8), dict(v=2 * P + 4), dict(kv_row=130), dict(kv_head=66),
                dict(page_stride=2050), dict(R=1 << 23), dict(B=1 << 22)]


@pytest.mark.parametrize("kw", TREE, ids=ids(TREE))
def test_attn_tree_refuses(sg, kw):
    L = sg.lib()
    for fn in ("sgpu_attn_tree", "sgpu_attn_tree_h"):
        assert getattr(L, fn)(ct.byref(tree(sg, **kw)), 16 * P, 1 << 50, None) == BAD
    assert L.sgpu_attn_tree_workspace(ct.byref(tree(sg, **kw))) == 0


def test_attn_tree_workspace_and_no_work(sg):
    L = sg.lib()
    assert L.sgpu_attn_tree(None, None, 0, None) == BAD and L.sgpu_attn_tree_workspace(None) == 0
    for kw in (dict(R=0), dict(B=0), dict(R=0, q=None, out=None, len=None)):
        assert L.sgpu_attn_tree(ct.byref(tree(sg, **kw)), None, 0, None) == 0
        assert L.sgpu_attn_tree_workspace(ct.byref(tree(sg, **kw))) == 0
    # fp16 pages: whole 16 bytes are 8 values
    for kw in (dict(kv_row=132), dict(kv_head=68), dict(page_stride=2052)):
        assert L.sgpu_attn_tree_h(ct.byref(tree(sg, **kw)), 16 * P, 1 << 50, None) == BAD
    for kw in (dict(max_kv=4096, table_pages=300, table_row=300, pages=1000), dict(max_q=0, max_kv=0), dict(pages=0, k=None, v=None, table=None)):
        a = tree(sg, **kw)
        need = L.sgpu_attn_tree_workspace(ct.byref(a))
        assert need >= 16
        for ws, n in ((None, need), (16 * P + 8, need), (16 * P, need - 1)):
            assert L.sgpu_attn_tree(ct.byref(a), ws, n, None) == BAD


def logits(sg, **kw):
    a = sg.LogitsArgs()
    base = dict(x=P, y=2 * P, x_row=1000, y_row=1000, rows=3, V=1000, tok=3 * P, n_tok=10, span=4 * P, rep=5 * P, freq=6 * P, pres=7 * P,
                bias_id=8 * P, bias=9 * P, n_bias=4, bias_span=10 * P, allow=11 * P, allow_row=32)
    for k, v in {**base, **kw}.items():
        setattr(a, k, v)
    return a


LOGITS = [dict(rows=-1), dict(rows=1 << 24), dict(V=0), dict(V=(1 << 30) + 1), dict(n_tok=-1), dict(n_bias=-1), dict(x=None), dict(y=None),
          dict(x=P + 1), dict(y=2 * P + 1), dict(x_row=999), dict(y_row=999), dict(x=P, y=P, y_row=1001), dict(tok=None), dict(span=4 * P + 2),
          dict(tok=3 * P + 2), dict(rep=5 * P + 1), dict(freq=6 * P + 2), dict(pres=7 * P + 3), dict(bias_id=None), dict(bias=None),
          dict(bias_span=10 * P + 2), dict(bias_id=8 * P + 2), dict(bias=9 * P + 2), dict(allow=11 * P + 1), dict(allow_row=31),
          dict(allow_row=-32), dict(rows=1 << 23, V=1 << 30, x_row=1 << 30, y_row=1 << 30, allow_row=1 << 25)]


@pytest.mark.parametrize("kw", LOGITS, ids=ids(LOGITS))
def test_logits_adjust_refuses(sg, kw):
    for fn in ("sgpu_logits_adjust", "sgpu_logits_adjust_h"):
        assert getattr(sg.lib(), fn)(ct.byref(logits(sg, **kw)), None) == BAD


def test_logits_adjust_without_work(sg):
    L = sg.lib()
    assert L.sgpu_logits_adjust(None, None) == BAD and L.sgpu_logits_adjust_h(None, None) == BAD
    assert L.sgpu_logits_adjust(ct.byref(logits(sg, rows=0, x=None, y=None)), None) == 0
    assert L.sgpu_logits_adjust(ct.byref(logits(sg, x=P + 2)), None) == BAD        # fp32


def test_qk_norm_rope_refuses(sg):
    L = sg.lib()

    def call(fn="sgpu_qk_norm_rope", x=P, xs=1024, y=2 * P, ys=1024, wq=3 * P, wk=3 * P, eps=1e-6, pos=P, turns=P, rot=64, T=2, NH=14,
             NKV=2, HD=64):
        return getattr(L, fn)(x, xs, y, ys, wq, wk, eps, pos, 0, turns, rot, 0, 1.0, T, NH, NKV, HD, None)

    for kw in (dict(T=-1), dict(T=(1 << 30) + 1), dict(NH=-1), dict(NKV=-1), dict(HD=0), dict(rot=-2), dict(rot=3), dict(rot=66), dict(xs=1023),
               dict(ys=1023), dict(x=None), dict(y=None), dict(turns=None), dict(x=P + 2), dict(y=2 * P + 2), dict(pos=P + 2),
               dict(turns=P + 4), dict(wq=P + 2), dict(wk=P + 1), dict(eps=-1e-9), dict(eps=math.nan), dict(eps=math.inf),
               dict(x=P, y=P, ys=2048), dict(HD=512, rot=258, xs=1 << 20, ys=1 << 20), dict(NH=1 << 17, xs=1 << 30, ys=1 << 30)):
        assert call(**kw) == BAD, kw
    assert call(fn="sgpu_qk_norm_rope_h", y=2 * P + 1) == BAD
    assert call(fn="sgpu_qk_norm_rope_h", y=P) == BAD                              # not in place
    assert call(T=0, x=None, y=None) == 0
    assert call(NH=0, NKV=0, x=None, y=None) == 0

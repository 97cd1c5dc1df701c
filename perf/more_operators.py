"""The operators that serve several requests from one paged cache and check tokens drafted ahead, as a
host calls them through include/switch_gpu.h (bound by switch-l4t-gpu_amd/sgpu.py), beside their plain
forms.

Kinds of case and the use each stands for:
  qkn     sgpu_qk_norm_rope / _h: the q and k heads of projected rows, each head's norm and the
          rotation of its position in one pass
  append  sgpu_kv_append / _h: projected rows of a batch: keys rotated (and normed) on their way into
          the pages of a cache, values beside them, queries rotated into a buffer
  tree    sgpu_attn_tree / _h: attention of each sequence's new rows over its pages: single tokens,
          drafted tokens in a row, or trees of them of which a row sees its ancestors only
  logits  sgpu_logits_adjust / _h: penalties for repeated tokens, biases and a grammar's mask on logits

Sizes are those of the repository's own engines (Qwen2.5-0.5B, GPT-2 124M) and generic ones.
"""
import math
import os
import random
import sys

import torch

own = False

V_QWEN, V_GPT2 = 151936, 50257


def listed():
    return [
        # one decode position: the q and k heads of a single row
        {"name": "qkn_step", "op": "qkn", "T": 1, "NH": 14, "NKV": 2, "HD": 64, "rot": 64, "inter": False, "first": 700,
         "gap": 1, "out": "f32"},
        # a long prompt's rows far into its context, half of each head rotated in neighbouring pairs, to fp16
        {"name": "qkn_prompt", "op": "qkn", "T": 4099, "NH": 32, "NKV": 8, "HD": 128, "rot": 64, "inter": True,
         "first": 100000, "gap": 3, "out": "f16"},
        # one token of one request
        {"name": "append_step", "op": "append", "B": 1, "ctx": 700, "q": 1, "NH": 14, "NKV": 2, "HD": 64, "rot": 64,
         "inter": False, "norm": False, "page": 16, "tree": False, "kv": "f32"},
        # the drafted tokens of a batch of requests
        {"name": "append_drafts", "op": "append", "B": 64, "ctx": 2000, "q": 17, "NH": 14, "NKV": 2, "HD": 64, "rot": 64,
         "inter": False, "norm": False, "page": 16, "tree": True, "kv": "f16"},
        # parts of three prompts, with the heads' norms
        {"name": "append_prompt", "op": "append", "B": 3, "ctx": 500, "q": 2731, "NH": 32, "NKV": 8, "HD": 128, "rot": 128,
         "inter": False, "norm": True, "page": 64, "tree": False, "kv": "f16"},
        # one token of one request, as the engines decode
        {"name": "tree_step", "op": "tree", "B": 1, "ctx": 700, "q": 1, "NH": 14, "NKV": 2, "HD": 64, "page": 16,
         "tree": False, "kv": "f32"},
        # a batch of requests of ragged lengths, one token each
        {"name": "tree_batch", "op": "tree", "B": 64, "ctx": 4096, "q": 1, "NH": 14, "NKV": 2, "HD": 64, "page": 16,
         "tree": False, "kv": "f16"},
        # trees of drafted tokens checked for a batch
        {"name": "tree_drafts", "op": "tree", "B": 32, "ctx": 3001, "q": 24, "NH": 14, "NKV": 2, "HD": 64, "page": 64,
         "tree": True, "kv": "f32"},
        # a few tokens drafted in a row behind two long contexts
        {"name": "tree_long", "op": "tree", "B": 2, "ctx": 50001, "q": 7, "NH": 32, "NKV": 8, "HD": 128, "page": 128,
         "tree": False, "kv": "f16"},
        # one sampled position, penalties only
        {"name": "logits_step", "op": "logits", "rows": 1, "V": V_QWEN, "prompt": 700, "out": 130, "share": 1, "bias": 0,
         "allow": 0.0, "x": "f32"},
        # the rows of four drafted trees, with a few biases and a grammar that allows half
        {"name": "logits_tree", "op": "logits", "rows": 68, "V": V_GPT2, "prompt": 300, "out": 500, "share": 17, "bias": 32,
         "allow": 0.5, "x": "f32"},
        # a large batch under a narrow grammar
        {"name": "logits_batch", "op": "logits", "rows": 512, "V": V_QWEN, "prompt": 2000, "out": 1000, "share": 1,
         "bias": 300, "allow": 0.02, "x": "f16"},
    ]


# The largest drawn costs: no drawn case costs more than the largest listed one of its kind.
QKN_VALUES = 4099 * 40 * 128
APPEND_VALUES = 3 * 2048 * 48 * 128
TREE_FLOPS, TREE_BYTES, TREE_SCORES = 7.8e9, 311e6, 1 << 26
LOGITS_VALUES = 512 * V_QWEN
_HEADS = [(14, 2, 64), (14, 2, 64), (12, 12, 64), (32, 8, 128), (8, 1, 64), (6, 2, 32), (9, 3, 128)]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["qkn", "append", "append", "tree", "tree", "tree", "logits", "logits"])
    while op == "qkn":
        HD = rng.choice([32, 64, 64, 80, 96, 128, 128, 256])
        NKV = _log(rng, 1, 16)
        c = {"op": op, "T": _log(rng, 1, 16384), "NH": NKV * rng.choice([1, 2, 4, 7]), "NKV": NKV, "HD": HD,
             "rot": rng.choice([HD, HD, HD // 2, HD // 4, 2 * rng.randint(1, HD // 2)]), "inter": rng.random() < 0.5,
             "first": _log(rng, 1, 500000), "gap": rng.randint(1, 7), "out": rng.choice(["f32", "f32", "f16"])}
        if c["T"] * (c["NH"] + NKV) * HD <= QKN_VALUES:
            return c
    page = rng.choice([16, 16, 32, 64, 128, 256, 8, 1, 24, 100])
    while op == "append":
        NH, NKV, HD = rng.choice(_HEADS)
        q = rng.choice([1, 1, _log(rng, 2, 64), _log(rng, 2, 4096)])
        c = {"op": op, "B": _log(rng, 1, 128), "ctx": _log(rng, 1, 4096), "q": q, "NH": NH, "NKV": NKV, "HD": HD,
             "rot": rng.choice([HD, HD, HD // 2]), "inter": rng.random() < 0.3, "norm": rng.random() < 0.4, "page": page,
             "tree": 1 < q <= 64 and rng.random() < 0.7, "kv": rng.choice(["f32", "f16"])}
        if c["B"] * q * (NH + 2 * NKV) * HD <= APPEND_VALUES and c["B"] * (c["ctx"] + q) * NKV * HD <= 1 << 27:
            return c
    while op == "tree":
        NH, NKV, HD = rng.choice(_HEADS)
        q = rng.choice([1, 1, _log(rng, 2, 8), _log(rng, 2, 64), _log(rng, 2, 64)])
        c = {"op": op, "B": _log(rng, 1, 128), "ctx": _log(rng, 1, 60000), "q": q, "NH": NH, "NKV": NKV, "HD": HD,
             "page": page, "tree": q > 1 and rng.random() < 0.7, "kv": rng.choice(["f32", "f16"])}
        w = work(c)
        if w["flops"] <= TREE_FLOPS and w["bytes"] <= TREE_BYTES and c["B"] * q * NH * (c["ctx"] + q) <= TREE_SCORES:
            return c
    while True:
        rows = _log(rng, 1, 1500)
        c = {"op": "logits", "rows": rows, "V": rng.choice([V_QWEN, V_GPT2, _log(rng, 100, 262144), _log(rng, 100, 262144)]),
             "prompt": rng.choice([0, _log(rng, 1, 8192), _log(rng, 1, 2048)]), "out": rng.choice([0, _log(rng, 1, 2048)]),
             "share": rng.choice([1, 1, 5, 24]), "bias": rng.choice([0, 0, 1, 32, 300]),
             "allow": rng.choice([0.0, 0.0, 0.001, 0.3, 0.97]), "x": rng.choice(["f32", "f32", "f16"])}
        if rows * c["V"] <= LOGITS_VALUES and c["bias"] <= c["V"]:
            return c


# ---- inputs ----
def _rng(seed, salt):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 1000003 + salt)


def _normal(shape, g, std=1.0):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).mul_(std)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _lengths(case):
    """(tokens in the cache, new rows) of each sequence: ragged, the first the longest."""
    r = random.Random(case["B"] * 7919 + case["q"] * 31 + case["ctx"])
    n = [case["q"] if b == 0 else r.randint((case["q"] + 1) // 2, case["q"]) for b in range(case["B"])]
    c = [case["ctx"] if b == 0 else r.randint((case["ctx"] + 3) // 4, case["ctx"]) for b in range(case["B"])]
    return c, n


def _trees(case, seed):
    """(depth, bits of the rows it sees: its ancestors and itself) of each new row."""
    r = random.Random(seed * 7 + 5)
    out = []
    for n in _lengths(case)[1]:
        depth, seen = [0], [1]
        for i in range(1, n):
            up = r.randint(max(0, i - 8), i - 1) if case["tree"] else i - 1
            depth.append(depth[up] + 1)
            seen.append(seen[up] | 1 << i)
        out += list(zip(depth, seen))
    return out


def _frequencies(rot):
    return [1e6 ** (-2.0 * i / rot) for i in range(rot // 2)]


def _paged(case, g):
    """A cache of pages in any order, and where each sequence's lie."""
    c, n = _lengths(case)
    page, NKV, HD = case["page"], case["NKV"], case["HD"]
    need = [(a + b + page - 1) // page for a, b in zip(c, n)]
    pages, most = sum(need) + 3, max(need)
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.full((case["B"], most), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, m in enumerate(need):
        table[b, :m] = order[at:at + m]
        at += m
    starts = [0]
    for m in n:
        starts.append(starts[-1] + m)
    size = torch.float16 if case["kv"] == "f16" else torch.float32
    k, v = (torch.randn((pages, page, NKV, HD), generator=g, device="cuda", dtype=size) for _ in range(2))
    return {"k": k, "v": v, "table": table, "len": _ints(c), "q_start": _ints(starts), "R": starts[-1], "pages": pages}


def _qkn_inputs(case, seed):
    g = _rng(seed, 1)
    T, n = case["T"], (case["NH"] + case["NKV"]) * case["HD"]
    x = _normal((T, n + case["NKV"] * case["HD"]), g, 3.0)      # values behind them, left alone
    return {"x": x[:, :n], "pos": case["first"] + case["gap"] * torch.arange(T, dtype=torch.int32, device="cuda"),
            "wq": 1.0 + _normal((case["HD"],), g, 0.2), "wk": 1.0 + _normal((case["HD"],), g, 0.2)}


def _append_inputs(case, seed):
    g = _rng(seed, 2)
    NH, NKV, HD = case["NH"], case["NKV"], case["HD"]
    s = _paged(case, g)
    rows = _normal((s["R"], (NH + 2 * NKV) * HD), g, 2.0)       # q, k, v side by side, as one projection left them
    c, n = _lengths(case)
    depth = [d for d, _ in _trees(case, seed)] if case["tree"] else [i for m in n for i in range(m)]
    at = [a for a, m in zip(c, n) for _ in range(m)]
    s.update(rows=rows, pos=_ints([a + d for a, d in zip(at, depth)]), wq=1.0 + _normal((HD,), g, 0.2),
             wk=1.0 + _normal((HD,), g, 0.2))
    return s


def _tree_inputs(case, seed):
    g = _rng(seed, 3)
    s = _paged(case, g)
    s["q"] = _normal((s["R"], case["NH"] * case["HD"]), g, 1.5)
    words = (case["q"] + 31) // 32
    s["mask"] = None
    if case["tree"]:
        bits = [[(m >> 32 * w) & 0xFFFFFFFF for w in range(words)] for _, m in _trees(case, seed)]
        s["mask"] = torch.tensor(bits, dtype=torch.int64).to(torch.int32).cuda()
    return s


def _logits_inputs(case, seed):
    g = _rng(seed, 4)
    rows, V = case["rows"], case["V"]
    x = _normal((rows, V), g, 3.0)
    r = random.Random(rows * 31 + case["out"])
    sets = (rows + case["share"] - 1) // case["share"]
    pn = [case["prompt"] if i == 0 else r.randint((case["prompt"] + 1) // 2, case["prompt"]) for i in range(sets)]
    on = [case["out"] if i == 0 else r.randint((case["out"] + 1) // 2, case["out"]) for i in range(rows)]
    starts = [0]
    for m in pn + on:
        starts.append(starts[-1] + m)
    span = [[starts[i // case["share"]], pn[i // case["share"]], starts[sets + i], on[i]] for i in range(rows)]
    # mostly frequent tokens, as texts have them
    tok = (torch.rand((max(starts[-1], 1),), generator=g, device="cuda", dtype=torch.float64) ** 3 * V).to(torch.int32)
    s = {"tok": tok, "n_tok": starts[-1], "span": _ints(span), "rep": 1.0 + 0.5 * torch.rand((rows,), generator=g, device="cuda"),
         "freq": 0.3 * torch.rand((rows,), generator=g, device="cuda"), "pres": torch.rand((rows,), generator=g, device="cuda"),
         "bias_id": None, "bias": None, "allow": None}
    if case["bias"]:
        step = max(1, V // case["bias"])                        # other tokens in each row, none twice
        at = torch.arange(case["bias"], device="cuda")[None] * step + torch.arange(rows, device="cuda")[:, None] % step
        s["bias_id"], s["bias"] = at.to(torch.int32), _normal((rows, case["bias"]), g, 5.0)
        s["bias_span"] = _ints([[i * case["bias"], case["bias"]] for i in range(rows)])
    if case["allow"]:
        words = (V + 31) // 32
        allow = torch.zeros((rows, words), dtype=torch.int64, device="cuda")
        for b in range(32):
            allow |= (torch.rand((rows, words), generator=g, device="cuda") < case["allow"]).long() << b
        s["allow"] = allow.to(torch.int32)
    s["x"] = x.half() if case["x"] == "f16" else x
    return s


_INPUTS = {"qkn": _qkn_inputs, "append": _append_inputs, "tree": _tree_inputs, "logits": _logits_inputs}


def prepare(case, seed):
    state = {"case": case, **_INPUTS[case["op"]](case, seed)}
    if case["op"] in ("qkn", "append"):
        state["freq"] = torch.tensor(_frequencies(case["rot"]), dtype=torch.float64, device="cuda")
    if case["op"] == "qkn":
        state["y"] = torch.empty(state["x"].shape, device="cuda", dtype=torch.float16 if case["out"] == "f16" else torch.float32)
    elif case["op"] in ("append", "tree"):
        state["out"] = torch.empty((state["R"], case["NH"] * case["HD"]), device="cuda")
    else:
        state["y"] = torch.empty_like(state["x"])
    return state


# ---- the framework's calls ----
_bound = None


def _sgpu():
    global _bound
    if _bound is None:
        sys.path.insert(0, os.path.join(os.getcwd(), "switch-l4t-gpu_amd"))
        import sgpu

        sgpu.init(0)
        _bound = sgpu
    return _bound


def _turns(s, case):
    if "turns" not in s:                                        # the table that a host uploads once
        s["turns"] = torch.from_numpy(_sgpu().rope_turns(case["rot"], 1e6)[0]).cuda()
    return s["turns"].data_ptr()


def _workspace(state, nbytes):
    """The caller's workspace of one call site, kept with its buffers."""
    if state.get("ws") is None or state["ws"].numel() < nbytes:
        state["ws"] = torch.empty((max(nbytes, 1),), dtype=torch.uint8, device="cuda")
    return state["ws"].data_ptr()


def _cache(s, case, c):
    c.k, c.v, c.table, c.len, c.q_start = (s[n].data_ptr() for n in ("k", "v", "table", "len", "q_start"))
    c.page_stride, c.kv_row, c.kv_head = s["k"].stride(0), s["k"].stride(1), s["k"].stride(2)
    c.pages, c.page, c.table_row, c.table_pages = s["pages"], case["page"], s["table"].stride(0), s["table"].shape[1]
    c.R, c.B = s["R"], case["B"]


def _own_qkn(s, case):
    _sgpu().call("sgpu_qk_norm_rope_h" if case["out"] == "f16" else "sgpu_qk_norm_rope", s["x"].data_ptr(), s["x"].stride(0),
                 s["y"].data_ptr(), s["y"].stride(0), s["wq"].data_ptr(), s["wk"].data_ptr(), 1e-6, s["pos"].data_ptr(), 0,
                 _turns(s, case), case["rot"], int(case["inter"]), 1.0, case["T"], case["NH"], case["NKV"], case["HD"],
                 torch.cuda.current_stream().cuda_stream)
    return s["y"]


def _own_append(s, case):
    sgpu = _sgpu()
    if "args" not in s:                                         # the description of its buffers that a host keeps
        a = s["args"] = sgpu.KvAppendArgs()
        _cache(s, case, a.c)
        NH, NKV, HD = case["NH"], case["NKV"], case["HD"]
        a.q, a.q_out, a.pos, a.turns = s["rows"].data_ptr(), s["out"].data_ptr(), s["pos"].data_ptr(), _turns(s, case)
        a.k, a.v = a.q + 4 * NH * HD, a.q + 4 * (NH + NKV) * HD
        a.q_row = a.k_row = a.v_row = s["rows"].stride(0)
        a.out_row = s["out"].stride(0)
        if case["norm"]:
            a.wq, a.wk = s["wq"].data_ptr(), s["wk"].data_ptr()
        a.eps, a.mscale, a.rot, a.neighbours, a.NH, a.NKV, a.HD = 1e-6, 1.0, case["rot"], int(case["inter"]), NH, NKV, HD
    sgpu.call("sgpu_kv_append_h" if case["kv"] == "f16" else "sgpu_kv_append", sgpu.byref(s["args"]),
              torch.cuda.current_stream().cuda_stream)
    return {"q": s["out"], "k": s["k"], "v": s["v"]}


def _own_tree(s, case):
    sgpu = _sgpu()
    if "args" not in s:
        a = s["args"] = sgpu.AttnTreeArgs()
        _cache(s, case, a.c)
        a.q, a.out = s["q"].data_ptr(), s["out"].data_ptr()
        a.q_row, a.out_row, a.q_head, a.out_head = s["q"].stride(0), s["out"].stride(0), case["HD"], case["HD"]
        if s["mask"] is not None:
            a.mask, a.mask_row = s["mask"].data_ptr(), s["mask"].stride(0)
        a.NH, a.NKV, a.HD, a.scale = case["NH"], case["NKV"], case["HD"], 1.0 / math.sqrt(case["HD"])
        a.max_q, a.max_kv = case["q"], case["ctx"] + case["q"]
        s["need"] = sgpu.lib().sgpu_attn_tree_workspace(sgpu.byref(a))
    sgpu.call("sgpu_attn_tree_h" if case["kv"] == "f16" else "sgpu_attn_tree", sgpu.byref(s["args"]),
              _workspace(s, s["need"]), s["need"], torch.cuda.current_stream().cuda_stream)
    return s["out"]


def _own_logits(s, case):
    sgpu = _sgpu()
    if "args" not in s:
        a = s["args"] = sgpu.LogitsArgs()
        a.x, a.y, a.x_row, a.y_row = s["x"].data_ptr(), s["y"].data_ptr(), s["x"].stride(0), s["y"].stride(0)
        a.rows, a.V, a.tok, a.n_tok, a.span = case["rows"], case["V"], s["tok"].data_ptr(), s["n_tok"], s["span"].data_ptr()
        a.rep, a.freq, a.pres = (s[n].data_ptr() for n in ("rep", "freq", "pres"))
        if s["bias"] is not None:
            a.bias_id, a.bias, a.n_bias = s["bias_id"].data_ptr(), s["bias"].data_ptr(), s["bias"].numel()
            a.bias_span = s["bias_span"].data_ptr()
        if s["allow"] is not None:
            a.allow, a.allow_row = s["allow"].data_ptr(), s["allow"].stride(0)
    sgpu.call("sgpu_logits_adjust_h" if case["x"] == "f16" else "sgpu_logits_adjust", sgpu.byref(s["args"]),
              torch.cuda.current_stream().cuda_stream)
    return s["y"]


# ---- the plain forms ----
def _norm(x, w):
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w


def _rotate(x, pos, freq, rot, inter):
    """Heads x[row, head, HD] turned by their rows' positions."""
    turn = pos.double()[:, None] * freq
    c, d = torch.cos(turn).float()[:, None, :], torch.sin(turn).float()[:, None, :]
    if inter:
        a, b = x[:, :, 0:rot:2], x[:, :, 1:rot:2]
        r = torch.stack((a * c - b * d, a * d + b * c), 3).reshape(x.shape[0], x.shape[1], rot)
    else:
        a, b = x[:, :, :rot // 2], x[:, :, rot // 2:rot]
        r = torch.cat((a * c - b * d, a * d + b * c), 2)
    return torch.cat((r, x[:, :, rot:]), 2)


def _plain_qkn(s, case):
    NH, HD = case["NH"], case["HD"]
    x = s["x"].reshape(case["T"], -1, HD)
    x = torch.cat((_norm(x[:, :NH], s["wq"]), _norm(x[:, NH:], s["wk"])), 1)
    return _rotate(x, s["pos"], s["freq"], case["rot"], case["inter"]).reshape(case["T"], -1).to(s["y"].dtype)


def _places(s, case):
    """Of each new row: its sequence and its number there."""
    start = s["q_start"].long()
    r = torch.arange(s["R"], device="cuda")
    b = (r[:, None] >= start[None, 1:]).sum(1)
    return b, r - start[b]


def _plain_append(s, case):
    NH, NKV, HD, R, page = case["NH"], case["NKV"], case["HD"], s["R"], case["page"]
    x = s["rows"].reshape(R, NH + 2 * NKV, HD)
    q, k, v = x[:, :NH], x[:, NH:NH + NKV], x[:, NH + NKV:]
    if case["norm"]:
        q, k = _norm(q, s["wq"]), _norm(k, s["wk"])
    q, k = (_rotate(t, s["pos"], s["freq"], case["rot"], case["inter"]) for t in (q, k))
    b, i = _places(s, case)
    at = s["len"].long()[b] + i
    to = s["table"].long()[b, at // page], at % page
    s["k"][to] = k.to(s["k"].dtype)
    s["v"][to] = v.to(s["v"].dtype)
    s["out"].copy_(q.reshape(R, NH * HD))
    return {"q": s["out"], "k": s["k"], "v": s["v"]}


def _plain_tree(s, case):
    NH, NKV, HD, R, B, page = case["NH"], case["NKV"], case["HD"], s["R"], case["B"], case["page"]
    G, nq, nk = NH // NKV, case["q"], case["ctx"] + case["q"]
    start, have = s["q_start"].long(), s["len"].long()
    n = start[1:] - start[:-1]
    i, j = torch.arange(nq, device="cuda"), torch.arange(nk, device="cuda")
    rows = (start[:-1, None] + torch.minimum(i, n[:, None] - 1))                        # padded to the longest
    keys = torch.minimum(j, (have + n)[:, None] - 1)
    to = s["table"].long().gather(1, keys // page), keys % page
    k = s["k"][to].float().permute(0, 2, 3, 1).reshape(B * NKV, HD, nk).contiguous()
    v = s["v"][to].float().permute(0, 2, 1, 3).reshape(B * NKV, nk, HD).contiguous()
    q = s["q"].reshape(R, NKV, G, HD)[rows].permute(0, 2, 1, 3, 4).reshape(B * NKV, nq * G, HD) * (1.0 / math.sqrt(HD))
    d = (j[None] - have[:, None])[:, None, :].expand(B, nq, nk)                         # number of a new key, negative: cached
    if s["mask"] is None:
        seen = d <= i[None, :, None]
    else:
        e = d.clamp(0, nq - 1)
        seen = (d < 0) | ((s["mask"][rows].gather(2, e // 32) >> (e % 32).int()) & 1).bool()
    seen = seen & (d < n[:, None, None])
    w = torch.bmm(q, k).reshape(B, NKV, nq, G, nk).masked_fill(~seen[:, None, :, None, :], -math.inf)
    w = torch.exp(w - w.amax(4, keepdim=True))
    w = w / w.sum(4, keepdim=True)
    o = torch.bmm(w.reshape(B * NKV, nq * G, nk), v).reshape(B, NKV, nq, G, HD).permute(0, 2, 1, 3, 4)
    return o[_places(s, case)].reshape(R, NH * HD)


def _counts(s, case, first, most):
    """How often each token is in the rows' spans."""
    out = torch.zeros((case["rows"], case["V"]), device="cuda")
    if most:
        j, span = torch.arange(most, device="cuda"), s["span"].long()
        inside = j < span[:, first + 1:first + 2]
        ids = s["tok"].long()[(span[:, first:first + 1] + j).clamp(max=s["n_tok"] - 1)]
        out.scatter_add_(1, ids, inside.float())
    return out


def _plain_logits(s, case):
    x = s["x"].float()
    out = _counts(s, case, 2, case["out"])
    seen = (_counts(s, case, 0, case["prompt"]) > 0) | (out > 0)
    rep, freq, pres = (s[n][:, None] for n in ("rep", "freq", "pres"))
    y = torch.where(seen, torch.where(x > 0, x / rep, x * rep), x) - freq * out - pres * (out > 0)
    if s["bias"] is not None:
        y.scatter_add_(1, s["bias_id"].long(), s["bias"])
    if s["allow"] is not None:
        v = torch.arange(case["V"], device="cuda")
        y.masked_fill_(((s["allow"][:, v // 32] >> (v % 32).int()) & 1) == 0, -math.inf)
    return y.to(s["y"].dtype)


def run(state):
    case = state["case"]
    if own:
        return {"qkn": _own_qkn, "append": _own_append, "tree": _own_tree, "logits": _own_logits}[case["op"]](state, case)
    return {"qkn": _plain_qkn, "append": _plain_append, "tree": _plain_tree, "logits": _plain_logits}[case["op"]](state, case)


# ---- work ----
def work(case):
    if case["op"] == "qkn":
        T, H, HD = case["T"], case["NH"] + case["NKV"], case["HD"]
        return {"bytes": T * H * HD * (4 + (2 if case["out"] == "f16" else 4)) + 4 * T, "flops": T * H * (4 * HD + 3 * case["rot"])}
    if case["op"] == "logits":
        rows, V = case["rows"], case["V"]
        size = 2 if case["x"] == "f16" else 4
        per = 2 * size * V + 4 * case["out"] + 8 * case["bias"] + (V // 8 if case["allow"] else 0) + 28
        return {"bytes": rows * per + 4 * case["prompt"] * ((rows + case["share"] - 1) // case["share"]), "flops": rows * V}
    c, n = _lengths(case)
    NH, NKV, HD, R = case["NH"], case["NKV"], case["HD"], sum(n)
    size = 2 if case["kv"] == "f16" else 4
    if case["op"] == "append":
        return {"bytes": R * HD * (8 * NH + 2 * NKV * (4 + size)) + 8 * R, "flops": R * (NH + NKV) * (3 * case["rot"] + (4 * HD if case["norm"] else 0))}
    # of a tree a row sees about half of the rows before it at most: counted as a chain
    seen = sum(a * b + a * (a + 1) // 2 for a, b in zip(n, c))
    return {"bytes": 2 * size * NKV * HD * (sum(c) + R) + 8 * R * NH * HD, "flops": 4 * HD * NH * seen}


# ---- the same in 64 bits ----
def _exact_heads(z, w, pos, case):
    """Heads in 64 bits: the norm, then each pair as one complex number, turned by a unit one."""
    z = z.double()
    if w is not None:
        z = z / torch.sqrt((z ** 2).sum(2, keepdim=True) / case["HD"] + 1e-6) * w.double()
    rot, half = case["rot"], case["rot"] // 2
    first = torch.arange(half, device="cuda") * 2 if case["inter"] else torch.arange(half, device="cuda")
    second = first + (1 if case["inter"] else half)
    angle = pos.double()[:, None] * torch.tensor(_frequencies(rot), dtype=torch.float64, device="cuda")[None]
    t = torch.complex(z[:, :, first], z[:, :, second]) * torch.polar(torch.ones_like(angle), angle)[:, None]
    out = z.clone()
    out[:, :, first], out[:, :, second] = t.real, t.imag
    return out


def _exact_qkn(case, seed):
    s = _qkn_inputs(case, seed)
    NH = case["NH"]
    x = s["x"].reshape(case["T"], -1, case["HD"])
    return torch.cat((_exact_heads(x[:, :NH], s["wq"], s["pos"], case), _exact_heads(x[:, NH:], s["wk"], s["pos"], case)),
                     1).reshape(case["T"], -1)


def _exact_append(case, seed):
    s = _append_inputs(case, seed)
    NH, NKV, HD, page = case["NH"], case["NKV"], case["HD"], case["page"]
    x = s["rows"].reshape(s["R"], NH + 2 * NKV, HD)
    wq, wk = (s["wq"], s["wk"]) if case["norm"] else (None, None)
    q, k = _exact_heads(x[:, :NH], wq, s["pos"], case), _exact_heads(x[:, NH:NH + NKV], wk, s["pos"], case)
    K, V = s["k"].double(), s["v"].double()
    c, n = _lengths(case)
    r0 = 0
    for b in range(case["B"]):
        at = torch.arange(c[b], c[b] + n[b], device="cuda")
        flat = s["table"][b].long()[at // page] * page + at % page
        K.view(-1, NKV, HD)[flat] = k[r0:r0 + n[b]]
        V.view(-1, NKV, HD)[flat] = x[r0:r0 + n[b], NH + NKV:].double()
        r0 += n[b]
    return {"q": q.reshape(s["R"], -1), "k": K, "v": V}


def _exact_tree(case, seed):
    s = _tree_inputs(case, seed)
    c, n = _lengths(case)
    NH, NKV, HD, page = case["NH"], case["NKV"], case["HD"], case["page"]
    G = NH // NKV
    seen_bits = _trees(case, seed) if case["tree"] else None
    out = torch.empty((s["R"], NKV, G, HD), dtype=torch.float64, device="cuda")
    K, V = s["k"].view(-1, NKV, HD), s["v"].view(-1, NKV, HD)
    r0 = 0
    for b in range(case["B"]):
        nb, N = n[b], c[b] + n[b]
        at = torch.arange(N, device="cuda")
        flat = s["table"][b].long()[at // page] * page + at % page
        if seen_bits:
            own_rows = torch.tensor([[bool(m >> j & 1) for j in range(nb)] for _, m in seen_bits[r0:r0 + nb]], device="cuda")
        else:
            own_rows = torch.ones((nb, nb), dtype=torch.bool, device="cuda").tril()
        see = torch.cat((torch.ones((nb, c[b]), dtype=torch.bool, device="cuda"), own_rows), 1)
        Q = s["q"][r0:r0 + nb].double().reshape(nb, NKV, G, HD)
        for g in range(NKV):
            k = K[flat, g].double().t().contiguous()
            w = (Q[:, g].reshape(nb * G, HD) @ k / math.sqrt(HD)).reshape(nb, G, N).masked_fill(~see[:, None], -math.inf)
            out[r0:r0 + nb, g] = (torch.softmax(w, 2).reshape(nb * G, N) @ V[flat, g].double()).reshape(nb, G, HD)
        r0 += nb
    return out.reshape(s["R"], NH * HD)


def _exact_logits(case, seed):
    s = _logits_inputs(case, seed)
    V, out = case["V"], torch.empty((case["rows"], case["V"]), dtype=torch.float64, device="cuda")
    span = s["span"].tolist()
    for r, (p0, pn, o0, on) in enumerate(span):
        y = s["x"][r].double()
        said = torch.bincount(s["tok"][o0:o0 + on].long(), minlength=V).double()
        seen = (torch.bincount(s["tok"][p0:p0 + pn].long(), minlength=V) + said) > 0
        rep, freq, pres = (s[n][r].double() for n in ("rep", "freq", "pres"))
        y = torch.where(seen, y * torch.where(y > 0, 1.0 / rep, rep), y)
        y = y - said * freq - torch.where(said > 0, pres, 0.0)
        if s["bias"] is not None:
            y[s["bias_id"][r].long()] += s["bias"][r].double()
        if s["allow"] is not None:
            words = s["allow"][r].long() & 0xFFFFFFFF
            y[((words[:, None] >> torch.arange(32, device="cuda")) & 1).reshape(-1)[:V] == 0] = -math.inf
        out[r] = y
    return out


def exact(case, seed):
    return {"qkn": _exact_qkn, "append": _exact_append, "tree": _exact_tree, "logits": _exact_logits}[case["op"]](case, seed)

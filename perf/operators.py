"""The operators that score and sample several continuations of one prompt, as a host calls them
through include/switch_gpu.h (bound by switch-l4t-gpu_amd/sgpu.py), beside their plain forms.

Kinds of case and the use each stands for:
  rope    sgpu_rope_rows / _h: the q and k heads of projected rows rotated at their positions,
          into another buffer (a query buffer, a cache): both pairings, part of the head,
          tables scaled for long contexts
  logp    sgpu_logprobs / _h: log probabilities of given tokens, the entropy of each row and its
          top alternatives, from logits
  attn    sgpu_attn_prefix / _h: attention of a batch whose sequences share a long prefix: one
          cache of the prefix, and each sequence's own rows after it (in slots of a cache, or
          packed as the projections left them)

Sizes are those of the repository's own engines (Qwen2.5-0.5B, GPT-2 124M) and generic ones.
"""
import math
import os
import random
import sys

import torch

own = False

V_QWEN, V_GPT2 = 151936, 50257

# The largest drawn costs: no drawn case costs more than the largest listed one of its kind.
ROPE_VALUES = 3001 * 40 * 128
LOGP_VALUES = 1024 * V_QWEN
ATTN_FLOPS = 26.4e9


def listed():
    return [
        # one decode position: the q and k heads of a single row
        {"name": "rope_step", "op": "rope", "T": 1, "H": 16, "HD": 64, "rot": 64, "inter": False, "scaling": "none",
         "theta": 1e6, "factor": 1.0, "first": 700, "gap": 1, "out": "f32"},
        # a prompt's rows, ragged length
        {"name": "rope_prompt", "op": "rope", "T": 3001, "H": 16, "HD": 64, "rot": 64, "inter": False, "scaling": "none",
         "theta": 1e6, "factor": 1.0, "first": 0, "gap": 1, "out": "f32"},
        # rows far into a long context, half of each head rotated in neighbouring pairs, to an fp16 cache
        {"name": "rope_far", "op": "rope", "T": 3001, "H": 40, "HD": 128, "rot": 64, "inter": True, "scaling": "yarn",
         "theta": 1e4, "factor": 16.0, "first": 100000, "gap": 3, "out": "f16"},
        # one sampled position: its token's log probability and 20 alternatives
        {"name": "logp_step", "op": "logp", "rows": 1, "V": V_QWEN, "nt": 1, "k": 20, "x": "f32", "masked": 0.0},
        # a batch of sampled positions
        {"name": "logp_batch", "op": "logp", "rows": 64, "V": V_QWEN, "nt": 1, "k": 5, "x": "f32", "masked": 0.0},
        # a scored text: rows of odd length
        {"name": "logp_text", "op": "logp", "rows": 2048, "V": V_GPT2, "nt": 1, "k": 1, "x": "f32", "masked": 0.0},
        # answers scored under a grammar that forbids half of the vocabulary, fp16 logits
        {"name": "logp_masked_h", "op": "logp", "rows": 1024, "V": V_QWEN, "nt": 4, "k": 8, "x": "f16", "masked": 0.5},
        # a few samples of a short prompt, one new row each
        {"name": "attn_small", "op": "attn", "B": 4, "P": 500, "q": 1, "hist": 30, "NH": 14, "NKV": 2, "HD": 64, "kv": "f32"},
        # many samples of a long prompt, one new row each
        {"name": "attn_samples", "op": "attn", "B": 64, "P": 7601, "q": 1, "hist": 500, "NH": 14, "NKV": 2, "HD": 64,
         "kv": "f32"},
        # samples of a long document from an fp16 cache
        {"name": "attn_document_h", "op": "attn", "B": 48, "P": 32768, "q": 1, "hist": 200, "NH": 32, "NKV": 8, "HD": 128,
         "kv": "f16"},
        # answers of up to 64 tokens scored after one question
        {"name": "attn_answers", "op": "attn", "B": 48, "P": 3001, "q": 64, "hist": 0, "NH": 14, "NKV": 2, "HD": 64,
         "kv": "f32"},
        # a few tokens a sequence at once, every head with keys of its own
        {"name": "attn_heads", "op": "attn", "B": 16, "P": 1000, "q": 8, "hist": 24, "NH": 12, "NKV": 12, "HD": 64,
         "kv": "f32"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope", "logp", "logp", "attn", "attn", "attn"])
    while op == "rope":
        HD = rng.choice([32, 64, 64, 80, 96, 128, 128, 256])
        rot = rng.choice([HD, HD, HD // 2, HD // 4, 2 * rng.randint(1, HD // 2)])
        c = {"op": op, "T": _log(rng, 1, 16384), "H": _log(rng, 1, 48), "HD": HD, "rot": rot, "inter": rng.random() < 0.5,
             "scaling": rng.choice(["none", "none", "linear", "base", "bands", "yarn"]), "theta": rng.choice([1e4, 5e5, 1e6]),
             "factor": rng.choice([2.0, 4.0, 8.0, 32.0]), "first": _log(rng, 1, 500000), "gap": rng.randint(1, 7),
             "out": rng.choice(["f32", "f32", "f16"])}
        if c["T"] * c["H"] * HD <= ROPE_VALUES:
            return c
    while op == "logp":
        c = {"op": op, "rows": _log(rng, 1, 3000), "V": rng.choice([V_QWEN, V_GPT2, _log(rng, 100, 262144), _log(rng, 100, 262144)]),
             "nt": rng.choice([0, 1, 1, 1, 4, 17]), "k": rng.choice([0, 1, 2, 5, 10, 20, 33, 64]), "x": rng.choice(["f32", "f32", "f16"]),
             "masked": rng.choice([0.0, 0.0, 0.3, 0.9])}
        if c["rows"] * c["V"] <= LOGP_VALUES:
            return c
    while True:
        NH, NKV, HD = rng.choice([(14, 2, 64), (14, 2, 64), (12, 12, 64), (32, 8, 128), (8, 1, 64), (6, 2, 32), (9, 3, 128)])
        q = rng.choice([1, 1, 1, _log(rng, 2, 100), _log(rng, 2, 100)])
        c = {"op": "attn", "B": _log(rng, 1, 128), "P": _log(rng, 1, 32768), "q": q,
             "hist": rng.choice([0, _log(rng, 1, 1000)]), "NH": NH, "NKV": NKV, "HD": HD, "kv": rng.choice(["f32", "f32", "f16"])}
        if work(c)["flops"] <= ATTN_FLOPS and c["B"] * q * NH * (c["P"] + q + c["hist"]) <= 1 << 28:
            return c


# ---- inputs ----
def _rng(seed, salt):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 1000003 + salt)


def _normal(shape, g, std=1.0):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).mul_(std)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _lengths(case):
    """(query rows, earlier rows of its own) of each sequence: ragged, the first the longest."""
    r = random.Random(case["B"] * 7919 + case["q"])
    q = [case["q"] if b == 0 else r.randint((case["q"] + 1) // 2, case["q"]) for b in range(case["B"])]
    h = [case["hist"] if b == 0 else r.randint(0, case["hist"]) for b in range(case["B"])]
    return q, h


def _frequencies(case):
    """Radians per position of each pair of a head, and the factor on the rotated values."""
    rot, theta, factor = case["rot"], case["theta"], case["factor"]
    ctx, low, high, fast, slow = 8192.0, 1.0, 4.0, 32.0, 1.0
    if case["scaling"] == "base" and rot > 2:
        theta *= factor ** (rot / (rot - 2))
    f = [theta ** (-2.0 * i / rot) for i in range(rot // 2)]
    if case["scaling"] == "linear":
        f = [v / factor for v in f]
    if case["scaling"] == "bands":                          # by wavelength: kept, divided, or between the two
        s = [min(1.0, max(0.0, (ctx * v / (2 * math.pi) - low) / (high - low))) for v in f]
        f = [v * (1 - w) / factor + v * w for v, w in zip(f, s)]
    scale = 1.0
    if case["scaling"] == "yarn":                           # by index: a ramp between two numbers of turns over ctx
        at = [rot * math.log(ctx / (n * 2 * math.pi)) / (2 * math.log(theta)) for n in (fast, slow)]
        lo, hi = max(math.floor(at[0]), 0), min(math.ceil(at[1]), rot - 1)
        s = [1 - min(1.0, max(0.0, (i - lo) / max(hi - lo, 1e-3))) for i in range(rot // 2)]
        f = [v * (1 - w) / factor + v * w for v, w in zip(f, s)]
        scale = 0.1 * math.log(factor) + 1.0
    return f, scale


def _rope_inputs(case, seed):
    g = _rng(seed, 1)
    T, n = case["T"], case["H"] * case["HD"]
    x = _normal((T, n + 128), g)                            # the heads to rotate, then others left alone
    pos = case["first"] + case["gap"] * torch.arange(T, dtype=torch.int32, device="cuda")
    return x[:, :n], pos


def _logp_inputs(case, seed):
    g = _rng(seed, 2)
    rows, V = case["rows"], case["V"]
    x = _normal((rows, V), g, 3.0)
    tok = torch.randint(0, V, (rows, case["nt"]), generator=g, device="cuda", dtype=torch.int32)
    if case["masked"]:
        x[torch.rand((rows, V), generator=g, device="cuda") < case["masked"]] = -math.inf
    x[torch.arange(rows, device="cuda"), (torch.arange(rows, device="cuda") * 31 + 7) % V] = 14.0   # what the model thinks likely
    return x.half() if case["x"] == "f16" else x, tok


def _attn_inputs(case, seed):
    g = _rng(seed, 3)
    NH, NKV, HD = case["NH"], case["NKV"], case["HD"]
    q, h = _lengths(case)
    half = case["kv"] == "f16"
    starts = [0]
    for n in q:
        starts.append(starts[-1] + n)
    R = starts[-1]
    s = {"R": R, "q_start": _ints(starts), "kv_len": _ints([a + b for a, b in zip(q, h)])}
    kp, vp = (_normal((case["P"], NKV * HD), g) for _ in range(2))
    if case["hist"] == 0 and not half:                      # rows as one projection left them: q, k, v side by side
        rows = _normal((R, (NH + 2 * NKV) * HD), g)
        s.update(q=rows[:, :NH * HD], ks=rows[:, NH * HD:(NH + NKV) * HD], vs=rows[:, (NH + NKV) * HD:],
                 kv_start=s["q_start"][:-1].clone())
    else:                                                   # a slot of the cache for each sequence
        cap = case["q"] + case["hist"]
        ks, vs = (_normal((case["B"] * cap, NKV * HD), g) for _ in range(2))
        s.update(q=_normal((R, NH * HD), g), ks=ks.half() if half else ks, vs=vs.half() if half else vs,
                 kv_start=_ints([cap * b for b in range(case["B"])]))
    s.update(kp=kp.half() if half else kp, vp=vp.half() if half else vp)
    return s


def prepare(case, seed):
    state = {"case": case}
    if case["op"] == "rope":
        x, pos = _rope_inputs(case, seed)
        f, scale = _frequencies(case)
        state.update(x=x, pos=pos, freq=torch.tensor(f, dtype=torch.float64, device="cuda"), mscale=scale,
                     y=torch.empty((case["T"], case["H"] * case["HD"]), device="cuda",
                                   dtype=torch.float16 if case["out"] == "f16" else torch.float32))
    elif case["op"] == "logp":
        x, tok = _logp_inputs(case, seed)
        rows, k = case["rows"], case["k"]
        state.update(x=x, tok=tok, logp=torch.empty((rows, case["nt"]), device="cuda"), entropy=torch.empty((rows,), device="cuda"),
                     top=torch.empty((rows, k), device="cuda"), ids=torch.empty((rows, k), device="cuda", dtype=torch.int32))
    else:
        state.update(_attn_inputs(case, seed))
        state["out"] = torch.empty((state["R"], case["NH"] * case["HD"]), device="cuda")
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


def _workspace(state, nbytes):
    """The caller's workspace of one call site, kept with its buffers."""
    if state.get("ws") is None or state["ws"].numel() < nbytes:
        state["ws"] = torch.empty((max(nbytes, 1),), dtype=torch.uint8, device="cuda")
    return state["ws"].data_ptr()


def _own_rope(s, case):
    sgpu = _sgpu()
    if "turns" not in s:                                    # the table that a host uploads once
        kind = {"none": sgpu.ROPE_PLAIN, "linear": sgpu.ROPE_LINEAR, "base": sgpu.ROPE_BASE, "bands": sgpu.ROPE_BANDS,
                "yarn": sgpu.ROPE_YARN}[case["scaling"]]
        lo, hi = (1.0, 4.0) if case["scaling"] == "bands" else (32.0, 1.0)
        turns, s["factor"] = sgpu.rope_turns(case["rot"], case["theta"], kind, case["factor"], 8192.0, lo, hi)
        s["turns"] = torch.from_numpy(turns).cuda()
    sgpu.call("sgpu_rope_rows_h" if case["out"] == "f16" else "sgpu_rope_rows", s["x"].data_ptr(), s["x"].stride(0),
              s["y"].data_ptr(), s["y"].stride(0), s["pos"].data_ptr(), 0, s["turns"].data_ptr(), case["rot"],
              int(case["inter"]), s["factor"], case["T"], case["H"], case["HD"], torch.cuda.current_stream().cuda_stream)
    return s["y"]


def _own_logp(s, case):
    sgpu = _sgpu()
    rows, V, k = case["rows"], case["V"], case["k"]
    if "need" not in s:
        s["need"] = sgpu.lib().sgpu_logprobs_workspace(rows, V, k)
    sgpu.call("sgpu_logprobs_h" if case["x"] == "f16" else "sgpu_logprobs", s["x"].data_ptr(), V, rows, V, s["tok"].data_ptr(),
              case["nt"], s["logp"].data_ptr(), s["entropy"].data_ptr(), k, s["top"].data_ptr(), s["ids"].data_ptr(),
              _workspace(s, s["need"]), s["need"], torch.cuda.current_stream().cuda_stream)
    return {"logp": s["logp"], "entropy": s["entropy"], "top": s["top"], "ids": s["ids"]}


def _own_attn(s, case):
    sgpu = _sgpu()
    if "args" not in s:                                     # the description of its buffers that a host keeps
        a = s["args"] = sgpu.AttnPrefixArgs()
        a.q, a.out, a.kp, a.vp, a.ks, a.vs = (s[n].data_ptr() for n in ("q", "out", "kp", "vp", "ks", "vs"))
        a.q_row, a.out_row, a.kp_row, a.ks_row = (s[n].stride(0) for n in ("q", "out", "kp", "ks"))
        a.q_head = a.out_head = a.kp_head = a.ks_head = case["HD"]
        a.q_start, a.kv_start, a.kv_len = (s[n].data_ptr() for n in ("q_start", "kv_start", "kv_len"))
        a.R, a.B, a.P, a.SR = s["R"], case["B"], case["P"], s["ks"].shape[0]
        a.NH, a.NKV, a.HD, a.scale = case["NH"], case["NKV"], case["HD"], 1.0 / math.sqrt(case["HD"])
        a.max_q, a.max_kv = case["q"], case["q"] + case["hist"]
        s["need"] = sgpu.lib().sgpu_attn_prefix_workspace(sgpu.byref(a))
    sgpu.call("sgpu_attn_prefix_h" if case["kv"] == "f16" else "sgpu_attn_prefix", sgpu.byref(s["args"]),
              _workspace(s, s["need"]), s["need"], torch.cuda.current_stream().cuda_stream)
    return s["out"]


# ---- the plain forms ----
def _plain_rope(s, case):
    T, H, HD, rot = case["T"], case["H"], case["HD"], case["rot"]
    x = s["x"].reshape(T, H, HD)
    turn = s["pos"].double()[:, None] * s["freq"]
    c, d = (v.float()[:, None, :] * s["mscale"] for v in (torch.cos(turn), torch.sin(turn)))
    if case["inter"]:
        a, b = x[:, :, 0:rot:2], x[:, :, 1:rot:2]
        r = torch.stack((a * c - b * d, a * d + b * c), 3).reshape(T, H, rot)
    else:
        a, b = x[:, :, :rot // 2], x[:, :, rot // 2:rot]
        r = torch.cat((a * c - b * d, a * d + b * c), 2)
    return torch.cat((r, x[:, :, rot:]), 2).reshape(T, H * HD).to(s["y"].dtype)


def _plain_logp(s, case):
    x, k, V = s["x"].float(), case["k"], case["V"]
    m = x.amax(1, keepdim=True)
    z = x - m
    e = torch.exp(z)
    Z = e.sum(1, keepdim=True)
    lnz = torch.log(Z)
    logp = z.gather(1, s["tok"].long()) - lnz
    entropy = (lnz - (e * torch.where(e > 0, z, 0.0)).sum(1, keepdim=True) / Z)[:, 0]
    # the k largest, the lowest id first among equals: one whole number orders both
    bits = (x + 0.0).view(torch.int32)
    key = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long() * (1 << 20) + (V - 1 - torch.arange(V, device=x.device))
    ids = V - 1 - (torch.topk(key, k, 1).values & ((1 << 20) - 1)) if k else torch.empty((case["rows"], 0), dtype=torch.long, device=x.device)
    return {"logp": logp, "entropy": entropy, "top": z.gather(1, ids) - lnz, "ids": ids.to(torch.int32)}


def _plain_attn(s, case):
    NH, NKV, HD, R, B, P = case["NH"], case["NKV"], case["HD"], s["R"], case["B"], case["P"]
    G, nq, nk = NH // NKV, case["q"], case["q"] + case["hist"]
    q = s["q"].float().reshape(R, NKV, G, HD) * (1.0 / math.sqrt(HD))
    # over the prefix: all rows as one matrix a key head
    qg = q.permute(1, 0, 2, 3).reshape(NKV, R * G, HD)
    kp = s["kp"].float().reshape(P, NKV, HD).permute(1, 2, 0).contiguous()
    vp = s["vp"].float().reshape(P, NKV, HD).permute(1, 0, 2).contiguous()
    s1 = torch.bmm(qg, kp)
    # over its own rows: each sequence's rows and keys padded to the longest
    start, length, first = s["q_start"].long(), s["kv_len"].long(), s["kv_start"].long()
    n = start[1:] - start[:-1]
    i, j = torch.arange(nq, device=q.device), torch.arange(nk, device=q.device)
    rows = (start[:-1, None] + i).clamp(max=R - 1)
    keys = (first[:, None] + torch.minimum(j, length[:, None] - 1)).reshape(-1)
    ks = s["ks"][keys].float().reshape(B, nk, NKV, HD).permute(0, 2, 3, 1).reshape(B * NKV, HD, nk).contiguous()
    vs = s["vs"][keys].float().reshape(B, nk, NKV, HD).permute(0, 2, 1, 3).reshape(B * NKV, nk, HD).contiguous()
    qs = q[rows].permute(0, 2, 1, 3, 4).reshape(B * NKV, nq * G, HD)
    hidden = (j[None, None, :] > (length - n)[:, None, None] + i[None, :, None])[:, None, :, None, :]
    s2 = torch.bmm(qs, ks).reshape(B, NKV, nq, G, nk).masked_fill(hidden, -math.inf)
    # back to rows, one softmax over both
    mine = torch.arange(R, device=q.device)
    b = (mine[:, None] >= start[None, 1:]).sum(1)
    at = mine - start[b]
    s2 = s2.permute(0, 2, 1, 3, 4)[b, at].permute(1, 0, 2, 3).reshape(NKV, R * G, nk)
    m = torch.maximum(s1.amax(2, keepdim=True), s2.amax(2, keepdim=True))
    p1, p2 = torch.exp(s1 - m), torch.exp(s2 - m)
    total = p1.sum(2, keepdim=True) + p2.sum(2, keepdim=True)
    o = torch.bmm(p1, vp)
    p2 = torch.zeros((B, nq, NKV, G, nk), device=q.device).index_put((b, at), p2.reshape(NKV, R, G, nk).permute(1, 0, 2, 3))
    o2 = torch.bmm(p2.permute(0, 2, 1, 3, 4).reshape(B * NKV, nq * G, nk), vs).reshape(B, NKV, nq, G, HD).permute(0, 2, 1, 3, 4)[b, at]
    o = (o + o2.permute(1, 0, 2, 3).reshape(NKV, R * G, HD)) / total
    return o.reshape(NKV, R, G, HD).permute(1, 0, 2, 3).reshape(R, NH * HD)


def run(state):
    case = state["case"]
    if own:
        return {"rope": _own_rope, "logp": _own_logp, "attn": _own_attn}[case["op"]](state, case)
    return {"rope": _plain_rope, "logp": _plain_logp, "attn": _plain_attn}[case["op"]](state, case)


# ---- work ----
def work(case):
    if case["op"] == "rope":
        n = case["T"] * case["H"] * case["HD"]
        return {"bytes": n * (4 + (2 if case["out"] == "f16" else 4)) + 4 * case["T"], "flops": 3 * case["T"] * case["H"] * case["rot"]}
    if case["op"] == "logp":
        rows, V = case["rows"], case["V"]
        return {"bytes": rows * (V * (2 if case["x"] == "f16" else 4) + 8 * case["nt"] + 4 + 8 * case["k"]), "flops": 5 * rows * V}
    q, h = _lengths(case)
    NH, NKV, HD, R = case["NH"], case["NKV"], case["HD"], sum(q)
    size = 2 if case["kv"] == "f16" else 4
    seen = R * case["P"] + sum(a * b + a * (a + 1) // 2 for a, b in zip(q, h))
    return {"bytes": 2 * size * NKV * HD * (case["P"] + sum(q) + sum(h)) + 8 * R * NH * HD, "flops": 4 * HD * NH * seen}


# ---- the same in 64 bits ----
def _exact_rope(case, seed):
    x, pos = _rope_inputs(case, seed)
    T, H, HD, rot = case["T"], case["H"], case["HD"], case["rot"]
    f, scale = _frequencies(case)
    z = x.double().reshape(T, H, HD)
    out = z.clone()
    half = rot // 2
    first = torch.arange(half, device="cuda") * 2 if case["inter"] else torch.arange(half, device="cuda")
    second = first + (1 if case["inter"] else half)
    # a pair as one complex number, turned by a unit one
    angle = pos.double()[:, None] * torch.tensor(f, dtype=torch.float64, device="cuda")[None]
    w = torch.complex(z[:, :, first], z[:, :, second]) * torch.polar(torch.full_like(angle, scale), angle)[:, None]
    out[:, :, first], out[:, :, second] = w.real, w.imag
    return out.reshape(T, H * HD)


def _exact_logp(case, seed):
    x, tok = _logp_inputs(case, seed)
    logp, entropy, top = [], [], []
    for r0 in range(0, case["rows"], 128):
        z = torch.log_softmax(x[r0:r0 + 128].double(), 1)
        logp.append(z.gather(1, tok[r0:r0 + 128].long()))
        entropy.append(-torch.where(z > -math.inf, z.exp() * z, 0.0).sum(1))
        top.append(torch.topk(z, case["k"], 1).values)
    return {"logp": torch.cat(logp), "entropy": torch.cat(entropy), "top": torch.cat(top), "ids": None}


def _exact_attn(case, seed):
    s = _attn_inputs(case, seed)
    q, h = _lengths(case)
    NH, NKV, HD, P = case["NH"], case["NKV"], case["HD"], case["P"]
    G = NH // NKV
    out = torch.empty((s["R"], NH * HD), dtype=torch.float64, device="cuda")
    r0 = 0
    for b in range(case["B"]):
        k0, n = int(s["kv_start"][b]), q[b] + h[b]
        Q = s["q"][r0:r0 + q[b]].double()
        see = torch.arange(n, device="cuda")[None] <= h[b] + torch.arange(q[b], device="cuda")[:, None]
        see = torch.cat((torch.ones((q[b], P), dtype=torch.bool, device="cuda"), see), 1)
        for g in range(NKV):
            cols = slice(g * HD, (g + 1) * HD)
            K = torch.cat((s["kp"][:, cols], s["ks"][k0:k0 + n, cols])).double()
            W = torch.cat((s["vp"][:, cols], s["vs"][k0:k0 + n, cols])).double()
            for e in range(g * G, (g + 1) * G):
                w = torch.softmax((Q[:, e * HD:(e + 1) * HD] @ K.t().contiguous() / math.sqrt(HD)).masked_fill(~see, -math.inf), 1)
                out[r0:r0 + q[b], e * HD:(e + 1) * HD] = w @ W
        r0 += q[b]
    return out


def exact(case, seed):
    return {"rope": _exact_rope, "logp": _exact_logp, "attn": _exact_attn}[case["op"]](case, seed)

"""Scoring of continuations of one prompt (sgpu_qwen_score): the engine path that runs the rotary rows,
the attention over a shared prefix and the log probabilities together, against the CPU golden run one
continuation and one position at a time.

Bars: the engine's logits are held to delta = 1e-4 of the logits' scale elsewhere.  Logits off by at most
delta move a log probability by at most 2 delta (its own logit, and the logarithm of the sum of
exponentials, a mean of the logits' changes), an entropy by at most 2 delta (H + 1) to first order, and
an ordering only among logits within 2 delta."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

NT = 8
PATHS = dict(reference=0, fused=1, graph=2)


def small(NH, NKV, HD, FC, CTX, NL=2, V=300):
    return dict(V=V, C=NH * HD, NL=NL, NH=NH, NKV=NKV, HD=HD, FC=FC, CTX=CTX)


def engine(gpu, cfg, seed=61, path="fused"):
    blob = gpu.qwen_random_blob(gpu.qwen_cfg(**cfg), seed=seed, std=0.15)
    return gpu.QwenEngine(gpu.qwen_cfg(**cfg), blob, PATHS[path]), blob


def check_row(got, j, z, tok, k):
    z = z.astype(np.float64)
    delta = 1e-4 * np.abs(z).max()
    lse = z.max() + np.log(np.exp(z - z.max()).sum())
    lp = z - lse
    H = -(np.exp(lp) * lp).sum()
    assert abs(got["logp"][j] - lp[tok]) <= 2 * delta, (j, got["logp"][j], lp[tok])
    assert abs(got["entropy"][j] - H) <= 2 * delta * (H + 1), (j, got["entropy"][j], H)
    if k:
        n = min(k, z.size)
        ids = got["top_id"][j][:n]
        assert len(set(ids.tolist())) == n and ids.min() >= 0
        best = np.sort(lp)[::-1][:n]
        assert np.abs(lp[ids] - best).max() <= 2 * delta, j
        assert np.abs(got["top_logp"][j][:n] - best).max() <= 2 * delta, j
        assert (got["top_id"][j][n:] == -1).all() and np.isneginf(got["top_logp"][j][n:]).all()


CASES = {
    "one-token": (small(4, 2, 32, 256, 64), 1, [1], 3),
    "hd32": (small(4, 2, 32, 256, 64), 40, [1, 2, 7, 1, 20, 24], 5),
    "first-tokens-only": (small(4, 2, 32, 256, 64), 9, [1] * 70, 2),
    "no-top": (small(2, 2, 64, 128, 64), 17, [5, 9], 0),
    "past-the-vocabulary": (small(2, 1, 64, 128, 64, V=37), 5, [3, 2], 64),
    "pieces": (small(14, 2, 64, 704, 120), 70, [1, 33, 2, 12, 50, 8, 3], 20),
    "pieces-hd128": (small(4, 2, 128, 1024, 150), 129, [20] * 6 + [1, 2], 4),
    "pieces-logits": (small(14, 2, 64, 704, 120, V=320), 30, [40, 33, 2, 12, 1], 20),
    "mha": (small(3, 3, 64, 192, 100), 30, [40, 41, 3], 1),
    "two-passes": (small(1, 1, 64, 64, 1400, NL=1), 3, [1301, 1299, 2], 1),
    "long": (small(1, 1, 64, 64, 2500, NL=1), 2, [1, 2400], 1),
}


@pytest.mark.parametrize("case", CASES.values(), ids=CASES.keys())
def test_score_matches_golden(gpu, og, case):
    cfg, T, lens, k = case
    print("score", cfg, T, lens[:8], k, flush=True)
    eng, blob = engine(gpu, cfg)
    rng = np.random.default_rng(T)
    prompt = rng.integers(0, cfg["V"], T)
    cont = [rng.integers(0, cfg["V"], n) for n in lens]
    got = eng.score(prompt, cont, k)
    gold = og.QwenGolden(og.qwen_cfg(**cfg), blob, NT)
    for p in range(T):
        first = gold.forward(int(prompt[p]), p, p == T - 1)
    first = np.array(first)
    for c, g in zip(cont, got):
        assert g["logp"].shape == g["entropy"].shape == (c.size,)
        z = first
        for j, tok in enumerate(c.tolist()):
            check_row(g, j, z, tok, k)
            if j + 1 < c.size:
                z = np.array(gold.forward(tok, T + j, True))
    eng.close()


@pytest.mark.parametrize("V", [300, 320], ids=["logits-in-tiles", "logits-in-pieces"])
def test_score_leaves_the_engine_as_prefill_does(gpu, V):
    cfg = small(14, 2, 64, 704, 200, V=V)
    rng = np.random.default_rng(5)
    prompt, cont = rng.integers(0, cfg["V"], 77), [rng.integers(0, cfg["V"], n) for n in (30, 1, 60)]
    a, _ = engine(gpu, cfg, path="graph")
    b, _ = engine(gpu, cfg, path="graph")
    want = b.prefill(prompt).copy()
    before = a.generate(prompt, 20)
    first = a.score(prompt, cont, 3)
    for j in range(3):                                             # no position of it reads what scoring left
        assert np.array_equal(a.forward(int(cont[0][j]), 77 + j), b.forward(int(cont[0][j]), 77 + j))
    second = a.score(prompt, cont, 3)
    for x, y in zip(first, second):                                # nothing depends on timing or on earlier calls
        for key in x:
            assert np.array_equal(x[key], y[key]), key
    # alone, in another order, beside others: the same tokens' scores (to the products' other tilings)
    alone = a.score(prompt, [cont[2]])[0]
    assert np.abs(alone["logp"] - first[2]["logp"]).max() <= 4e-4 * np.abs(want).max()
    assert np.array_equal(a.generate(prompt, 20), before)
    a.close()
    b.close()


def test_score_of_nothing_primes_the_prompt(gpu):
    cfg = small(4, 2, 32, 256, 64)
    a, _ = engine(gpu, cfg)
    b, _ = engine(gpu, cfg)
    prompt = np.arange(11)
    assert a.score(prompt, []) == []
    b.prefill(prompt)
    assert np.array_equal(a.forward(3, 11), b.forward(3, 11))
    a.close()
    b.close()


def test_score_refusals(gpu):
    cfg = small(4, 2, 32, 256, 64)
    eng, _ = engine(gpu, cfg)
    ok = [np.array([1, 2]), np.array([3])]
    bad = [lambda: eng.score([], ok), lambda: eng.score([300], ok), lambda: eng.score([-1], ok),
           lambda: eng.score([1], ok + [np.array([], np.int32)]), lambda: eng.score([1], [np.array([1, 300])]),
           lambda: eng.score([1], [np.array([-1])]), lambda: eng.score([1], ok, -1), lambda: eng.score([1], ok, 65),
           lambda: eng.score(np.zeros(60, int), [np.zeros(6, int)]), lambda: eng.score(np.zeros(65, int), ok)]
    for i, f in enumerate(bad):
        with pytest.raises(gpu.SgpuError) as err:
            f()
        assert err.value.status == gpu.SGPU_ERR_INVALID_ARG, i
    assert len(eng.score(np.zeros(60, int), [np.zeros(5, int)])[0]["logp"]) == 5       # the last row at the last position
    call = gpu.lib().sgpu_qwen_score
    i1, f1 = np.ones(1, np.int32), np.zeros(4, np.float32)
    p = lambda a: a.ctypes.data
    for args in [(None, p(i1), 1, p(i1), p(i1), 1, p(f1), None, 0, None, None),
                 (eng.h, None, 1, p(i1), p(i1), 1, p(f1), None, 0, None, None),
                 (eng.h, p(i1), 1, None, p(i1), 1, p(f1), None, 0, None, None),
                 (eng.h, p(i1), 1, p(i1), None, 1, p(f1), None, 0, None, None),
                 (eng.h, p(i1), 1, p(i1), p(i1), 1, None, None, 0, None, None),
                 (eng.h, p(i1), 1, p(i1), p(i1), -1, p(f1), None, 0, None, None),
                 (eng.h, p(i1), 1, p(i1), p(i1), 1, p(f1), None, 1, None, p(i1)),
                 (eng.h, p(i1), 1, p(i1), p(i1), 1, p(f1), None, 1, p(f1), None)]:
        assert call(*args) == gpu.SGPU_ERR_INVALID_ARG
    assert call(eng.h, p(i1), 1, p(i1), p(i1), 1, p(f1), None, 0, None, None) == 0 and f1[0] < 0
    eng.close()


def test_score_refuses_other_rotation_tables(gpu):
    """The rotation is computed from cfg.theta: a file that brings other tables is not scored."""
    cfg = small(4, 2, 32, 256, 64)
    blob = gpu.qwen_random_blob(gpu.qwen_cfg(**cfg), seed=1, std=0.15).copy()
    at = cfg["V"] * cfg["C"] * 2
    table = blob.view(np.uint8)[at:at + cfg["CTX"] * 16 * 4].view(np.float32)
    table[5 * 16 + 3] += 1e-3
    eng = gpu.QwenEngine(gpu.qwen_cfg(**cfg), blob, 1)
    with pytest.raises(gpu.SgpuError):
        eng.score([1, 2], [[3]])
    eng.generate([1, 2], 3)
    eng.close()


def test_score_of_very_many_one_token_continuations(gpu):
    """They have no rows, and take no part in a launch: two longer ones among them are scored as by themselves."""
    cfg = small(64, 64, 32, 64, 64, NL=1)
    eng, _ = engine(gpu, cfg)
    rng = np.random.default_rng(9)
    prompt, long = rng.integers(0, cfg["V"], 5), [rng.integers(0, cfg["V"], n) for n in (3, 2)]
    ones = rng.integers(0, cfg["V"], (140000, 1)).astype(np.int32)
    cont = [*ones[:70000], long[0], *ones[70000:], long[1]]
    got, alone = eng.score(prompt, cont, 1), eng.score(prompt, long + [np.array([t]) for t in range(cfg["V"])], 1)
    for a, b in ((got[70000], alone[0]), (got[-1], alone[1])):
        for key in a:
            assert np.array_equal(a[key], b[key]), key
    first = np.array([r["logp"][0] for r in alone[2:]])
    for i in (*range(70000), *range(70001, len(cont) - 1)):
        assert got[i]["logp"][0] == first[cont[i][0]]
    eng.close()


# sgpu_malloc as the engine calls it, refusing what is larger than `limit` bytes as a full device would; `largest`:
# of what it gave.
SHIM = """
#include <stddef.h>
extern int hipMalloc(void **p, size_t n);
size_t limit = (size_t)-1, largest = 0;
int sgpu_malloc(void **p, size_t n) {
    *p = 0;
    if (n > limit) return 2;                                               /* hipErrorOutOfMemory */
    if (n > largest && n != (32u << 20)) largest = n;
    return n ? hipMalloc(p, n) : 0;
}
"""
SHIM_RUN = """
import ctypes, sys
sys.path.insert(0, sys.argv[2])
shim = ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)               # found before the library's own
import numpy as np
import sgpu
cfg = dict(V=320, C=128, NL=2, NH=2, NKV=1, HD=64, FC=192, CTX=300)
blob = sgpu.qwen_random_blob(sgpu.qwen_cfg(**cfg), seed=51, std=0.15)
limit, largest = (ctypes.c_size_t.in_dll(shim, n) for n in ("limit", "largest"))
ids = [(7 * i) % 320 for i in range(100)]
rng = np.random.default_rng(1)
cont = [rng.integers(0, 320, n) for n in [66] * 29 + [1, 200, 3]]
def run(lim):
    limit.value = 2**64 - 1
    e = sgpu.QwenEngine(sgpu.qwen_cfg(**cfg), blob, sgpu.QWEN_PATH_FUSED)
    e.prefill(ids)
    limit.value, largest.value = lim, 0
    got = e.score(ids, cont, 5)
    limit.value = 2**64 - 1
    after = e.forward(5, 100).copy()
    again = e.score(ids, cont, 5)
    e.close()
    return got, after, again, largest.value
want, after, _, n = run(2**64 - 1)
scale = np.abs(after).max()
for lim in (n - 1, (32 << 20) - 1):                                    # smaller passes; no room for the partials either
    got, a, again, m = run(lim)
    print("limit", lim, "largest", m, flush=True)
    assert np.array_equal(a, after)
    for w, g, s in zip(want, got, again):
        assert np.abs(g["logp"] - w["logp"]).max() <= 4e-4 * scale and np.abs(g["entropy"] - w["entropy"]).max() <= 4e-3 * scale
        assert all(np.array_equal(s[k], w[k]) for k in w)
limit.value = 2**64 - 1
e = sgpu.QwenEngine(sgpu.qwen_cfg(**cfg), blob, sgpu.QWEN_PATH_FUSED)
e.prefill(ids)
limit.value = 1000                                                     # no room at all: an error, and the engine as before
try:
    e.score(ids, cont, 5)
    raise SystemExit("scored without room")
except sgpu.SgpuError as err:
    assert err.status == 2, err
limit.value = 2**64 - 1
e.prefill(ids)
assert np.array_equal(e.forward(5, 100), after)
assert all(np.array_equal(s[k], w[k]) for s, w in zip(e.score(ids, cont, 5), want) for k in w)
print("done", flush=True)
"""


def test_score_without_room_for_its_buffers(gpu, tmp_path):
    """Smaller passes, then the form on fp32 tiles, where the device has no room; then an error of its own."""
    import os
    import subprocess
    import sys

    (tmp_path / "shim.c").write_text(SHIM)
    so = str(tmp_path / "shim.so")
    subprocess.run(["gcc", "-shared", "-fPIC", "-o", so, str(tmp_path / "shim.c"), "-L/opt/rocm/lib", "-lamdhip64",
                    "-Wl,-rpath,/opt/rocm/lib"], check=True)
    out = subprocess.run([sys.executable, "-c", SHIM_RUN, so, os.path.dirname(gpu.__file__)], capture_output=True, text=True,
                         timeout=100)
    assert out.returncode == 0 and out.stdout.endswith("done\n"), out.stdout + out.stderr[-2000:]

"""Attention over a shared prefix with NaN and infinities in keys and values, in every form of the kernel: rows and heads
that do not see them are as if they were not there, and what sees them says so.

An infinite key whose score is -infinity may count as a key without weight."""
import numpy as np
import pytest

from test_gpu_score import Attn, cut_case, renew

pytestmark = pytest.mark.gpu

HEADS = {32: (6, 2, 32), 64: (14, 2, 64), 128: (4, 2, 128)}
# (query rows, earlier own rows): the longest own keys take several splits
SEQS = {"few": [(3, 700), (1, 5)], "step": [(4, 700)] + [(2, 9)] * 20, "rows": [(50, 700), (70, 3), (1, 0)]}
SEQS.update(cut_step=SEQS["step"], cut_rows=SEQS["rows"])
FORMS = [(f, half) for f in SEQS for half in (False, True) if not (half and f in ("cut_step", "cut_rows", "step"))]
DIM, KV = 5, 1                                                 # the poisoned dim and KV head


def case(gpu, form, half, HD, P, seed):
    if form.startswith("cut"):
        return cut_case(gpu, SEQS[form], P + 400, *HEADS[HD], seed=seed)
    return Attn(gpu, SEQS[form], P, *HEADS[HD], half=half, seed=seed)


def check(gpu, c, where, at, value, sees):
    """`sees`: the rows that see the poisoned key or value."""
    t, G = getattr(c, where), c.NH // c.NKV
    clean, bar = c.want()
    before = t[at, KV, DIM]
    t[at, KV, DIM] = value
    renew(gpu, c, where)
    c.call()
    gpu.synchronize()
    got = c.out()
    hit = np.zeros(got.shape, bool)
    hit[sees, KV * G:(KV + 1) * G, DIM if where in ("vp", "vs") else slice(None)] = True
    diff = np.abs(np.where(hit, 0.0, got - clean))
    assert np.all(diff <= bar), np.argwhere(~(diff <= bar))[:3].tolist()
    fine = np.isfinite(got)
    if where in ("kp", "ks") and np.isinf(value):              # one or the other, for the whole head
        t[at, KV, DIM] = before
        keep = c.q[..., DIM] * np.sign(value) < 0              # the score is -infinity
        t[at, KV] = 0
        t[at, KV, DIM] = np.sign(value) * 6e4                  # as good as no weight: q is not small where it is kept
        gone, bar = c.want()
        for r in np.flatnonzero(sees):
            for h in range(KV * G, (KV + 1) * G):
                if not fine[r, h].any():
                    continue
                assert keep[r, h] and fine[r, h].all(), (r, h)
                if c.q[r, h, DIM] * np.sign(value) * 6e4 * c.scale < -200:
                    assert np.all(np.abs(got[r, h] - gone[r, h]) <= bar[r, h]), (r, h)
    else:
        assert not fine[hit].any(), np.argwhere(hit & fine)[:3].tolist()


@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf], ids=str)
@pytest.mark.parametrize("where", ["ks", "vs"])
@pytest.mark.parametrize("HD", list(HEADS))
@pytest.mark.parametrize("form,half", FORMS, ids=str)
def test_attn_own_keys_not_finite(gpu, form, half, HD, where, value):
    """In one of the newest own keys of the first sequence, which its earlier rows do not see."""
    print("own", form, half, HD, where, value, flush=True)
    c = case(gpu, form, half, HD, 210, seed=HD)
    q0, n, nq = int(c.q_start[0]), int(c.kv_len[0]), SEQS[form][0][0]
    at = n - 2                                                 # the last two rows see it
    sees = np.zeros(c.R, bool)
    sees[q0 + nq - 2:q0 + nq] = True
    check(gpu, c, where, int(c.kv_start[0]) + at, value, sees)


@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf], ids=str)
@pytest.mark.parametrize("where", ["kp", "vp"])
@pytest.mark.parametrize("HD", list(HEADS))
@pytest.mark.parametrize("form,half", FORMS, ids=str)
def test_attn_prefix_keys_not_finite(gpu, form, half, HD, where, value):
    print("prefix", form, half, HD, where, value, flush=True)
    c = case(gpu, form, half, HD, 210, seed=HD + 1)
    sees = np.zeros(c.R, bool)
    sees[int(c.q_start[0]):int(c.q_start[-1])] = True
    check(gpu, c, where, 201, value, sees)

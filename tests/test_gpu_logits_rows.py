"""Adjusted logits of more rows than one launch holds blocks for."""
import numpy as np
import pytest

from test_gpu_paged import dev

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("same", [False, True])
def test_logits_adjust_of_five_million_rows(gpu, same):
    """Each row penalised, biased and masked by its own numbers."""
    rows, V = 5_000_011, 6
    r = np.arange(rows)
    x = ((r[:, None] * 7 + np.arange(V)) % 64 - 31).astype(np.float16)
    rep, freq, pres = 1 + (r % 4).astype(np.float32), (r % 5).astype(np.float32), (r % 3).astype(np.float32)
    tok = (np.arange(64) * 5 % V).astype(np.int32)      # row r: prompt tok[r % 61], output tok[r % 59 .. + 2]
    span = np.stack([r % 61, np.ones_like(r), r % 59, np.full_like(r, 2)], 1).astype(np.int32)
    bias_id, bias = (np.arange(7) % V).astype(np.int32), np.arange(7).astype(np.float32) - 3
    bias_span = np.stack([r % 7, r % 2], 1).astype(np.int32)
    allow = (r % 64).astype(np.uint32)
    want = x.astype(np.float64)
    seen, said = np.zeros((rows, V), bool), np.zeros((rows, V))
    seen[r, tok[span[:, 0]]] = True
    for i in range(2):
        seen[r, tok[span[:, 2] + i]] = True
        said[r, tok[span[:, 2] + i]] += 1
    want = np.where(seen, np.where(want > 0, want / rep[:, None], want * rep[:, None]), want)
    want -= said * freq[:, None] + (said > 0) * pres[:, None]
    some = r[r % 2 == 1]
    want[some, bias_id[some % 7]] += bias[some % 7]
    want = np.where(allow[:, None] >> np.arange(V, dtype=np.uint32) & 1, want, -np.inf).astype(np.float16)
    a = gpu.LogitsArgs()
    d = [dev(gpu, v) for v in (x, tok, span, rep, freq, pres, bias_id, bias, bias_span, allow)]
    y = d[0] if same else gpu.DeviceArray((rows, V), np.float16)
    for n, v in zip(("x", "tok", "span", "rep", "freq", "pres", "bias_id", "bias", "bias_span", "allow"), d):
        setattr(a, n, v.ptr)
    a.y, a.x_row, a.y_row, a.rows, a.V, a.n_tok, a.n_bias, a.allow_row = y.ptr, V, V, rows, V, tok.size, bias.size, 1
    gpu.call("sgpu_logits_adjust_h", gpu.byref(a), None)
    gpu.synchronize()
    assert np.array_equal(y.to_host(), want)

"""Norms of heads (sgpu_qk_norm_rope, sgpu_kv_append) at the ends of the fp32 range, against 64 bits; the bars are
test_gpu_paged's."""
import numpy as np
import pytest

from test_gpu_paged import Append, dev, heads64, rounded, turns_of

pytestmark = pytest.mark.gpu

SIZES = [2.0**-149, 1e-42, 1e-40, 2.0**-128, 1e-38, 1e-30, 1.0, 1e30, 3e37, 1e38, 3e38]


def norm(gpu, x, w, eps, rot, nb, half=False):
    """[T][1][HD] through sgpu_qk_norm_rope / _h: one query head a row, rows at positions 0, 1, .."""
    T, _, HD = x.shape
    d, dw, dt = dev(gpu, x), dev(gpu, w), dev(gpu, turns_of(rot))
    y = gpu.DeviceArray(x.shape, np.float16 if half else np.float32)
    gpu.call("sgpu_qk_norm_rope_h" if half else "sgpu_qk_norm_rope", d.ptr, HD, y.ptr, HD, dw.ptr, None, eps, None, 0, dt.ptr, rot, nb, 1.0,
             T, 1, 0, HD, None)
    gpu.synchronize()
    return y.to_host().astype(np.float64)


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("eps", [0.0, 2.0**-149])
@pytest.mark.parametrize("HD,rot,nb", [(64, 2, 0), (64, 64, 0), (128, 64, 1), (33, 2, 0), (40, 6, 1), (512, 256, 0)])
def test_norm_of_values_of_any_size(gpu, HD, rot, nb, eps, half):
    """Heads whose root mean square has no fp32 inverse, or one with few digits, give values of order 1."""
    rng = np.random.default_rng(HD)
    x = np.stack([rng.uniform(0.3, 1.0, (1, HD)) * rng.choice([-1, 1], (1, HD)) * s for s in SIZES]).astype(np.float32)
    x[0] = np.where(rng.random((1, HD)) < 0.5, 1, -2) * np.float32(2.0**-149)
    w = (1 + 0.3 * rng.standard_normal(HD)).astype(np.float32)
    want, bar = heads64(x, w, eps, np.arange(len(x)), turns_of(rot), rot, nb, 1.0)
    got = norm(gpu, x, w, eps, rot, nb, half)
    assert np.isfinite(got).all()
    assert np.all(np.abs(got - want) <= rounded(want, bar + 2.0**-149, half))


@pytest.mark.parametrize("half", [False, True])
def test_appended_keys_and_queries_of_any_size(gpu, half):
    """The same through the append: rows of any size, their keys and queries normed without eps."""
    a = Append(gpu, [(17, 5), (3, 6)], 6, 2, 64, 16, half)
    a.a.eps = 0.0
    n = 8 * 64                                          # q and k; the values stay
    a.x[:, :n] = (a.x[:, :n].astype(np.float64) / 10 * np.array(SIZES)[:, None]).astype(np.float32)
    a.x[0, :n] = np.float32(2.0**-149)
    gpu.call("sgpu_memcpy_htod", a.keep["x"].ptr, a.x.ctypes.data, a.x.nbytes)
    a.call()
    gpu.synchronize()
    x = a.x[:, :n].reshape(11, 8, 64)
    at = np.concatenate([17 + np.arange(5), 3 + np.arange(6)])
    want, bar = heads64(x[:, :6], a.w[0], 0.0, at, a.turns, 64, 0, 1.0)
    got = a.keep["out"].to_host()[:, :-4].reshape(want.shape)
    assert np.all(np.abs(got - want) <= bar + 2.0**-149)
    want, bar = heads64(x[:, 6:], a.w[1], 0.0, at, a.turns, 64, 0, 1.0)
    c = a.c
    c.buf[0] = c.keep["k"].to_host()
    for r, (b, t) in enumerate([(0, 17 + i) for i in range(5)] + [(1, 3 + i) for i in range(6)]):
        k = c.at(0, b, t).astype(np.float64)
        assert np.all(np.abs(k - want[r]) <= rounded(want[r], bar[r] + 2.0**-149, half)), r


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("HD,rot,nb", [(64, 2, 0), (64, 64, 0), (128, 64, 1), (33, 2, 0), (40, 6, 1), (512, 256, 0)])
def test_norm_of_an_infinite_value(gpu, HD, rot, nb, half):
    """An infinite value has no norm: it is NaN, with what it is rotated into; the head's others are 0, other heads as ever."""
    rng = np.random.default_rng(HD + 1)
    x = rng.standard_normal((6, 1, HD)).astype(np.float32)
    x[1, 0, 0], x[2, 0, HD - 1], x[3, 0, 4] = np.inf, -np.inf, np.inf
    x[4, 0, 1], x[4, 0, HD // 2] = np.inf, -np.inf
    w = (1 + 0.3 * rng.standard_normal(HD)).astype(np.float32)
    with np.errstate(invalid="ignore"):
        want, bar = heads64(x, w, 1e-6, np.arange(6), turns_of(rot), rot, nb, 1.0)
    got = norm(gpu, x, w, 1e-6, rot, nb, half)
    fine = np.isfinite(want)
    assert (~fine).any() and np.array_equal(np.isnan(got), ~fine)
    assert np.all(np.abs(got - want)[fine] <= rounded(want, bar, half)[fine])

"""How near the residual tower's operators come to their definitions where f32 formulas usually lose: the activations' tails, rows far
from zero with little or no variance.  The bounds are derived here, beside each test."""
import numpy as np
import pytest
from scipy.special import erfc

import tower_ref as R
from test_gpu_tower import EPS, Pool, within

pytestmark = pytest.mark.gpu
f32, U = np.float32, R.U
TYPES = [R.F32, R.BF16, R.F16]


@pytest.fixture
def pool():
    p = Pool()
    yield p
    p.close()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("D", [3, 7, 24, 49, 107, 300, 429, 512, 1001, 1024, 2051, 4099, 8191, 9001])
def test_ln_of_constant_rows_is_beta(pool, t, D):
    """a row of one value has no variance: whatever the value, y is beta (the mean of equal f32 numbers is that number, and x - mean is 0
    exactly), and 1 / sqrt(var + eps) that of eps.  A mean that is a step off is divided by sqrt(eps) = 0.003 and shows."""
    from ps_amd import native as N
    L, kv = N.lib(), pool.kv
    rng = np.random.default_rng(D)
    c = np.array([1.0, -3.5, 0.1, 1000.0, 1e5 if t != R.F16 else 6e4, -12345.678, 3e-3, 77.7])
    B = c.size
    v = np.tile(c[:, None], (1, D))
    g, b = (1 + 0.2 * rng.standard_normal(D)).astype(f32), (0.2 * rng.standard_normal(D)).astype(f32)
    kv.create_ln(0, D)
    kv.put("ln0.weights", g)
    kv.put("ln0.bias", b)
    xr, yr, st = pool.rows(t, B, D, values=v), pool.rows(t, B, D), pool.rows(R.F32, B, 2)
    N.check(L.ps_ln_forward(kv.h, 0, t, xr.p, D, B, EPS, yr.p, D, st.p))
    np.testing.assert_array_equal(yr.get(), np.tile(R.rounded(b, t), (B, 1)))
    s = st.get()
    np.testing.assert_array_equal(s[:, 0], R.rounded(c, t))
    within(s[:, 1], np.full(B, 1 / np.sqrt(np.float64(f32(EPS)))), 3 * U / np.sqrt(EPS), "rstd")


@pytest.mark.parametrize("t", [R.F32, R.BF16])
@pytest.mark.parametrize("D", [24, 300, 1024, 2051, 9001])
def test_ln_far_from_zero(pool, t, D):
    """rows whose mean is far larger than their spread: what is lost is the rounding of the mean to f32 (u |mean|), not a whole sum's.
    d = x - m is exact up to u |d| for any m near the values, m' = m + mean(d) is off by u |mean| and the chain of d's sum, (c + 2) u
    mean|d| -- c the longest chain of adds, ln_chain -- and y carries that over the spread."""
    from ps_amd import native as N
    L, kv = N.lib(), pool.kv
    rng = np.random.default_rng(D + 1)
    B = 5
    x = rng.standard_normal((B, D)) * (1.0 if t == R.F32 else 400.0) + np.array([1e4, -3e4, 1e5, 7e3, 12.0])[:, None]
    kv.create_ln(0, D)
    xr, yr, st = pool.rows(t, B, D, values=x), pool.rows(t, B, D), pool.rows(R.F32, B, 2)
    N.check(L.ps_ln_forward(kv.h, 0, t, xr.p, D, B, EPS, yr.p, D, st.p))
    x = R.rounded(x, t)
    y, mean, rstd = R.ln_forward(x, 1.0, 0.0, f32(EPS))
    c = R.ln_chain(D)
    spread = np.abs(x - mean).mean(1, keepdims=True)
    # the first mean m is off by at most (c + 2) u mean|x|, which d's sum then carries in every term
    d = spread + (c + 2) * U * np.abs(x).mean(1, keepdims=True)
    e = U * np.abs(mean) + (c + 4) * U * d
    rel = 0.5 * (2 * d * d * (c + 8) * U * rstd ** 2 + (c + 4) * U) + 6 * U
    tol = e * rstd + np.abs(y) * (rel + 4 * U)
    s = st.get()
    within(s[:, :1], mean, e, "mean")
    within(yr.get(), y, tol + R.store_tol(np.abs(y) + tol, t), "y")


def through_one(pool, t, a, z):
    """(z as the type has it, act(z), act'(z)) by a product with the number 1"""
    from ps_amd import native as N
    L, kv = N.lib(), pool.kv
    kv.create_fc(0, 1, 1)
    kv.put("fc0.weights", [1.0])
    kv.put("fc0.bias", [0.0])
    B = z.size
    zr, y, dy = pool.rows(t, B, 1, values=z[:, None]), pool.rows(t, B, 1), pool.rows(t, B, 1, values=np.ones((B, 1)))
    dx, g = pool.rows(t, B, 1), pool.rows(R.F32, 2, 1)
    N.check(L.ps_fc_res_forward(kv.h, 0, t, a, zr.p, 1, B, None, 0, None, 0, y.p, 1))
    N.check(L.ps_fc_res_backward(kv.h, 0, t, a, zr.p, 1, zr.p, 1, dy.p, 1, B, None, 0, dx.p, 1, g.p))
    return R.rounded(z, t), y.get()[:, 0], dx.get()[:, 0]


def test_silu_f32_is_accurate_relative_to_itself(pool):
    """z / (1 + e^-z) in f32, from e = e^-|z|: e is off by 3 u (the exponential a step, its correction half of one), 1 + e by u and its
    reciprocal by u, and a value below 0 has two products more: 7 u of the value.  Beyond -87.3 e is below f32's normal numbers and the
    value, less than 1.1e-36, becomes 0.  (e^0 is exact, the value at 0 too.)"""
    z = np.concatenate([-np.logspace(-6, np.log10(120), 3000), np.logspace(-6, 2, 1000), np.random.default_rng(0).standard_normal(4000) * 3])
    zv, y, _ = through_one(pool, R.F32, R.SILU, z)
    e = np.exp(-np.abs(zv))
    want = zv * np.where(zv < 0, e, 1.0) / (1 + e)
    within(y, want, 7.01 * U * np.abs(want) + 1.1e-36, "silu")


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("a", [R.GELU, R.SILU])
def test_activations_at_minus_infinity_are_their_limits(pool, t, a):
    _, y, slope = through_one(pool, t, a, np.array([-np.inf, -1e30, -3e4, np.nan, 1.0]))
    assert (y[:3] == 0).all() and (slope[:3] == 0).all() and np.isnan(y[3]) and abs(y[4]) > 0.5


@pytest.mark.parametrize("t", TYPES)
def test_gelu_tail_is_rounded_once(pool, t):
    """z Phi(z) for z < 0 is -|z| Q(|z|).  Q's polynomial in f32 arithmetic (test_tower_accuracy_cpu.py evaluates it) is within 5e-8 of Q
    and, down to -8, within 4e-4 of it relatively; the exponential adds a step (2 u) and the product half of one.  In 16 bits that is the
    storing's rounding and a fifth of it, down to -8, where the value is 5e-15; from there on it is smaller than that."""
    z = -np.concatenate([np.linspace(0.01, 14, 3000), np.random.default_rng(1).random(1000) * 8])
    zv, y, slope = through_one(pool, t, R.GELU, z)
    q = 0.5 * erfc(-zv / np.sqrt(2.0))
    off = np.where(zv >= -8, np.minimum(5e-8, 4e-4 * q), q)
    tol = np.abs(zv) * off + 4 * U * np.abs(zv) * q
    within(y, zv * q, tol + R.store_tol(np.abs(zv * q) + tol, t), "gelu")
    # the slope Q - |z| phi: Q as above; |z| phi by an exponential of z^2 log2(e) / 2, whose argument carries 2 u of itself
    p = np.abs(zv) * np.exp(-zv * zv / 2) / np.sqrt(2 * np.pi)
    want = q - p
    tol = off + 4 * U * q + (zv * zv + 6) * U * p + 2e-37
    within(slope, want, tol + R.store_tol(np.abs(want) + tol, t), "slope")

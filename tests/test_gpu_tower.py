"""The residual tower's operators through the C ABI (ps_ln_*, ps_fc_res_*) against their definitions in 64 bits (tower_ref.py, where the
tolerances are derived): every type, row strides and alignments of every kind, sizes around the kernels' tiles, what lies behind a row
and behind the last row left alone; the pending gradient, the updaters, the keys and the checkpoint; a block of them trained; recorded
into a HIP graph; and the calls that are refused."""
import ctypes as C

import numpy as np
import pytest

import tower_ref as R

pytestmark = pytest.mark.gpu
f32 = np.float32
EPS = 1e-5
TYPES = [R.F32, R.BF16, R.F16]
SENTINEL = 0x5A


class Rows:
    """[B][w] values of a type in rows of ld elements, `shift` elements into a device allocation; guard rows behind."""

    def __init__(self, kv, t, B, w, ld=None, shift=0, values=None):
        from ps_amd import native as N
        self.N, self.kv, self.t, self.B, self.w, self.ld, self.shift = N, kv, t, B, w, ld or w, shift
        self.dt = np.float32 if t == R.F32 else np.float16 if t == R.F16 else np.uint16
        self.n = shift + (B + 2) * self.ld + 8
        self.host = np.frombuffer(bytes([SENTINEL]) * (self.n * np.dtype(self.dt).itemsize), self.dt).copy()
        if values is not None:
            self.view(self.host)[:] = R.encode(values, t)
        self.buf = C.c_void_p()
        N.check(N.lib().ps_dev_alloc(kv.h, max(self.host.nbytes, 16), C.byref(self.buf)))
        N.check(N.lib().ps_dev_upload(kv.h, self.buf, self.host.ctypes.data, self.host.nbytes))
        self.p = self.buf.value + shift * self.host.itemsize

    def view(self, a):
        return np.lib.stride_tricks.as_strided(a[self.shift:], (self.B, self.w), (self.ld * a.itemsize, a.itemsize))

    def raw(self):
        out = np.empty_like(self.host)
        self.N.check(self.N.lib().ps_dev_download(self.kv.h, out.ctypes.data, self.buf, out.nbytes))
        return out

    def get(self, untouched=True):
        """the values, float64; everything else in the allocation has to be as it was"""
        raw = self.raw()
        vals = R.decode(np.ascontiguousarray(self.view(raw)), self.t)
        if untouched:
            rest = raw.copy()
            self.view(rest)[:] = np.ascontiguousarray(self.view(self.host))
            np.testing.assert_array_equal(rest.view(np.uint8), self.host.view(np.uint8), err_msg="written outside the rows")
        return vals

    def free(self):
        self.N.lib().ps_dev_free(self.kv.h, self.buf)


class Pool:
    """the device buffers of one test"""

    def __init__(self):
        import ps_amd
        self.kv, self.all = ps_amd.KVStore(0, 0x5EED), []

    def rows(self, *a, **k):
        r = Rows(self.kv, *a, **k)
        self.all.append(r)
        return r

    def close(self):
        for r in self.all:
            r.free()
        self.kv.close()


@pytest.fixture
def pool():
    p = Pool()
    yield p
    p.close()


def within(got, want, tol, what):
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), "%s: %d of %d off, worst %.3g of its tolerance, first at %s" % (
        what, bad.sum(), bad.size, np.nanmax(np.abs(got - want)[bad] / np.broadcast_to(tol, got.shape)[bad]), np.argwhere(bad)[0])


def p_(r):
    return None if r is None else r.p


def ld_(r):
    return 0 if r is None else r.ld


# rows of every lane layout: 4, 16, 64 lanes, a workgroup, the walking kernel; odd ends; one and many rows
LN_SIZES = [(1, 1), (3, 5), (70, 8), (5, 16), (130, 29), (257, 64), (33, 65), (100, 128), (9, 250), (40, 275), (64, 429), (17, 512),
            (300, 700), (21, 1024), (7, 2047), (6, 2049), (5, 4100), (3, 8192), (2, 8193), (3, 20011)]


def ln_case(pool, t, B, D, pad, shift, seed=0):
    rng = np.random.default_rng(B * 31 + D + seed)
    x = rng.standard_normal((B, D)) * (0.5 + rng.random(D)) + rng.standard_normal(D)
    g, b = (1 + 0.2 * rng.standard_normal(D)).astype(f32), (0.2 * rng.standard_normal(D)).astype(f32)
    pool.kv.create_ln(3, D)
    pool.kv.put("ln3.weights", g)
    pool.kv.put("ln3.bias", b)
    xr = pool.rows(t, B, D, D + pad, shift, x)
    return rng, xr, R.rounded(x, t), g.astype(np.float64), b.astype(np.float64)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("B,D", LN_SIZES)
def test_ln_forward_and_backward(pool, t, B, D):
    from ps_amd import native as N
    L = N.lib()
    pad, shift = ((0, 0), (3, 1), (8, 8), (1, 5))[(B + D) % 4]
    rng, xr, x, g, b = ln_case(pool, t, B, D, pad, shift)
    yr, st = pool.rows(t, B, D, D + pad, shift), pool.rows(R.F32, B, 2)
    N.check(L.ps_ln_forward(pool.kv.h, 3, t, xr.p, xr.ld, B, EPS, yr.p, yr.ld, st.p))
    y, mean, rstd = R.ln_forward(x, g, b, f32(EPS))
    ty, tm, tr = R.ln_forward_tol(x, g, b, f32(EPS), t)
    within(yr.get(), y, ty, "y")
    got = st.get()
    within(got[:, :1], mean, tm, "mean")
    within(got[:, 1:], rstd, tr, "rstd")
    # without statistics, and in place: the same values
    ip = pool.rows(t, B, D, D + pad, shift, x)
    N.check(L.ps_ln_forward(pool.kv.h, 3, t, ip.p, ip.ld, B, EPS, ip.p, ip.ld, None))
    np.testing.assert_array_equal(ip.get(untouched=False), yr.get())
    # backward from the statistics as they lie in memory
    dy, sk = rng.standard_normal((B, D)), rng.standard_normal((B, D))
    dyr, skr = pool.rows(t, B, D, D, 0, dy), pool.rows(t, B, D, D + pad, shift, sk)
    dy, sk = R.rounded(dy, t), R.rounded(sk, t)
    for skip in (None, skr):
        dxr, gr = pool.rows(t, B, D, D + pad, shift), pool.rows(R.F32, 2, D)
        N.check(L.ps_ln_backward(pool.kv.h, 3, t, xr.p, xr.ld, st.p, dyr.p, dyr.ld, B, p_(skip), ld_(skip), dxr.p, dxr.ld, gr.p))
        args = (x, got[:, :1], got[:, 1:], g, dy, sk if skip else None)
        dx, grad = R.ln_backward(*args)
        tdx, tg = R.ln_backward_tol(*args, t)
        within(dxr.get(), dx, tdx, "dx")
        within(gr.get(), grad, tg, "gamma / beta gradient")
    # dx over dy, and gradients alone
    N.check(L.ps_ln_backward(pool.kv.h, 3, t, xr.p, xr.ld, st.p, dyr.p, dyr.ld, B, skr.p, skr.ld, dyr.p, dyr.ld, gr.p))
    np.testing.assert_array_equal(dyr.get(untouched=False), dxr.get())
    dyr2, g2 = pool.rows(t, B, D, D, 0, dy), pool.rows(R.F32, 2, D)
    N.check(L.ps_ln_backward(pool.kv.h, 3, t, xr.p, xr.ld, st.p, dyr2.p, dyr2.ld, B, None, 0, None, 0, g2.p))
    np.testing.assert_array_equal(g2.get(), gr.get())


@pytest.mark.parametrize("t", TYPES)
def test_ln_many_rows(pool, t):
    """more rows than workgroups: the loops over rows, the column sums over several rows a lane"""
    from ps_amd import native as N
    L = N.lib()
    for B, D in ((20011, 24), (9000, 130), (2600, 1030)):
        rng, xr, x, g, b = ln_case(pool, t, B, D, 0, 0)
        yr, st = pool.rows(t, B, D), pool.rows(R.F32, B, 2)
        N.check(L.ps_ln_forward(pool.kv.h, 3, t, xr.p, D, B, EPS, yr.p, D, st.p))
        within(yr.get(), R.ln_forward(x, g, b, f32(EPS))[0], R.ln_forward_tol(x, g, b, f32(EPS), t)[0], "y")
        s = st.get()
        dy = rng.standard_normal((B, D)) + 0.1
        dyr, dxr, gr = pool.rows(t, B, D, values=dy), pool.rows(t, B, D), pool.rows(R.F32, 2, D)
        args = (x, s[:, :1], s[:, 1:], g, R.rounded(dy, t), None)
        N.check(L.ps_ln_backward(pool.kv.h, 3, t, xr.p, D, st.p, dyr.p, D, B, None, 0, dxr.p, D, gr.p))
        tdx, tg = R.ln_backward_tol(*args, t)
        within(dxr.get(), R.ln_backward(*args)[0], tdx, "dx")
        within(gr.get(), R.ln_backward(*args)[1], tg, "grad")
        first = gr.raw()
        N.check(L.ps_ln_backward(pool.kv.h, 3, t, xr.p, D, st.p, dyr.p, D, B, None, 0, dxr.p, D, gr.p))
        np.testing.assert_array_equal(gr.raw(), first)            # the order of every sum is fixed
        pool.close()
        pool.__init__()


@pytest.mark.parametrize("t", TYPES)
def test_ln_far_from_zero_constant_rows_and_bad_values(pool, t):
    """a large common offset (the variance from differences survives it), constant rows (variance 0), and rows of infinities and NaN
    that must not reach their neighbours"""
    from ps_amd import native as N
    L = N.lib()
    B, D = 6, 300
    rng, xr, x, g, b = ln_case(pool, t, B, D, 0, 0)
    v = rng.standard_normal((B, D))
    v[0] += 1000
    v[1] = 3.5
    v[2, 7] = np.inf
    v[3, 299] = np.nan
    xr = pool.rows(t, B, D, values=v)
    x = R.rounded(v, t)
    yr, st = pool.rows(t, B, D), pool.rows(R.F32, B, 2)
    N.check(L.ps_ln_forward(pool.kv.h, 3, t, xr.p, D, B, EPS, yr.p, D, st.p))
    y, ok = yr.get(), [0, 1, 4, 5]
    within(y[ok], R.ln_forward(x[ok], g, b, f32(EPS))[0], R.ln_forward_tol(x[ok], g, b, f32(EPS), t)[0], "y")
    assert np.isnan(y[2]).all() and np.isnan(y[3]).all()


# around the tiles of every product kernel, skinny and wide, one column, one row
FC_SIZES = [(1, 1, 1), (1, 429, 512), (2, 7, 3), (5, 33, 130), (15, 64, 16), (16, 65, 17), (17, 16, 100), (31, 200, 40), (33, 129, 65),
            (64, 64, 64), (65, 63, 129), (130, 275, 150), (257, 40, 300), (600, 150, 10), (1000, 37, 1), (300, 257, 260)]


def fc_case(pool, t, B, K, N_, pad, shift):
    rng = np.random.default_rng(B * 7 + K * 3 + N_)
    w, b = (rng.standard_normal((K, N_)) / np.sqrt(K)).astype(f32), (0.3 * rng.standard_normal(N_)).astype(f32)
    pool.kv.create_fc(2, K, N_)
    pool.kv.put("fc2.weights", w)
    pool.kv.put("fc2.bias", b)
    x = rng.standard_normal((B, K))
    return rng, pool.rows(t, B, K, K + pad, shift, x), R.rounded(x, t), w.astype(np.float64), b.astype(np.float64)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("B,K,N_", FC_SIZES)
def test_fc_res_forward_and_backward(pool, t, B, K, N_):
    from ps_amd import native as N
    L = N.lib()
    acts = (R.NONE, R.RELU, R.GELU, R.SILU)
    for i, (pad, shift) in enumerate(((0, 0), (3, 1), (8, 8), (5, 2))):
        a = acts[(i + B + K) % 4]
        rng, xr, x, w, b = fc_case(pool, t, B, K, N_, pad, shift)
        r = rng.standard_normal((B, N_)) if i % 2 else None
        rr = None if r is None else pool.rows(t, B, N_, N_ + pad, shift, r)
        r = None if r is None else R.rounded(r, t)
        yr, zr = pool.rows(t, B, N_, N_ + pad, shift), pool.rows(t, B, N_, N_ + (7 if i == 3 else 0), 0)
        N.check(L.ps_fc_res_forward(pool.kv.h, 2, t, a, xr.p, xr.ld, B, p_(rr), ld_(rr), zr.p, zr.ld, yr.p, yr.ld))
        y, z, ty, tz = R.fc_forward(x, w, b, a, r, t)
        within(yr.get(), y, ty, "y act %d" % a)
        within(zr.get(), z, tz, "z")
        y2 = pool.rows(t, B, N_, N_ + pad, shift)
        N.check(L.ps_fc_res_forward(pool.kv.h, 2, t, a, xr.p, xr.ld, B, p_(rr), ld_(rr), None, 0, y2.p, y2.ld))
        np.testing.assert_array_equal(y2.get(), yr.get())
        if rr is not None:                                        # over the residual
            N.check(L.ps_fc_res_forward(pool.kv.h, 2, t, a, xr.p, xr.ld, B, rr.p, rr.ld, None, 0, rr.p, rr.ld))
            np.testing.assert_array_equal(rr.get(untouched=False), yr.get())
        dy, sk = rng.standard_normal((B, N_)), rng.standard_normal((B, K))
        dyr = pool.rows(t, B, N_, N_ + pad, shift, dy)
        skr = pool.rows(t, B, K, K + pad, shift, sk) if i % 2 == 0 else None
        dxr, gr = pool.rows(t, B, K, K + pad, shift), pool.rows(R.F32, K + 1, N_)
        N.check(L.ps_fc_res_backward(pool.kv.h, 2, t, a, xr.p, xr.ld, zr.p if a else None, zr.ld, dyr.p, dyr.ld, B, p_(skr), ld_(skr), dxr.p, dxr.ld, gr.p))
        dx, grad, tdx, tg = R.fc_backward(x, w, zr.get(), R.rounded(dy, t), a, R.rounded(sk, t) if skr else None, t)
        within(dxr.get(), dx, tdx, "dx act %d" % a)
        within(gr.get(), grad, tg, "gradient act %d" % a)
        if skr is not None:                                       # over the skip's gradient
            N.check(L.ps_fc_res_backward(pool.kv.h, 2, t, a, xr.p, xr.ld, zr.p if a else None, zr.ld, dyr.p, dyr.ld, B, skr.p, skr.ld, skr.p, skr.ld, gr.p))
            np.testing.assert_array_equal(skr.get(untouched=False), dxr.get())
        g2 = pool.rows(R.F32, K + 1, N_)                          # gradients alone
        N.check(L.ps_fc_res_backward(pool.kv.h, 2, t, a, xr.p, xr.ld, zr.p if a else None, zr.ld, dyr.p, dyr.ld, B, None, 0, None, 0, g2.p))
        np.testing.assert_array_equal(g2.get(), gr.get())


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("B,K,N_,a", [(4096, 429, 512, R.RELU), (2000, 1024, 2048, R.GELU), (8191, 520, 264, R.NONE), (16, 2048, 2048, R.NONE),
                                      (20000, 64, 1, R.SILU), (48, 4096, 1000, R.NONE), (1, 4096, 4096, R.SILU),
                                      (40000, 72, 200, R.GELU), (33000, 64, 256, R.RELU), (40000, 40, 296, R.NONE), (35003, 328, 77, R.SILU), (33100, 200, 128, R.GELU),
                                      (10950, 520, 776, R.GELU), (7301, 2056, 264, R.NONE), (4000, 1032, 2000, R.RELU),
                                      (700, 2051, 700, R.SILU), (130, 4099, 640, R.GELU), (17000, 603, 517, R.GELU), (17001, 517, 603, R.NONE), (20001, 301, 333, R.SILU)])
def test_fc_res_large(pool, t, B, K, N_, a):
    """sizes at which the split products, the large tiles and the few-row kernels run"""
    from ps_amd import native as N
    L = N.lib()
    rng, xr, x, w, b = fc_case(pool, t, B, K, N_, 0, 0)
    yr, zr = pool.rows(t, B, N_), pool.rows(t, B, N_)
    N.check(L.ps_fc_res_forward(pool.kv.h, 2, t, a, xr.p, K, B, None, 0, zr.p, N_, yr.p, N_))
    y, z, ty, tz = R.fc_forward(x, w, b, a, None, t)
    within(yr.get(), y, ty, "y")
    within(zr.get(), z, tz, "z")
    dy = rng.standard_normal((B, N_))
    dyr, dxr, gr = pool.rows(t, B, N_, values=dy), pool.rows(t, B, K), pool.rows(R.F32, K + 1, N_)
    N.check(L.ps_fc_res_backward(pool.kv.h, 2, t, a, xr.p, K, zr.p if a else None, N_, dyr.p, N_, B, None, 0, dxr.p, K, gr.p))
    dx, grad, tdx, tg = R.fc_backward(x, w, zr.get(), R.rounded(dy, t), a, None, t)
    within(dxr.get(), dx, tdx, "dx")
    within(gr.get(), grad, tg, "gradient")
    first = gr.raw()
    N.check(L.ps_fc_res_backward(pool.kv.h, 2, t, a, xr.p, K, zr.p if a else None, N_, dyr.p, N_, B, None, 0, dxr.p, K, gr.p))
    np.testing.assert_array_equal(gr.raw(), first)                # the order of every sum is fixed


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("B", [3, 40, 300])
def test_fc_bad_values_stay_in_their_row(pool, t, B):
    """an infinity and a NaN in one row of x, and whatever lies behind the rows' ends, must not reach other rows"""
    from ps_amd import native as N
    L = N.lib()
    K, N_ = 70, 90
    rng, xr, x, w, b = fc_case(pool, t, B, K, N_, 0, 0)
    v = rng.standard_normal((B, K + 9))
    v[:, K:] = np.nan                                             # behind every row
    v[1, 3], v[2, 69] = np.inf, np.nan
    wide = pool.rows(t, B, K + 9, values=v)
    yr = pool.rows(t, B, N_)
    N.check(L.ps_fc_res_forward(pool.kv.h, 2, t, R.RELU, wide.p, K + 9, B, None, 0, None, 0, yr.p, N_))
    got = yr.get()
    ok = [i for i in range(B) if i not in (1, 2)]
    x = R.rounded(v[:, :K], t)
    y, _, ty, _ = R.fc_forward(x[ok], w, b, R.RELU, None, t)
    within(got[ok], y, ty, "y")
    assert np.isnan(got[2]).all() and not np.isfinite(got[1][w[3] > 0]).any()
    # backward: a gradient that is blocked by relu stays blocked, whatever it is
    z = rng.standard_normal((B, N_)); z[0, 0] = -1.0
    dy = rng.standard_normal((B, N_)); dy[0, 0] = np.inf
    zr, dyr, dxr, gr = pool.rows(t, B, N_, values=z), pool.rows(t, B, N_, values=dy), pool.rows(t, B, K), pool.rows(R.F32, K + 1, N_)
    xf = pool.rows(t, B, K, values=np.where(np.isfinite(v[:, :K]), v[:, :K], 0))
    N.check(L.ps_fc_res_backward(pool.kv.h, 2, t, R.RELU, xf.p, K, zr.p, N_, dyr.p, N_, B, None, 0, dxr.p, K, gr.p))
    dy[0, 0] = 0
    dx, grad, tdx, tg = R.fc_backward(R.rounded(np.where(np.isfinite(v[:, :K]), v[:, :K], 0), t), w, R.rounded(z, t), R.rounded(dy, t), R.RELU, None, t)
    within(dxr.get(), dx, tdx, "dx")
    within(gr.get(), grad, tg, "gradient")


@pytest.mark.parametrize("t", TYPES)
def test_activations_at_their_ends(pool, t):
    """z from far below to far above, the borders, infinities and a NaN, through a product by one: values and slopes"""
    from ps_amd import native as N
    L, kv = N.lib(), pool.kv
    kv.create_fc(0, 1, 1)
    kv.put("fc0.weights", [1.0]); kv.put("fc0.bias", [0.0])
    z = np.array([-np.inf, -1e4, -200, -100, -64, -30, -13, -6, -4, -3, -1, -1e-3, -1e-7, 0, 1e-7, 1e-3, 0.5, 1, 3, 4, 6, 13, 30, 64, 100, 200, 1e4, np.inf, np.nan])
    B = z.size
    zr, y, dy = pool.rows(t, B, 1, values=z[:, None]), pool.rows(t, B, 1), pool.rows(t, B, 1, values=np.ones((B, 1)))
    dx, g = pool.rows(t, B, 1), pool.rows(R.F32, 2, 1)
    zv = R.rounded(z, t)
    fin = np.isfinite(zv)
    for a in (R.RELU, R.GELU, R.SILU):
        N.check(L.ps_fc_res_forward(kv.h, 0, t, a, zr.p, 1, B, None, 0, None, 0, y.p, 1))
        N.check(L.ps_fc_res_backward(kv.h, 0, t, a, zr.p, 1, zr.p, 1, dy.p, 1, B, None, 0, dx.p, 1, g.p))
        got, slope = y.get()[:, 0], dx.get()[:, 0]
        with np.errstate(all="ignore"):
            want, dwant = R.act(zv, a), R.act_grad(zv, a)
        tol = (0 if a == R.RELU else 8 * R.U) * np.abs(zv[fin]) + R.store_tol(np.abs(want[fin]) * 1.001, t) + 1e-37
        within(got[fin], want[fin], tol, "act %d" % a)
        tol = (0 if a == R.RELU else 14 * R.U) * (1 + np.minimum(np.abs(zv[fin]), 8)) + R.store_tol(np.abs(dwant[fin]) * 1.001, t)
        within(slope[fin], dwant[fin], tol, "slope %d" % a)
        up = zv == np.inf
        assert (got[up] == np.inf).all() and (slope[up] == 1).all() and np.isnan(got[-1])
        if a != R.SILU:
            assert (got[zv == -np.inf] == 0).all()
        assert (slope[zv == -np.inf] == 0).all()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("a", [R.GELU, R.SILU])
def test_infinite_gradients_behind_a_slope(pool, t, a):
    """an infinite dy is infinite behind a slope that is not zero, with the product's sign; its neighbours are what they were"""
    from ps_amd import native as N
    L, kv = N.lib(), pool.kv
    kv.create_fc(0, 1, 1)
    kv.put("fc0.weights", [1.0])
    z = np.tile([-3.0, -0.5, 0.25, 1.0, 2.0, 5.0, -1e4, 1e4], 3)
    dy = np.ones_like(z)
    dy[8:16], dy[16] = np.inf, -np.inf
    B = z.size
    x, zr, d = (pool.rows(t, B, 1, values=v[:, None]) for v in (np.ones(B), z, dy))
    dx, g = pool.rows(t, B, 1), pool.rows(R.F32, 2, 1)
    N.check(L.ps_fc_res_backward(kv.h, 0, t, a, x.p, 1, zr.p, 1, d.p, 1, B, None, 0, dx.p, 1, g.p))
    with np.errstate(over="ignore"):
        got, slope = dx.get()[:, 0], R.act_grad(R.rounded(z, t), a)
    for i in range(B):
        if np.isfinite(dy[i]):
            within(got[i], slope[i], 14 * R.U * (1 + min(abs(z[i]), 8)) + R.store_tol(abs(slope[i]) * 1.001, t), "row %d" % i)
        elif abs(z[i]) < 100:
            assert got[i] == dy[i] * np.sign(slope[i]), (i, got[i])
        else:
            assert got[i] == np.inf if z[i] > 0 else np.isnan(got[i])         # (infinity times 0)


def test_pending_gradients_updaters_and_keys(pool, orc):
    """two backward calls add up in the store's pending gradients (KVStore.sum), dense_update divides by their number and runs every
    tensor's own updater; the keys are read, written, pushed and sized like the FC layers'"""
    import ps_amd
    from ps_amd import native as N
    L, kv = N.lib(), pool.kv
    B, D, N_ = 50, 48, 20
    rng = np.random.default_rng(5)
    kv.create_ln(0, D); kv.create_ln(0, D); kv.create_fc(0, D, N_)
    assert np.array_equal(kv.get("ln0.weights"), np.ones(D, f32)) and not kv.get("ln0.bias").any()
    assert kv.get("ln1.weights") is None and kv.key_length("ln0.bias") == D
    kv.set_updater("ln0.bias", ps_amd.SimpleUpdater(0.5))
    assert L.ps_ln_update(kv.h, 0) == N.PS_MISSING and L.ps_ln_update(kv.h, 7) == N.PS_MISSING
    cnt = C.c_int(-1)
    out = np.empty(D, f32)
    fp = out.ctypes.data_as(C.POINTER(C.c_float))
    assert L.ps_ln_pending_grad(kv.h, 0, 0, fp, D, C.byref(cnt)) == N.PS_MISSING and cnt.value == 0
    x = pool.rows(R.F32, B, D, values=rng.standard_normal((B, D)))
    y, st = pool.rows(R.F32, B, D), pool.rows(R.F32, B, 2)
    N.check(L.ps_ln_forward(kv.h, 0, R.F32, x.p, D, B, EPS, y.p, D, st.p))
    sums, fsums = np.zeros((2, D), f32), np.zeros((D + 1, N_), f32)
    for _ in range(2):
        dy, g = pool.rows(R.F32, B, D, values=rng.standard_normal((B, D))), pool.rows(R.F32, 2, D)
        N.check(L.ps_ln_backward(kv.h, 0, R.F32, x.p, D, st.p, dy.p, D, B, None, 0, None, 0, g.p))
        N.check(L.ps_ln_backward(kv.h, 0, R.F32, x.p, D, st.p, dy.p, D, B, None, 0, None, 0, None))
        sums = sums + g.get().astype(f32)
        d2, fg = pool.rows(R.F32, B, N_, values=rng.standard_normal((B, N_))), pool.rows(R.F32, D + 1, N_)
        N.check(L.ps_fc_res_backward(kv.h, 0, R.F32, R.NONE, y.p, D, None, 0, d2.p, N_, B, None, 0, None, 0, fg.p))
        N.check(L.ps_fc_res_backward(kv.h, 0, R.F32, R.NONE, y.p, D, None, 0, d2.p, N_, B, None, 0, None, 0, None))
        fsums = fsums + fg.get().astype(f32)
    for bias in (0, 1):
        N.check(L.ps_ln_pending_grad(kv.h, 0, bias, fp, D, C.byref(cnt)))
        assert cnt.value == 2 and np.array_equal(out, sums[bias])
    assert L.ps_ln_pending_grad(kv.h, 0, 0, fp, D - 1, None) == N.PS_E_BAD_ARG
    w0, fw, fb = kv.get("ln0.weights"), kv.get("fc0.weights"), kv.get("fc0.bias")
    step = kv.global_step()
    kv.dense_update()
    assert kv.global_step() == step + 1 and L.ps_ln_update(kv.h, 0) == N.PS_MISSING
    z = np.zeros(D, f32)
    np.testing.assert_array_equal(kv.get("ln0.weights"), orc.adam_update(w0, sums[0] / f32(2), z, z)[0])
    np.testing.assert_array_equal(kv.get("ln0.bias"), ((sums[1] / f32(2)) * f32(-0.5)).astype(f32))
    zf = np.zeros(D * N_, f32)
    np.testing.assert_array_equal(kv.get("fc0.weights"), orc.adam_update(fw, (fsums[:-1] / f32(2)).ravel(), zf, zf)[0])
    np.testing.assert_array_equal(kv.get("fc0.bias"), orc.adam_update(fb, fsums[-1] / f32(2), np.zeros(N_, f32), np.zeros(N_, f32))[0])
    # pushed by key, like a server's (KVStore.sum / count, one updater step)
    before = kv.get("ln0.bias")
    g1, g2 = rng.standard_normal(D).astype(f32), rng.standard_normal(D).astype(f32)
    kv.push_update([("ln0.bias", g1), ("ln0.bias", g2)])
    np.testing.assert_array_equal(kv.get("ln0.bias"), ((g1 + g2) / f32(2)) * f32(-0.5) + before)
    with pytest.raises(N.PsError):
        kv.push_update([("ln0.bias", g1[:-1])])
    # the changed parameters are what the next forward uses
    N.check(L.ps_ln_forward(kv.h, 0, R.F32, x.p, D, B, EPS, y.p, D, None))
    g, b, xv = kv.get("ln0.weights").astype(np.float64), kv.get("ln0.bias").astype(np.float64), x.get()
    within(y.get(), R.ln_forward(xv, g, b, f32(EPS))[0], R.ln_forward_tol(xv, g, b, f32(EPS), R.F32)[0], "y")


def test_checkpoint_keeps_the_normalisations(pool, tmp_path):
    import ps_amd
    from ps_amd import native as N
    rng = np.random.default_rng(2)
    pool.kv.create_fc(0, 12, 7); pool.kv.create_ln(2, 12)
    pool.kv.put("ln2.weights", rng.standard_normal(12)); pool.kv.put("ln2.bias", rng.standard_normal(12))
    pool.kv.push_update([("ln2.weights", rng.standard_normal(12))])          # updater state too
    pool.kv.save(tmp_path / "a.ck")
    other = ps_amd.KVStore(0, 1)
    other.create_fc(0, 12, 7); other.create_ln(2, 12)
    other.load(tmp_path / "a.ck")
    for k in ("ln2.weights", "ln2.bias", "fc0.weights", "fc0.bias"):
        np.testing.assert_array_equal(other.get(k), pool.kv.get(k))
    g = rng.standard_normal(12)
    other.push_update([("ln2.weights", g)]); pool.kv.push_update([("ln2.weights", g)])
    np.testing.assert_array_equal(other.get("ln2.weights"), pool.kv.get("ln2.weights"))
    other.close()
    for make in (lambda k: k.create_fc(0, 12, 7), lambda k: (k.create_fc(0, 12, 7), k.create_ln(2, 13)), lambda k: (k.create_fc(0, 12, 7), k.create_ln(1, 12))):
        other = ps_amd.KVStore(0, 1)
        make(other)
        with pytest.raises(N.PsError) as e:
            other.load(tmp_path / "a.ck")
        assert e.value.code == N.PS_E_BAD_ARG
        other.close()


@pytest.mark.parametrize("t", TYPES)
def test_a_block_forward_backward_update(pool, t, orc):
    """y = r + W2 gelu(W1 LN(r) + b1) + b2, its gradients with the skip's added on the way down, and one update of every tensor: each
    operator against its definition on what the one before it left in memory."""
    from ps_amd import native as N
    L, kv = N.lib(), pool.kv
    B, D, H = 333, 100, 260
    rng = np.random.default_rng(8)
    kv.create_ln(0, D); kv.create_fc(0, D, H); kv.create_fc(1, H, D)
    kv.put("ln0.weights", 1 + 0.1 * rng.standard_normal(D)); kv.put("ln0.bias", 0.1 * rng.standard_normal(D))
    for k, s in (("fc0", (D, H)), ("fc1", (H, D))):
        kv.put(k + ".weights", rng.standard_normal(s) / np.sqrt(s[0])); kv.put(k + ".bias", 0.1 * rng.standard_normal(s[1]))

    def P(k, *s):
        return kv.get(k).astype(np.float64).reshape(s)
    r = pool.rows(t, B, D, values=rng.standard_normal((B, D)))
    x, st, z, h, y = pool.rows(t, B, D), pool.rows(R.F32, B, 2), pool.rows(t, B, H), pool.rows(t, B, H), pool.rows(t, B, D)
    N.check(L.ps_ln_forward(kv.h, 0, t, r.p, D, B, EPS, x.p, D, st.p))
    N.check(L.ps_fc_res_forward(kv.h, 0, t, R.GELU, x.p, D, B, None, 0, z.p, H, h.p, H))
    N.check(L.ps_fc_res_forward(kv.h, 1, t, R.NONE, h.p, H, B, r.p, D, None, 0, y.p, D))
    dy = pool.rows(t, B, D, values=rng.standard_normal((B, D)))
    dh, dx, dr = pool.rows(t, B, H), pool.rows(t, B, D), pool.rows(t, B, D)
    N.check(L.ps_fc_res_backward(kv.h, 1, t, R.NONE, h.p, H, None, 0, dy.p, D, B, None, 0, dh.p, H, None))
    N.check(L.ps_fc_res_backward(kv.h, 0, t, R.GELU, x.p, D, z.p, H, dh.p, H, B, None, 0, dx.p, D, None))
    N.check(L.ps_ln_backward(kv.h, 0, t, r.p, D, st.p, dx.p, D, B, dy.p, D, dr.p, D, None))
    rv, xv, zv, hv, sv, dyv, dhv, dxv = (b.get() for b in (r, x, z, h, st, dy, dh, dx))
    g, b = P("ln0.weights", D), P("ln0.bias", D)
    within(xv, R.ln_forward(rv, g, b, f32(EPS))[0], R.ln_forward_tol(rv, g, b, f32(EPS), t)[0], "LN(r)")
    ya, za, ta, tza = R.fc_forward(xv, P("fc0.weights", D, H), P("fc0.bias", H), R.GELU, None, t)
    within(hv, ya, ta, "h"); within(zv, za, tza, "z")
    yb, _, tb, _ = R.fc_forward(hv, P("fc1.weights", H, D), P("fc1.bias", D), R.NONE, rv, t)
    within(y.get(), yb, tb, "y")
    want, gb, tw, tgb = R.fc_backward(hv, P("fc1.weights", H, D), None, dyv, R.NONE, None, t)
    within(dhv, want, tw, "dh")
    want, ga, tw, tga = R.fc_backward(xv, P("fc0.weights", D, H), zv, dhv, R.GELU, None, t)
    within(dxv, want, tw, "dx")
    args = (rv, sv[:, :1], sv[:, 1:], g, dxv, dyv)
    tw, tgl = R.ln_backward_tol(*args, t)
    want, gl = R.ln_backward(*args)
    within(dr.get(), want, tw, "dr")
    # every tensor moves by its updater's first step from the pending gradient
    buf = {}
    for name, fn, l, rows, cols, ref, tol in (("fc1", L.ps_fc_pending_grad, 1, H, D, gb, tgb), ("fc0", L.ps_fc_pending_grad, 0, D, H, ga, tga),
                                              ("ln0", L.ps_ln_pending_grad, 0, 1, D, gl, tgl)):
        for bias in (0, 1):
            o = np.empty(cols if bias else rows * cols, f32)
            N.check(fn(kv.h, l, bias, o.ctypes.data_as(C.POINTER(C.c_float)), o.size, None))
            within(o.astype(np.float64).reshape(-1, cols), ref[-1:] if bias else ref[:-1], tol[-1:] if bias else tol[:-1], name)
            buf[name + (".bias" if bias else ".weights")] = o
    before = {k: kv.get(k) for k in buf}
    kv.dense_update()
    for k, o in buf.items():
        np.testing.assert_array_equal(kv.get(k), orc.adam_update(before[k], o, np.zeros_like(o), np.zeros_like(o))[0], err_msg=k)


class Hip:
    """the runtime the library is linked to, for a stream and a graph of the test's own"""

    def __init__(self):
        self.L = C.CDLL("libamdhip64.so.7")

    def __call__(self, name, *a):
        rc = getattr(self.L, name)(*a)
        assert rc == 0, "%s -> %d" % (name, rc)


@pytest.mark.parametrize("t", [R.F32, R.BF16])
def test_recorded_and_replayed(pool, t):
    """a block's forward and backward in a HIP graph: replays with new inputs in the same buffers give what eager calls give; a second
    graph of other shapes shares the workspace; what cannot be recorded is refused and leaves the recording whole"""
    from ps_amd import native as N
    L, kv, hip = N.lib(), pool.kv, Hip()
    B, D, H = 200, 96, 130
    rng = np.random.default_rng(1)
    kv.create_ln(0, D); kv.create_fc(0, D, H)
    stream = C.c_void_p()
    hip("hipStreamCreateWithFlags", C.byref(stream), 1)
    kv.set_stream(stream)

    def make(B):
        return {k: pool.rows(ty, b, w, values=rng.standard_normal((b, w))) for k, ty, b, w in
                (("x", t, B, D), ("n", t, B, D), ("st", R.F32, B, 2), ("z", t, B, H), ("y", t, B, H), ("dy", t, B, H), ("dn", t, B, D), ("dx", t, B, D),
                 ("gf", R.F32, D + 1, H), ("gl", R.F32, 2, D))}

    def go(s):
        B = s["x"].B
        N.check(L.ps_ln_forward(kv.h, 0, t, s["x"].p, D, B, EPS, s["n"].p, D, s["st"].p))
        N.check(L.ps_fc_res_forward(kv.h, 0, t, R.SILU, s["n"].p, D, B, None, 0, s["z"].p, H, s["y"].p, H))
        N.check(L.ps_fc_res_backward(kv.h, 0, t, R.SILU, s["n"].p, D, s["z"].p, H, s["dy"].p, H, B, None, 0, s["dn"].p, D, s["gf"].p))
        N.check(L.ps_ln_backward(kv.h, 0, t, s["x"].p, D, s["st"].p, s["dn"].p, D, B, s["x"].p, D, s["dx"].p, D, s["gl"].p))
    outs = ("n", "st", "z", "y", "dn", "dx", "gf", "gl")
    small, big = make(B), make(3 * B)
    # recording a first call would have to make the workspace: refused
    hip("hipStreamBeginCapture", stream, 2)
    assert L.ps_ln_backward(kv.h, 0, t, small["x"].p, D, small["st"].p, small["dn"].p, D, B, None, 0, small["dx"].p, D, small["gl"].p) == N.PS_E_STATE
    assert L.ps_ln_backward(kv.h, 0, t, small["x"].p, D, small["st"].p, small["dn"].p, D, B, None, 0, small["dx"].p, D, None) == N.PS_E_UNSUPPORTED
    g = C.c_void_p()
    hip("hipStreamEndCapture", stream, C.byref(g))
    execs = []
    for s in (small, big):                                        # the second one's workspace is larger: the first graph keeps its own
        go(s)
        kv.sync()
        hip("hipStreamBeginCapture", stream, 2)
        go(s)
        assert L.ps_fc_res_backward(kv.h, 0, t, R.NONE, s["n"].p, D, None, 0, s["dy"].p, H, s["x"].B, None, 0, None, 0, None) == N.PS_E_UNSUPPORTED
        hip("hipStreamEndCapture", stream, C.byref(g))
        e = C.c_void_p()
        hip("hipGraphInstantiate", C.byref(e), g, None, None, C.c_size_t(0))
        execs.append(e)
    for rnd in range(4):
        for s, e in zip((small, big), execs):
            for k in ("x", "dy"):
                s[k].view(s[k].host)[:] = R.encode(rng.standard_normal((s[k].B, s[k].w)), t)
                N.check(L.ps_dev_upload(kv.h, s[k].buf, s[k].host.ctypes.data, s[k].host.nbytes))
            hip("hipGraphLaunch", e, stream)
            kv.sync()
            replay = {k: s[k].raw() for k in outs}
            go(s)
            kv.sync()
            for k in outs:
                np.testing.assert_array_equal(s[k].raw().view(np.uint8), replay[k].view(np.uint8), err_msg=k)
    for e in execs:
        hip("hipGraphExecDestroy", e)
    for r in pool.all:
        r.free()
    pool.all = []
    kv.close()
    hip("hipStreamDestroy", stream)


def test_recording_behind_a_training_step(pool):
    """a fused step's last join lies outside a graph: the call is refused while recording, the join is not lost, and what follows is whole"""
    import ps_amd
    from ps_amd import native as N
    L, kv, hip = N.lib(), pool.kv, Hip()
    F, D, X, V, B = 4, 8, 5, 50, 512
    rng = np.random.default_rng(3)
    kv.create_embedding([V] * F, D)
    m = ps_amd.DNN.buildModel(F, D, X, [32, 16, 1], store=kv, max_batch=B)
    kv.create_ln(0, 32)
    x, y = pool.rows(R.F32, B, 32, values=rng.standard_normal((B, 32))), pool.rows(R.F32, B, 32)
    stream = C.c_void_p()
    hip("hipStreamCreateWithFlags", C.byref(stream), 1)
    kv.set_stream(stream)
    b = ps_amd.DeviceBatch(kv, rng.integers(0, V, (B, F)), rng.standard_normal((B, X)), (rng.random(B) < 0.3).astype(f32))
    for _ in range(3):
        m.train_async(b)
    hip("hipStreamBeginCapture", stream, 2)
    rc = L.ps_ln_forward(kv.h, 0, R.F32, x.p, 32, B, EPS, y.p, 32, None)
    g = C.c_void_p()
    hip("hipStreamEndCapture", stream, C.byref(g))
    assert rc in (N.PS_OK, N.PS_E_STATE)                          # (a store that joins by events has nothing left to join)
    kv.sync()
    N.check(L.ps_ln_forward(kv.h, 0, R.F32, x.p, 32, B, EPS, y.p, 32, None))
    xv = x.get()
    within(y.get(), R.ln_forward(xv, 1.0, 0.0, f32(EPS))[0], R.ln_forward_tol(xv, np.ones(32), np.zeros(32), f32(EPS), R.F32)[0], "y")
    assert np.isfinite(m.train(b))
    b.close()
    m.close()
    for r in pool.all:
        r.free()
    pool.all = []
    kv.close()
    hip("hipStreamDestroy", stream)


def test_refusals(pool):
    from ps_amd import native as N
    L, kv = N.lib(), pool.kv
    kv.create_ln(0, 16); kv.create_fc(0, 16, 8)
    B = 4
    x, y, n, st, z, g = (pool.rows(R.F32, B, w) for w in (16, 16, 8, 2, 8, 200))
    big = pool.rows(R.F32, B, 64)

    def lnf(layer=0, ty=0, xp=x.p, ldx=16, B=B, eps=EPS, yp=y.p, ldy=16, sp=st.p):
        return L.ps_ln_forward(kv.h, layer, ty, xp, ldx, B, eps, yp, ldy, sp)

    def lnb(layer=0, ty=0, xp=x.p, sp=st.p, dp=y.p, B=B, kp=None, dxp=big.p, lddx=16, gp=g.p):
        return L.ps_ln_backward(kv.h, layer, ty, xp, 16, sp, dp, 16, B, kp, 16, dxp, lddx, gp)

    def fcf(layer=0, ty=0, act=0, xp=x.p, ldx=16, B=B, rp=None, ldr=8, zp=None, yp=n.p, ldy=8):
        return L.ps_fc_res_forward(kv.h, layer, ty, act, xp, ldx, B, rp, ldr, zp, 8, yp, ldy)

    def fcb(layer=0, ty=0, act=0, xp=x.p, zp=None, dp=n.p, B=B, kp=None, dxp=big.p, lddx=16, gp=g.p):
        return L.ps_fc_res_backward(kv.h, layer, ty, act, xp, 16, zp, 8, dp, 8, B, kp, 16, dxp, lddx, gp)
    assert (lnf(), lnb(), fcf(), fcb()) == (0, 0, 0, 0)
    for f in (lnf, lnb, fcf, fcb):
        assert f(layer=1) == N.PS_MISSING and f(layer=-1) == N.PS_MISSING
        assert f(ty=3) == N.PS_E_BAD_ARG and f(ty=-1) == N.PS_E_BAD_ARG
        assert f(B=0) == N.PS_E_BAD_ARG and f(B=-5) == N.PS_E_BAD_ARG and f(xp=None) == N.PS_E_BAD_ARG
        assert f(xp=x.p + 2) == N.PS_E_BAD_ARG and f(ty=1, xp=x.p + 1) == N.PS_E_BAD_ARG
    assert lnf(yp=None) == fcf(yp=None) == lnb(dp=None) == fcb(dp=None) == lnb(sp=None) == N.PS_E_BAD_ARG
    assert lnf(ldx=15) == lnf(ldy=15) == fcf(ldx=15) == fcf(ldy=7) == lnb(lddx=15) == fcb(lddx=3) == fcf(rp=big.p, ldr=7) == N.PS_E_BAD_ARG
    assert lnf(eps=-1.0) == lnf(eps=float("nan")) == N.PS_E_BAD_ARG and lnf(eps=0.0) == 0
    assert fcf(act=2) == fcb(act=2) == N.PS_E_UNSUPPORTED and fcf(act=5) == fcb(act=-1) == N.PS_E_BAD_ARG
    for a in (1, 3, 4):
        assert fcb(act=a) == N.PS_E_BAD_ARG and fcb(act=a, zp=z.p) == 0
    assert lnb(kp=x.p, dxp=None) == fcb(kp=x.p, dxp=None) == N.PS_E_BAD_ARG
    # overlaps: in place only where it is allowed, and views into the same rows may interleave
    assert lnf(yp=x.p, ldy=16) == 0 and lnf(xp=big.p, ldx=16, yp=big.p + 64, ldy=16) == N.PS_E_BAD_ARG
    assert lnf(xp=big.p, ldx=32, yp=big.p + 64, ldy=32, B=2) == 0 and lnf(xp=big.p, ldx=32, yp=big.p + 60, ldy=32, B=2) == N.PS_E_BAD_ARG
    assert lnf(xp=big.p + 64, ldx=32, yp=big.p, ldy=32, B=2) == 0 and lnf(xp=big.p + 60, ldx=32, yp=big.p, ldy=32, B=2) == N.PS_E_BAD_ARG
    assert fcf(yp=x.p) == N.PS_E_BAD_ARG and fcf(rp=n.p) == 0 and fcf(zp=n.p) == N.PS_E_BAD_ARG and fcf(zp=x.p) == N.PS_E_BAD_ARG
    assert fcb(dxp=x.p) == fcb(dxp=n.p) == N.PS_E_BAD_ARG and fcb(kp=big.p) == 0 and lnb(dxp=x.p) == N.PS_E_BAD_ARG
    assert lnb(gp=big.p) == fcb(gp=x.p) == lnf(sp=x.p) == lnb(sp=big.p) == N.PS_E_BAD_ARG
    assert lnb(gp=g.p + 1) == lnf(sp=st.p + 2) == N.PS_E_BAD_ARG
    assert lnb(gp=st.p) == lnb(gp=st.p + 4) == N.PS_E_BAD_ARG             # the gradient over the statistics
    assert L.ps_store_create_ln(kv.h, 0, 17) == N.PS_E_STATE
    for layer, dims in ((-1, 8), (64, 8), (1, 0), (1, -3), (1, (1 << 20) + 1)):
        assert L.ps_store_create_ln(kv.h, layer, dims) == N.PS_E_BAD_ARG
    # nothing of the above has left a pending gradient
    assert L.ps_ln_update(kv.h, 0) == N.PS_MISSING and L.ps_dense_update(kv.h, 0) == N.PS_MISSING

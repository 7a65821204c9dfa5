"""Every product kernel of the residual tower with everything a call can ask of it -- the pre-activation kept, a residual, a skipped
gradient, results over their own residual or skip, rows at any stride and alignment -- and its gradients over many rows.

All values are small integers, so that every sum is exact in f32 in any order (below 2^24) and a result is the exact one rounded once:
the comparisons are for equality, and one row too few, one too many or one taken twice is seen however many rows there are.  (Gradients
are means: the exact sum divided by the batch, one more f32 rounding.)"""
import numpy as np
import pytest

import tower_ref as R
from test_gpu_tower import Pool, ld_, p_

pytestmark = pytest.mark.gpu
f32 = np.float32
T16 = [R.BF16, R.F16]


@pytest.fixture
def pool():
    p = Pool()
    yield p
    p.close()


def ints(rng, *shape):
    return rng.integers(-2, 3, shape).astype(np.float64)


def same(got, want, t, what):
    """want: exact; stored in the type with one rounding"""
    want = R.rounded(want, t)
    bad = got != want
    assert not bad.any(), "%s: %d of %d wrong, first at %s: %s for %s" % (what, bad.sum(), bad.size, np.argwhere(bad)[0], got[bad][0], want[bad][0])


def mean(total, B):
    return total.astype(f32) / f32(B)


# the kernel that each size is there for (kernels_fcres.hip nt_plan, nt_kind, fc_tn_plan): forward, or dx where the name says so
SIZES = [
    ("few_4rows", R.F32, 150, 61, 800), ("few_2rows", R.F32, 146, 130, 330), ("few_dx", R.F32, 90, 246, 19),
    ("tiles64", R.F32, 1300, 37, 650), ("tiles64_dx_both", R.F32, 1500, 650, 700), ("tiles128", R.F32, 4100, 48, 4000), ("tiles128_dx", R.F32, 4100, 4001, 45),
] + [(n, t, *s) for t in T16 for n, s in (
    ("few_4rows", (150, 61, 800)), ("few_dx", (90, 246, 19)), ("tiles64", (1000, 200, 500)), ("tiles64_dx_both", (1000, 500, 520)),
    ("split", (700, 2051, 700)), ("split_dx", (690, 700, 2056)), ("tiles128", (65600, 33, 200)), ("tiles128_dx", (65600, 200, 33)),
    ("big128", (8200, 200, 600)), ("big128_whole_steps", (8200, 192, 641)), ("big256", (16400, 200, 603)), ("big256_dx", (16400, 603, 200)),
    ("big256_one_step", (16500, 40, 520)), ("big128_narrow", (33000, 64, 100)), ("big128_dx_narrow", (33000, 100, 64)), ("big128_under_a_piece", (33000, 7, 5)))]


@pytest.mark.parametrize("pad,shift", [(0, 0), (8, 8), (5, 3)])
@pytest.mark.parametrize("name,t,B,K,N_", SIZES)
def test_every_product_with_everything(pool, name, t, B, K, N_, pad, shift):
    from ps_amd import native as N
    L, kv = N.lib(), pool.kv
    rng = np.random.default_rng(B + 3 * K + N_ + pad)
    w, b = ints(rng, K, N_), ints(rng, N_)
    kv.create_fc(2, K, N_)
    kv.put("fc2.weights", w)
    kv.put("fc2.bias", b)
    x, r, dy, sk = ints(rng, B, K), ints(rng, B, N_), ints(rng, B, N_), ints(rng, B, K)
    a = R.NONE if name == "tiles128_dx" else R.RELU          # (dz behind an activation lies in aligned rows, which take the big tiles)
    rows = lambda w, v=None: pool.rows(t, B, w, w + pad, shift, v)       # noqa: E731
    xr, rr, zr, yr = rows(K, x), rows(N_, r), rows(N_), rows(N_)
    z = x @ w + b
    y = np.maximum(z, 0) if a else z
    N.check(L.ps_fc_res_forward(kv.h, 2, t, a, xr.p, xr.ld, B, rr.p, rr.ld, zr.p, zr.ld, yr.p, yr.ld))
    same(yr.get(), y + r, t, "y with a residual")
    same(zr.get(), z, t, "z")
    N.check(L.ps_fc_res_forward(kv.h, 2, t, a, xr.p, xr.ld, B, rr.p, rr.ld, None, 0, rr.p, rr.ld))
    same(rr.get(untouched=False), y + r, t, "y over the residual")
    N.check(L.ps_fc_res_forward(kv.h, 2, t, a, xr.p, xr.ld, B, None, 0, None, 0, yr.p, yr.ld))
    same(yr.get(), y, t, "y")
    dyr, skr, dxr, gr = rows(N_, dy), rows(K, sk), rows(K), pool.rows(R.F32, K + 1, N_)
    dz = dy * (R.rounded(z, t) > 0) if a else dy
    dx, total = dz @ w.T, np.concatenate([x, np.ones((B, 1))], 1).T @ dz

    def back(skip, out, grad):
        N.check(L.ps_fc_res_backward(kv.h, 2, t, a, xr.p, xr.ld, zr.p if a else None, zr.ld, dyr.p, dyr.ld, B, p_(skip), ld_(skip), p_(out), ld_(out), grad.p))
    back(skr, dxr, gr)
    same(dxr.get(), dx + sk, t, "dx with a skip")
    np.testing.assert_array_equal(gr.get(), mean(total, B))
    back(skr, skr, gr)
    same(skr.get(untouched=False), dx + sk, t, "dx over the skip")
    back(None, dxr, gr)
    same(dxr.get(), dx, t, "dx")
    g2 = pool.rows(R.F32, K + 1, N_)
    back(None, None, g2)
    np.testing.assert_array_equal(g2.get(), mean(total, B))
    for what, q in (("x", xr), ("dy", dyr), ("z", zr)):          # inputs are inputs, and what lies around them is nobody's
        q.get() if q is zr else np.testing.assert_array_equal(q.raw().view(np.uint8), q.host.view(np.uint8), err_msg=what)


@pytest.mark.parametrize("t", [R.F32, R.BF16, R.F16])
@pytest.mark.parametrize("B,K,N_", [(1, 64, 64), (31, 64, 64), (33, 70, 20), (63, 64, 130), (65, 40, 9), (257, 300, 260), (1025, 429, 512), (4096, 429, 512),
                                    (20000, 64, 1), (8191, 520, 264), (40000, 72, 200), (33000, 64, 256), (40000, 40, 296), (35003, 328, 77), (33100, 200, 128),
                                    (10950, 520, 776), (17000, 603, 517), (20001, 301, 333), (100000, 64, 64), (65537, 5, 3), (70001, 33, 17)])
def test_gradients_count_every_row_once(pool, t, B, K, N_):
    """parts of the batch, their borders, and the ragged last step of each kernel for dW and db"""
    from ps_amd import native as N
    L, kv = N.lib(), pool.kv
    rng = np.random.default_rng(B + K)
    kv.create_fc(0, K, N_)
    x, dy = ints(rng, B, K), ints(rng, B, N_)
    want = mean(np.concatenate([x, np.ones((B, 1))], 1).T @ dy, B)
    for pad in (0, 3):
        xr, dyr, gr = pool.rows(t, B, K, K + pad, pad, x), pool.rows(t, B, N_, N_ + pad, pad, dy), pool.rows(R.F32, K + 1, N_)
        N.check(L.ps_fc_res_backward(kv.h, 0, t, R.NONE, xr.p, xr.ld, None, 0, dyr.p, dyr.ld, B, None, 0, None, 0, gr.p))
        np.testing.assert_array_equal(gr.get(), want)
    # into the pending sum, twice: f32 adds of what the first call left
    for _ in range(2):
        N.check(L.ps_fc_res_backward(kv.h, 0, t, R.NONE, xr.p, xr.ld, None, 0, dyr.p, dyr.ld, B, None, 0, None, 0, None))
    import ctypes as C
    cnt, out = C.c_int(), np.empty((K, N_), f32)
    N.check(L.ps_fc_pending_grad(kv.h, 0, 0, out.ctypes.data_as(C.POINTER(C.c_float)), out.size, C.byref(cnt)))
    assert cnt.value == 2
    np.testing.assert_array_equal(out, want[:-1] + want[:-1])


@pytest.mark.parametrize("t", [R.F32, R.BF16, R.F16])
@pytest.mark.parametrize("B,D", [(1, 8), (3, 5), (255, 24), (257, 31), (70001, 9), (20011, 24), (9000, 130), (4097, 512), (2600, 1030), (513, 2048), (700, 4100), (300, 8192),
                                 (2049, 8200), (520, 9001)])
def test_ln_gradients_count_every_row_once(pool, t, B, D):
    """dgamma and dbeta: with mean 0 and 1 / sqrt(var + eps) = 1 given as the statistics, x is its own normalised value"""
    from ps_amd import native as N
    L, kv = N.lib(), pool.kv
    rng = np.random.default_rng(B + D)
    kv.create_ln(0, D)
    x, dy = ints(rng, B, D), ints(rng, B, D)
    want = mean(np.stack([(x * dy).sum(0), dy.sum(0)]), B)
    st = pool.rows(R.F32, B, 2, values=np.tile([0.0, 1.0], (B, 1)))
    for pad in (0, 3):
        xr, dyr, gr = pool.rows(t, B, D, D + pad, pad, x), pool.rows(t, B, D, D + pad, pad, dy), pool.rows(R.F32, 2, D)
        N.check(L.ps_ln_backward(kv.h, 0, t, xr.p, xr.ld, st.p, dyr.p, dyr.ld, B, None, 0, None, 0, gr.p))
        np.testing.assert_array_equal(gr.get(), want)

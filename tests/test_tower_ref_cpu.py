"""tests/tower_ref.py against itself on the CPU: its gradients against differences of its forward passes, its rounding against the
types' definitions; and the refusals of the residual tower's entry points that need no device."""
import numpy as np
import pytest

import tower_ref as R


@pytest.mark.parametrize("a", [R.NONE, R.RELU, R.GELU, R.SILU])
def test_fc_gradients_are_the_differences(a):
    rng = np.random.default_rng(a)
    B, K, N, h = 5, 7, 6, 1e-6
    x, w, b = rng.standard_normal((B, K)), R.rounded(rng.standard_normal((K, N)), R.F32), rng.standard_normal(N)      # (the store's weights are f32)
    r, c = rng.standard_normal((B, N)), rng.standard_normal((B, N))

    def loss(x, w, b):
        return (c * (R.act(x @ w + b, a) + r)).sum()
    dx, grad, _, _ = R.fc_backward(x, w, x @ w + b, c, a, None, R.F32)
    for _ in range(4):
        vx, vw, vb = rng.standard_normal(x.shape), rng.standard_normal(w.shape), rng.standard_normal(N)
        num = (loss(x + h * vx, w + h * vw, b + h * vb) - loss(x - h * vx, w - h * vw, b - h * vb)) / (2 * h)
        got = (dx * vx).sum() + B * ((grad[:-1] * vw).sum() + (grad[-1] * vb).sum())
        assert abs(num - got) < 1e-7 * (1 + abs(num))


def test_ln_gradients_are_the_differences():
    rng = np.random.default_rng(1)
    B, D, h, eps = 4, 9, 1e-6, 1e-5
    x, g, b, c = rng.standard_normal((B, D)), rng.standard_normal(D), rng.standard_normal(D), rng.standard_normal((B, D))
    _, mean, rstd = R.ln_forward(x, g, b, eps)
    dx, grad = R.ln_backward(x, mean, rstd, g, c, None)
    for _ in range(4):
        vx, vg, vb = rng.standard_normal(x.shape), rng.standard_normal(D), rng.standard_normal(D)
        num = ((c * R.ln_forward(x + h * vx, g + h * vg, b + h * vb, eps)[0]).sum() - (c * R.ln_forward(x - h * vx, g - h * vg, b - h * vb, eps)[0]).sum()) / (2 * h)
        assert abs(num - ((dx * vx).sum() + B * ((grad[0] * vg).sum() + (grad[1] * vb).sum()))) < 1e-7 * (1 + abs(num))


def test_types_round_to_nearest_even():
    one = np.float32(1)
    steps = np.array([1, 1 + 2.0 ** -8, 1 + 3 * 2.0 ** -8, 1 + 2.0 ** -8 + 2.0 ** -20], np.float32)
    np.testing.assert_array_equal(R.rounded(steps, R.BF16), [1, 1, 1 + 2.0 ** -6, 1 + 2.0 ** -7])
    np.testing.assert_array_equal(R.rounded(np.array([one + 2.0 ** -11, one + 3 * 2.0 ** -11]), R.F16), [1, 1 + 2.0 ** -9])
    assert np.isnan(R.rounded(np.array([np.nan]), R.BF16))[0] and np.isinf(R.rounded(np.array([1e6]), R.F16))[0]


def test_refusals_without_a_store():
    from ps_amd import native as N
    L = N.lib()
    p = 64                                     # a non-null pointer that nothing follows
    assert L.ps_store_create_ln(None, 0, 8) == N.PS_E_BAD_ARG
    assert L.ps_ln_forward(None, 0, 0, p, 8, 1, 1e-5, p, 8, None) == N.PS_E_BAD_ARG
    assert L.ps_ln_backward(None, 0, 0, p, 8, p, p, 8, 1, None, 0, None, 0, None) == N.PS_E_BAD_ARG
    assert L.ps_fc_res_forward(None, 0, 0, 0, p, 8, 1, None, 0, None, 0, p, 8) == N.PS_E_BAD_ARG
    assert L.ps_fc_res_backward(None, 0, 0, 0, p, 8, None, 0, p, 8, 1, None, 0, None, 0, None) == N.PS_E_BAD_ARG
    assert L.ps_ln_update(None, 0) == N.PS_E_BAD_ARG
    assert b"NULL" in L.ps_last_error()


def test_python_layers_refuse_what_they_cannot_pass_on():
    torch = pytest.importorskip("torch")
    import ps_amd
    from ps_amd import api, native as N

    class Store:                               # stands for a store on device 0; none of these calls gets as far as the library
        h, device = None, 0

        def create_ln(self, *a):
            pass

        def create_fc(self, *a):
            pass
    ln, fc = ps_amd.LnLayer(Store(), 0, 8), ps_amd.FcResLayer(Store(), 0, 8, 4)
    x = torch.zeros(3, 8)
    for call in (lambda: ln.forward(x), lambda: fc.forward(x),                      # host memory
                 lambda: ln.forward(x.double()), lambda: fc.forward(x.int())):      # a type that is none of the three
        with pytest.raises(N.PsError) as e:
            call()
        assert e.value.code == N.PS_E_BAD_ARG
    assert api._mat(torch.zeros(3, 11)[:, :8], "x", 3, 8)[1] == 11
    assert api._mat(torch.zeros(1, 11)[:, :8], "x", 1, 8)[1] == 8
    for t in (torch.zeros(3, 7), torch.zeros(2, 8), torch.zeros(3, 8, 1), torch.zeros(8, 3).t(), torch.zeros(3, 16)[:, ::2]):
        with pytest.raises(N.PsError):
            api._mat(t, "x", 3, 8)
    with pytest.raises(N.PsError):
        api._mat(x.half(), "dy", 3, 8, x)
    with pytest.raises(N.PsError):
        api._f32(torch.zeros(3, 4)[:, :2], "stats", (3, 2), x)

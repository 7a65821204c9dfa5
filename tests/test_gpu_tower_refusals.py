"""Calls beside the residual tower's that its names make possible: refused, not answered as something else."""
import ctypes as C

import numpy as np
import pytest

import tower_ref as R
from test_gpu_tower import EPS, Hip, Pool

pytestmark = pytest.mark.gpu


@pytest.fixture
def pool():
    p = Pool()
    yield p
    p.close()


def test_the_reference_layers_refuse_the_towers_activations(pool):
    """ps_fc_forward and its like know relu, the clipped sigmoid and none; GELU and SiLU had passed for none"""
    from ps_amd import native as N
    L, kv = N.lib(), pool.kv
    kv.create_fc(0, 16, 8)
    kv.create_embedding([10, 10], 8)
    B, k = 4, 32                                             # (in + 1 rounded up to 16)
    x, y, d = pool.rows(R.F32, B, k), pool.rows(R.F32, B, 16), pool.rows(R.F32, B, 16)
    ids = pool.rows(R.F32, B, 4)                             # (never read: the call is refused before)
    for a in (N.PS_ACT_GELU, N.PS_ACT_SILU):
        assert L.ps_fc_forward(kv.h, 0, a, x.p, k, B, y.p, 16) == N.PS_E_UNSUPPORTED
        assert L.ps_fc_backward(kv.h, 0, a, x.p, k, y.p, 16, d.p, 16, B, None, 0) == N.PS_E_UNSUPPORTED
        assert L.ps_emb_forward(kv.h, ids.p, None, B, a, y.p, 16) == N.PS_E_UNSUPPORTED
        assert L.ps_emb_backward_update(kv.h, ids.p, None, 2 * B, B, a, y.p, 16, d.p, 16, 0, 0, 1) == N.PS_E_UNSUPPORTED
    assert L.ps_dense_update(kv.h, 0) == N.PS_MISSING        # nothing was added up
    for r in (x, y, d, ids):
        assert (r.raw().view("u1") == r.host.view("u1")).all()


def test_an_update_of_a_pending_gradient_is_not_recorded(pool):
    """what adds to a normalisation's pending gradient is refused while a graph is recorded; an update in the graph would apply the one
    that lay there at every replay.  The refusal leaves the recording whole and the gradient pending."""
    from ps_amd import native as N
    L, kv, hip = N.lib(), pool.kv, Hip()
    B, D = 8, 24
    kv.create_ln(0, D)
    x, y, st = pool.rows(R.F32, B, D, values=np.arange(B * D).reshape(B, D)), pool.rows(R.F32, B, D), pool.rows(R.F32, B, 2)
    stream, g = C.c_void_p(), C.c_void_p()
    hip("hipStreamCreateWithFlags", C.byref(stream), 1)
    kv.set_stream(stream)
    N.check(L.ps_ln_forward(kv.h, 0, R.F32, x.p, D, B, EPS, y.p, D, st.p))
    N.check(L.ps_ln_backward(kv.h, 0, R.F32, x.p, D, st.p, x.p, D, B, None, 0, None, 0, None))
    before, step = kv.get("ln0.weights"), kv.global_step()
    hip("hipStreamBeginCapture", stream, 2)
    assert L.ps_ln_update(kv.h, 0) == N.PS_E_UNSUPPORTED and L.ps_dense_update(kv.h, -1) == N.PS_E_UNSUPPORTED
    N.check(L.ps_ln_forward(kv.h, 0, R.F32, x.p, D, B, EPS, y.p, D, st.p))
    hip("hipStreamEndCapture", stream, C.byref(g))
    assert g.value and kv.global_step() == step
    np.testing.assert_array_equal(kv.get("ln0.weights"), before)
    kv.dense_update()
    assert kv.global_step() == step + 1 and (kv.get("ln0.weights") != before).any() and L.ps_ln_update(kv.h, 0) == N.PS_MISSING
    hip("hipGraphDestroy", g)
    for r in pool.all:
        r.free()
    pool.all = []
    kv.close()
    hip("hipStreamDestroy", stream)

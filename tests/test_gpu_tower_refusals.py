"""Calls beside the residual tower's that its names make possible: refused, not answered as something else."""
import pytest

import tower_ref as R
from test_gpu_tower import Pool

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

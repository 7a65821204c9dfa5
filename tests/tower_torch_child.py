"""Run by test_gpu_tower_torch.py in a process of its own: torch has to come first, so that it and libps_amd share one HIP runtime."""
import os
import sys

import torch

HERE = os.path.dirname(os.path.abspath(__file__))
sys.path[:0] = [os.path.dirname(HERE), HERE]
import numpy as np  # noqa: E402

import ps_amd  # noqa: E402
import tower_ref as R  # noqa: E402
from ps_amd import native as N  # noqa: E402

TYPES = {R.F32: torch.float32, R.BF16: torch.bfloat16, R.F16: torch.float16}


def n64(t):
    return t.detach().double().cpu().numpy()


def ok(got, want, tol, what):
    bad = ~(np.abs(n64(got) - want) <= tol)
    assert not bad.any(), (what, int(bad.sum()), bad.size)
    print("ok", what, flush=True)


def refused(code, f):
    try:
        f()
    except N.PsError as e:
        assert e.code == code, (e.code, code, e)
        return
    raise AssertionError("not refused")


def block(kv, t):
    """one pre-norm block on strided tensors: forward, backward against the definitions, and against autograd in 64 bits"""
    dt, B, D, H = TYPES[t], 77, 96, 136
    ln = ps_amd.LnLayer(kv, 0, D)
    up, down = ps_amd.FcResLayer(kv, 0, D, H, act=N.PS_ACT_GELU), ps_amd.FcResLayer(kv, 1, H, D)
    buf = torch.randn(B, D + 5, device="cuda").to(dt)
    r = buf[:, 3:3 + D]
    st, z = torch.empty(B, 2, device="cuda"), torch.empty(B, H + 2, dtype=dt, device="cuda")[:, :H]
    x = ln.forward(r, stats=st)
    h = up.forward(x, z=z)
    y = down.forward(h, res=r)
    w = {k: kv.get(k).astype(np.float64) for k in ("ln0.weights", "ln0.bias", "fc0.weights", "fc0.bias", "fc1.weights", "fc1.bias")}
    w["fc0.weights"] = w["fc0.weights"].reshape(D, H); w["fc1.weights"] = w["fc1.weights"].reshape(H, D)
    ok(x, R.ln_forward(n64(r), w["ln0.weights"], w["ln0.bias"], np.float32(1e-5))[0], R.ln_forward_tol(n64(r), w["ln0.weights"], w["ln0.bias"], np.float32(1e-5), t)[0], "ln")
    yy, zz, ty, tz = R.fc_forward(n64(x), w["fc0.weights"], w["fc0.bias"], R.GELU, None, t)
    ok(h, yy, ty, "up"); ok(z, zz, tz, "z")
    yy, _, ty, _ = R.fc_forward(n64(h), w["fc1.weights"], w["fc1.bias"], R.NONE, n64(r), t)
    ok(y, yy, ty, "down")
    dy = torch.randn(B, D, device="cuda").to(dt)
    g1, g0, gl = torch.empty(H + 1, D, device="cuda"), torch.empty(D + 1, H, device="cuda"), torch.empty(2, D, device="cuda")
    dh = down.backward(h, None, dy, grad=g1)
    dx = up.backward(x, z, dh, grad=g0)
    dr = ln.backward(r, st, dx, skip=dy, grad=gl)
    assert down.backward(h, None, dy, want_dx=False) is None
    pend, cnt = down.pending_grad()
    assert cnt == 1 and np.array_equal(pend, n64(g1)[:-1].astype(np.float32)) and ln.pending_grad() == (None, 0)
    down.update()
    assert down.pending_grad(bias=True) == (None, 0)
    if t == R.F32:
        p = {k: torch.tensor(v, requires_grad=True) for k, v in w.items()}
        rr = torch.tensor(n64(r), requires_grad=True)
        xx = torch.nn.functional.layer_norm(rr, (D,), p["ln0.weights"], p["ln0.bias"], 1e-5)
        out = rr + torch.nn.functional.gelu(xx @ p["fc0.weights"] + p["fc0.bias"]) @ p["fc1.weights"] + p["fc1.bias"]
        out.backward(torch.tensor(n64(dy)))
        # a chain of four f32 operators of up to 136 terms each: 1e-4 of the largest gradient is far above their roundings and far
        # below any term left out
        for got, want in ((dr, rr.grad), (gl[0] * B, p["ln0.weights"].grad), (gl[1] * B, p["ln0.bias"].grad), (g0[:-1] * B, p["fc0.weights"].grad),
                          (g0[-1] * B, p["fc0.bias"].grad), (g1[:-1] * B, p["fc1.weights"].grad), (g1[-1] * B, p["fc1.bias"].grad)):
            assert np.abs(n64(got) - want.numpy()).max() <= 1e-4 * want.abs().max().item()
        print("ok autograd", flush=True)


def refusals(kv):
    ln, fc = ps_amd.LnLayer(kv, 0, 96), ps_amd.FcResLayer(kv, 0, 96, 136, act=N.PS_ACT_RELU)
    x = torch.zeros(4, 96, device="cuda")
    st, z = torch.zeros(4, 2, device="cuda"), torch.zeros(4, 136, device="cuda")
    refused(N.PS_E_BAD_ARG, lambda: ln.forward(x.cpu()))
    refused(N.PS_E_BAD_ARG, lambda: ln.forward(x.double()))
    refused(N.PS_E_BAD_ARG, lambda: ln.forward(x[:0]))
    refused(N.PS_E_BAD_ARG, lambda: ln.forward(x, y=torch.zeros(4, 96, device="cuda", dtype=torch.bfloat16)))
    refused(N.PS_E_BAD_ARG, lambda: ln.forward(x, stats=torch.zeros(4, 4, device="cuda")[:, :2]))
    refused(N.PS_E_BAD_ARG, lambda: ln.backward(x, st.double(), x))
    refused(N.PS_E_BAD_ARG, lambda: fc.backward(x, None, z))
    refused(N.PS_E_BAD_ARG, lambda: fc.backward(x, z, z, grad=torch.zeros(96, 136, device="cuda")))
    refused(N.PS_E_BAD_ARG, lambda: fc.forward(x, y=x))
    refused(N.PS_E_STATE, lambda: ps_amd.LnLayer(kv, 0, 97))
    print("ok refusals", flush=True)


def streams(kv):
    """the store's stream is torch's current one; work behind it on that stream sees the results"""
    s = torch.cuda.Stream()
    kv.set_stream(s.cuda_stream)
    fc = ps_amd.FcResLayer(kv, 0, 96, 136, act=N.PS_ACT_GELU)
    with torch.cuda.stream(s):
        x = torch.randn(3000, 96, device="cuda")
        outs = [fc.forward(x * k) for k in range(1, 5)]
        sums = [o.sum() for o in outs]
    s.synchronize()
    for o, t in zip(outs, sums):
        assert torch.allclose(o.sum(), t)
    # recorded with torch's own graphs
    y, g, dx = torch.empty(3000, 136, device="cuda"), torch.empty(97, 136, device="cuda"), torch.empty(3000, 96, device="cuda")
    z = torch.empty_like(y)
    with torch.cuda.stream(s):
        def go():
            fc.forward(x, z=z, y=y)
            fc.backward(x, z, y, dx=dx, grad=g)
        go()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            go()
        for k in range(3):
            x.normal_()
            graph.replay()
            got = [t.clone() for t in (y, z, dx, g)]
            go()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, (y, z, dx, g)))
    kv.set_stream(torch.cuda.current_stream().cuda_stream)
    print("ok streams", flush=True)


def cases():
    """the listed calls' small relatives: the timed file's own path through the layers agrees with its plain path"""
    import random

    from perf import operators as P
    rng = random.Random(5)
    for i in range(24):
        case = P.draw(rng)
        case["B"] = min(case["B"], 500)
        for k in ("K", "N"):
            if k in case:
                case[k] = min(case[k], 700)
        P.own = False
        plain, exact = P.run(P.prepare(case, i)), P.exact(case, i)
        P.own = True
        here = P.run(P.prepare(case, i))
        P.own = False
        for a, b, e in zip(plain, here, exact):
            assert a.shape == b.shape and a.dtype == b.dtype, case
            na, nb, ne = n64(a), n64(b), n64(e)
            scale = np.sqrt((ne ** 2).mean()) + 1e-30
            ea, eb = np.sqrt(((na - ne) ** 2).mean()) / scale, np.sqrt(((nb - ne) ** 2).mean()) / scale
            # no worse than the plain form by more than an f32 sum's own noise
            assert eb <= 1.2 * ea + 2e-6, (case, ea, eb)
    print("ok cases", flush=True)


if __name__ == "__main__":
    torch.manual_seed(1)
    store = ps_amd.KVStore(0, 7)
    store.set_stream(torch.cuda.current_stream().cuda_stream)
    for ty in TYPES:
        block(store, ty)
    refusals(store)
    streams(store)
    cases()
    store.close()
    print("all done", flush=True)

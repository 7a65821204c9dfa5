"""Run by test_gpu_tower_streams.py in a process of its own: torch has to come first, so that it and libps_amd share one HIP runtime."""
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import ps_amd  # noqa: E402
from ps_amd import native as N  # noqa: E402

B, D, H = 2048, 512, 384


def block(ln, up, down, x, dy):
    """forward and backward of a block in fresh tensors, every temporary dropped at once: torch hands its memory on"""
    st, z = torch.empty(B, 2, device="cuda"), torch.empty(B, H, device="cuda")
    h = up.forward(ln.forward(x, stats=st), z=z)
    y = down.forward(h, res=x)
    g1, g0, gl = torch.empty(H + 1, D, device="cuda"), torch.empty(D + 1, H, device="cuda"), torch.empty(2, D, device="cuda")
    n = ln.forward(x)
    dx = up.backward(n, z, down.backward(h, None, dy, grad=g1), grad=g0)
    del n, h
    return [y, ln.backward(x, st, dx, skip=dy, grad=gl), g1, g0, gl]


def late(a, k):
    """a tensor that is there only after some milliseconds of work on the current stream"""
    m = a
    for _ in range(k):
        m = torch.mm(m, EYE)
    return m


def check(kv, what):
    ln, up, down = ps_amd.LnLayer(kv, 0, D), ps_amd.FcResLayer(kv, 0, D, H, act=N.PS_ACT_GELU), ps_amd.FcResLayer(kv, 1, H, D)
    src = [torch.randn(B, D, device="cuda") for _ in range(6)]
    dy = torch.randn(B, D, device="cuda")
    torch.cuda.synchronize()
    # what a program that waits after every step gets
    want = []
    for a in src:
        w = block(ln, up, down, a, dy)
        torch.cuda.synchronize()
        want.append([t.clone() for t in w])
        torch.cuda.synchronize()
    # one that waits for nothing: inputs still being made, outputs used at once, memory handed on
    got = []
    for a in src:
        outs = block(ln, up, down, late(a, 40), dy)
        got.append([t * 1.0 for t in outs])
        del outs
        junk = [torch.full((B, D), float("nan"), device="cuda") for _ in range(8)]
        del junk
    torch.cuda.synchronize()
    for w, g in zip(want, got):
        assert all(torch.equal(p, q) for p, q in zip(w, g)), what
    print("ok", what, flush=True)


if __name__ == "__main__":
    torch.manual_seed(3)
    EYE = torch.eye(D, device="cuda")
    own = ps_amd.KVStore(0, 7)                     # on a stream of its own
    check(own, "a store on its own stream, torch on the default one")
    s, other = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(s):
        check(own, "a store on its own stream, torch on another")
    kv = ps_amd.KVStore(0, 7)
    kv.set_stream(other.cuda_stream)
    with torch.cuda.stream(s):
        check(kv, "a store on a stream that torch has left")
    with torch.cuda.stream(other):
        check(kv, "a store on torch's stream")
    check(kv, "torch back on the default stream")
    # a recording torch stream that is not the store's: refused, and the graph is whole
    ln = ps_amd.LnLayer(kv, 0, D)
    x, y, n = torch.randn(B, D, device="cuda"), torch.empty(B, D, device="cuda"), torch.zeros(4, device="cuda")
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        with torch.cuda.graph(g, stream=s):
            n.add_(1)
            try:
                ln.forward(x, y=y)
                raise SystemExit("not refused")
            except N.PsError as e:
                assert e.code == N.PS_E_STATE, e
    for _ in range(3):
        g.replay()
    torch.cuda.synchronize()
    assert n.tolist() == [3.0] * 4
    # adopted, it is recorded
    kv.set_stream(s.cuda_stream)
    with torch.cuda.stream(s):
        ln.forward(x, y=y)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            ln.forward(x, y=y)
        for _ in range(3):
            x.normal_()
            g.replay()
            got = y.clone()
            assert torch.equal(got, ln.forward(x))
    assert N.lib().ps_store_order(kv.h, s.cuda_stream, 0) == N.PS_OK and N.lib().ps_store_order(None, None, 0) == N.PS_E_BAD_ARG
    print("ok graphs", flush=True)
    torch.cuda.synchronize()
    own.close()
    kv.close()
    print("all done", flush=True)

"""Run by test_gpu_tower_large.py in a process of its own: torch has to come first, so that it and libps_amd share one HIP runtime."""
import os
import sys

import torch

import numpy as np

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import ps_amd  # noqa: E402
from ps_amd import native as N  # noqa: E402

T = torch.bfloat16


def ints(*shape):
    """-1, 0, 1: sums of 4.3 million products of them are exact in f32"""
    return torch.randint(-1, 2, shape, device="cuda", dtype=torch.int8).to(T)


def column_sums(x, dy):
    """the exact sums over the rows of x * dy and of dy"""
    a, b = 0, 0
    for i in range(0, x.shape[0], 1 << 19):
        p, q = x[i:i + (1 << 19)].float(), dy[i:i + (1 << 19)].float()
        a, b = a + (p * q).sum(0, dtype=torch.float64), b + q.sum(0, dtype=torch.float64)
    return a, b


def mean(total, B):
    """divided in f32, once (torch multiplies by a number's reciprocal)"""
    return total.cpu().numpy().astype(np.float32) / np.float32(B)


def layer_norm(kv, B, D):
    ln = ps_amd.LnLayer(kv, 0, D)
    x, dy = ints(B, D), ints(B, D)
    st = torch.empty(B, 2, device="cuda")
    y = ln.forward(x, stats=st)
    for rows in (slice(0, 1000), slice(B // 2, B // 2 + 1000), slice(B - 1000, B)):
        s2 = torch.empty(1000, 2, device="cuda")
        assert torch.equal(ln.forward(x[rows].clone(), stats=s2), y[rows]) and torch.equal(s2, st[rows])      # a row's result is its own
    st[:, 0] = 0
    st[:, 1] = 1
    g = torch.empty(2, D, device="cuda")
    dx = ln.backward(x, st, dy, grad=g, dx=y)
    a, b = column_sums(x, dy)
    assert (g.cpu().numpy() == mean(torch.stack([a, b]), B)).all()
    for rows in (slice(0, 1000), slice(B - 1000, B)):
        assert torch.equal(ln.backward(x[rows].clone(), st[rows].clone(), dy[rows].clone(), grad=torch.empty_like(g)), dx[rows])
    print("ok ln", B, D, flush=True)


def fc(kv, layer, B, K, H):
    up = ps_amd.FcResLayer(kv, layer, K, H, act=N.PS_ACT_RELU)
    w, b = torch.randint(-1, 2, (K, H)).float(), torch.randint(-1, 2, (H,)).float()
    kv.put("fc%d.weights" % layer, w.numpy())
    kv.put("fc%d.bias" % layer, b.numpy())
    w, b = w.cuda(), b.cuda()
    x, r, dy = ints(B, K), ints(B, H), ints(B, H)
    z = torch.empty(B, H, device="cuda", dtype=T)
    y = up.forward(x, res=r, z=z)
    g = torch.empty(K + 1, H, device="cuda")
    dx = up.backward(x, z, dy, grad=g)
    total = torch.zeros(K + 1, H, device="cuda", dtype=torch.float64)
    for i in range(0, B, 1 << 19):
        rows = slice(i, min(B, i + (1 << 19)))
        xf = x[rows].float()
        zz = xf @ w + b
        assert torch.equal(zz.to(T), z[rows]) and torch.equal((torch.relu(zz) + r[rows].float()).to(T), y[rows]), i
        dz = dy[rows].float() * (z[rows] > 0)
        assert torch.equal((dz @ w.t()).to(T), dx[rows]), i
        total[:K] += (xf.t() @ dz).double()
        total[K] += dz.sum(0)
    assert (g.cpu().numpy() == mean(total, B)).all()
    print("ok fc", B, K, H, flush=True)


def recorded(kv, layer, s, B, K, H):
    """the 256-wide kernels with their workspace (cast weights, dz, slabs): replays give what eager calls between them give"""
    up = ps_amd.FcResLayer(kv, layer, K, H, act=N.PS_ACT_GELU)
    x, dy, sk = (torch.randn(B, n, device="cuda").to(T) for n in (K, H, K))
    z, y, dx, g = torch.empty(B, H, device="cuda", dtype=T), torch.empty(B, H, device="cuda", dtype=T), torch.empty_like(x), torch.empty(K + 1, H, device="cuda")

    def go():
        up.forward(x, z=z, y=y)
        up.backward(x, z, dy, skip=sk, dx=dx, grad=g)
    go()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        go()
    for k in range(4):
        x.normal_()
        dy.normal_()
        graph.replay()
        got = [t.clone() for t in (y, z, dx, g)]
        torch.cuda.synchronize()
        for t in (y, z, dx, g):
            t.zero_()
        go()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, (y, z, dx, g))), k
    print("ok recorded", B, K, H, flush=True)


if __name__ == "__main__":
    torch.manual_seed(4)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        kv = ps_amd.KVStore(0, 7)
        kv.set_stream(s.cuda_stream)
        recorded(kv, 3, s, 16500, 600, 520)
        recorded(kv, 4, s, 9001, 603, 517)       # off the 16-byte grid: copies in the workspace
        layer_norm(kv, 4300001, 1001)
        torch.cuda.empty_cache()
        fc(kv, 0, 4300001, 1001, 16)
        torch.cuda.empty_cache()
        fc(kv, 1, 4200001, 1024, 24)
        torch.cuda.synchronize()
        kv.close()
    print("all done", flush=True)

"""What is timed of the residual tower's operators: layer normalisation (LnLayer) and the fully connected layer with bias,
activation and residual in one call (FcResLayer), each forward and backward.

Both keep f32 parameters in the store; the activations are f32, bf16 or f16 ("type").  By definition a 16-bit product takes
the weights, and in the backward pass the gradient behind the activation, rounded to the activations' type; everything else is
f32 and rounded once.  Parameter gradients are means over the batch, as everywhere in this framework.

    ln_fwd   y = (x - mean) / sqrt(var + eps) * gamma + beta, and (mean, 1 / sqrt(var + eps)) of every row when training
    ln_bwd   dx (plus the gradient that came round the skip connection), dgamma, dbeta
    fc_fwd   z = x W + b, y = act(z) + r
    fc_bwd   dz = dy act'(z), dx = dz W^T (plus the skip's gradient), dW = x^T dz / B, db = mean of dz
"""
import math

import numpy as np
import torch

own = False

EPS = 1e-5
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
ACTS = {"none": 0, "relu": 1, "gelu": 3, "silu": 4}


def _ln(name, op, B, D, type, train=True, skip=False, pad=0):
    return {"name": name, "op": op, "B": B, "D": D, "type": type, "train": train, "skip": skip, "pad": pad}


def _fc(name, op, B, K, N, type, act, train=False, skip=False, pad=0):
    return {"name": name, "op": op, "B": B, "K": K, "N": N, "type": type, "act": act, "train": train, "skip": skip, "pad": pad}


def listed():
    return [
        # one request being answered: nothing but latency
        _ln("ln_fwd_one", "ln_fwd", 1, 512, "f32", train=False),
        # the concatenated input of Wide&Deep (26 fields x 16 + 13 dense columns) at its batch: an odd width
        _ln("ln_fwd_ctr", "ln_fwd", 4096, 429, "f32"),
        # a wide tower over a large batch of stored activations
        _ln("ln_fwd_wide", "ln_fwd", 65536, 1024, "bf16"),
        # the CTR example's input (23 fields x 10 + 45 dense columns) at its batch of 1000, training
        _ln("ln_bwd_ctr", "ln_bwd", 1000, 275, "f32"),
        # the wide tower's training step: the gradient that skipped the block is added on the way
        _ln("ln_bwd_wide", "ln_bwd", 65536, 1024, "bf16", skip=True),
        # one request through Wide&Deep's first layer
        _fc("fc_fwd_one", "fc_fwd", 1, 429, 512, "f32", "relu"),
        # a handful of candidates through a wide block's second product
        _fc("fc_fwd_few", "fc_fwd", 16, 2048, 2048, "bf16", "none", skip=True),
        # Wide&Deep's first layer at the training batch, in the framework's own type
        _fc("fc_fwd_ctr", "fc_fwd", 4096, 429, 512, "f32", "relu", train=True),
        # the expanding product of a wide block in training: the pre-activation is kept
        _fc("fc_fwd_wide", "fc_fwd", 32768, 1024, 4096, "bf16", "gelu", train=True),
        # its contracting product, which closes the residual; a ragged last batch
        _fc("fc_fwd_down", "fc_fwd", 8191, 4096, 1024, "f16", "none", skip=True),
        # Wide&Deep's second layer, mixed precision
        _fc("fc_bwd_ctr", "fc_bwd", 4096, 512, 256, "bf16", "relu"),
        # the expanding product's gradients: the largest case
        _fc("fc_bwd_wide", "fc_bwd", 32768, 1024, 4096, "bf16", "gelu", skip=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["ln_fwd", "ln_bwd", "fc_fwd", "fc_bwd"])
    type = rng.choice(["f32", "bf16", "f16"])
    pad = rng.choice([0, 0, 0, 3, 8])
    B = _log(rng, 1, 65536)
    if op.startswith("ln"):
        D = _log(rng, 8, 8192)
        B = min(B, 65536 * 1024 // D)
        return dict(_ln("", op, B, D, type, train=op == "ln_bwd" or rng.random() < 0.5, skip=op == "ln_bwd" and rng.random() < 0.5, pad=pad))
    K, N = _log(rng, 8, 4096), _log(rng, 8, 4096)
    # f32 products run at a sixteenth of the 16-bit rate: the same time, not the same size
    most = 32768 * 1024 * 4096 // (16 if type == "f32" else 1)
    B = max(1, min(B, most // (K * N)))
    act = rng.choice(["none", "relu", "gelu", "silu"])
    train = act != "none" and (op == "fc_bwd" or rng.random() < 0.5)
    return dict(_fc("", op, B, K, N, type, act, train=train, skip=rng.random() < 0.5, pad=pad))


def _rows(g, B, D, t, pad):
    """[B][D] normal values inside rows of D + pad"""
    return torch.randn(B, D + pad, generator=g, device="cuda").to(t)[:, :D]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    t, pad, B = TYPES[case["type"]], case["pad"], case["B"]
    s = {"case": case, "type": t}
    if case["op"].startswith("ln"):
        D = case["D"]
        s["gamma"] = 1 + 0.2 * torch.randn(D, generator=g, device="cuda")
        s["beta"] = 0.2 * torch.randn(D, generator=g, device="cuda")
        # columns of different scale and offset, as concatenated embeddings and dense features have
        scale = 0.5 + torch.rand(D + pad, generator=g, device="cuda")
        offset = 0.5 * torch.randn(D + pad, generator=g, device="cuda")
        s["x"] = (torch.randn(B, D + pad, generator=g, device="cuda") * scale + offset).to(t)[:, :D]
        if case["op"] == "ln_bwd":
            xf = s["x"].float()
            mean = xf.mean(1, keepdim=True)
            rstd = 1 / torch.sqrt(((xf - mean) ** 2).mean(1, keepdim=True) + EPS)
            s["stats"] = torch.cat([mean, rstd], 1).contiguous()       # what the forward pass left
            s["dy"] = _rows(g, B, D, t, pad)
            s["skip"] = _rows(g, B, D, t, pad) if case["skip"] else None
    else:
        K, N = case["K"], case["N"]
        s["w"] = torch.randn(K, N, generator=g, device="cuda") / math.sqrt(K)
        s["b"] = 0.2 * torch.randn(N, generator=g, device="cuda")
        s["x"] = _rows(g, B, K, t, pad)
        if case["op"] == "fc_fwd":
            s["r"] = _rows(g, B, N, t, pad) if case["skip"] else None
        else:
            s["z"] = _rows(g, B, N, t, pad) if case["act"] != "none" else None
            s["dy"] = _rows(g, B, N, t, pad)
            s["skip"] = _rows(g, B, K, t, pad) if case["skip"] else None
    if own:
        # the store that holds the layer's parameters, on this program's stream
        import ps_amd
        kv = ps_amd.KVStore(0, 1)
        kv.set_stream(torch.cuda.current_stream().cuda_stream)
        if case["op"].startswith("ln"):
            s["layer"] = ps_amd.LnLayer(kv, 0, case["D"], eps=EPS)
            kv.put("ln0.weights", s["gamma"].cpu().numpy())
            kv.put("ln0.bias", s["beta"].cpu().numpy())
        else:
            s["layer"] = ps_amd.FcResLayer(kv, 0, case["K"], case["N"], act=ACTS[case["act"]])
            kv.put("fc0.weights", s["w"].cpu().numpy())
            kv.put("fc0.bias", s["b"].cpu().numpy())
    return s


def _act(z, act):
    if act == "relu":
        return torch.maximum(z, torch.zeros_like(z))
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if act == "silu":
        return z / (1 + torch.exp(-z))
    return z


def _act_grad(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    p = 1 / (1 + torch.exp(-z))
    return p * (1 + z * (1 - p))


def _plain(s):
    case, t, op = s["case"], s["type"], s["case"]["op"]
    x = s["x"].float()
    if op == "ln_fwd":
        mean = x.mean(1, keepdim=True)
        d = x - mean
        rstd = 1 / torch.sqrt((d * d).mean(1, keepdim=True) + EPS)
        y = (d * rstd * s["gamma"] + s["beta"]).to(t)
        return [y, torch.cat([mean, rstd], 1)] if case["train"] else [y]
    if op == "ln_bwd":
        dy, mean, rstd = s["dy"].float(), s["stats"][:, :1], s["stats"][:, 1:]
        h = (x - mean) * rstd
        p = dy * s["gamma"]
        dx = rstd * (p - p.mean(1, keepdim=True) - h * (p * h).mean(1, keepdim=True))
        if s["skip"] is not None:
            dx = dx + s["skip"].float()
        return [dx.to(t), torch.stack([(dy * h).mean(0), dy.mean(0)])]
    w = s["w"].to(t).float()
    if op == "fc_fwd":
        z = x @ w + s["b"]
        y = _act(z, case["act"])
        if s["r"] is not None:
            y = y + s["r"].float()
        return [y.to(t), z.to(t)] if case["train"] else [y.to(t)]
    dz = s["dy"].float()
    if s["z"] is not None:
        dz = (dz * _act_grad(s["z"].float(), case["act"])).to(t).float()
    dx = dz @ w.t()
    if s["skip"] is not None:
        dx = dx + s["skip"].float()
    B = case["B"]
    return [dx.to(t), torch.cat([(x.t() @ dz) / B, dz.sum(0, keepdim=True) / B])]


def run(state):
    if not own:
        return _plain(state)
    case, layer, x = state["case"], state["layer"], state["x"]
    op, B = case["op"], case["B"]
    if op == "ln_fwd":
        if not case["train"]:
            return [layer.forward(x)]
        stats = torch.empty(B, 2, device=x.device)
        return [layer.forward(x, stats=stats), stats]
    if op == "ln_bwd":
        grad = torch.empty(2, case["D"], device=x.device)
        return [layer.backward(x, state["stats"], state["dy"], skip=state["skip"], grad=grad), grad]
    if op == "fc_fwd":
        if not case["train"]:
            return [layer.forward(x, res=state["r"])]
        z = torch.empty(B, case["N"], dtype=x.dtype, device=x.device)
        return [layer.forward(x, res=state["r"], z=z), z]
    grad = torch.empty(case["K"] + 1, case["N"], device=x.device)
    return [layer.backward(x, state["z"], state["dy"], skip=state["skip"], grad=grad), grad]


def work(case):
    es, B = 4 if case["type"] == "f32" else 2, case["B"]
    if case["op"].startswith("ln"):
        D = case["D"]
        if case["op"] == "ln_fwd":
            return {"bytes": 2 * B * D * es + 8 * D + (8 * B if case["train"] else 0), "flops": 8 * B * D}
        return {"bytes": (3 + case["skip"]) * B * D * es + 8 * B + 12 * D, "flops": 16 * B * D}
    K, N = case["K"], case["N"]
    if case["op"] == "fc_fwd":
        return {"bytes": es * B * (K + N * (1 + case["train"] + case["skip"])) + 4 * (K + 1) * N, "flops": 2 * B * K * N}
    return {"bytes": es * B * (K * (2 + case["skip"]) + N * (1 + (case["act"] != "none"))) + 4 * (2 * K + 1) * N, "flops": 4 * B * K * N}


def exact(case, seed):
    """The same from the definitions in 64 bits: matrix forms with a centring matrix's effect written out, erfc for the normal law"""
    s = prepare(case, seed)
    t, B = s["type"], case["B"]
    x = s["x"].double()
    if case["op"] == "ln_fwd":
        var, mean = torch.var_mean(x, dim=1, correction=0, keepdim=True)
        rstd = (var + EPS).pow(-0.5)
        y = torch.addcmul(s["beta"].double(), (x - mean) * s["gamma"].double(), rstd)
        return [y, torch.cat([mean, rstd], 1)] if case["train"] else [y]
    if case["op"] == "ln_bwd":
        D = case["D"]
        st = s["stats"].double()
        h = torch.addcmul(-st[:, :1] * st[:, 1:], x, st[:, 1:])
        dy = s["dy"].double()
        p = dy * s["gamma"].double()
        c1, c2 = p.sum(1) / D, torch.linalg.vecdot(p, h) / D
        dx = st[:, 1:] * (p - (c1[:, None] + h * c2[:, None]))
        if case["skip"]:
            dx += s["skip"].double()
        return [dx, torch.stack([torch.linalg.vecdot(dy, h, dim=0), dy.sum(0)]) / B]
    w = s["w"].to(t).double()
    if case["op"] == "fc_fwd":
        z = torch.addmm(s["b"].double(), x, w)
        y = z
        if case["act"] == "relu":
            y = z.clamp(min=0)
        elif case["act"] == "gelu":
            y = 0.5 * z * torch.special.erfc(-z / math.sqrt(2.0))
        elif case["act"] == "silu":
            y = z * torch.special.expit(z)
        if case["skip"]:
            y = y + s["r"].double()
        return [y, z] if case["train"] else [y]
    dz = s["dy"].double()
    if case["act"] != "none":
        z = s["z"].double()
        if case["act"] == "relu":
            d = torch.where(z > 0, 1.0, 0.0)
        elif case["act"] == "gelu":
            d = 0.5 * torch.special.erfc(-z / math.sqrt(2.0)) + z * torch.exp(-z.square() / 2) / math.sqrt(2 * np.pi)
        else:
            e = torch.special.expit(z)
            d = e + z * e * torch.special.expit(-z)
        dz = (dz * d).to(t).double()
    dx = torch.matmul(dz, w.transpose(0, 1))
    if case["skip"]:
        dx = dx + s["skip"].double()
    ones = torch.ones(B, 1, dtype=torch.float64, device=x.device)
    return [dx, torch.matmul(torch.cat([x, ones], 1).transpose(0, 1), dz) / B]

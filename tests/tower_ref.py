"""The residual tower's operators restated in 64 bits (numpy), with the error bounds their tests use.

u = 2^-24 is half a step of f32, half(t) half a step of the activations' type (bf16 2^-8, fp16 2^-11, f32 u).  A sum of n terms
formed in f32 in any order is off by at most (n - 1) u times the sum of the terms' magnitudes; a product and each further operation
add one u.  A result that is stored in a 16-bit type is rounded once more: half(t) times its magnitude (f16 below 2^-14: half of 2^-24)."""
import numpy as np
from scipy.special import erf

U = 2.0 ** -24
F32, BF16, F16 = 0, 1, 2
HALF = {F32: 0.0, BF16: 2.0 ** -8, F16: 2.0 ** -11}        # beyond the f32 arithmetic itself
TINY = {F32: 0.0, BF16: 0.0, F16: 2.0 ** -25}
NONE, RELU, GELU, SILU = 0, 1, 3, 4


def encode(a, t):
    """float array -> the type's bits (round to nearest even)"""
    a = np.ascontiguousarray(a, np.float32)
    if t == F32:
        return a
    if t == F16:
        with np.errstate(over="ignore"):
            return a.astype(np.float16)
    b = a.view(np.uint32)
    r = ((b + np.uint32(0x7FFF) + ((b >> np.uint32(16)) & np.uint32(1))) >> np.uint32(16)).astype(np.uint16)
    return np.where(np.isnan(a), np.uint16(0x7FC0), r)


def decode(a, t):
    """the type's bits -> float64"""
    if t == BF16:
        return (a.astype(np.uint32) << np.uint32(16)).view(np.float32).astype(np.float64)
    return a.astype(np.float64)


def rounded(a, t):
    """a (any float) as the nearest value of the type, float64"""
    return decode(encode(a, t), t)


def store_tol(y, t):
    return HALF[t] * np.abs(y) + TINY[t]


# ---- layer normalisation
def ln_forward(x, gamma, beta, eps):
    mean = x.mean(1, keepdims=True)
    rstd = 1 / np.sqrt(((x - mean) ** 2).mean(1, keepdims=True) + eps)
    return (x - mean) * rstd * gamma + beta, mean, rstd


def ln_chain(D):
    """longest chain of dependent adds of a row's sum: a lane's own elements (at most 32; D / 256 in the walking kernel), 6 steps
    over the lanes, 2 over the waves"""
    return max(32, D // 256 + 8) + 8


def ln_forward_tol(x, gamma, beta, eps, t):
    """mean: (c + 2) u mean|x|.  d = x - mean carries that shift e and u |d|; the variance's first-order change by a common shift
    vanishes (sum d = 0), so var is off by e^2 + (c + 4) u var, rstd by half of that relative plus 2 u.  y = d rstd gamma + beta."""
    c = ln_chain(x.shape[1])
    y, mean, rstd = ln_forward(x, gamma, beta, eps)
    e = (c + 2) * U * np.abs(x).mean(1, keepdims=True)
    var = ((x - mean) ** 2).mean(1, keepdims=True)
    rel = 0.5 * (e * e / (var + eps) + (c + 4) * U) + 3 * U
    h = np.abs(x - mean) * rstd
    ty = np.abs(gamma) * (h * (rel + 3 * U) + e * rstd * (1 + rel)) + 2 * U * (np.abs(y) + np.abs(beta))
    return ty + store_tol(np.abs(y) + ty, t), e + U * np.abs(mean), rel * rstd


def ln_backward(x, mean, rstd, gamma, dy, skip):
    h, p = (x - mean) * rstd, dy * gamma
    dx = rstd * (p - p.mean(1, keepdims=True) - h * (p * h).mean(1, keepdims=True)) + (0 if skip is None else skip)
    return dx, np.stack([(dy * h).mean(0), dy.mean(0)])


def ln_backward_tol(x, mean, rstd, gamma, dy, skip, t):
    """h: 2 u |h| (the statistics are inputs); p: u |p|; the two row means: (c + 6) u of their magnitudes; then five operations.
    Column sums: a chain of at most min(B, rows a lane group sees + 64 groups of a workgroup + 1024 slabs) adds."""
    B, D = x.shape
    c = ln_chain(D)
    h, p = np.abs(x - mean) * rstd, np.abs(dy * gamma)
    mag = rstd * (p + p.mean(1, keepdims=True) + h * (p * h).mean(1, keepdims=True)) + (0 if skip is None else np.abs(skip))
    dx, _ = ln_backward(x, mean, rstd, gamma, dy, skip)
    tol = (c + 12) * U * mag
    n = min(B, B // 256 + 64 + 1024) + 6
    return tol + store_tol(np.abs(dx) + tol, t), n * U * np.stack([(np.abs(dy) * h).mean(0), np.abs(dy).mean(0)])


# ---- FC with bias, activation, residual
def act(z, a):
    if a == RELU:
        return np.where(z < 0, 0.0, z)
    if a == GELU:
        return 0.5 * z * (1 + erf(z / np.sqrt(2.0)))
    if a == SILU:
        return z / (1 + np.exp(-z))
    return z


def act_grad(z, a):
    if a == RELU:
        return (z > 0).astype(np.float64)
    if a == GELU:
        return 0.5 * (1 + erf(z / np.sqrt(2.0))) + z * np.exp(-z * z / 2) / np.sqrt(2 * np.pi)
    if a == SILU:
        p = 1 / (1 + np.exp(-z))
        return p * (1 + z * (1 - p))
    return np.ones_like(z)


def fc_forward(x, w, b, a, r, t):
    """(y, z, tol_y, tol_z); w as the store holds it (f32): the product takes it rounded to the type"""
    w = rounded(w, t)
    z = x @ w + b
    tz = (x.shape[1] + 2) * U * (np.abs(x) @ np.abs(w) + np.abs(b))
    y = act(z, a) + (0 if r is None else r)
    # |act'| < 1.13 for all four; the function itself: a few operations and a library call of at most 4 u relative to |z|, then r's add
    ty = 1.13 * tz + (0 if a in (NONE, RELU) else 8 * U * np.abs(z)) + 2 * U * (np.abs(y) + (0 if r is None else np.abs(r)))
    return y, z, ty + store_tol(np.abs(y) + ty, t), tz + store_tol(np.abs(z) + tz, t)


def fc_backward(x, w, z, dy, a, skip, t):
    """(dx, grad [K + 1][N], tol_dx, tol_grad).  dz is rounded to the type; where it was computed rather than selected (GELU, SILU) the
    f32 value may fall to the other side of a border, so it counts as the unrounded value off by half a step plus its f32 error."""
    B = x.shape[0]
    w = rounded(w, t)
    if a in (NONE, RELU):
        dz, tdz = dy * act_grad(z, a), 0.0 * dy
    else:
        dz = dy * act_grad(z, a)
        f = np.abs(dy) * 12 * U * (1 + np.abs(z))          # p (1 + z (1 - p)) and Phi + z phi: operations on terms of at most 1 + |z|
        tdz = f + (HALF[t] if t != F32 else 0) * (np.abs(dz) + f) + TINY[t]
    N = dz.shape[1]
    dx = dz @ w.T + (0 if skip is None else skip)
    mag = np.abs(dz) @ np.abs(w).T + (0 if skip is None else np.abs(skip))
    tdx = (N + 2) * U * mag + tdz @ np.abs(w).T * (1 + (N + 2) * U)
    ones = np.concatenate([x, np.ones((B, 1))], 1)
    grad = ones.T @ dz / B
    tg = ((B + 3) * U * (np.abs(ones).T @ np.abs(dz)) + np.abs(ones).T @ tdz * (1 + (B + 3) * U)) / B
    return dx, grad, tdx + store_tol(np.abs(dx) + tdx, t), tg

"""The polynomial behind GELU's kernels, read from their source and evaluated in f32 arithmetic, against the normal law's tail."""
import os
import re

import numpy as np
from scipy.special import ndtr

f32 = np.float32


def tail(x):
    """kernels_fcres.hip normal_tail: a multiply-add rounds once (the double arithmetic in between is exact to far below f32's step)"""
    src = open(os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "ps_amd", "csrc", "kernels_fcres.hip")).read()
    body = re.search(r"float normal_tail\(float z\) \{(.*?)\n\}", src, re.S).group(1)
    number = r"(-?[0-9.]+(?:e-?[0-9]+)?)f"
    lead, second = re.search(r"float p = fmaf\(%s, x, %s\);" % (number, number), body).groups()
    rest = re.findall(r"p = fmaf\(p, x, %s\);" % number, body)
    last = re.search(r"exp2f\(fmaf\(p, x, %s\)\)" % number, body).group(1)
    x = x.astype(f32).astype(np.float64)
    p = np.full_like(x, f32(float(lead)))
    for c in [second] + rest + [last]:
        with np.errstate(over="ignore"):          # (far beyond 8: to minus infinity)
            p = (p * x + float(f32(float(c)))).astype(f32).astype(np.float64)
    return np.exp2(p).astype(f32).astype(np.float64), len(rest) + 2


def test_gelu_tail_keeps_its_bounds():
    x = np.linspace(0, 13, 260001).astype(f32)
    q, n = tail(x)
    assert n == 10
    want = ndtr(-x.astype(np.float64))
    err = np.abs(q - want)
    assert err.max() < 5e-8
    for top, rel in ((2, 1e-6), (3, 6e-6), (4, 4e-5), (8, 4e-4)):
        assert (err / want)[x <= top].max() < rel, top
    # beyond 8 it is smaller than it should be, and falls to 0
    far, _ = tail(np.concatenate([np.linspace(8.01, 70, 10000), [1e3, 1e10, 3e38]]).astype(f32))
    assert (np.diff(far) <= 0).all() and far[0] < 7e-16 and far[-1] == 0 and (q[x > 8] <= want[x > 8] * 1.0005).all()

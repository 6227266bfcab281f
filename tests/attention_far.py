"""Inputs whose scores are whole numbers that fp32 holds exactly, however they are summed, and whose scale makes the kernels'
exponents (base 2) exact too: q = (2^12, b, 0, ..), k = (+-2^11, t, 0, ..) with small whole b and t, so that a score is +-2^23 +
b t. log2(e) is folded into the scale in fp32, and fp32(ln 2) times fp32(log2 e) rounds to 1: the scale ln 2 times a power of
two gives exponents of that power of two times whole numbers.

Bound of an output, u half a step of the values' type: probabilities are rounded to the type (u, and fp16 ones below 2^-14 by up
to 2^-25 each), exponentials and fp32 sums over n keys are off by 2^-20 + n 2^-24 relative, the output is rounded (u, at least
2^-25 for fp16).
"""
import math

import numpy as np
import torch

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
LN2 = float(np.float32(math.log(2)))
assert np.float32(LN2) * np.float32(1.4426950408889634) == np.float32(1)


def scale_of(power):
    """the scale whose exponents are 2^power times the scores"""
    return LN2 * 2.0 ** power


def fill_queries(q, g):
    q.zero_()
    q[..., 0] = 4096
    q[..., 1] = torch.randint(-1, 3, q.shape[:-1], device=q.device, generator=g).to(q.dtype)


def fill_keys(k, t, sign=1):
    """t: whole numbers, of k's shape without its last dimension"""
    k.zero_()
    k[..., 0] = sign * 2048
    k[..., 1] = t.to(k.dtype)


def rows(q, k, v, seen, power):
    """q [r][d], k, v [n][d], seen [r][n] -> (o, bound of o, lse, bound of lse) in 64 bits"""
    n = k.shape[0]
    s = (q.double() @ k.double().T).masked_fill(~seen, -math.inf)
    top = s.amax(1, keepdim=True)
    p = torch.exp2((s - top) * 2.0 ** power)
    l = p.sum(1, keepdim=True)
    vd = v.double()
    o, a = p @ vd / l, p @ vd.abs() / l
    u, e = HALF_STEP[q.dtype], 2.0 ** -20 + n * 2.0 ** -24
    small = (n * 2.0 ** -25 * vd.abs().max() + 2.0 ** -25) if q.dtype == torch.float16 else 0.0
    lse = (top * 2.0 ** power + torch.log2(l)) * math.log(2)
    return o, (u + 2 * e) * 1.02 * a + u * o.abs() * 1.02 + small, lse[:, 0], 2.0 ** -22 * (1 + lse.abs())[:, 0] + e


def check(out, lse, want, what):
    o, ob, l, lb = want
    assert torch.isfinite(out).all() and torch.isfinite(lse).all(), what
    assert ((out.double() - o).abs() <= ob).all(), f"{what}: off by {((out.double() - o).abs() / ob).max().item():.3f} bounds"
    assert ((lse.double() - l).abs() <= lb).all(), f"{what}: lse off by {((lse.double() - l).abs() / lb).max().item():.3f} bounds"

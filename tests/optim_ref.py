"""Plain float64 restatement of the list optimizer step (include/prl_optim.h) on CPU tensors, and
the bounds on how far a float32 evaluation of it may be off: used by test_optim_gpu.py and checked by
itself in test_optim_cpu.py."""
import math

import torch

U32 = 2.0 ** -24          # half a float32 step, relative
HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def norm64(grads):
    return math.sqrt(sum(float(g.double().square().sum()) for g in grads))


def clip64(norm, max_norm):
    if max_norm is None:
        return 1.0
    c = max_norm / (norm + 1e-6)
    return c if math.isnan(c) else min(1.0, c)


def draws(n, t, first=0):
    """The two 16-bit draws of values first .. first + n - 1 of a tensor at step t."""
    i = torch.arange(first, first + n, dtype=torch.int64)
    M = 2 ** 32
    h = ((i % M) + (i // M) * 0x85EBCA77) % M
    h = h ^ (t * 0x9E3779B1 % M)
    h = (h ^ (h // 2 ** 16)) * 0x7FEB352D % M
    h = (h ^ (h // 2 ** 15)) % M
    h = torch.tensor([int(x) * 0x846CA68B % M for x in h.tolist()], dtype=torch.int64)
    h = h ^ (h // 2 ** 16)
    return h % 65536, h // 65536


def quantise(x, draw, least, err=None):
    """(scales, codes' values, least, most) of the flat float64 x in blocks of 256: the values that may
    be held where x is known up to an error of `err` lie between the last two (rounding with a
    given draw is monotonous), signs taken off."""
    n = x.numel()
    pad = torch.zeros(-(-n // 256) * 256, dtype=torch.float64)
    pad[:n] = x
    A = pad.view(-1, 256).abs().amax(1)
    A = torch.where(A < 2.0 ** -118, torch.zeros_like(A), A)
    k = torch.where(A > 0, 256.0 / A, torch.zeros_like(A)).repeat_interleave(256)[:n]

    def code(y):
        unit = torch.exp2(torch.floor(torch.log2(y.clamp(min=2.0 ** -6))) - 3)
        q = torch.floor(y / unit + draw.double() / 65536) * unit
        return torch.where((y > 0) & (q < least), torch.full_like(q, least), q)
    y = (x.abs() * k).clamp(max=256.0)
    q = code(y)
    # x's own error and the rounding of the scale and of two products
    d = (0.0 if err is None else err * k) + 4 * U32 * y + 2.0 ** -30
    return A, torch.where(x < 0, -q, q), code((y - d).clamp(min=0.0)), code((y + d).clamp(max=256.0))


def step64(w, g, m, v, t, lr, betas, eps, wd, c):
    """One step in float64; returns (w', m', v', bound on a float32 evaluation's error of each)."""
    b1, b2 = betas
    gc = g * c
    m1 = m + (1 - b1) * (gc - m)
    v1 = b2 * v + (1 - b2) * gc * gc
    step_size, bc2 = lr / (1 - b1 ** t), 1 - b2 ** t
    denom = (v1 / bc2).sqrt() + eps
    w1 = w * (1 - lr * wd) - step_size * m1 / denom
    # c: a norm rounded, a sum, a quotient (3 U); c g: 1; the difference 1, the coefficient 1, the
    # product 1, the sum 1: at most 8 U of the operands' sizes
    em = 8 * U32 * (m.abs() + gc.abs())
    # products and a sum of positive terms: c twice (6 U) + its products (2) + square, coefficients,
    # products, sum (4): at most 12 U of the result; the smallest steps of a float32 below 2^-126
    ev = 12 * U32 * v1 + 2.0 ** -148
    # the quotient takes m's error, half of v's (a root), and its own roundings: root, two coefficients,
    # product, sum, the reciprocal (1 ulp: 2 U), two products (9 U); then the decayed weight (3 U) and
    # the sum
    part = step_size * m1.abs() / denom
    ew = (step_size * em / denom + (6 + 9) * U32 * part + step_size * m1.abs() / denom ** 2 * 2.0 ** -74
          + 3 * U32 * w.abs() + U32 * w1.abs())
    return w1, m1, v1, ew, em, ev

"""64-bit references of the training-step operators and the error bounds their
tests use.

U is half a step of f32 relative to the value.  A sum of n terms whose longest
chain of additions is d long is off by at most d * U * (sum of magnitudes).
The layer norm kernels add at most N / 8 terms of a row in sequence up to 256
columns (8 lanes at least), N / 32 beyond (a warp at least), then a tree."""
from __future__ import annotations

import math

import torch

U = 2.0 ** -24
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}


def chain(n: int) -> int:
    return (n // 8 if n <= 256 else n // 32) + 16


def rounded(v: torch.Tensor, dtype) -> torch.Tensor:
    """Half a step of `dtype` at v (half the smallest subnormal at least)."""
    return v.abs() * (torch.finfo(dtype).eps / 2) + TINY[dtype] / 2


def norm_ref(x, w, b, eps):
    """(y, mean, rstd, bounds of mean and rstd and y before its rounding), 64 bits."""
    x = x.double()
    n = x.shape[-1]
    mean = x.mean(-1, keepdim=True)
    off = x - mean
    var = off.square().mean(-1, keepdim=True)
    rstd = 1 / (var + eps).sqrt()
    d = chain(n)
    e_mean = (d + 2) * U * x.abs().mean(-1, keepdim=True)
    # Each deviation is off by e_mean + U |off|; squares, their sum, the division, eps, root and reciprocal follow.
    e_var = 2 * e_mean * off.abs().mean(-1, keepdim=True) + e_mean ** 2 + (d + 6) * U * var
    r_rstd = (e_var / (var + eps)).clamp(max=1e3) * 0.5 / (1 - (e_var / (var + eps)).clamp(max=0.5)) + 6 * U
    xh = off * rstd
    e_xh = (rstd * (e_mean + U * off.abs())) * (1 + r_rstd) + xh.abs() * (r_rstd + 2 * U)
    wd = torch.ones(n, dtype=torch.float64, device=x.device) if w is None else w.double()
    y = xh * wd + (0 if b is None else b.double())
    e_y = wd.abs() * e_xh + 2 * U * ((xh * wd).abs() + y.abs())
    return y, mean[..., 0], rstd[..., 0], e_mean[..., 0], rstd[..., 0] * r_rstd[..., 0], e_y


def norm_back_ref(dy, x, mean, rstd, w):
    """(dx, dw, db, bounds of the three before their rounding), 64 bits, for the given statistics."""
    dy, x = dy.double(), x.double()
    n = x.shape[-1]
    mean, rstd = mean.double()[..., None], rstd.double()[..., None]
    xh = (x - mean) * rstd
    a = dy if w is None else dy * w.double()
    c1 = a.mean(-1, keepdim=True)
    c2 = (a * xh).mean(-1, keepdim=True)
    dx = (a - c1 - xh * c2) * rstd
    d = chain(n)
    e_c1 = (d + 3) * U * a.abs().mean(-1, keepdim=True)
    e_c2 = (d + 7) * U * (a * xh).abs().mean(-1, keepdim=True)
    e_dx = rstd * (e_c1 + xh.abs() * e_c2 + 6 * U * (a.abs() + c1.abs() + (xh * c2).abs())) + 2 * U * dx.abs()
    rows = math.prod(x.shape[:-1])
    flat = lambda t: t.reshape(rows, n)  # noqa: E731
    p = flat(dy * xh)
    dw, db = p.sum(0), flat(dy).sum(0)
    return dx, dw, db, e_dx, (rows + 20) * U * p.abs().sum(0), (rows + 16) * U * flat(dy).abs().sum(0)


def assert_within(got, want, bound, what):
    got = got.double()
    bad = ~((got - want).abs() <= bound)
    bad &= ~(got.isnan() & want.isnan())
    if bool(bad.any()):
        k = int(bad.reshape(-1).int().argmax())
        g, v, e = (t.expand(bad.shape).reshape(-1)[k].item() for t in (got, want, bound))
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} outside; first at {k}: {g!r}, exact {v!r}, bound {e:.3g}")


def adam_ref(p, g, m, v, *, step, lr, betas, eps, decay, scale=1.0):
    """(p, m, v, bounds of the three before p's rounding) after one step, 64 bits."""
    b1, b2 = betas
    p, m, v = p.double(), m.double(), v.double()
    g = g.double() * scale
    m1, v1 = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    # The factors are off by U each, g by U, products and the sum by U each.
    e_m = U * (2 * (b1 * m).abs() + 4 * ((1 - b1) * g).abs() + m1.abs()) + 2.0 ** -148
    e_v = U * (2 * (b2 * v).abs() + 7 * ((1 - b2) * g * g).abs() + v1.abs()) + 2.0 ** -148
    c1, c2 = 1 - b1 ** step, 1 - b2 ** step
    root = (v1 / c2).sqrt()
    den = root + eps
    change = lr / c1 * m1 / den
    # sqrt(v +- e) moves by at most min(e / sqrt(v), sqrt(e)).
    e_root = torch.minimum(e_v / v1.clamp(min=1e-300).sqrt(), e_v.sqrt()) / math.sqrt(c2) + 6 * U * root
    r_den = (e_root + U * den) / den
    e_change = lr / c1 * e_m / den * (1 + 2 * r_den.clamp(max=1)) + change.abs() * (8 * U + r_den / (1 - r_den.clamp(max=0.5)))
    p1 = p * (1 - lr * decay) - change
    return p1, m1, v1, 4 * U * p.abs() + e_change + 2 * U * p1.abs(), e_m, e_v

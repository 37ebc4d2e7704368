"""The row-wise operators in 64 bits, with bounds on what a kernel may be off by.

Bounds count roundings: half a step (``finfo(type).eps / 2`` of the value) for each result that is stored in fewer bits, and
for fp32 arithmetic 2^-24 for every rounding on the longest chain, relative to the sum of magnitudes that passes it.  A sum
of a row is 32 additions in a thread, 5 in a warp and 8 over the warps of a team: 45 roundings.  The mean is therefore off
by 45 * 2^-24 * mean|x| at most, the variance (second order in that) relatively by 45 * 2^-24 plus the square's 2, its root
by half of that plus 2 units, so that a normalised value is off by 64 * 2^-24 * A with A = rstd (|x| + mean|x|) >= |xh|.
"""
from __future__ import annotations

import torch

U = 2.0 ** -24
GROUP = 128
TINY = 2.0 ** -119
MAX_SCALE = float.fromhex("0x1.020406p121")     # the largest fp32 value with a finite product with 127


def half_step(dtype):
    return 0.0 if dtype == torch.float64 else torch.finfo(dtype).eps / 2


def pack(x):
    """``(codes, scales, values)`` in 64 bits; the two factors of a group are fp32 values by definition."""
    rows, cols = x.shape
    groups = -(-cols // GROUP)
    p = torch.zeros(rows, groups * GROUP, dtype=torch.float64)
    p[:, :cols] = x.double()
    p = p.view(rows, groups, GROUP)
    a = p.abs().amax(-1, keepdim=True)          # (a NaN stays)
    bad = ~torch.isfinite(a)
    empty = a < TINY
    safe = torch.where(bad | empty, 1.0, a)
    up = torch.where(empty, 0.0, 127.0 / safe).float().double()
    down = torch.where(empty, 0.0, safe / 127.0).float().double().clamp(max=MAX_SCALE)
    codes = torch.round(torch.where(bad, 0.0, p) * up)
    down = torch.where(bad, float("nan"), down)
    return (codes.view(rows, -1)[:, :cols], down.view(rows, groups), (codes * down).view(rows, -1)[:, :cols])


def pack_off(x, dtype):
    """What the values given back in ``dtype`` may be off by from x itself.  With f = (127 / a)(1 + e1), s = (a / 127)(1 + e2), code =
    x f + d, |d| <= 1/2, the value is (x (1 + e1)(1 + e2) + d (a / 127)(1 + e2))(1 + e3); |e1|, |e3| <= U, |e2| <= 2 U (U, but for the
    largest scale), |x| <= a: off by a (1 / 254 + 5 U) in fp32, below a (1 / 254 + 2^-21).  Then half a step of the type, of a
    subnormal the smallest normal's.  Groups below the smallest amax are off by all they have."""
    rows, cols = x.shape
    groups = -(-cols // GROUP)
    p = torch.zeros(rows, groups * GROUP, dtype=torch.float64)
    p[:, :cols] = x.double().abs()
    a = p.view(rows, groups, GROUP).amax(-1, keepdim=True).expand(-1, -1, GROUP).reshape(rows, -1)[:, :cols]
    off = torch.where(a < TINY, a, a * (1 / 254 + 2.0 ** -21))
    if dtype == torch.float32:
        return off
    return off + half_step(dtype) * torch.clamp(x.double().abs() + off, min=torch.finfo(dtype).tiny)


def layer_norm(x, w, b, eps):
    """``y``, ``mean``, ``rstd`` and the bound on y before it is rounded."""
    x = x.double()
    w = torch.ones(x.shape[1], dtype=torch.float64) if w is None else w.double()
    b = torch.zeros(x.shape[1], dtype=torch.float64) if b is None else b.double()
    mean = x.mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt(((x - mean) ** 2).mean(-1, keepdim=True) + eps)
    y = (x - mean) * rstd * w + b
    A = rstd * (x.abs() + x.abs().mean(-1, keepdim=True))
    return y, mean, rstd, 68 * U * (A * w.abs() + b.abs())


def layer_norm_backward(dy, kept, mean, rstd, w, dy_off=0.0):
    """Gradients and their bounds before they are rounded.  ``kept``: x as the backward pass knows it; ``dy_off``: what the
    incoming gradient itself may be off by (same shape as dy)."""
    dy, kept = dy.double(), kept.double()
    w = torch.ones(dy.shape[1], dtype=torch.float64) if w is None else w.double()
    xh = (kept - mean) * rstd
    wd = dy * w
    m = lambda t: t.mean(-1, keepdim=True)  # noqa: E731
    dx = rstd * (wd - m(wd) - xh * m(wd * xh))
    # statistics come from the true x: |mean| is at most what |kept| says up to half a step of the codes; both are covered
    A = rstd * (kept.abs() + mean.abs() + m(kept.abs()))
    off = wd.abs()
    dx_off = 192 * U * rstd * (off + m(off) + A * m(off * A))
    e = w.abs() * torch.as_tensor(dy_off, dtype=torch.float64)
    dx_off = dx_off + rstd * (e + m(e.expand_as(dy)) + A * m(e * A))
    # a column's sum: rows of a thread, teams of a CTA, CTAs: fewer than 192 additions for the sizes tested, and 64 for xh
    dw_off = ((256 * U * dy.abs() + dy_off) * A).sum(0)
    db_off = (192 * U * dy.abs() + dy_off).sum(0)
    return dict(dx=dx, dw=(dy * xh).sum(0), db=dy.sum(0), dx_off=dx_off, dw_off=dw_off, db_off=db_off)


def check(got, ref, off, name=""):
    """Every element of ``got`` within half a step of its type and ``off`` of ``ref``."""
    g, r = got.detach().cpu().double(), ref.double()
    assert g.shape == r.shape, (name, g.shape, r.shape)
    bound = off + half_step(got.dtype) * (r.abs() + off) + torch.finfo(got.dtype).tiny
    bad = (g - r).abs() > bound
    bad |= torch.isnan(g) != torch.isnan(r)
    assert not bool(bad.any()), (name, int(bad.sum()), float(((g - r).abs() / bound).nan_to_num().max()))

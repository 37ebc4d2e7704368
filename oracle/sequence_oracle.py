"""Dropout, the position rotation of heads and the window attention in 64 bits, with bounds on what a kernel may be off by.

Bounds count roundings as oracle/rows_oracle.py does: half a step of the stored type, and U = 2^-24 for each fp32 rounding on the
longest chain, relative to the sum of magnitudes that passes it.
"""
from __future__ import annotations

import math

import numpy as np
import torch

U = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def check(got, ref, off, name):
    """|got - ref| <= half a step of got's type + off, element by element; half a step of the smallest number of a type counts as well."""
    got64 = got.detach().double().to(ref.device)
    room = half_step(got.dtype) * (ref.abs() + off) + off + torch.finfo(got.dtype).smallest_normal
    bad = ~((got64 - ref).abs() <= room)
    assert not bad.any(), f"{name}: {int(bad.sum())} of {bad.numel()} values off, by up to {((got64 - ref).abs() / room).max():.3g} of their room"


# ---- dropout ---------------------------------------------------------------------------------------
def philox(seed, offset, group):
    """Philox 4x32-10 of the counter (group, offset) under the key ``seed``, in Python's whole numbers: four 32-bit words."""
    low = 2 ** 32 - 1
    c = [group & low, group >> 32, offset & low, (offset >> 32) & low]
    k = [seed & low, (seed >> 32) & low]
    for _ in range(10):
        a, b = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
        c = [(b >> 32) ^ c[1] ^ k[0], b & low, (a >> 32) ^ c[3] ^ k[1], a & low]
        k = [(k[0] + 0x9E3779B9) & low, (k[1] + 0xBB67AE85) & low]
    return c


def dropout_mask(shape, p, seed, offset=0, shared_dim=None):
    """Which elements are kept, as a bool tensor of ``shape``; group by group with numpy's 64-bit words."""
    sizes = list(shape)
    if shared_dim is not None:
        sizes[shared_dim] = 1
    count = math.prod(sizes)
    low, s32 = np.uint64(2 ** 32 - 1), np.uint64(32)
    n = np.arange(-(-count // 8), dtype=np.uint64)
    offset %= 2 ** 64
    seed %= 2 ** 64
    c = [n & low, n >> s32, np.full_like(n, offset & 0xFFFFFFFF), np.full_like(n, offset >> 32)]
    k = [seed & 0xFFFFFFFF, seed >> 32]
    for _ in range(10):
        a, b = np.uint64(0xD2511F53) * c[0], np.uint64(0xCD9E8D57) * c[2]
        c = [(b >> s32) ^ c[1] ^ np.uint64(k[0]), b & low, (a >> s32) ^ c[3] ^ np.uint64(k[1]), a & low]
        k = [(k[0] + 0x9E3779B9) % 2 ** 32, (k[1] + 0xBB67AE85) % 2 ** 32]
    halves = np.stack([h for w in c for h in (w & np.uint64(0xFFFF), w >> np.uint64(16))], 1).reshape(-1)[:count]
    kept = torch.from_numpy(halves.astype(np.int64) >= round(65536 * p))
    return kept.view(sizes).expand(shape)


def dropout(x, kept, p, residual=None):
    """``(out, off)``: the product and the sum are rounded to fp32, and so is the scale."""
    t = round(65536 * p)
    scale = 65536.0 / (65536 - t) if t < 65536 else 0.0
    y = torch.where(kept, x.double() * scale, 0.0)
    r = 0.0 if residual is None else residual.double()
    return y + r, 2 * U * y.abs() + U * (y + r).abs()


# ---- rotation --------------------------------------------------------------------------------------
def radians(dim, base=10000.0):
    return torch.tensor([base ** (-2.0 * i / dim) for i in range(dim // 2)], dtype=torch.float64)


def pairs(rot, half):
    at = torch.arange(rot)
    return (at[:rot // 2], at[rot // 2:]) if half else (at[0::2], at[1::2])


def rotate(x, f, positions, half, magnitude=1.0, back=False):
    """x ``[..., N, H, D]``, positions ``[..., N]`` (whole numbers), f radians a position."""
    a, b = pairs(2 * f.numel(), half)
    t = positions.double()[..., None, None] * f.to(x.device)
    c, s = magnitude * torch.cos(t), magnitude * torch.sin(t) * (-1 if back else 1)
    y = x.double().clone()
    y[..., a] = x[..., a].double() * c - x[..., b].double() * s
    y[..., b] = x[..., a].double() * s + x[..., b].double() * c
    return y


def pair_size(x, rot, half, magnitude=1.0):
    """|a| + |b| of every rotated element, |x| of the others: what the roundings of a rotation are relative to."""
    a, b = pairs(rot, half)
    m = x.double().abs()
    r = m.clone()
    r[..., a] = r[..., b] = magnitude * (m[..., a] + m[..., b])
    return r


# A cosine or sine: the phase is cut off at 2^-32 of a turn (0.03 U) and rounded to fp32 (half turns up to 1: pi / 2 * 2 U = 3.2 U at
# most), sincospi is good to 2 U, the magnitude's two roundings 2 U: 7.2 U; the rotation adds a product and a sum: 10 U.
ROTATE = 10 * U
# The sum of up to 256 squares: 16 in a thread, 4 by shuffles, 22 roundings with the mean and eps; half of that in the root, 2 for
# rsqrt, 2 products: 15 U; with the conversion of 1 / D 16 U.
NORM = 16 * U


def rms(x, eps):
    return torch.rsqrt((x.double() ** 2).mean(-1, keepdim=True) + eps)


def qk_norm_rotary(x, w, f, positions, half, eps, magnitude=1.0):
    """``(y, off)``"""
    w = torch.ones(x.shape[-1], dtype=torch.float64, device=x.device) if w is None else w.double()
    z = x.double() * rms(x, eps) * w
    return rotate(z, f, positions, half, magnitude), (ROTATE + NORM) * pair_size(z, 2 * f.numel(), half, magnitude)


def qk_norm_rotary_backward(d, x, w, f, positions, half, eps, magnitude=1.0, adds=200):
    """``adds``: additions on the longest way to a weight's gradient."""
    w = torch.ones(x.shape[-1], dtype=torch.float64, device=x.device) if w is None else w.double()
    x, r = x.double(), rms(x, eps)
    g = rotate(d, f, positions, half, magnitude, back=True)
    size = pair_size(d, 2 * f.numel(), half, magnitude)
    t, big = g * w, size * w.abs()
    dx = r * (t - x * r * r * (t * x).mean(-1, keepdim=True))
    # ROTATE in t; NORM and 4 products on one side, 2 NORM, 24 for the sum and 6 products on the other
    off = r * (big * (ROTATE + NORM + 4 * U) + x.abs() * r * r * (big * x.abs()).mean(-1, keepdim=True) * (ROTATE + 3 * NORM + 30 * U))
    lead = tuple(range(x.dim() - 1))
    return dict(dx=dx, dx_off=off, dw=(g * x * r).sum(lead), dw_off=(size * (x * r).abs()).sum(lead) * (ROTATE + NORM + adds * U))


# ---- window attention ------------------------------------------------------------------------------
def seen(n, m, window, sinks, offset, length, device="cpu"):
    """Bool ``[n, m]`` of one sequence."""
    pos = offset + torch.arange(n, device=device)[:, None]
    j = torch.arange(m, device=device)[None]
    left, right = window
    ok = (j < length).expand(n, m)
    if right is not None:
        ok = ok & (j <= pos + right)
    if left is not None:
        ok = ok & ((j >= pos - left) | (j < sinks))
    return ok


def window_attention(q, k, v, window, sinks=0, offsets=None, lengths=None, scale=None, d_out=None):
    """One batch ``q [B, N, H, D]``, ``k, v [B, M, HK, D]`` of 16-bit tensors: ``out, lse`` and, for a ``d_out``, the gradients, each with
    its bound.

    e: half a step of the type, once for P (and dS) as an operand.  A logit is off by D roundings of its products' magnitudes (the order
    of a product's sum is not known) and 3 of its own, and an exponential by 2^-22; a row's probabilities are off by twice the
    largest of these, with the sum's 64 roundings.  An exponential below 2^-126 is zero in fp32 without subnormal numbers, which its
    product with dP - delta (or dO), of any size, shows.
    """
    B, N, H, D = q.shape
    M, HK = k.shape[1:3]
    scale = D ** -0.5 if scale is None else scale
    e = half_step(q.dtype)
    q, k, v = (t.double().transpose(1, 2) for t in (q, k, v))
    k, v = (t.repeat_interleave(H // HK, 1) for t in (k, v))
    ok = torch.stack([seen(N, M, window, sinks, 0 if offsets is None else int(offsets[b]),
                           M if lengths is None else min(max(int(lengths[b]), 0), M), q.device) for b in range(B)])[:, None]
    # (what is behind the last key does not count)
    there = ok.any(2)[..., None] | torch.zeros_like(k[..., :1], dtype=torch.bool)
    k, v = torch.where(there, k, 0.0), torch.where(there, v, 0.0)
    s = (q @ k.transpose(-1, -2)) * scale
    s_off = torch.where(ok, (q.abs() @ k.abs().transpose(-1, -2)) * scale * D * U + 3 * U * s.abs(), 0.0)
    s = s.masked_fill(~ok, -math.inf)
    lse = torch.logsumexp(s, -1)
    p = torch.where(ok, torch.exp(s - torch.where(lse == -math.inf, 0.0, lse)[..., None]), 0.0)
    rel = 2 * (s_off.amax(-1, keepdim=True) if M else 0.0) + 2 * 2.0 ** -22 + 64 * U
    out = p @ v
    out_off = (p * (e + rel)) @ v.abs()
    back = lambda t: t.transpose(1, 2)  # noqa: E731
    res = dict(out=back(out), out_off=back(out_off), lse=lse, lse_off=(rel.squeeze(-1) if M else rel) + 4 * U * lse.abs())
    if d_out is None:
        return res
    g = d_out.double().transpose(1, 2)
    # the backward makes P from the rounded log-sum-exp; delta from the stored output
    dp = g @ v.transpose(-1, -2)
    delta = (g * out).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    rel = rel + 4 * U * torch.where(lse == -math.inf, 0.0, lse).abs()[..., None]
    dp_off = (g.abs() @ v.abs().transpose(-1, -2)) * D * U
    delta_off = (g.abs() * (e * out.abs() + (1 + e) * out_off + D * U * out.abs())).sum(-1, keepdim=True)
    least = torch.where(ok, 2.0 ** -126, 0.0)
    ds_off = p * (dp_off + delta_off) + ds.abs() * (e + rel + 4 * U) + least * (dp - delta).abs()
    fold = lambda t: back(t.unflatten(1, (HK, H // HK)).sum(2))  # noqa: E731
    sums = 512 * U     # of a gradient over the rows of its tiles
    res.update(dq=back(ds @ k) * scale, dq_off=back((ds_off + sums * ds.abs()) @ k.abs()) * scale,
               dk=fold(ds.transpose(-1, -2) @ q) * scale, dk_off=fold((ds_off + sums * ds.abs()).transpose(-1, -2) @ q.abs()) * scale,
               dv=fold(p.transpose(-1, -2) @ g), dv_off=fold((p * (e + rel + sums) + least).transpose(-1, -2) @ g.abs()))
    return res

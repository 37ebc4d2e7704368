"""Workloads of the row-wise operators: layer norm, 8-bit activation checkpoints, and the normalised projection.

Four public entry points: :func:`turbo_layer_norm`, :func:`pack_activation` with :func:`unpack_activation`, and
:func:`turbo_norm_linear`; the first and the last as inference (no gradients) and as one training pass (forward, then the
gradients of every differentiable input for a given output gradient), with the saved activation kept whole or in 8 bits.

Where the sizes come from: rows are the N * N entries of a pair tensor (N = 257, 384, 768 are the lengths of the benchmark
and the parity tests, C in {32, 64, 96, 128} their channels) or the tokens of a sequence; the other widths are generic.
"""
from __future__ import annotations

import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_EPS = 1e-5
_GROUP = 128            # elements of a row that share one scale of an 8-bit checkpoint
_TINY = 2.0 ** -119     # a group whose largest magnitude is below this is kept as zeros

_MOST_ELEMENTS = 589824 * 128
_MOST_PRODUCTS = 589824 * 128 * 512


def _norm(name, mode, rows, cols, dtype="bf16", keep="whole"):
    return dict(name=name, op="layer_norm", mode=mode, rows=rows, cols=cols, dtype=dtype, keep=keep)


def _pack(name, rows, cols, dtype="bf16"):
    return dict(name=name, op="pack", rows=rows, cols=cols, dtype=dtype)


def _linear(name, mode, rows, cols, outs, keep="whole"):
    return dict(name=name, op="norm_linear", mode=mode, rows=rows, cols=cols, outs=outs, keep=keep)


def listed():
    return [
        # one token of a sequence: the call is latency, not work
        _norm("norm_infer_token", "infer", 1, 384),
        # the pair tensor of the training crop, inference
        _norm("norm_infer_n384_c128", "infer", 384 * 384, 128),
        # a ragged pair tensor in fp32
        _norm("norm_train_n257_c96_fp32", "train", 257 * 257, 96, "fp32"),
        # tokens of a width that no vector divides
        _norm("norm_train_4099x1001_fp16", "train", 4099, 1001, "fp16"),
        # wide tokens
        _norm("norm_train_8192x4096", "train", 8192, 4096),
        # the pair tensor of the larger crop, its input kept in 8 bits until the backward pass
        _norm("norm_train_n768_c128_int8", "train", 768 * 768, 128, keep="int8"),
        # the pair tensor of the larger crop put away in 8 bits and taken out again
        _pack("pack_n768_c128", 768 * 768, 128),
        # a ragged fp32 activation of an odd width
        _pack("pack_66049x97_fp32", 257 * 257, 97, "fp32"),
        # one pair row's entry through a stacked projection: latency
        _linear("norm_linear_infer_token", "infer", 1, 128, 512),
        # stacked projections of a ragged pair tensor, inputs kept whole
        _linear("norm_linear_train_n257_c96", "train", 257 * 257, 96, 384),
        # tokens of a wide layer
        _linear("norm_linear_train_4099x1024_int8", "train", 4099, 1024, 4096, keep="int8"),
        # stacked q / k / v / gate projections of the larger crop
        _linear("norm_linear_train_n768_c128_int8", "train", 768 * 768, 128, 512, keep="int8"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["layer_norm", "layer_norm", "pack", "norm_linear", "norm_linear"])
    mode, keep = rng.choice(["infer", "train", "train"]), rng.choice(["whole", "int8"])
    if mode == "infer":
        keep = "whole"
    if op == "norm_linear":
        cols, outs = 8 * _log(rng, 2, 128), 8 * _log(rng, 2, 512)
        rows = _log(rng, 1, max(1, min(600000, _MOST_PRODUCTS // (cols * outs), _MOST_ELEMENTS // cols)))
        return dict(op=op, mode=mode, rows=rows, cols=cols, outs=outs, keep=keep)
    cols = _log(rng, 4, 8192)
    if rng.random() < 0.6:
        cols = (cols + 7) // 8 * 8
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    rows = _log(rng, 1, max(1, min(600000, _MOST_ELEMENTS // 2 // cols)))
    if op == "pack":
        return dict(op=op, rows=rows, cols=cols, dtype=dtype)
    return dict(op=op, mode=mode, rows=rows, cols=cols, dtype=dtype, keep=keep)


def prepare(case, seed):
    """Activations whose channels differ in scale and whose rows differ in mean, the last rows padding (zeros, without a
    gradient); norms near one and zero; Xavier-normal projections.  The projection's parameters are bf16, a plain layer norm
    has fp32 masters."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    rn = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    rows, cols, dtype = case["rows"], case["cols"], _DTYPES[case.get("dtype", "bf16")]
    pad = rows // 20
    x = rn(rows, cols).mul_(torch.exp(0.5 * rn(cols))).add_(0.3 * rn(rows, 1))
    x[rows - pad:] = 0
    state = dict(case=dict(case), x=x.to(dtype))
    if case["op"] == "pack":
        return state
    params = torch.bfloat16 if case["op"] == "norm_linear" else torch.float32
    state["norm_weight"] = (1 + 0.1 * rn(cols)).to(params)
    state["norm_bias"] = (0.1 * rn(cols)).to(params)
    outs = cols
    if case["op"] == "norm_linear":
        outs = case["outs"]
        state["weight"] = (rn(outs, cols) * math.sqrt(2.0 / (outs + cols))).to(params)
    if case["mode"] == "train":
        d_out = rn(rows, outs)
        d_out[rows - pad:] = 0
        state["d_out"] = d_out.to(dtype)
        for name in ("x", "norm_weight", "norm_bias", "weight"):
            if name in state:
                state[name].requires_grad_(True)
    return state


# ---- plain forms ---------------------------------------------------------------------------------
def _kept(x):
    """``(values, scales)`` of x in 8 bits: per 128 elements of a row code = rint(x * fl32(127 / amax)), value = code * scale,
    scale = fl32(amax / 127).  The codes are rounded in 64 bits, where the product is exact; the quotients likewise, because
    a device's division by a constant is a product."""
    rows, cols = x.shape
    groups = -(-cols // _GROUP)
    xp = torch.nn.functional.pad(x.float(), (0, groups * _GROUP - cols)).view(rows, groups, _GROUP)
    amax = xp.abs().amax(-1, keepdim=True)
    empty = amax < _TINY
    ratio = (127.0 / torch.where(empty, 1.0, amax).double()).float()
    ratio = torch.where(empty, 0.0, ratio)
    scale = torch.where(empty, 0.0, (amax.double() / 127.0).float())
    code = torch.round(xp.double() * ratio.double()).float()
    return (code * scale).view(rows, -1)[:, :cols], scale.view(rows, groups)


def _normalise(x):
    mean = x.mean(-1, keepdim=True)
    centred = x - mean
    rstd = torch.rsqrt((centred * centred).mean(-1, keepdim=True) + _EPS)
    return centred * rstd, mean, rstd


def _norm_grads(dy, kept, mean, rstd, weight):
    xhat = (kept - mean) * rstd
    wdy = dy * weight
    dx = rstd * (wdy - wdy.mean(-1, keepdim=True) - xhat * (wdy * xhat).mean(-1, keepdim=True))
    return dx, (dy * xhat).sum(0), dy.sum(0), xhat


def _plain(state):
    case, x = state["case"], state["x"].detach()
    if case["op"] == "pack":
        values, scales = _kept(x)
        return dict(values=values.to(x.dtype), scales=scales)
    w, b = state["norm_weight"].detach(), state["norm_bias"].detach()
    xhat, mean, rstd = _normalise(x.float())
    y = xhat * w.float() + b.float()
    linear = case["op"] == "norm_linear"
    weight = state["weight"].detach().float() if linear else None
    out = (y @ weight.t() if linear else y).to(x.dtype)
    if case["mode"] == "infer":
        return dict(out=out)
    kept = _kept(x)[0] if case["keep"] == "int8" else x.float()
    d_out = state["d_out"].float()
    dy = d_out @ weight if linear else d_out
    dx, dw, db, xhat = _norm_grads(dy, kept, mean, rstd, w.float())
    res = dict(out=out, d_x=dx.to(x.dtype), d_norm_weight=dw.to(w.dtype), d_norm_bias=db.to(b.dtype))
    if linear:
        res["d_weight"] = (d_out.t() @ (xhat * w.float() + b.float())).to(w.dtype)
    return res


def _own(state):
    import openfold3_triangle_kernel_b200 as tk

    case, x = state["case"], state["x"]
    if case["op"] == "pack":
        codes, scales = tk.pack_activation(x)
        return dict(values=tk.unpack_activation(codes, scales, x.dtype), scales=scales)
    keep = "int8" if case["keep"] == "int8" else None
    leaves = [x, state["norm_weight"], state["norm_bias"]]
    names = ["d_x", "d_norm_weight", "d_norm_bias"]
    if case["op"] == "norm_linear":
        leaves.append(state["weight"])
        names.append("d_weight")
        out = tk.turbo_norm_linear(*leaves, checkpoint=keep)
    else:
        out = tk.turbo_layer_norm(*leaves, checkpoint=keep)
    if case["mode"] == "infer":
        return dict(out=out)
    return dict(out=out.detach(), **dict(zip(names, torch.autograd.grad(out, leaves, state["d_out"]))))


def run(state):
    return _own(state) if own else _plain(state)


def work(case):
    """Inputs read once, outputs written once (gradients among them); what is kept between the passes is not counted."""
    rows, cols = case["rows"], case["cols"]
    size = 4 if case.get("dtype") == "fp32" else 2
    if case["op"] == "pack":
        return {"bytes": rows * cols * 2 * size + rows * -(-cols // _GROUP) * 4, "flops": 3 * rows * cols}
    if case["op"] == "layer_norm":
        passes = 1 if case["mode"] == "infer" else 2
        return {"bytes": passes * (2 * rows * cols * size + 2 * cols * 4), "flops": (8 if passes == 1 else 24) * rows * cols}
    outs = case["outs"]
    passes = 1 if case["mode"] == "infer" else 2
    return {"bytes": passes * 2 * (rows * (cols + outs) + cols * outs + 2 * cols),
            "flops": (2 if passes == 1 else 6) * rows * cols * outs}


# ---- the definitions in 64 bits ------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    x = s["x"].detach().double()
    rows, cols = x.shape

    def eight_bits():
        out, scales = torch.empty_like(x), []
        for g in range(0, cols, _GROUP):
            part = x[:, g:g + _GROUP]
            top = part.abs().max(dim=1).values
            live = top >= _TINY
            # the factors are defined as fp32 values
            up = torch.where(live, 127.0 / torch.where(live, top, 1.0), 0.0).float().double()
            down = torch.where(live, top / 127.0, 0.0).float().double()
            out[:, g:g + _GROUP] = (part * up[:, None]).round() * down[:, None]
            scales.append(down)
        return out, torch.stack(scales, 1)

    if case["op"] == "pack":
        values, scales = eight_bits()
        return dict(values=values, scales=scales)
    gamma, beta = s["norm_weight"].detach().double(), s["norm_bias"].detach().double()
    mu = x.sum(1, keepdim=True) / cols
    var = ((x - mu) ** 2).sum(1, keepdim=True) / cols
    sigma = torch.sqrt(var + _EPS)
    y = (x - mu) / sigma * gamma + beta
    linear = case["op"] == "norm_linear"
    w = s["weight"].detach().double() if linear else None
    out = torch.einsum("rc,oc->ro", y, w) if linear else y
    if case["mode"] == "infer":
        return dict(out=out)
    z = (((eight_bits()[0] if case["keep"] == "int8" else x) - mu) / sigma)
    g = s["d_out"].double()
    gy = torch.einsum("ro,oc->rc", g, w) if linear else g
    t = gy * gamma
    d_x = (t - t.sum(1, keepdim=True) / cols - z * ((t * z).sum(1, keepdim=True) / cols)) / sigma
    res = dict(out=out, d_x=d_x, d_norm_weight=(gy * z).sum(0), d_norm_bias=gy.sum(0))
    if linear:
        res["d_weight"] = torch.einsum("ro,rc->oc", g, z * gamma + beta)
    return res

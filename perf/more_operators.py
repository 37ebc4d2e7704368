"""Workloads of the operators around a sequence attention and of dropout.

Four public entry points, in the order in which a layer calls them: :func:`turbo_qk_norm_rotary` (norm of every head of q and k,
and the position rotation) or :func:`turbo_rotary` (the rotation alone), :func:`turbo_window_attention` (a sliding window and a
few first tokens that stay visible), and :func:`turbo_dropout` with the residual.  Each as inference or as one training pass:
forward, then the gradients of every differentiable input for a given output gradient.

Where the sizes come from: N = 257, 384 and 20 with 64 or 128 channels are pair tensors of the benchmark and the tests; lengths and
head layouts of the sequence operators are generic.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_EPS = 1e-6

_MOST_ELEMENTS = 384 * 384 * 128
_MOST_HEAD_ELEMENTS = 8192 * 40 * 128
_MOST_ATTENTION = 8192 * 1024 * 32 * 128     # visible pairs x heads x head dimension, a training pass


def _dropout(name, shape, dtype="bf16", shared=0, residual=True, p=0.25):
    """``shared``: the dimension, from the end, along which the mask is shared; 0: none."""
    return dict(name=name, op="dropout", shape="x".join(map(str, shape)), dtype=dtype, shared=shared, residual=residual, p=p)


def _rotary(name, op, mode, batch, tokens, heads, kv_heads, dim, rot, layout="half", dtype="bf16", first=0, factor=1.0):
    """``first``: position of the first token; ``factor``: how far the context is stretched (YaRN)."""
    return dict(name=name, op=op, mode=mode, batch=batch, tokens=tokens, heads=heads, kv_heads=kv_heads, dim=dim, rot=rot,
                layout=layout, dtype=dtype, first=first, factor=factor)


def _attention(name, mode, batch, queries, keys, heads, kv_heads, dim, left, right, sinks, ragged=False, dtype="bf16"):
    """``left``, ``right``: reach of the window, -1: unlimited.  ``ragged``: sequences of different lengths in one batch."""
    return dict(name=name, op="attention", mode=mode, batch=batch, queries=queries, keys=keys, heads=heads, kv_heads=kv_heads,
                dim=dim, left=left, right=right, sinks=sinks, ragged=ragged, dtype=dtype)


def listed():
    return [
        # the update of a small pair tensor: latency
        _dropout("dropout_n20_c64", (1, 20, 20, 64), shared=3),
        # tokens of a width that no vector divides, every element on its own
        _dropout("dropout_4099x1001_fp16", (4099, 1001), "fp16", residual=False, p=0.1),
        # row-wise dropout of a pair update, added to the residual
        _dropout("dropout_rows_n384_c128", (1, 384, 384, 128), shared=3),
        # part of every head in the interleaved order, fp32, far into a long context
        _rotary("rotary_train_part_fp32", "rotary", "train", 2, 1021, 8, 0, 96, 64, "interleaved", "fp32", first=100000),
        # keys and queries of a stretched context
        _rotary("rotary_infer_8192x32", "rotary", "infer", 1, 8192, 32, 0, 128, 128, first=122880, factor=8.0),
        # q and k of one token: latency
        _rotary("qk_norm_infer_token", "qk_norm_rotary", "infer", 1, 1, 16, 4, 128, 128, first=4096),
        # a ragged number of tokens, part of a head of 80 elements
        _rotary("qk_norm_train_4099_d80_fp16", "qk_norm_rotary", "train", 1, 4099, 12, 12, 80, 32, "half", "fp16"),
        # q and k as they lie in a stacked projection, shared key heads
        _rotary("qk_norm_train_8192_d128", "qk_norm_rotary", "train", 1, 8192, 32, 8, 128, 128),
        # a batch of sequences of different lengths, one new token each, over their caches
        _attention("attention_token_b16", "token", 16, 1, 8192, 32, 8, 128, 1023, 0, 4, ragged=True),
        # a long prompt
        _attention("attention_infer_16384", "infer", 1, 16384, 16384, 16, 4, 128, 1023, 0, 4),
        # a padded batch of sequences that look both ways
        _attention("attention_train_both_ways_d64", "train", 2, 2053, 2053, 16, 16, 64, 128, 128, 1, ragged=True),
        # a training sequence, causal, shared key heads
        _attention("attention_train_8192", "train", 1, 8192, 8192, 32, 8, 128, 1023, 0, 4),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def _draw_dropout(rng):
    shared, dtype = rng.choice([0, 2, 3]), rng.choice(["bf16", "bf16", "fp16", "fp32"])
    cols = _log(rng, 8, 2048)
    if rng.random() < 0.6:
        cols = (cols + 7) // 8 * 8
    if shared:
        side = _log(rng, 1, min(600, math.isqrt(_MOST_ELEMENTS // 2 // cols)))
        shape = (1, side, side, cols)
    else:
        shape = (_log(rng, 1, _MOST_ELEMENTS // 2 // cols), cols)
    return _dropout("", shape, dtype, shared, rng.random() < 0.7, rng.choice([0.1, 0.15, 0.25, 0.5]))


def _draw_rotary(rng):
    op = rng.choice(["rotary", "qk_norm_rotary"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    dim = 8 * rng.randint(2, 32) if rng.random() < 0.8 else 2 * rng.randint(8, 100)
    rot = dim if rng.random() < 0.6 else 2 * rng.randint(4, dim // 2)
    heads = _log(rng, 1, 40)
    kv_heads = 0 if op == "rotary" else rng.choice([h for h in range(1, heads + 1) if heads % h == 0])
    batch = rng.choice([1, 1, 2, 3])
    tokens = _log(rng, 1, max(1, _MOST_HEAD_ELEMENTS // 2 // (batch * (heads + kv_heads) * dim)))
    return _rotary("", op, rng.choice(["infer", "train", "train"]), batch, min(tokens, 200000), heads, kv_heads, dim, rot,
                   rng.choice(["half", "interleaved"]), dtype, rng.choice([0, _log(rng, 1, 500000)]),
                   rng.choice([1.0, 1.0, 4.0, 8.0]))


def _draw_attention(rng):
    mode = rng.choice(["token", "infer", "train", "train"])
    dim = rng.choice([32, 64, 64, 80, 96, 128, 128])
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 4])
    left, right = _log(rng, 1, 4096), 0
    if rng.random() < 0.4:
        right = left
    sinks = rng.choice([0, 1, 4, rng.randint(1, 64)])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    batch = rng.choice([1, 2, 3, 8])
    if mode == "token":
        queries = rng.choice([1, 1, 2, 5])
        keys = _log(rng, 16, 32768)
        return _attention("", mode, batch, queries, max(keys, 2 * queries), heads, kv_heads, dim, left, 0, sinks, True, dtype)
    keys = _log(rng, 1, 8192)
    most = _MOST_ATTENTION // 2 // (heads * dim * batch)
    keys = min(keys, max(1, most // min(keys, left + right + 1 + sinks)))
    return _attention("", mode, batch, keys, keys, heads, kv_heads, dim, left, right, sinks, rng.random() < 0.5, dtype)


def draw(rng):
    case = rng.choice([_draw_dropout, _draw_rotary, _draw_attention, _draw_attention])(rng)
    del case["name"]
    return case


# ---- inputs --------------------------------------------------------------------------------------
def _shape(case):
    return tuple(int(n) for n in case["shape"].split("x"))


def _radians(case):
    """Radians a position, one number a pair, and the factor of the rotated values.  YaRN (Peng et al. 2023): pairs that turn
    often over the original 16384 positions keep their frequency, pairs that turn less than once are slowed down by the
    factor, with a ramp between."""
    rot, factor, base, length = case["rot"], case["factor"], 10000.0, 16384
    f = [base ** (-2.0 * i / rot) for i in range(rot // 2)]
    if factor == 1.0:
        return f, 1.0
    pair = lambda turns: rot * math.log(length / (2 * math.pi * turns)) / (2 * math.log(base))  # noqa: E731
    low, high = max(math.floor(pair(32.0)), 0), min(math.ceil(pair(1.0)), rot - 1)
    ramp = [min(max((i - low) / max(high - low, 1e-3), 0.0), 1.0) for i in range(rot // 2)]
    return [x * (1 - r) + x / factor * r for x, r in zip(f, ramp)], 0.1 * math.log(factor) + 1.0


def _lengths(case):
    """Keys of each sequence."""
    batch, keys = case["batch"], case["keys"]
    return [max(case["queries"] if case["mode"] == "token" else 1, keys - b * keys // (2 * batch)) if case["ragged"] else keys
            for b in range(batch)]


def prepare(case, seed):
    """Activations of a standard deviation of about one; heads differ in scale before their norm; padding has no gradient."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    rn = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    dtype = _DTYPES[case["dtype"]]
    state = dict(case=dict(case))
    train = case.get("mode", "train") == "train"
    if case["op"] == "dropout":
        shape = _shape(case)
        state["x"] = rn(*shape).to(dtype)
        if case["residual"]:
            state["residual"] = rn(*shape).to(dtype)
        state["d_out"] = rn(*shape).to(dtype)
        state["seed"] = torch.randint(-2 ** 62, 2 ** 62, (2,), device="cuda", generator=g, dtype=torch.int64)
        leaves = ["x", "residual"]
    elif case["op"] == "attention":
        batch, n, m, h, hk, d = (case[x] for x in ("batch", "queries", "keys", "heads", "kv_heads", "dim"))
        state["q"], state["k"], state["v"] = rn(batch, n, h, d).to(dtype), rn(batch, m, hk, d).to(dtype), rn(batch, m, hk, d).to(dtype)
        lengths = torch.tensor(_lengths(case), dtype=torch.int32, device="cuda")
        state["lengths"] = lengths
        state["offset"] = lengths - n if case["mode"] == "token" else torch.zeros_like(lengths)
        if train:
            d_out = rn(batch, n, h, d)
            d_out[torch.arange(n, device="cuda")[None, :] >= lengths[:, None]] = 0
            state["d_out"] = d_out.to(dtype)
        leaves = ["q", "k", "v"]
    else:
        batch, n, h, hk, d = (case[x] for x in ("batch", "tokens", "heads", "kv_heads", "dim"))
        total = h + 2 * hk if hk else h
        stacked = (rn(batch, n, total, d) * torch.exp(0.5 * rn(total, 1))).to(dtype)     # v follows q and k
        state["q"] = stacked[:, :, :h]
        state["positions"] = (case["first"] + torch.arange(n, device="cuda")).expand(batch, n).contiguous()
        state["radians"], state["magnitude"] = _radians(case)
        leaves = ["q"]
        if hk:
            state["k"] = stacked[:, :, h:h + hk]
            state["q_weight"], state["k_weight"] = 1 + 0.1 * rn(d), 1 + 0.1 * rn(d)
            leaves += ["k", "q_weight", "k_weight"]
        if train:
            state["d_q"] = rn(batch, n, h, d).to(dtype)
            if hk:
                state["d_k"] = rn(batch, n, hk, d).to(dtype)
        if own:
            import openfold3_triangle_kernel_b200 as tk
            scaling = None if case["factor"] == 1.0 else "yarn"
            state["frequencies"] = tk.rotary_frequencies(case["rot"], scaling=scaling, factor=case["factor"],
                                                         original_length=16384, device="cuda")
    if train:
        for name in leaves:
            if name in state:
                state[name] = state[name].detach().requires_grad_(True)
    return state


# ---- plain forms ---------------------------------------------------------------------------------
def _philox(seed, groups):
    """Philox 4x32-10 (Salmon, Moraes, Dror, Shaw 2011) of the counters (group, offset) under the key ``seed``: int64 tensors
    that hold 32 bits each.  Products wrap at 64 bits, which leaves both of their halves right."""
    low = 0xFFFFFFFF
    word = lambda x: (x & low, (x >> 32) & low)  # noqa: E731
    k0, k1 = word(seed[0])
    c0, c1 = word(groups)
    c2, c3 = (x.expand_as(groups) for x in word(seed[1]))
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((b >> 32) & low) ^ c1 ^ k0, b & low, ((a >> 32) & low) ^ c3 ^ k1, a & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    return c0, c1, c2, c3


def _plain_dropout(state):
    case, x = state["case"], state["x"].detach()
    shape = list(x.shape)
    if case["shared"]:
        shape[-case["shared"]] = 1
    count = math.prod(shape)
    words = _philox(state["seed"], torch.arange(-(-count // 8), device=x.device))
    halves = torch.stack([h for w in words for h in (w & 0xFFFF, w >> 16)], 1).reshape(-1)[:count].view(shape)
    threshold = round(65536 * case["p"])
    kept = halves >= threshold
    scale = 65536.0 / (65536 - threshold)
    out = torch.where(kept, x.float() * scale, 0.0)
    if case["residual"]:
        out = out + state["residual"].detach().float()
    d_x = torch.where(kept, state["d_out"].float() * scale, 0.0)
    res = dict(out=out.to(x.dtype), d_x=d_x.to(x.dtype))
    if case["residual"]:
        res["d_residual"] = state["d_out"]
    return res


def _turn(x, cos, sin, rot, layout):
    """The first ``rot`` elements of x rotated; cos, sin: [batch, tokens, 1, rot / 2]."""
    if layout == "half":
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        turned = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    else:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    return torch.cat([turned, x[..., rot:]], -1)


def _plain_rotary(state):
    case = state["case"]
    radians = torch.tensor(state["radians"], dtype=torch.float64, device="cuda")
    angle = state["positions"].double()[..., None] * radians
    cos, sin = ((f(angle) * state["magnitude"]).float()[:, :, None] for f in (torch.cos, torch.sin))
    rot, layout = case["rot"], case["layout"]
    res = {}
    for name in ("q", "k"):
        if name not in state:
            continue
        x = state[name].detach()
        z, w = x.float(), None
        if case["op"] == "qk_norm_rotary":
            w = state[name + "_weight"].detach()
            rstd = torch.rsqrt((z * z).mean(-1, keepdim=True) + _EPS)
            hat = z * rstd
            z = hat * w
        res[name] = _turn(z, cos, sin, rot, layout).to(x.dtype)
        if case["mode"] != "train":
            continue
        d = _turn(state["d_" + name].float(), cos, -sin, rot, layout)
        if w is not None:
            res["d_" + name + "_weight"] = (d * hat).sum((0, 1, 2))
            t = d * w
            d = rstd * (t - hat * (t * hat).mean(-1, keepdim=True))
        res["d_" + name] = d.to(x.dtype)
    return res


def _plain_attention(state):
    case = state["case"]
    q, k, v = (state[n].detach().float().transpose(1, 2) for n in "qkv")
    group, dim, m = case["heads"] // case["kv_heads"], case["dim"], case["keys"]
    k, v = (t.repeat_interleave(group, 1) for t in (k, v))
    scale = dim ** -0.5
    train = case["mode"] == "train"
    d_out = state["d_out"].float().transpose(1, 2) if train else None
    at = torch.arange(m, device=q.device)
    out, d_q = torch.empty_like(q), torch.empty_like(q)
    d_k, d_v = torch.zeros_like(k), torch.zeros_like(v)
    step = max(1, 2 ** 31 // (q.shape[0] * q.shape[1] * m))
    for i in range(0, q.shape[2], step):
        qi = q[:, :, i:i + step]
        pos = state["offset"][:, None, None] + torch.arange(i, i + qi.shape[2], device=q.device)[:, None]
        seen = at < state["lengths"][:, None, None]
        if case["right"] >= 0:
            seen = seen & (at <= pos + case["right"])
        if case["left"] >= 0:
            seen = seen & ((at >= pos - case["left"]) | (at < case["sinks"]))
        s = torch.where(seen[:, None], qi @ k.transpose(-1, -2) * scale, -math.inf)
        top = s.amax(-1, keepdim=True)
        p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
        total = p.sum(-1, keepdim=True)
        p = p / torch.where(total == 0, 1.0, total)
        o = p @ v
        out[:, :, i:i + step] = o
        if train:
            do = d_out[:, :, i:i + step]
            ds = p * (do @ v.transpose(-1, -2) - (do * o).sum(-1, keepdim=True)) * scale
            d_q[:, :, i:i + step] = ds @ k
            d_k += ds.transpose(-1, -2) @ qi
            d_v += p.transpose(-1, -2) @ do
    back = lambda t: t.transpose(1, 2).contiguous().to(state["q"].dtype)  # noqa: E731
    res = dict(out=back(out))
    if train:
        shared = lambda t: back(t.unflatten(1, (-1, group)).sum(2))  # noqa: E731
        res.update(d_q=back(d_q), d_k=shared(d_k), d_v=shared(d_v))
    return res


# ---- the framework's calls -----------------------------------------------------------------------
def _grads(outs, names, leaves, d_outs):
    return dict(zip(names, torch.autograd.grad(outs, leaves, d_outs)))


def _own(state):
    import openfold3_triangle_kernel_b200 as tk

    case = state["case"]
    if case["op"] == "dropout":
        x, residual = state["x"], state.get("residual")
        out = tk.turbo_dropout(x, case["p"], state["seed"], shared_dim=-case["shared"] if case["shared"] else None,
                               residual=residual)
        names, leaves = (["d_x"], [x]) if residual is None else (["d_x", "d_residual"], [x, residual])
        return dict(out=out.detach(), **_grads(out, names, leaves, state["d_out"]))
    if case["op"] == "rotary":
        q = state["q"]
        out = tk.turbo_rotary(q, state["frequencies"], state["positions"], layout=case["layout"])
        if case["mode"] != "train":
            return dict(q=out)
        return dict(q=out.detach(), **_grads(out, ["d_q"], [q], state["d_q"]))
    if case["op"] == "qk_norm_rotary":
        leaves = [state[n] for n in ("q", "k", "q_weight", "k_weight")]
        q, k = tk.turbo_qk_norm_rotary(*leaves, state["frequencies"], state["positions"], eps=_EPS, layout=case["layout"])
        if case["mode"] != "train":
            return dict(q=q, k=k)
        return dict(q=q.detach(), k=k.detach(), **_grads([q, k], ["d_q", "d_k", "d_q_weight", "d_k_weight"], leaves,
                                                         [state["d_q"], state["d_k"]]))
    leaves = [state[n] for n in "qkv"]
    reach = tuple(None if case[n] < 0 else case[n] for n in ("left", "right"))
    out = tk.turbo_window_attention(*leaves, window=reach, sinks=case["sinks"],
                                    query_offset=state["offset"] if case["mode"] == "token" else 0,
                                    key_lengths=state["lengths"] if case["ragged"] else None)
    if case["mode"] != "train":
        return dict(out=out)
    return dict(out=out.detach(), **_grads(out, ["d_q", "d_k", "d_v"], leaves, state["d_out"]))


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    return _plain_dropout(state) if op == "dropout" else _plain_attention(state) if op == "attention" else _plain_rotary(state)


# ---- what a pass cannot do without ---------------------------------------------------------------
def _seen(case):
    """Visible pairs of queries and keys, and keys that some query sees, over the batch."""
    pairs = keys = 0
    for length in _lengths(case):
        first = length - case["queries"] if case["mode"] == "token" else 0
        pos = first + np.arange(case["queries"], dtype=np.int64)
        upper = np.minimum(length, pos + case["right"] + 1) if case["right"] >= 0 else np.full_like(pos, length)
        lower = np.maximum(pos - case["left"], 0) if case["left"] >= 0 else np.zeros_like(pos)
        pairs += int((np.maximum(upper - lower, 0) + np.maximum(np.minimum(case["sinks"], np.minimum(lower, upper)), 0)).sum())
        low, high = int(lower.min()), int(upper.max())
        keys += max(high - low, 0) + max(min(case["sinks"], low, high), 0)
    return pairs, keys


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "dropout":
        count = math.prod(_shape(case))
        # x, residual -> out; d_out -> d_x (the residual's gradient is the output's)
        return {"bytes": count * size * (5 if case["residual"] else 4), "flops": 4 * count}
    if case["op"] == "attention":
        pairs, keys = _seen(case)
        q = case["batch"] * case["queries"] * case["heads"] * case["dim"]
        kv = keys * case["kv_heads"] * case["dim"]
        train = case["mode"] == "train"
        # q, k, v -> out; q, k, v, out, d_out -> their gradients
        return {"bytes": size * ((2 * q + 2 * kv) + (train and 4 * q + 4 * kv)),
                "flops": (14 if train else 4) * pairs * case["heads"] * case["dim"]}
    count = case["batch"] * case["tokens"] * (case["heads"] + case["kv_heads"]) * case["dim"]
    if case["op"] == "rotary":      # a rotation's gradient needs no input
        return {"bytes": count * size * (4 if case["mode"] == "train" else 2), "flops": 6 * count}
    return {"bytes": count * size * (5 if case["mode"] == "train" else 2), "flops": (26 if case["mode"] == "train" else 8) * count}


# ---- the definitions in 64 bits ------------------------------------------------------------------
def _exact_dropout(case, s):
    shape = list(_shape(case))
    if case["shared"]:
        shape[len(shape) - case["shared"]] = 1
    count = int(np.prod(shape))
    seed, offset = (int(n) % 2 ** 64 for n in s["seed"].tolist())
    u32 = np.uint64(0xFFFFFFFF)
    n = np.arange((count + 7) // 8, dtype=np.uint64)
    c = [n & u32, n >> np.uint64(32), np.full_like(n, offset % 2 ** 32), np.full_like(n, offset // 2 ** 32)]
    key = [seed % 2 ** 32, seed // 2 ** 32]
    for _ in range(10):
        left, right = np.uint64(0xD2511F53) * c[0], np.uint64(0xCD9E8D57) * c[2]
        c = [(right >> np.uint64(32)) ^ c[1] ^ np.uint64(key[0]), right & u32,
             (left >> np.uint64(32)) ^ c[3] ^ np.uint64(key[1]), left & u32]
        key = [(key[0] + 0x9E3779B9) % 2 ** 32, (key[1] + 0xBB67AE85) % 2 ** 32]
    words = np.stack(c, 1).astype(np.uint32)
    bits = words.view(np.uint16).reshape(-1)[:count].reshape(shape)     # (little-endian: the low half first)
    dropped = int(np.rint(case["p"] * 65536))
    factor = torch.from_numpy((bits.astype(np.int64) >= dropped) * (65536.0 / (65536 - dropped))).cuda()
    out = s["x"].detach().double() * factor
    grads = dict(d_x=s["d_out"].double() * factor)
    if case["residual"]:
        out = out + s["residual"].detach().double()
        grads["d_residual"] = s["d_out"].double()
    return dict(out=out, **grads)


def _exact_rotary(case, s):
    rot = case["rot"]
    angle = torch.einsum("bt,p->btp", s["positions"].double(), torch.tensor(s["radians"], dtype=torch.float64, device="cuda"))
    turn = torch.polar(torch.full_like(angle, s["magnitude"]), angle)[:, :, None]     # complex [batch, tokens, 1, pairs]
    first, second = (torch.arange(rot, device="cuda").view(2, -1) if case["layout"] == "half"
                     else torch.arange(rot, device="cuda").view(-1, 2).t())

    def rotate(x, by):
        z = torch.complex(x[..., first].contiguous(), x[..., second].contiguous()) * by
        y = x.clone()
        y[..., first], y[..., second] = z.real, z.imag
        return y

    res = {}
    for name in ("q", "k"):
        if name not in s:
            continue
        x = s[name].detach().double()
        y, norm = x, case["op"] == "qk_norm_rotary"
        if norm:
            w = s[name + "_weight"].detach().double()
            size = torch.sqrt(torch.linalg.vecdot(x, x)[..., None] / case["dim"] + _EPS)
            y = x / size * w
        res[name] = rotate(y, turn)
        if case["mode"] == "train":
            g = rotate(s["d_" + name].double(), turn.conj())
            if norm:
                res["d_" + name + "_weight"] = torch.einsum("bthd,bthd->d", g, x / size)
                h = g * w
                g = h / size - x * torch.linalg.vecdot(h, x)[..., None] / (case["dim"] * size ** 3)
            res["d_" + name] = g
    return res


def _exact_attention(case, s):
    heads, group, dim = case["heads"], case["heads"] // case["kv_heads"], case["dim"]
    q, k, v = (s[n].detach().double() for n in "qkv")
    train = case["mode"] == "train"
    g = s["d_out"].double() if train else None
    out, dq, dk, dv = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    for b, (length, first) in enumerate(zip(s["lengths"].tolist(), s["offset"].tolist())):
        for i in range(0, case["queries"], 512):
            rows = slice(i, min(i + 512, case["queries"]))
            pos = torch.arange(first + rows.start, first + rows.stop, device="cuda")[:, None]
            last = length if case["right"] < 0 else min(length, first + rows.stop + case["right"])
            start = 0 if case["left"] < 0 else min(max(first + rows.start - case["left"], 0), max(last, 0))
            cols = torch.cat([torch.arange(0, max(min(case["sinks"], start, last), 0), device="cuda"),
                              torch.arange(start, max(last, start), device="cuda")])
            if cols.numel() == 0:
                continue
            ok = torch.ones(len(pos), len(cols), dtype=torch.bool, device="cuda")
            if case["right"] >= 0:
                ok &= cols - pos <= case["right"]
            if case["left"] >= 0:
                ok &= (pos - cols <= case["left"]) | (cols < case["sinks"])
            kc, vc = k[b, cols], v[b, cols]
            qg = q[b, rows].unflatten(1, (-1, group))                                # [rows, kv heads, group, dim]
            logits = torch.einsum("ihgd,jhd->hgij", qg, kc) / math.sqrt(dim)
            logits.masked_fill_(~ok, -math.inf)
            p = torch.softmax(logits, -1)
            p = torch.where(ok.any(1)[:, None], p, 0.0)
            out[b, rows] = torch.einsum("hgij,jhd->ihgd", p, vc).flatten(1, 2)
            if train:
                gg = g[b, rows].unflatten(1, (-1, group))
                dp = torch.einsum("ihgd,jhd->hgij", gg, vc)
                t = p * (dp - (p * dp).sum(-1, keepdim=True)) / math.sqrt(dim)
                dq[b, rows] = torch.einsum("hgij,jhd->ihgd", t, kc).flatten(1, 2)
                dk[b].index_add_(0, cols, torch.einsum("hgij,ihgd->jhd", t, qg))
                dv[b].index_add_(0, cols, torch.einsum("hgij,ihgd->jhd", p, gg))
    return dict(out=out, d_q=dq, d_k=dk, d_v=dv) if train else dict(out=out)


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    return _exact_dropout(case, s) if op == "dropout" else _exact_attention(case, s) if op == "attention" else _exact_rotary(case, s)

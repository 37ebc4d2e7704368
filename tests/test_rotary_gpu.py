"""turbo_rotary and turbo_qk_norm_rotary on a B200 against the 64-bit oracle (bounds derived in oracle/sequence_oracle.py)."""
import math

import pytest
import torch

import openfold3_triangle_kernel_b200 as tk
from oracle import sequence_oracle as so

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA device")]

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _rn(*s, seed=0, dtype=torch.float32):
    return torch.randn(*s, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)).to(dtype)


def _freq(rot, **kw):
    return tk.rotary_frequencies(rot, device="cuda", **kw)


def _check_rotary(x, rot, layout="half", positions=None, first=0):
    half = layout == "half"
    pos = positions if positions is not None else first + torch.arange(x.shape[-3], device="cuda")
    leaf = x.detach().requires_grad_(True)
    out = tk.turbo_rotary(leaf, _freq(rot), positions if positions is not None else first, layout=layout)
    assert out.dtype == x.dtype and out.shape == x.shape and out.is_contiguous()
    f = so.radians(rot)
    full = pos.expand(x.shape[:-2])
    so.check(out, so.rotate(x, f, full, half), so.ROTATE * so.pair_size(x, rot, half), "out")
    d = _rn(*x.shape, seed=9, dtype=x.dtype)
    g, = torch.autograd.grad(out, leaf, d)
    so.check(g, so.rotate(d, f, full, half, back=True), so.ROTATE * so.pair_size(d, rot, half), "d_x")
    with torch.no_grad():
        assert torch.equal(tk.turbo_rotary(leaf, _freq(rot), positions if positions is not None else first, layout=layout), out)


def _check_norm(q, k, rot, layout="half", first=0, weights=(torch.float32, torch.float32), eps=1e-6, positions=None, adds=200, fr=None):
    half = layout == "half"
    pos = (positions if positions is not None else first + torch.arange(q.shape[-3], device="cuda")).expand(q.shape[:-2])
    w = [None if t is None else (1 + 0.2 * _rn(q.shape[-1], seed=20 + i)).to(t).requires_grad_(True) for i, t in enumerate(weights)]
    leaves = [q.detach().requires_grad_(True), k.detach().requires_grad_(True)]
    f = so.radians(rot)
    outs = tk.turbo_qk_norm_rotary(*leaves, *w, _freq(rot), positions if positions is not None else first, eps=eps, layout=layout)
    ds = [_rn(*t.shape, seed=30 + i, dtype=t.dtype) for i, t in enumerate(outs)]
    wanted = leaves + [t for t in w if t is not None]
    grads = torch.autograd.grad(outs, wanted, ds)
    at = 2
    for i in range(2):
        assert outs[i].dtype == q.dtype and outs[i].shape == leaves[i].shape and outs[i].is_contiguous()
        ref, off = so.qk_norm_rotary(leaves[i].detach(), w[i], f, pos, half, eps)
        so.check(outs[i], ref, off, f"out {i}")
        back = so.qk_norm_rotary_backward(ds[i], leaves[i].detach(), w[i], f, pos, half, eps, adds=adds)
        so.check(grads[i], back["dx"], back["dx_off"], f"dx {i}")
        if w[i] is not None:
            assert grads[at].dtype == w[i].dtype
            so.check(grads[at], back["dw"], back["dw_off"], f"dw {i}")
            at += 1
    with torch.no_grad():
        again = tk.turbo_qk_norm_rotary(*leaves, *w, _freq(rot), positions if positions is not None else first, eps=eps, layout=layout)
    assert all(torch.equal(a, b) for a, b in zip(outs, again))
    return outs, grads


# head sizes: every team width, their borders, sizes that no vector divides; parts that no piece fits
SIZES = [(2, 2), (8, 8), (16, 16), (16, 8), (24, 24), (32, 32), (40, 16), (40, 40), (64, 64), (64, 32), (64, 20), (72, 48), (80, 32), (96, 64), (96, 96),
         (100, 50), (126, 126), (128, 128), (128, 64), (128, 120), (136, 136), (192, 128), (256, 256), (256, 2), (254, 100), (250, 250)]


@pytest.mark.parametrize("dim, rot", SIZES)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_rotary_sizes(dim, rot, layout, dtype):
    _check_rotary(_rn(2, 7, 3, dim, seed=dim, dtype=DT[dtype]), rot, layout, first=5)


@pytest.mark.parametrize("dim, rot", SIZES)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_norm_sizes(dim, rot, layout, dtype):
    _check_norm(_rn(2, 7, 4, dim, seed=dim, dtype=DT[dtype]), _rn(2, 7, 2, dim, seed=dim + 1, dtype=DT[dtype]), rot, layout, first=3)


@pytest.mark.parametrize("tokens", [1, 2, 31, 33, 300, 3000])
@pytest.mark.parametrize("heads, kv", [(1, 1), (5, 1), (12, 4), (32, 8)])
def test_norm_tokens_and_heads(tokens, heads, kv):
    # a thread's additions: the items of a block's team (fewer than 3000 * 40 / 296 / 16 + 40) and the fold
    _check_norm(_rn(1, tokens, heads, 64, seed=tokens).bfloat16(), _rn(1, tokens, kv, 64, seed=heads).bfloat16(), 64, adds=400)


@pytest.mark.parametrize("weights", [(None, None), (torch.bfloat16, torch.float16), (None, torch.float32), (torch.float32, None)])
def test_norm_weights(weights):
    _check_norm(_rn(2, 19, 4, 96).half(), _rn(2, 19, 2, 96, seed=1).half(), 96, weights=weights)


@pytest.mark.parametrize("first", [0, 1, 2 ** 20 - 3, 2 ** 31 + 5, -7])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_far_positions(first, layout):
    """In fp32; the oracle's angles, in 64 bits, are off by 2^-53 of themselves, 2^-22 at 2^31 radians: 4 U of the bound's 10."""
    _check_rotary(_rn(1, 9, 2, 64), 64, layout, first=first)
    _check_norm(_rn(1, 9, 2, 64), _rn(1, 9, 1, 64, seed=4), 64, layout, first=first)


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_positions(dtype):
    x = _rn(3, 11, 2, 32)
    pos = torch.randint(0, 5000, (3, 11), device="cuda", dtype=dtype)
    _check_rotary(x, 32, positions=pos)
    _check_rotary(x, 32, positions=pos[0])
    _check_rotary(x, 32, positions=pos[:, :1])
    _check_rotary(x, 32, positions=pos.t().contiguous().t())
    _check_rotary(_rn(11, 2, 32), 32, positions=pos[1])
    _check_rotary(_rn(2, 3, 5, 2, 32), 32, positions=pos[:, :5])
    _check_norm(x, _rn(3, 11, 1, 32, seed=2), 32, positions=pos)


def test_strides():
    """q, k as slices of a stacked projection, head-major tensors, tokens at an odd pitch, a misaligned start, expanded heads."""
    stacked = _rn(2, 13, 10, 64).bfloat16()
    _check_norm(stacked[:, :, :6], stacked[:, :, 6:8], 64)
    _check_norm(_rn(2, 6, 13, 64).bfloat16().transpose(1, 2), _rn(2, 2, 13, 64, seed=1).bfloat16().transpose(1, 2), 64)
    odd = _rn(2, 13, 6 * 64 + 1).bfloat16()
    _check_norm(odd[..., :384].unflatten(-1, (6, 64)), odd[..., 1:129].unflatten(-1, (2, 64)), 64)
    _check_norm(_rn(2, 13, 1, 64).bfloat16().expand(2, 13, 4, 64), stacked[:, :, :2], 64)
    _check_rotary(stacked[:, :, 3:5], 32)
    _check_rotary(_rn(2, 3, 13, 4, 64).transpose(0, 1), 64, "interleaved")
    _check_rotary(_rn(4, 13, 64, 5).transpose(2, 3)[..., ::1], 64)


def test_infinities_stay_in_their_pairs():
    for layout in ("half", "interleaved"):
        x = torch.zeros(1, 1, 1, 64, device="cuda")
        x[..., 40] = math.inf     # not rotated
        x[..., 3] = 1.0
        out = tk.turbo_rotary(x, _freq(32), 1, layout=layout)
        assert out[..., 40].item() == math.inf and torch.isfinite(out[..., :40]).all() and torch.isfinite(out[..., 41:]).all()
        # a head with an infinity is lost, its neighbours are not
        q = _rn(1, 5, 4, 64)
        q[:, 2, 1, 7] = math.inf
        a, b = tk.turbo_qk_norm_rotary(q, q[:, :, :2], None, None, _freq(64), layout=layout)
        assert not torch.isfinite(a[:, 2, 1]).all()
        a = a.clone()
        a[:, 2, 1] = 0
        assert torch.isfinite(a).all()


def test_zeros():
    """A head of zeros with no eps is a NaN, with one it is zeros, and its gradient is that of the formula."""
    q = torch.zeros(1, 3, 2, 64, device="cuda")
    a, _ = tk.turbo_qk_norm_rotary(q, q, None, None, _freq(64), eps=0.0)
    assert a.isnan().all()
    _check_norm(q, q[:, :, :1], 64, eps=1e-4)


def test_nothing():
    for shape in ((0, 5, 2, 32), (2, 0, 2, 32), (2, 5, 0, 32)):
        x = torch.zeros(shape, device="cuda", requires_grad=True)
        out = tk.turbo_rotary(x, _freq(32))
        assert out.shape == shape
        out.sum().backward()
    q = torch.zeros(0, 5, 2, 32, device="cuda", requires_grad=True)
    w = torch.ones(32, device="cuda", requires_grad=True)
    a, b = tk.turbo_qk_norm_rotary(q, q, w, None, _freq(32))
    (a.sum() + b.sum()).backward()
    assert (w.grad == 0).all()


def test_keys_without_heads():
    q, k = _rn(2, 9, 4, 64).requires_grad_(True), _rn(2, 9, 0, 64).requires_grad_(True)
    qw, kw = (_rn(64, seed=2) + 1).requires_grad_(True), (_rn(64, seed=3) + 1).requires_grad_(True)
    fill = [torch.full((1 << 18,), float("nan"), device="cuda") for _ in range(4)]   # what workspaces then hold
    del fill
    a, b = tk.turbo_qk_norm_rotary(q, k, qw, kw, _freq(64))
    g = torch.autograd.grad([a, b], [q, k, qw, kw], [torch.ones_like(a), torch.ones_like(b)])
    assert torch.equal(g[3], torch.zeros_like(kw)) and g[1].shape == k.shape and g[2].isfinite().all()


def test_magnitudes_that_are_no_numbers_are_refused():
    x = _rn(1, 3, 2, 64)
    for magnitude in (float("nan"), float("inf"), 1e300, "one", torch.ones((), device="cuda")):
        f = tk.RotaryFrequencies(_freq(64).turns, magnitude)
        with pytest.raises(ValueError, match="frequencies"):
            tk.turbo_rotary(x, f)
        with pytest.raises(ValueError, match="frequencies"):
            tk.turbo_qk_norm_rotary(x, x, None, None, f)


def test_one_output_used():
    """A gradient that never came counts as zeros."""
    q, k = _rn(1, 9, 4, 64).requires_grad_(True), _rn(1, 9, 2, 64, seed=1).requires_grad_(True)
    qw, kw = (_rn(64, seed=2) + 1).requires_grad_(True), (_rn(64, seed=3) + 1).requires_grad_(True)
    d = _rn(1, 9, 4, 64, seed=4)
    a, _ = tk.turbo_qk_norm_rotary(q, k, qw, kw, _freq(64))
    g = torch.autograd.grad(a, [q, qw, k, kw], d, allow_unused=True)
    back = so.qk_norm_rotary_backward(d, q.detach(), qw.detach(), so.radians(64), torch.arange(9, device="cuda").expand(1, 9), True, 1e-6)
    so.check(g[0], back["dx"], back["dx_off"], "dq")
    so.check(g[1], back["dw"], back["dw_off"], "dqw")
    assert g[2] is None and (g[3] is None or (g[3] == 0).all())
    _, b = tk.turbo_qk_norm_rotary(q, k, qw, kw, _freq(64))
    assert torch.autograd.grad(b.sum(), k)[0].abs().sum() > 0


def test_differences():
    """The gradients are those of the computed function: central differences in fp32 with steps of 2^-7, whose error is third order
    (2^-14 of the third derivative) plus the function's own rounding, 2^-20 / 2^-6."""
    q, k = _rn(1, 3, 2, 16).requires_grad_(True), _rn(1, 3, 1, 16, seed=1).requires_grad_(True)
    w = (1 + 0.1 * _rn(16, seed=2)).requires_grad_(True)
    d = [_rn(1, 3, 2, 16, seed=3), _rn(1, 3, 1, 16, seed=4)]

    def f():
        a, b = tk.turbo_qk_norm_rotary(q, k, w, w, _freq(16), 7)
        return (a * d[0]).double().sum() + (b * d[1]).double().sum()

    grads = torch.autograd.grad(f(), [q, k, w])
    with torch.no_grad():
        for leaf, g in zip((q, k, w), grads):
            step = _rn(*leaf.shape, seed=5)
            leaf.add_(step * 2.0 ** -7)
            up = f()
            leaf.sub_(step * 2.0 ** -6)
            down = f()
            leaf.add_(step * 2.0 ** -7)
            slope = (g.double() * step).sum()
            assert abs((up - down) * 64 - slope) <= 0.02 * (g.double().abs() * step.abs()).sum() + 1e-3


@pytest.mark.parametrize("scaling, kw", [("linear", dict(factor=4.0)), ("ntk", dict(factor=4.0)),
                                         ("yarn", dict(factor=8.0, original_length=1024))])
def test_scaled_frequencies(scaling, kw):
    fr = _freq(64, scaling=scaling, **kw)
    x = _rn(1, 50, 2, 64)
    f = (fr.turns.double() % 2.0 ** 64).cpu() * 2 * math.pi / 2.0 ** 64
    pos = torch.arange(50, device="cuda").expand(1, 50)
    so.check(tk.turbo_rotary(x, fr), so.rotate(x, f, pos, True, fr.magnitude), so.ROTATE * so.pair_size(x, 64, True, fr.magnitude), "out")


def test_captured_replays():
    q, k = _rn(1, 40, 4, 64).bfloat16().requires_grad_(True), _rn(1, 40, 2, 64, seed=1).bfloat16().requires_grad_(True)
    w = (1 + 0.1 * _rn(64, seed=2)).requires_grad_(True)
    pos = torch.arange(40, device="cuda").expand(1, 40).contiguous()
    d = [_rn(1, 40, 4, 64, seed=3).bfloat16(), _rn(1, 40, 2, 64, seed=4).bfloat16()]
    fr = _freq(64)

    def step():
        outs = tk.turbo_qk_norm_rotary(q, k, w, w, fr, pos)
        return [*(o.detach() for o in outs), *torch.autograd.grad(outs, [q, k, w], d)]

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = step()
    for shift in (0, 1000):
        with torch.no_grad():
            pos.add_(shift)
            q.mul_(1.5)
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(res, step()))


def test_traced_calls():
    torch.compiler.reset()
    fr = _freq(32)
    w = (1 + 0.1 * _rn(64, seed=2)).requires_grad_(True)
    f = lambda q, k, p: tk.turbo_qk_norm_rotary(q, k, w, None, fr, p)  # noqa: E731
    g = lambda x: tk.turbo_rotary(x, fr, 9, layout="interleaved")  # noqa: E731
    cf, cg = (torch.compile(h, fullgraph=True, dynamic=True, backend="aot_eager") for h in (f, g))
    for n in (5, 12):
        q, k = _rn(2, n, 4, 64).bfloat16().requires_grad_(True), _rn(2, n, 2, 64, seed=1).bfloat16().requires_grad_(True)
        pos = torch.arange(n, device="cuda").expand(2, n)
        d = [_rn(2, n, 4, 64, seed=3).bfloat16(), _rn(2, n, 2, 64, seed=4).bfloat16()]
        res = []
        for call, rot in ((f, g), (cf, cg)):
            outs = call(q, k, pos)
            r = rot(q)
            res.append([*outs, r, *torch.autograd.grad([*outs, r], [q, k, w], [*d, d[0]])])
        assert all(torch.equal(a, b) for a, b in zip(*res))
    x = _rn(1, 4, 2, 64, dtype=torch.bfloat16).requires_grad_(True)
    torch.library.opcheck(torch.ops.tpf_b200.rotary_fwd, (x, x.detach()[:, :, :1].clone().requires_grad_(True), None, None, fr.turns, None, 3, 1.0, True,
                                                          True, 1e-6))


def test_second_derivatives_and_changed_inputs_raise():
    q = _rn(1, 4, 2, 64).requires_grad_(True)
    a, b = tk.turbo_qk_norm_rotary(q, q, None, None, _freq(64))
    g, = torch.autograd.grad(a.sum(), q, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        g.sum().backward()
    x = q * 1.0
    a, _ = tk.turbo_qk_norm_rotary(x, x, None, None, _freq(64))
    x.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        a.sum().backward()


@pytest.mark.parametrize("norm", [False, True])
def test_saved_tensors_of_other_layouts(norm):
    """A hook of the caller's may hand back any strides of the positions and the frequencies, too: transposed, spread out, expanded."""
    q, k = (_rn(3, 50, h, 64, seed=h, dtype=torch.bfloat16).requires_grad_(True) for h in (4, 2))
    fr = _freq(32)
    row = torch.randint(0, 10 ** 6, (1, 50), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    positions = torch.cat([row, row, row])
    d = [_rn(3, 50, h, 64, seed=h + 10, dtype=torch.bfloat16) for h in (4, 2)]

    def call():
        if norm:
            return tk.turbo_qk_norm_rotary(q, k, None, None, fr, positions)
        return tk.turbo_rotary(q, fr, positions), tk.turbo_rotary(k, fr, positions)

    want = torch.autograd.grad(call(), [q, k], d)
    turned = lambda t: t.transpose(0, 1).contiguous().transpose(0, 1) if t.ndim > 1 else t  # noqa: E731
    spread = lambda t: torch.stack([t, t + 1], -1)[..., 0]  # noqa: E731
    once = lambda t: t[:1].clone().expand(t.shape) if t.ndim == 2 else t  # noqa: E731
    for hook in (turned, spread, once):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach(), hook):
            outs = call()
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(outs, [q, k], d), want))


@pytest.mark.parametrize("dim", [2, 64])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_angles_of_any_position(dim, layout):
    """Sines and cosines of the exact phase, by whole numbers: an angle off by 2^-26 of a turn for its rounding to fp32 and 2^-32 for the
    bits that are cut off, and 2^-23 for sincospi (two steps of a number below one)."""
    import random
    rng = random.Random(5)
    rates = [rng.randrange(-2 ** 63, 2 ** 63) for _ in range(dim // 2 - 1)] + [2 ** 32 + 1]
    at = [0, 1, -1, 2 ** 62, -2 ** 62, 2 ** 63 - 1, -2 ** 63] + [rng.randrange(-2 ** 63, 2 ** 63) for _ in range(300)]
    fr = tk.RotaryFrequencies(torch.tensor(rates, device="cuda"))
    x = torch.zeros(1, len(at), 1, dim, device="cuda")
    first, second = so.pairs(dim, layout == "half")
    x[..., first] = 1.0
    out = tk.turbo_rotary(x, fr, torch.tensor([at], device="cuda"), layout=layout)[0, :, 0].double().cpu()
    t = torch.tensor([[(r * p % 2 ** 64) / 2 ** 64 for r in rates] for p in at], dtype=torch.float64) * 2 * math.pi
    room = 2 * math.pi * (2.0 ** -26 + 2.0 ** -32) + 2.0 ** -23
    assert (out[:, first] - t.cos()).abs().max() <= room and (out[:, second] - t.sin()).abs().max() <= room

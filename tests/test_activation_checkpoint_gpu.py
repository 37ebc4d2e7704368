"""8-bit activation checkpoints on a B200: codes and scales equal the 64-bit definition's bit by bit."""
import pytest
import torch

import openfold3_triangle_kernel_b200 as tk
from oracle import rows_oracle as ro

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA device")]

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _x(rows, cols, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(rows, cols, generator=g) * torch.exp(0.5 * torch.randn(cols, generator=g))).to(dtype)


def _same(a, b):  # a NaN equals a NaN
    return torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(a.nan_to_num(), b.nan_to_num())


def _check(x, x_cuda=None):
    codes, scales = tk.pack_activation(x.cuda() if x_cuda is None else x_cuda)
    c, s, v = ro.pack(x.reshape(-1, x.shape[-1]))
    assert codes.dtype == torch.int8 and codes.shape == x.shape
    assert torch.equal(codes.cpu().double().view(c.shape), c)
    assert _same(scales.cpu().double().view(s.shape), s)
    for dt in (torch.bfloat16, torch.float16, torch.float32):
        back = tk.unpack_activation(codes, scales, dt)
        assert back.dtype == dt and back.shape == x.shape
        # fl32(code * scale), rounded to the type
        assert _same(back.cpu().view(c.shape), v.float().to(dt))
    return codes, scales


@pytest.mark.parametrize("rows, cols", [(1, 1), (5, 8), (33, 24), (65, 32), (7, 40), (70, 64), (9, 96), (21, 97), (300, 128),
                                        (3, 129), (5, 136), (17, 200), (4, 1000), (3, 1001), (2, 4096), (1, 5003), (1, 70001),
                                        (257, 4)])
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_pack_and_unpack(rows, cols, dtype):
    _check(_x(rows, cols, DT[dtype], seed=rows + cols))


@pytest.mark.parametrize("cols", [5, 97, 128, 200, 1000])
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_values_are_near_what_was_put_away(cols, dtype):
    """The bound that the documents give, against x itself."""
    for scale in (1.0, 1.0625, 2.0 ** -10, 300.0):
        x = _x(200, cols, DT[dtype], seed=cols) * scale
        x[::7, cols // 2] = scale * 1.0625
        back = tk.unpack_activation(*tk.pack_activation(x.cuda()), DT[dtype])
        assert ((back.cpu().double() - x.double()).abs() <= ro.pack_off(x, DT[dtype])).all()


@pytest.mark.parametrize("cols", [1, 3, 5, 7, 9, 17, 30, 60, 63, 97, 121, 127, 130, 131, 135, 250, 259, 381, 1029, 4099])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_odd_widths_of_many_rows(cols, dtype):
    _check(_x(max(3, 20011 // cols), cols, DT[dtype], seed=cols))


@pytest.mark.parametrize("cols", [5, 30, 97, 131])
def test_unpacking_from_and_to_odd_addresses(cols):
    codes, scales = _check(_x(50, cols, torch.bfloat16, seed=cols))
    buf = torch.empty(50 * cols + 1, device="cuda", dtype=torch.int8)
    buf[1:] = codes.view(-1)
    assert torch.equal(tk.unpack_activation(buf[1:].view(50, cols), scales), tk.unpack_activation(codes, scales))


def test_ties_go_to_the_even_code():
    # amax 127 makes the factor exactly 1, so that halves are ties
    x = torch.zeros(1, 128)
    x[0, 0] = 127
    x[0, 1:9] = torch.tensor([0.5, 1.5, 2.5, -0.5, -1.5, -2.5, 63.5, -126.5])
    codes, _ = _check(x)
    assert codes[0, 1:9].tolist() == [0, 2, 2, 0, -2, -2, 64, -126]


def test_extremes():
    x = torch.zeros(8, 128)
    x[1, 5] = 3.4e38
    x[2, 5] = 2.0 ** -119
    x[2, 6] = -(2.0 ** -120)
    x[3, 5] = 1.99 * 2.0 ** -120   # below the smallest amax that is kept
    x[4, 5] = 1e-42
    x[5] = -7
    _, scales = _check(x)
    assert scales[3, 0] == 0 and scales[4, 0] == 0 and scales[0, 0] == 0
    _check(x.bfloat16())


@pytest.mark.parametrize("cols", [128, 200, 97])
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_the_largest_values_stay_finite(cols, dtype):
    """finfo.max and finfo.min fill masks.  127 scales of FLT_MAX / 127, rounded up, would be infinity."""
    info = torch.finfo(DT[dtype])
    x = _x(5, cols, DT[dtype])
    x[1], x[2, 3], x[3, 7], x[3, 8] = info.min, info.max, info.min, info.max
    codes, scales = _check(x)
    back = tk.unpack_activation(codes, scales, DT[dtype])
    assert torch.isfinite(back).all() and codes[1].eq(-127).all()
    assert ((back[1].cpu().double() / x[1].double() - 1).abs() <= 2.0 ** -23 + ro.half_step(DT[dtype])).all()


@pytest.mark.parametrize("cols", [128, 200, 97])
@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
def test_infinities_mark_their_group(cols, value):
    x = _x(6, cols, torch.bfloat16)
    x[2, 50] = value
    codes, scales = tk.pack_activation(x.cuda())
    back = tk.unpack_activation(codes, scales)
    assert torch.isnan(back[2, :min(128, cols)].float()).all()
    x[2, :128] = 0
    clean = tk.unpack_activation(*tk.pack_activation(x.cuda()))
    assert torch.equal(back[[0, 1, 3, 4, 5]], clean[[0, 1, 3, 4, 5]]) and torch.equal(back[2, 128:], clean[2, 128:])


def test_layouts():
    x = _x(30, 256, torch.bfloat16)
    wide = torch.full((30, 400), float("nan"), device="cuda", dtype=torch.bfloat16)
    for first in (0, 8, 5):
        wide[:, first:first + 256] = x.cuda()
        _check(x, wide[:, first:first + 256])
    _check(x.view(5, 6, 256).transpose(0, 1).contiguous(), x.view(5, 6, 256).cuda().transpose(0, 1))
    _check(x[4].expand(9, 256).contiguous(), x[4].cuda().expand(9, 256))
    _check(x[7])
    codes, scales = tk.pack_activation(x.cuda())
    c2 = torch.empty(30, 300, device="cuda", dtype=torch.int8)
    c2[:, 3:259] = codes
    assert torch.equal(tk.unpack_activation(c2[:, 3:259], scales), tk.unpack_activation(codes, scales))
    for shape in ((0, 128), (4, 0)):
        codes, scales = tk.pack_activation(torch.empty(shape, device="cuda"))
        assert tk.unpack_activation(codes, scales).shape == shape


def test_more_than_2_31_elements():
    x = torch.zeros(2 ** 24 + 3, 128, device="cuda", dtype=torch.bfloat16)
    tail = _x(5, 128, torch.bfloat16)
    x[-5:] = tail.cuda()
    codes, scales = tk.pack_activation(x)
    back = tk.unpack_activation(codes, scales)
    c, s, v = ro.pack(tail)
    assert torch.equal(codes[-5:].cpu().double(), c) and torch.equal(back[-5:].cpu(), v.float().bfloat16())
    assert not codes[:-5].any() and not back[:-5].any()


def test_no_gradient_passes():
    x = torch.randn(4, 128, device="cuda", requires_grad=True)
    codes, scales = tk.pack_activation(x)
    assert not scales.requires_grad and not tk.unpack_activation(codes, scales).requires_grad


def test_traced_route_matches_eager():
    x = _x(10, 200, torch.float16).cuda()
    f = lambda t: tk.unpack_activation(*tk.pack_activation(t), torch.float16)  # noqa: E731
    assert torch.equal(torch.compile(f, fullgraph=True, backend="aot_eager")(x), f(x))
    torch.library.opcheck(torch.ops.tpf_b200.int8_pack, (x,), test_utils=("test_schema", "test_faketensor"))


# ---- int8_activations ----------------------------------------------------------------------------
def _value_of(t):
    """What the context gives back for t: groups in memory order."""
    flat = t.detach().cpu().as_strided((t.numel(),), (1,))
    rows = flat.view(-1, 128) if flat.numel() % 128 == 0 else flat.view(1, -1)
    return ro.pack(rows)[2].float().to(t.dtype).view(-1).as_strided(t.size(), t.stride()).cuda()


@pytest.mark.parametrize("shape", [(64, 128), (33, 77)])
@pytest.mark.parametrize("transposed", [False, True])
def test_context_gives_back_the_kept_values(shape, transposed):
    x = _x(*shape, torch.bfloat16).cuda()
    x = (x.t() if transposed else x).detach().requires_grad_(True)
    with tk.int8_activations(min_elements=1):
        h = x * 1.0
        y = h * h                       # keeps h
    (g,) = torch.autograd.grad(y.sum(), x)
    assert torch.equal(g, _value_of(h) * 2)


def test_context_keeps_parameters_statistics_and_small_tensors_whole():
    seen = []
    w = torch.randn(256, 256, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    x = torch.randn(64, 256, device="cuda", dtype=torch.bfloat16)
    with tk.int8_activations(min_elements=1, keep_whole=lambda t: seen.append(tuple(t.shape)) or False):
        y = torch.nn.functional.linear(x, w)
        z = (y.float() * y.float()).sum()
    (g,) = torch.autograd.grad(z, w)
    assert (256, 256) not in seen and (64, 256) in seen
    ref = (2 * y.float()).bfloat16().t().float() @ _value_of(x).float()
    # one rounding to bf16 at the end (and fp32 sums of 64 terms)
    assert ((g.float() - ref).abs() <= 2.0 ** -8 * ref.abs() + 1e-3).all()
    with tk.int8_activations(min_elements=64 * 256 + 1):
        y = torch.nn.functional.linear(x, w)
    (g1,) = torch.autograd.grad(y.sum(), w)
    (g2,) = torch.autograd.grad(torch.nn.functional.linear(x, w).sum(), w)
    assert torch.equal(g1, g2)
    with tk.int8_activations(min_elements=1, keep_whole=lambda t: True):
        y = torch.nn.functional.linear(x, w)
    assert torch.equal(torch.autograd.grad(y.sum(), w)[0], g2)


@pytest.mark.parametrize("frozen", [True, False])
def test_context_leaves_weights_alone(frozen):
    """A frozen weight, or autocast's copy of a trained one: the input's gradient is that without the context, bit by bit,
    and nothing more is kept."""
    g = torch.Generator(device="cuda").manual_seed(4)
    w = torch.randn(256, 256, device="cuda", generator=g)
    w = torch.nn.Parameter(w.bfloat16() if frozen else w, requires_grad=not frozen)
    x = torch.randn(512, 256, device="cuda", generator=g).bfloat16().requires_grad_(True)
    d = torch.randn(512, 256, device="cuda", generator=g).bfloat16()

    def run(context):
        h = x * 1.0
        before = torch.cuda.memory_allocated()
        with torch.autocast("cuda", torch.bfloat16, enabled=not frozen), context:
            y = torch.nn.functional.linear(h, w)
        kept = torch.cuda.memory_allocated() - before
        return torch.autograd.grad(y, x, d)[0], kept

    import contextlib
    run(contextlib.nullcontext())
    g0, m0 = run(contextlib.nullcontext())
    g1, m1 = run(tk.int8_activations(min_elements=1))
    assert torch.equal(g0, g1)
    if frozen:
        assert m1 == m0
    w8 = _value_of(w.detach().bfloat16().t())
    assert not torch.equal(g0, (d.float() @ w8.t().float()).bfloat16())   # (the codes would have been seen)


def test_what_the_context_keeps():
    """Bytes of one tensor of 2^20 elements with one, two and four nodes that keep it, each with codes of its own; without the
    context autograd holds it once."""
    import contextlib
    n = 2 ** 20
    packed = n + 4 * n // 128
    x = torch.randn(4096, 256, device="cuda").bfloat16()
    ws = [torch.nn.Parameter(torch.randn(8, 256, device="cuda").bfloat16()) for _ in range(4)]
    linears = lambda k: (lambda h: [torch.nn.functional.linear(h, w) for w in ws[:k]])  # noqa: E731

    def kept(f, context):
        with context:
            h = x * 1.0
            before = torch.cuda.memory_allocated()
            out = f(h)
        size = sum(t.numel() * t.element_size() for t in out)
        del h
        return torch.cuda.memory_allocated() - before - size    # of h and of what is kept, but for h's 2 n

    slack = 4096
    for f, codes in ((linears(1), 1), (linears(2), 2), (linears(4), 4)):
        assert abs(kept(f, contextlib.nullcontext())) <= slack
        assert abs(kept(f, tk.int8_activations(min_elements=n)) - (codes * packed - 2 * n)) <= slack * codes


def test_context_keeps_what_a_tensor_held_when_it_was_kept():
    """A buffer that is written behind autograd's back (a replayed graph, a kernel) between two nodes that keep it."""
    x = torch.nn.Parameter(torch.zeros(256, device="cuda", dtype=torch.bfloat16))
    buf = torch.empty(64, 256, device="cuda", dtype=torch.bfloat16)
    parts = [_x(64, 256, torch.bfloat16, seed=s).cuda() for s in (1, 2)]
    with tk.int8_activations(min_elements=1):
        out = []
        for p in parts:
            buf.data.copy_(p)
            out.append((buf * x).float().sum())
    (g,) = torch.autograd.grad(out[0] + out[1], x)
    ref = sum(_value_of(p).double().sum(0) for p in parts)
    # two bf16 gradients (sums of 64 terms in fp32), and their bf16 sum
    mags = sum(_value_of(p).double().abs().sum(0) for p in parts)
    assert ((g.double() - ref).abs() <= 2.0 ** -8 * 3 * mags + 64 * 2.0 ** -24 * mags).all()


def test_context_around_the_framework_operators():
    """TriMul, layer norm and projection inside the context: gradients near those without it, less memory kept."""
    from openfold3_triangle_kernel_b200.synthetic import trimul_inputs

    t = trimul_inputs(1, 64, 64, seed=3)
    w = {k: v.cuda() for k, v in t["weights"].items()}
    wo = (torch.randn(128, 64, generator=torch.Generator().manual_seed(1)) / 8).bfloat16().cuda()

    def run(context):
        z = t["z"].cuda().requires_grad_(True)
        before = torch.cuda.memory_allocated()
        with context:
            u = z + tk.turbo_trimul(z, "outgoing", t["mask"].cuda(), **w)
            v = torch.nn.functional.silu(tk.turbo_norm_linear(u, None, None, wo))
        kept = torch.cuda.memory_allocated() - before
        (g,) = torch.autograd.grad(v.float().square().mean() * 100, z)
        return g.float(), kept

    import contextlib
    g0, m0 = run(contextlib.nullcontext())
    g1, m1 = run(tk.int8_activations(min_elements=1024))
    assert m1 < m0
    # each kept value is off by a / 254 of its group, about 1 % of a typical one; three of them enter each gradient
    assert (g1 - g0).norm() / g0.norm() < 0.04


def test_context_around_a_masked_attention():
    """The additive mask is fp32 and stays whole, its infinities with it.  At logits of a standard deviation of 1 each kept value
    is off by 0.6 % (root mean square), a logit by 0.006 sqrt(2), and P, v and the output by as much again: below 4 % in all."""
    import contextlib
    g = torch.Generator(device="cuda").manual_seed(2)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g).bfloat16().requires_grad_(True)  # noqa: E731
    q, k, v, bias = r(1, 16, 4, 96, 32), r(1, 16, 4, 96, 32), r(1, 16, 4, 96, 32), r(1, 1, 4, 96, 96)
    mask = torch.zeros(1, 16, 1, 1, 96, device="cuda")
    mask[:, :, ..., 80:] = -float("inf")
    mask[:, 3] = -float("inf")      # a row without a key
    d = r(1, 16, 96, 4, 32).detach()

    def run(context):
        with context:
            o = tk.turbo_attention(q * 1, k * 1, v * 1, pair_bias=bias * 1, res_mask=mask)
        return torch.autograd.grad(o, (q, k, v, bias), d)

    for a, b in zip(run(contextlib.nullcontext()), run(tk.int8_activations(min_elements=1))):
        assert torch.isfinite(b).all()
        assert 0 < (a.float() - b.float()).norm() / a.float().norm() < 0.04


def test_context_inside_a_capture():
    """What is packed while a graph is captured is packed again by every replay."""
    w = torch.randn(64, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    x = torch.randn(100, 64, device="cuda", dtype=torch.bfloat16)
    d = torch.randn(100, 64, device="cuda", dtype=torch.bfloat16)

    def step():
        with tk.int8_activations(min_elements=1000):
            y = torch.tanh(x * 2) @ w
        return torch.autograd.grad(y, w, d)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for seed in (1, 2):
        x.copy_(torch.randn(100, 64, generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, step())

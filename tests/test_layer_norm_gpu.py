"""turbo_layer_norm on a B200 against the 64-bit oracle (bounds derived in oracle/rows_oracle.py)."""
import pytest
import torch

import openfold3_triangle_kernel_b200 as tk
from openfold3_triangle_kernel_b200 import _cabi as C
from oracle import rows_oracle as ro

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA device")]

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _inputs(rows, cols, dtype, seed=0, wdtype=torch.float32, offset=0.3):
    g = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    x = (rn(rows, cols) * torch.exp(0.5 * rn(cols)) + offset * rn(rows, 1)).to(dtype)
    return dict(x=x, w=(1 + 0.2 * rn(cols)).to(wdtype), b=(0.2 * rn(cols)).to(wdtype), dy=rn(rows, cols).to(dtype))


def _check(i, eps=1e-5, checkpoint=None, use_w=True, use_b=True, x_cuda=None):
    w, b = (i["w"] if use_w else None), (i["b"] if use_b else None)
    x = (i["x"].cuda() if x_cuda is None else x_cuda).detach().requires_grad_(True)
    p = [t.cuda().requires_grad_(True) if t is not None else None for t in (w, b)]
    y = tk.turbo_layer_norm(x, *p, eps=eps, checkpoint=checkpoint)
    assert y.dtype == x.dtype and y.shape == x.shape and y.is_contiguous()
    leaves = [t for t in (x, *p) if t is not None]
    grads = torch.autograd.grad(y, leaves, i["dy"].cuda().view(x.shape))
    rows = i["x"].reshape(-1, i["x"].shape[-1])
    ref, mean, rstd, off = ro.layer_norm(rows, w, b, eps)
    kept = ro.pack(rows)[2] if checkpoint else rows
    back = ro.layer_norm_backward(i["dy"].view(rows.shape), kept, mean, rstd, w)
    ro.check(y.reshape(rows.shape), ref, off, "y")
    ro.check(grads[0].reshape(rows.shape), back["dx"], back["dx_off"], "dx")
    k = 1
    if use_w:
        assert grads[k].dtype == w.dtype
        ro.check(grads[k], back["dw"], back["dw_off"], "dw")
        k += 1
    if use_b:
        ro.check(grads[k], back["db"], back["db_off"], "db")
    with torch.no_grad():
        assert torch.equal(tk.turbo_layer_norm(x, *p, eps=eps), y)
    return y, grads


# every width class of the two layouts, their borders, one column, rows that fill no block
@pytest.mark.parametrize("cols", [1, 7, 8, 32, 33, 40, 64, 72, 97, 128, 129, 136, 256, 257, 264, 384, 512, 513, 1001, 1024,
                                  1032, 2000, 2048, 2049, 4096, 4097, 5000, 8191, 8192])
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_widths(cols, dtype):
    _check(_inputs(37, cols, DT[dtype], seed=cols))


@pytest.mark.parametrize("cols", [1, 8, 24, 32, 64, 96, 97, 128, 136, 200, 384, 1000, 1001, 2048, 3000, 4099, 8192])
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_int8_checkpoint(cols, dtype):
    _check(_inputs(41, cols, DT[dtype], seed=cols + 1), checkpoint="int8")


@pytest.mark.parametrize("cols", [9, 17, 31, 57, 58, 63, 121, 122, 127, 130, 249, 250, 255, 301, 505, 511, 513, 1018, 1022, 2049, 4090,
                                  8185, 8191])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("checkpoint", [None, "int8"])
def test_odd_widths_of_many_rows(cols, dtype, checkpoint):
    _check(_inputs(3001 if cols < 600 else 301, cols, DT[dtype], seed=cols + 2), checkpoint=checkpoint)


@pytest.mark.parametrize("rows", [63, 64, 65, 66, 71, 72, 120, 1001])
@pytest.mark.parametrize("cols", [9, 93, 517])
def test_odd_widths_of_some_rows(rows, cols):
    _check(_inputs(rows, cols, torch.bfloat16, seed=rows))


@pytest.mark.parametrize("cols", [9, 45, 333, 1001])
def test_odd_widths_keep_rows_apart(cols):
    """Infinities and NaN of a row stay in it where rows begin at any address, and nothing behind the last row is read or written."""
    rows = 200
    i = _inputs(rows, cols, torch.bfloat16)
    bad = list(range(0, rows, 3)) + [rows - 1]
    good = [r for r in range(rows) if r not in bad]

    def run(x, dy):
        buf = torch.full((rows * cols + 64,), float("nan"), device="cuda", dtype=torch.bfloat16)
        xc = buf[:rows * cols].view(rows, cols).copy_(x.cuda()).requires_grad_(True)
        y = tk.turbo_layer_norm(xc, i["w"].cuda(), i["b"].cuda())
        (g,) = torch.autograd.grad(y, xc, dy.cuda())
        assert torch.isnan(buf[rows * cols:].float()).all()
        return y, g

    y0, g0 = run(i["x"], i["dy"])
    x, dy = i["x"].clone(), i["dy"].clone()
    x[bad, 0], x[bad, cols - 1] = float("inf"), float("nan")
    dy[bad, 0], dy[bad, cols - 1] = float("nan"), float("inf")
    y1, g1 = run(x, dy)
    assert torch.equal(y0[good], y1[good]) and torch.equal(g0[good], g1[good])
    assert torch.isnan(y1[bad].float()).all() and torch.isnan(g1[bad].float()).all()


@pytest.mark.parametrize("rows", [1, 2, 3, 31, 33, 64, 65, 97, 257, 4099])
@pytest.mark.parametrize("cols", [96, 128, 384, 1001])
@pytest.mark.parametrize("checkpoint", [None, "int8"])
def test_row_counts(rows, cols, checkpoint):
    _check(_inputs(rows, cols, torch.bfloat16, seed=rows), checkpoint=checkpoint)


@pytest.mark.parametrize("use_w, use_b", [(True, False), (False, True), (False, False)])
@pytest.mark.parametrize("cols", [128, 100])
def test_absent_parameters(use_w, use_b, cols):
    _check(_inputs(50, cols, torch.bfloat16), use_w=use_w, use_b=use_b)


@pytest.mark.parametrize("wdtype", ["bf16", "fp16", "fp32"])
def test_parameter_types(wdtype):
    _check(_inputs(300, 128, torch.bfloat16, wdtype=DT[wdtype]))


def test_large_mean_and_eps():
    # a mean that is 3000 times the spread: squares are summed after it is taken off
    i = _inputs(64, 384, torch.float32, offset=0.0)
    i["x"] = i["x"] + 3000
    _check(i)
    _check(_inputs(64, 384, torch.float32), eps=0.5)


def test_constant_rows():
    i = _inputs(20, 128, torch.bfloat16)
    i["x"][3] = 0
    i["x"][4] = 2.5
    i["dy"][3] = 0
    _check(i)
    _check(i, checkpoint="int8")


def test_layouts():
    i = _inputs(48, 128, torch.bfloat16)
    x = i["x"].cuda()
    ref = tk.turbo_layer_norm(x, i["w"].cuda(), i["b"].cuda())
    wide = torch.full((48, 300), float("nan"), device="cuda", dtype=torch.bfloat16)
    for first in (0, 8, 3):   # aligned rows at a pitch; a misaligned start
        wide[:, first:first + 128] = x
        _check(i, x_cuda=wide[:, first:first + 128])
        _check(i, x_cuda=wide[:, first:first + 128], checkpoint="int8")
    odd = torch.empty(48, 301, device="cuda", dtype=torch.bfloat16)
    odd[:, :128] = x
    _check(i, x_cuda=odd[:, :128])
    # leading dimensions that do not collapse: a copy
    t = x.view(6, 8, 128).transpose(0, 1)
    assert torch.equal(tk.turbo_layer_norm(t, i["w"].cuda(), i["b"].cuda()), ref.view(6, 8, 128).transpose(0, 1))
    assert torch.equal(tk.turbo_layer_norm(x.t().contiguous().t(), i["w"].cuda(), i["b"].cuda()), ref)
    # one row for all, parameters with strides
    row = x[5]
    assert torch.equal(tk.turbo_layer_norm(row.expand(7, 128), i["w"].cuda()), tk.turbo_layer_norm(row, i["w"].cuda()).expand(7, 128))
    w2 = torch.stack([i["w"], i["w"]], 1).cuda()[:, 0]
    assert torch.equal(tk.turbo_layer_norm(x, w2, i["b"].cuda()), ref)


def test_expanded_incoming_gradient_and_broadcast_input():
    x = torch.randn(5, 1, 128, device="cuda", requires_grad=True)
    w = torch.randn(128, device="cuda", requires_grad=True)
    tk.turbo_layer_norm(x.expand(5, 9, 128), w).sum().backward()
    x2, w2 = x.detach().double().requires_grad_(True), w.detach().double().requires_grad_(True)
    torch.nn.functional.layer_norm(x2.expand(5, 9, 128), (128,), w2).sum().backward()
    # dx of a sum: terms of size w rstd that cancel; 9 of them are added
    scale = float(w2.detach().abs().max() * 10)
    assert (x.grad.double() - x2.grad).abs().max() < 9 * 1024 * ro.U * scale
    assert (w.grad.double() - w2.grad).abs().max() < 45 * 256 * ro.U * 10


def test_no_rows():
    x = torch.empty(0, 128, device="cuda", requires_grad=True)
    w = torch.ones(128, device="cuda", requires_grad=True)
    for keep in (None, "int8"):
        y = tk.turbo_layer_norm(x, w, checkpoint=keep)
        gx, gw = torch.autograd.grad(y.sum(), (x, w))
        assert y.shape == (0, 128) and gx.shape == (0, 128) and torch.equal(gw, torch.zeros_like(w))


@pytest.mark.parametrize("checkpoint", [None, "int8"])
def test_infinities_stay_in_their_rows(checkpoint):
    i = _inputs(40, 128, torch.bfloat16)
    x = i["x"].clone()
    x[7, 3], x[9, 100], x[11, 0] = float("inf"), float("nan"), float("-inf")
    w = i["w"].cuda().requires_grad_(True)
    xc = x.cuda().requires_grad_(True)
    y = tk.turbo_layer_norm(xc, w, i["b"].cuda(), checkpoint=checkpoint)
    (gx,) = torch.autograd.grad(y, xc, i["dy"].cuda())
    good = [r for r in range(40) if r not in (7, 9, 11)]
    clean = i["x"].cuda().requires_grad_(True)
    yc = tk.turbo_layer_norm(clean, w, i["b"].cuda(), checkpoint=checkpoint)
    (gc,) = torch.autograd.grad(yc, clean, i["dy"].cuda())
    assert torch.equal(y[good], yc[good]) and torch.equal(gx[good], gc[good])
    for r in (7, 9, 11):
        assert torch.isnan(y[r].float()).all() and torch.isnan(gx[r].float()).all()


def test_some_gradients_only():
    i = _inputs(100, 128, torch.bfloat16)
    x, w, b = i["x"].cuda(), i["w"].cuda(), i["b"].cuda()
    full = [t.clone().requires_grad_(True) for t in (x, w, b)]
    ref = torch.autograd.grad(tk.turbo_layer_norm(*full), full, i["dy"].cuda())
    for which in ([0], [1], [2], [0, 2], [1, 2]):
        leaves = [t.clone().requires_grad_(k in which) for k, t in enumerate((x, w, b))]
        got = torch.autograd.grad(tk.turbo_layer_norm(*leaves), [leaves[k] for k in which], i["dy"].cuda())
        for k, g in zip(which, got):
            assert torch.equal(g, ref[k])
    # asked for some, with all wanting one; the bias alone, without a weight
    got = torch.autograd.grad(tk.turbo_layer_norm(*full), full[2], i["dy"].cuda())
    assert torch.equal(got[0], ref[2])
    b2 = b.clone().requires_grad_(True)
    assert torch.equal(torch.autograd.grad(tk.turbo_layer_norm(x, None, b2), b2, i["dy"].cuda())[0], ref[2])


def test_kept_input_is_watched():
    x = torch.randn(8, 128, device="cuda", requires_grad=True)
    h = x * 2
    y = tk.turbo_layer_norm(h)
    h.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    h = x * 2
    y = tk.turbo_layer_norm(h, checkpoint="int8")   # the codes were written in the forward pass
    h.add_(1)
    y.sum().backward()


def test_second_derivative_raises():
    x = torch.randn(8, 128, device="cuda", requires_grad=True)
    (g,) = torch.autograd.grad(tk.turbo_layer_norm(x).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        g.sum().backward()


def test_gradient_against_differences():
    # central differences of the 64-bit definition, from the operator's own gradient in fp32
    i = _inputs(3, 40, torch.float32)
    x = i["x"].cuda().requires_grad_(True)
    (g,) = torch.autograd.grad(tk.turbo_layer_norm(x, i["w"].cuda(), i["b"].cuda()), x, i["dy"].cuda())
    f = lambda t: float((ro.layer_norm(t, i["w"], i["b"], 1e-5)[0] * i["dy"].double()).sum())  # noqa: E731
    h = 2.0 ** -13
    for r, c in ((0, 0), (1, 17), (2, 39)):
        e = torch.zeros(3, 40, dtype=torch.float64)
        e[r, c] = h
        slope = (f(i["x"].double() + e) - f(i["x"].double() - e)) / (2 * h)
        # h^2 / 6 times a third derivative of order |dy| rstd^3 per element, 40 elements
        assert abs(float(g[r, c]) - slope) < 40 * h * h * 20 + 192 * ro.U * 40


def test_same_bits_every_time():
    i = _inputs(5000, 384, torch.bfloat16)
    a = _check(i, checkpoint="int8")
    b = _check(i, checkpoint="int8")
    assert torch.equal(a[0], b[0]) and all(torch.equal(s, t) for s, t in zip(a[1], b[1]))


def test_more_than_2_31_elements():
    rows = 2 ** 24 + 5
    x = torch.zeros(rows, 128, device="cuda", dtype=torch.bfloat16)
    tail = _inputs(9, 128, torch.bfloat16)
    x[-9:] = tail["x"].cuda()
    x.requires_grad_(True)
    w = tail["w"].cuda().requires_grad_(True)
    for keep in (None, "int8"):
        y = tk.turbo_layer_norm(x, w, checkpoint=keep)
        dy = torch.zeros_like(y)
        dy[-9:] = tail["dy"].cuda()
        gx, gw = torch.autograd.grad(y, (x, w), dy)
        ref, mean, rstd, off = ro.layer_norm(tail["x"], tail["w"], None, 1e-5)
        kept = ro.pack(tail["x"])[2] if keep else tail["x"]
        back = ro.layer_norm_backward(tail["dy"], kept, mean, rstd, tail["w"])
        ro.check(y[-9:], ref, off, "y")
        ro.check(gx[-9:], back["dx"], back["dx_off"], "dx")
        ro.check(gw, back["dw"], back["dw_off"], "dw")
        assert not gx[:-9].any()
        del y, dy, gx


def test_streams_and_two_calls_at_once():
    i = _inputs(3000, 384, torch.bfloat16)
    ref = _check(i)
    torch.cuda.synchronize()
    x, w, b, dy = (i[n].cuda() for n in ("x", "w", "b", "dy"))
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            for _ in range(5):
                y = tk.turbo_layer_norm(*leaves)
                got.append((y, torch.autograd.grad(y, leaves, dy)))
    torch.cuda.synchronize()
    for y, g in got:
        assert torch.equal(y, ref[0]) and all(torch.equal(s, t) for s, t in zip(g, ref[1]))


@pytest.mark.parametrize("checkpoint", [None, "int8"])
def test_captured_training_pass(checkpoint):
    i, j = _inputs(500, 128, torch.bfloat16, seed=1), _inputs(500, 128, torch.bfloat16, seed=2)
    ref = [_check(k, checkpoint=checkpoint) for k in (i, j)]
    x, w, b, dy = (i[n].cuda() for n in ("x", "w", "b", "dy"))
    leaves = [t.requires_grad_(True) for t in (x, w, b)]

    def step():
        y = tk.turbo_layer_norm(*leaves, checkpoint=checkpoint)
        return (y.detach(), *torch.autograd.grad(y, leaves, dy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k, r in zip((i, j), ref):
        with torch.no_grad():
            for t, n in ((x, "x"), (w, "w"), (b, "b"), (dy, "dy")):
                t.copy_(k[n].cuda())
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[0], r[0]) and all(torch.equal(s, t) for s, t in zip(out[1:], r[1]))


@pytest.mark.parametrize("checkpoint", [None, "int8"])
def test_traced_route_matches_eager(checkpoint):
    i = _inputs(60, 96, torch.bfloat16)
    leaves = [i[n].cuda().requires_grad_(True) for n in ("x", "w", "b")]
    f = lambda x, w, b: tk.turbo_layer_norm(x, w, b, checkpoint=checkpoint)  # noqa: E731
    y = f(*leaves)
    g = torch.autograd.grad(y, leaves, i["dy"].cuda())
    yc = torch.compile(f, fullgraph=True, backend="aot_eager")(*leaves)
    gc = torch.autograd.grad(yc, leaves, i["dy"].cuda())
    assert torch.equal(y, yc) and all(torch.equal(a, b) for a, b in zip(g, gc))
    args = (leaves[0].detach().requires_grad_(True), leaves[1], None, 1e-5, checkpoint == "int8")
    torch.library.opcheck(torch.ops.tpf_b200.layer_norm_fwd, args,
                          test_utils=("test_schema", "test_autograd_registration", "test_faketensor"))


def test_a_traced_graph_meets_the_contract_when_it_runs():
    """Sizes and devices that differ from the traced ones are refused before a launch."""
    x, w = torch.randn(6, 64, device="cuda"), torch.ones(64, device="cuda")
    wide, mat = torch.randn(6, 128, device="cuda"), torch.zeros(16, 64, device="cuda")
    norm = torch.jit.trace(lambda t: tk.turbo_layer_norm(t, w), (x,), check_trace=False)
    proj = torch.jit.trace(lambda t: tk.turbo_norm_linear(t.bfloat16(), None, None, mat), (x,), check_trace=False)
    unpack = torch.jit.trace(lambda c, s: tk.unpack_activation(c, s), tuple(tk.pack_activation(x)), check_trace=False)
    codes, scales = tk.pack_activation(wide)
    more = torch.randn(9, 64, device="cuda")
    assert torch.equal(norm(more), tk.turbo_layer_norm(more, w))
    ops = torch.ops.tpf_b200
    dy, stats = torch.zeros(6, 64, device="cuda"), torch.zeros(2, 6, device="cuda")
    none = torch.empty(0, device="cuda", dtype=torch.int8)
    before = C.load().tpf_launch_count()
    for call in (lambda: norm(wide), lambda: proj(wide), lambda: unpack(codes, scales[:1]),
                 lambda: ops.layer_norm_fwd(x, w.cpu(), None, 1e-5, False),
                 lambda: ops.norm_linear_fwd(x.bfloat16(), None, None, mat.cpu(), 1e-5, False),
                 lambda: ops.layer_norm_bwd(dy, None, stats, none, scales, w, None),
                 lambda: ops.layer_norm_bwd(dy, x, stats[:, :3], none, scales, w, None),
                 lambda: ops.norm_linear_bwd(dy, x.bfloat16(), stats, none, scales, None, None, mat)):
        with pytest.raises(Exception, match=r"unsupported \["):
            call()
    with pytest.raises(Exception):
        norm(x.cpu())
    kernels = C.load().tpf_launch_count() - before
    assert kernels == 0


def test_backward_operators_take_strided_statistics():
    i = _inputs(40, 96, torch.bfloat16)
    x, w, b, dy = (i[n].cuda() for n in ("x", "w", "b", "dy"))
    ops = torch.ops.tpf_b200
    for int8 in (False, True):
        y, stats, codes, scales = ops.layer_norm_fwd(x, w, b, 1e-5, int8)
        both = torch.stack([stats, stats], 2)[..., 0]
        wide = torch.cat([codes, codes], -1)[..., :codes.shape[-1]]
        ref = ops.layer_norm_bwd(dy, None if int8 else x, stats, codes, scales, w, b)
        got = ops.layer_norm_bwd(dy, None if int8 else x, both, wide, scales, w, b)
        assert not both.is_contiguous() and all(torch.equal(s, t) for s, t in zip(ref, got))


def test_refusals_leave_no_launch():
    before = C.load().tpf_launch_count()
    x = torch.zeros(4, 128, device="cuda")
    for bad in (dict(x=x.double()), dict(x=x, weight=torch.ones(128)), dict(x=x, weight=torch.ones(64, device="cuda")),
                dict(x=x, checkpoint="int4"), dict(x=torch.zeros(1, 8200, device="cuda")), dict(x=x, eps=-1e-5)):
        with pytest.raises(ValueError, match="turbo_layer_norm unsupported"):
            tk.turbo_layer_norm(**bad)
    assert C.load().tpf_launch_count() == before

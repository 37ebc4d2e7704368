"""turbo_norm_linear on a B200 against the 64-bit oracle.

Bounds: the normalised rows y and the gradient dy are rounded to bf16 (half a step, 2^-8 of the value) on their way into
products, an fp32 or fp16 weight likewise; the products' sums are fp32, at most K roundings.  The gradients of narrow rows
come from G = d_out^T xh and s = d_out^T 1: there xh is rounded in the place of y, and the norm's gradients are
sum_o W_oc G_oc and sum_o W_oc s_o: their first error is sum_r dy_rc (what xh_rc is off by), as before, and the sums over r and
o are fp32 chains of R + O roundings, relative to the magnitudes |d_out|, |W| and |xh| of their terms."""
import pytest
import torch

import openfold3_triangle_kernel_b200 as tk
from openfold3_triangle_kernel_b200 import _cabi as C
from oracle import rows_oracle as ro

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA device")]

H = 2.0 ** -8


def _inputs(rows, cols, outs, seed=0, wdtype=torch.bfloat16):
    g = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    x = (rn(rows, cols) * torch.exp(0.5 * rn(cols)) + 0.3 * rn(rows, 1)).bfloat16()
    return dict(x=x, nw=(1 + 0.2 * rn(cols)).to(wdtype), nb=(0.2 * rn(cols)).to(wdtype),
                w=(rn(outs, cols) * (2.0 / (cols + outs)) ** 0.5).to(wdtype), d_out=rn(rows, outs).bfloat16())


def _run(i, checkpoint=None, eps=1e-5, x_cuda=None, use=(True, True)):
    x = (i["x"].cuda() if x_cuda is None else x_cuda).detach().requires_grad_(True)
    p = [i[n].cuda().requires_grad_(True) if u else None for n, u in (("nw", use[0]), ("nb", use[1]), ("w", True))]
    out = tk.turbo_norm_linear(x, *p, eps=eps, checkpoint=checkpoint)
    leaves = [t for t in (x, *p) if t is not None]
    names = [n for n, t in zip(("dx", "dnw", "dnb", "dw"), (x, *p)) if t is not None]
    grads = torch.autograd.grad(out, leaves, i["d_out"].cuda().view(out.shape))
    with torch.no_grad():
        assert torch.equal(tk.turbo_norm_linear(x, *p, eps=eps), out)
    return out, dict(zip(names, grads))


def _check(i, checkpoint=None, eps=1e-5, x_cuda=None, use=(True, True)):
    out, g = _run(i, checkpoint, eps, x_cuda, use)
    rows = i["x"].reshape(-1, i["x"].shape[-1])
    nw, nb = (i["nw"] if use[0] else None), (i["nb"] if use[1] else None)
    R, Cc = rows.shape
    W, O = i["w"].double(), i["w"].shape[0]
    d = i["d_out"].double().view(R, O)
    hw = 0.0 if i["w"].dtype == torch.bfloat16 else H
    y, mean, rstd, y_off = ro.layer_norm(rows, nw, nb, eps)
    y_off = y_off + H * (y.abs() + y_off)
    out_off = y_off @ W.abs().t() * (1 + hw) + (hw + (Cc + 8) * ro.U) * (y.abs() @ W.abs().t())
    ro.check(out.reshape(R, O), y @ W.t(), out_off, "out")
    kept = ro.pack(rows)[2] if checkpoint else rows
    dy = d @ W
    dy_off = (hw + (O + 8) * ro.U) * (d.abs() @ W.abs())
    dy_off = dy_off + H * (dy.abs() + dy_off)
    back = ro.layer_norm_backward(dy, kept, mean, rstd, nw, dy_off)
    ro.check(g["dx"].reshape(R, Cc), back["dx"], back["dx_off"], "dx")
    xk = (kept.double() - mean) * rstd
    A = rstd * (kept.double().abs() + mean.abs() + kept.double().abs().mean(-1, keepdim=True))
    xk_off = 68 * ro.U * A
    terms = d.abs() @ W.abs()
    chain = (R + O + 64) * ro.U
    if use[0]:
        ro.check(g["dnw"], back["dw"], back["dw_off"] + chain * (terms * xk.abs()).sum(0), "dnw")
    if use[1]:
        ro.check(g["dnb"], back["db"], back["db_off"] + chain * terms.sum(0), "dnb")
    # the kept rows, normalised again: off as y is, with the kept values in the place of x
    one = torch.ones(Cc, dtype=torch.float64)
    nwd, nbd = (one if nw is None else nw.double()), (0 * one if nb is None else nb.double())
    yk = xk * nwd + nbd
    if Cc <= 128 and -(-O // 64) * -(-Cc // 64) <= 16:   # (the weight stays in shared memory)
        yk_off = nwd.abs() * (xk_off + H * (xk.abs() + xk_off))
    else:
        yk_off = 68 * ro.U * (A * nwd.abs() + nbd.abs())
        yk_off = yk_off + H * (yk.abs() + yk_off)
    dw_off = d.abs().t() @ yk_off + (R + 64) * ro.U * (d.abs().t() @ ((xk * nwd).abs() + nbd.abs()))
    assert g["dw"].dtype == i["w"].dtype
    ro.check(g["dw"], d.t() @ yk, dw_off, "dw")
    # The bounds above are for the worst signs, and wide where many rows are added.  Roundings are as often up as down: with
    # at most three on a way, each H / sqrt(3) of its value in the root mean square, a whole result is off by about H.
    for name, got, ref in (("out", out, y @ W.t()), ("dx", g["dx"], back["dx"]), ("dnw", g.get("dnw"), back["dw"]),
                           ("dnb", g.get("dnb"), back["db"]), ("dw", g["dw"], d.t() @ yk)):
        if got is not None:
            off = (got.detach().cpu().double().view(ref.shape) - ref).norm() / ref.norm()
            assert off < 2 * H, (name, float(off))
    assert C.device_status() == 0
    return out, g


@pytest.mark.parametrize("cols", [8, 16, 32, 40, 64, 96, 104, 128, 136, 200, 256, 264, 384, 512, 1000, 1024, 2048])
@pytest.mark.parametrize("checkpoint", [None, "int8"])
def test_widths(cols, checkpoint):
    _check(_inputs(150, cols, 136, seed=cols), checkpoint)


@pytest.mark.parametrize("outs", [8, 16, 24, 64, 120, 128, 136, 256, 384, 512, 520, 1024, 2056])
@pytest.mark.parametrize("cols", [32, 128, 264])
def test_outputs(outs, cols):
    _check(_inputs(140, cols, outs, seed=outs), "int8")


@pytest.mark.parametrize("rows", [1, 2, 7, 16, 17, 63, 64, 65, 127, 128, 129, 300, 1000, 4099, 20000])
@pytest.mark.parametrize("cols, outs", [(128, 512), (96, 64), (264, 136)])
@pytest.mark.parametrize("checkpoint", [None, "int8"])
def test_row_counts(rows, cols, outs, checkpoint):
    _check(_inputs(rows, cols, outs, seed=rows), checkpoint)


@pytest.mark.parametrize("rows, cols, outs", [(66049, 96, 384), (66049, 64, 1024), (50000, 128, 512), (70001, 128, 104),
                                              (9001, 200, 512)])
@pytest.mark.parametrize("checkpoint", [None, "int8"])
def test_many_rows(rows, cols, outs, checkpoint):
    """Every stage of the rings is used many times over; several runs, since what goes wrong there goes wrong now and then."""
    i = _inputs(rows, cols, outs, seed=rows)
    out, g = _check(i, checkpoint)
    for _ in range(5):
        again, h = _run(i, checkpoint)
        assert torch.equal(out, again) and all(torch.equal(g[n], h[n]) for n in g)


@pytest.mark.parametrize("rows", [1, 33, 64, 257, 320, 1281])
@pytest.mark.parametrize("cols, outs", [(64, 64), (128, 128), (40, 1024), (128, 512)])
@pytest.mark.parametrize("checkpoint", [None, "int8"])
def test_ranges_of_one_step(rows, cols, outs, checkpoint):
    """Up to 64 rows in a range, or in its last: of the two groups of warps that make xh, the second has no step.  The sums
    are staged over its buffer, so nothing may be on its way there; what could go wrong would do so now and then."""
    i = _inputs(rows, cols, outs, seed=rows)
    out, g = _check(i, checkpoint)
    for _ in range(20):
        again, h = _run(i, checkpoint)
        assert torch.equal(out, again) and all(torch.equal(g[n], h[n]) for n in g)


@pytest.mark.parametrize("rows", [1, 2, 3, 4, 5])
@pytest.mark.parametrize("cols, outs", [(8, 8), (40, 2504), (136, 24), (1000, 4096), (1024, 520), (8192, 40)])
@pytest.mark.parametrize("checkpoint", [None, "int8"])
def test_few_rows(rows, cols, outs, checkpoint):
    _check(_inputs(rows, cols, outs, seed=rows + cols), checkpoint)


@pytest.mark.parametrize("wdtype", [torch.float32, torch.float16])
def test_parameter_types(wdtype):
    _check(_inputs(200, 128, 256, wdtype=wdtype), "int8")


@pytest.mark.parametrize("use", [(True, False), (False, True), (False, False)])
@pytest.mark.parametrize("checkpoint", [None, "int8"])
def test_absent_parameters(use, checkpoint):
    _check(_inputs(200, 128, 64), checkpoint, use=use)


def test_wide_rows():
    _check(_inputs(70, 8192, 64), "int8")


def test_more_than_2_31_elements():
    rows = 2 ** 24 + 5
    x = torch.zeros(rows, 128, device="cuda", dtype=torch.bfloat16)
    i = _inputs(9, 128, 8)
    x[-9:] = i["x"].cuda()
    d = torch.zeros(rows, 8, device="cuda", dtype=torch.bfloat16)
    d[-9:] = i["d_out"].cuda()
    nw, w = (i[n].cuda().requires_grad_(True) for n in ("nw", "w"))
    x.requires_grad_(True)
    for keep in (None, "int8"):
        # the nine rows by themselves give the same products in another order of sums
        small, g = _run(i, keep, use=(True, False))
        out = tk.turbo_norm_linear(x, nw, None, w, checkpoint=keep)
        gx, gn, gw = torch.autograd.grad(out, (x, nw, w), d)
        assert torch.equal(out[-9:], small) and not out[:-9].any()
        assert torch.equal(gx[-9:], g["dx"]) and not gx[:-9].any()
        for a, b in ((gn, g["dnw"]), (gw, g["dw"])):
            assert ((a.float() - b.float()).abs() <= 2 * H * b.float().abs() + 2 * 64 * ro.U * 9 * 16).all()
        del out, gx


def test_host_threads():
    """Four threads with a stream each, different sizes at once."""
    import threading

    cases = [_inputs(r, c, o, seed=r) for r, c, o in ((700, 128, 512), (333, 64, 128), (90, 256, 136), (3, 128, 64))]
    ref = [_run(c, "int8") for c in cases]
    torch.cuda.synchronize()
    bad = []

    def work(k):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(10):
                out, g = _run(cases[k], "int8")
                stream.synchronize()
                if not (torch.equal(out, ref[k][0]) and all(torch.equal(g[n], ref[k][1][n]) for n in g)):
                    bad.append(k)

    threads = [threading.Thread(target=work, args=(k,)) for k in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def test_layouts():
    i = _inputs(60, 128, 64)
    for first, pitch in ((0, 256), (8, 264), (3, 256), (0, 301)):
        wide = torch.full((60, pitch), float("nan"), device="cuda", dtype=torch.bfloat16)
        wide[:, first:first + 128] = i["x"].cuda()
        _check(i, None, x_cuda=wide[:, first:first + 128])
        _check(i, "int8", x_cuda=wide[:, first:first + 128])
    ref = tk.turbo_norm_linear(i["x"].cuda(), None, None, i["w"].cuda())
    t = i["x"].cuda().view(6, 10, 128).transpose(0, 1)
    got = tk.turbo_norm_linear(t, None, None, i["w"].cuda())
    assert torch.equal(got, ref.view(6, 10, 64).transpose(0, 1))
    wt = i["w"].cuda().t().contiguous().t()
    assert torch.equal(tk.turbo_norm_linear(i["x"].cuda(), None, None, wt), ref)
    flat = torch.empty(64 * 128 + 1, device="cuda", dtype=torch.bfloat16)
    flat[1:] = i["w"].cuda().view(-1)
    assert torch.equal(tk.turbo_norm_linear(i["x"].cuda(), None, None, flat[1:].view(64, 128)), ref)


def test_expanded_and_odd_gradients():
    i = _inputs(100, 128, 64)
    x, w = i["x"].cuda().requires_grad_(True), i["w"].cuda().requires_grad_(True)
    ref = torch.autograd.grad(tk.turbo_norm_linear(x, None, None, w), (x, w), torch.ones(100, 64, device="cuda").bfloat16())
    got = torch.autograd.grad(tk.turbo_norm_linear(x, None, None, w).sum(), (x, w))
    assert all(torch.equal(a, b) for a, b in zip(ref, got))
    d = torch.zeros(100 * 64 + 1, device="cuda", dtype=torch.bfloat16)[1:].view(100, 64).add_(1)   # misaligned
    got = torch.autograd.grad(tk.turbo_norm_linear(x, None, None, w), (x, w), d)
    assert all(torch.equal(a, b) for a, b in zip(ref, got))


def test_no_rows():
    x = torch.empty(0, 128, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    w = torch.ones(64, 128, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    nw = torch.ones(128, device="cuda", requires_grad=True)
    for keep in (None, "int8"):
        out = tk.turbo_norm_linear(x, nw, None, w, checkpoint=keep)
        g = torch.autograd.grad(out.sum(), (x, nw, w))
        assert out.shape == (0, 64) and not g[1].any() and not g[2].any()


def test_some_gradients_only():
    i = _inputs(300, 128, 192)
    _, ref = _run(i)
    names = ["dx", "dnw", "dnb", "dw"]
    base = [i[n].cuda() for n in ("x", "nw", "nb", "w")]
    for which in ([0], [1], [2], [3], [0, 3], [1, 2]):
        leaves = [t.clone().requires_grad_(k in which) for k, t in enumerate(base)]
        got = torch.autograd.grad(tk.turbo_norm_linear(*leaves), [leaves[k] for k in which], i["d_out"].cuda())
        for k, g in zip(which, got):
            assert torch.equal(g, ref[names[k]]), names[k]
        leaves = [t.clone().requires_grad_(True) for t in base]
        got = torch.autograd.grad(tk.turbo_norm_linear(*leaves), [leaves[k] for k in which], i["d_out"].cuda())
        for k, g in zip(which, got):
            assert torch.equal(g, ref[names[k]]), names[k]


@pytest.mark.parametrize("checkpoint", [None, "int8"])
def test_infinities_stay_in_their_rows(checkpoint):
    i = _inputs(200, 128, 64)
    clean, g0 = _run(i, checkpoint)
    i["x"][30, 5], i["x"][150, 100] = float("nan"), float("inf")
    out, g1 = _run_nan(i, checkpoint)
    good = [r for r in range(200) if r not in (30, 150)]
    assert torch.equal(out[good], clean[good]) and torch.equal(g1[good], g0["dx"][good])
    assert torch.isnan(out[[30, 150]].float()).all() and torch.isnan(g1[[30, 150]].float()).all()


def _run_nan(i, checkpoint):
    x = i["x"].cuda().requires_grad_(True)
    out = tk.turbo_norm_linear(x, i["nw"].cuda(), i["nb"].cuda(), i["w"].cuda(), checkpoint=checkpoint)
    return out, torch.autograd.grad(out, x, i["d_out"].cuda())[0]


def test_kept_input_is_watched_and_second_derivative_raises():
    x = torch.randn(8, 128, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    w = torch.randn(64, 128, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    h = x * 2
    out = tk.turbo_norm_linear(h, None, None, w)
    h.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()
    (g,) = torch.autograd.grad(tk.turbo_norm_linear(x, None, None, w).float().square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        g.sum().backward()


def test_same_bits_every_time_and_on_two_streams():
    i = _inputs(5000, 128, 256)
    ref = _run(i, "int8")
    torch.cuda.synchronize()
    got = []
    for s in [torch.cuda.Stream() for _ in range(2)]:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got += [_run(i, "int8") for _ in range(3)]
    torch.cuda.synchronize()
    for out, g in got:
        assert torch.equal(out, ref[0]) and all(torch.equal(g[n], ref[1][n]) for n in g)


@pytest.mark.parametrize("checkpoint", [None, "int8"])
def test_two_captured_training_passes(checkpoint):
    """Two graphs of the same operator, replayed one after the other and on new inputs."""
    cases = [_inputs(700, 128, 192, seed=s) for s in (1, 2, 3)]
    ref = [_run(c, checkpoint) for c in cases]
    made = []
    for c in cases[:2]:
        t = [c[n].cuda() for n in ("x", "nw", "nb", "w")]
        leaves, d = [v.requires_grad_(True) for v in t], c["d_out"].cuda()

        def step(leaves=leaves, d=d):
            out = tk.turbo_norm_linear(*leaves, checkpoint=checkpoint)
            return (out.detach(), *torch.autograd.grad(out, leaves, d))

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        made.append((graph, out, leaves, d))
    for first, second in ((0, 1), (1, 0)):
        made[first][0].replay()
        made[second][0].replay()
        torch.cuda.synchronize()
        for k in (0, 1):
            got, (out, g) = made[k][1], ref[k]
            assert torch.equal(got[0], out) and all(torch.equal(a, g[n]) for a, n in zip(got[1:], ("dx", "dnw", "dnb", "dw")))
    graph, got, leaves, d = made[0]
    with torch.no_grad():
        for v, n in zip(leaves, ("x", "nw", "nb", "w")):
            v.copy_(cases[2][n].cuda())
        d.copy_(cases[2]["d_out"].cuda())
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got[0], ref[2][0]) and torch.equal(got[4], ref[2][1]["dw"])


@pytest.mark.parametrize("rows, cols, outs", [(3, 200, 72), (1500, 264, 136), (900, 64, 1024)])
def test_captured_replays_follow_the_inputs(rows, cols, outs):
    """The route of a few rows, of wide ones, and of a weight that fills shared memory; other work runs between the replays."""
    cases = [_inputs(rows, cols, outs, seed=s) for s in (1, 2)]
    ref = [_run(c, "int8") for c in cases]
    leaves = [cases[0][n].cuda().requires_grad_(True) for n in ("x", "nw", "nb", "w")]
    d = cases[0]["d_out"].cuda()

    def step():
        out = tk.turbo_norm_linear(*leaves, checkpoint="int8")
        return (out.detach(), *torch.autograd.grad(out, leaves, d))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for k in (0, 1, 0):
        with torch.no_grad():
            for v, n in zip(leaves, ("x", "nw", "nb", "w")):
                v.copy_(cases[k][n].cuda())
            d.copy_(cases[k]["d_out"].cuda())
        graph.replay()
        other = _run(cases[1 - k], "int8")
        torch.cuda.synchronize()
        for have, (out, g) in ((got, ref[k]), ((other[0], *(other[1][n] for n in ("dx", "dnw", "dnb", "dw"))), ref[1 - k])):
            assert torch.equal(have[0], out)
            assert all(torch.equal(a, g[n]) for a, n in zip(have[1:], ("dx", "dnw", "dnb", "dw")))


@pytest.mark.parametrize("checkpoint", [None, "int8"])
def test_traced_route_matches_eager(checkpoint):
    i = _inputs(60, 96, 64)
    leaves = [i[n].cuda().requires_grad_(True) for n in ("x", "nw", "nb", "w")]
    f = lambda *a: tk.turbo_norm_linear(*a, checkpoint=checkpoint)  # noqa: E731
    out, g = _run(i, checkpoint)
    oc = torch.compile(f, fullgraph=True, backend="aot_eager")(*leaves)
    gc = torch.autograd.grad(oc, leaves, i["d_out"].cuda())
    assert torch.equal(out, oc) and all(torch.equal(g[n], b) for n, b in zip(("dx", "dnw", "dnb", "dw"), gc))
    torch.library.opcheck(torch.ops.tpf_b200.norm_linear_fwd, (leaves[0], leaves[1], None, leaves[3], 1e-5, checkpoint == "int8"),
                          test_utils=("test_schema", "test_autograd_registration", "test_faketensor"))


def test_a_transition_of_the_operators():
    """Norm -> stacked gate and value projections -> gated product -> norm, as a transition uses them, one 8-bit copy of each
    input: gradients near those with whole inputs."""
    g = torch.Generator().manual_seed(5)
    x0 = torch.randn(2, 40, 40, 64, generator=g).bfloat16().cuda()
    nw, nb = torch.ones(64, device="cuda"), torch.zeros(64, device="cuda")
    w = (torch.randn(512, 64, generator=g) / 17).bfloat16().cuda()

    def run(keep):
        x, wl = x0.clone().requires_grad_(True), w.clone().requires_grad_(True)
        a, b = tk.turbo_norm_linear(x, nw, nb, wl, checkpoint=keep).chunk(2, -1)
        h = torch.nn.functional.silu(a) * b
        y = tk.turbo_layer_norm(h, checkpoint=keep)
        return (y.detach(), *torch.autograd.grad((y.float() ** 3).mean() * 1000, (x, wl)))

    whole, kept = run(None), run("int8")
    assert torch.equal(whole[0], kept[0])     # the forward does not depend on what is kept
    for a, b in zip(whole[1:], kept[1:]):
        # kept values are off by a / 254 of their group at most, about 1 % of a typical value
        assert (a.float() - b.float()).norm() / a.float().norm() < 0.03


def test_refusals_leave_no_launch():
    before = C.load().tpf_launch_count()
    x = torch.zeros(4, 128, device="cuda", dtype=torch.bfloat16)
    w = torch.zeros(64, 128, device="cuda", dtype=torch.bfloat16)
    for bad in ((x.float(), None, None, w), (x[:, :100], None, None, w[:, :100]), (x, None, None, w[:60]), (x, None, None, w.cpu()),
                (x, w[0, :64], None, w), (x, None, None, w.double())):
        with pytest.raises(ValueError, match="turbo_norm_linear unsupported"):
            tk.turbo_norm_linear(*bad)
    with pytest.raises(ValueError, match=r"\[checkpoint\]"):
        tk.turbo_norm_linear(x, None, None, w, checkpoint="e4m3")
    assert C.load().tpf_launch_count() == before

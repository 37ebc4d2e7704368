"""turbo_window_attention on a B200 against the 64-bit oracle (bounds derived in oracle/sequence_oracle.py)."""
import math

import pytest
import torch

import openfold3_triangle_kernel_b200 as tk
from openfold3_triangle_kernel_b200 import _cabi as C
from oracle import sequence_oracle as so

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA device")]

BF, FP16 = torch.bfloat16, torch.float16


def _rn(*s, seed=0, dtype=BF):
    return torch.randn(*s, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)).to(dtype)


def _inputs(B, N, M, H, HK, D, dtype=BF, seed=0):
    return _rn(B, N, H, D, seed=seed, dtype=dtype), _rn(B, M, HK, D, seed=seed + 1, dtype=dtype), _rn(B, M, HK, D, seed=seed + 2, dtype=dtype)


def _check(q, k, v, window, sinks=0, offset=0, lengths=None, scale=None, train=True):
    B, N, H, D = q.shape
    kw = dict(window=window, sinks=sinks, scale=scale)
    dev = lambda t: None if t is None else torch.tensor(t, dtype=torch.int32, device="cuda")  # noqa: E731
    kw["query_offset"] = dev(offset) if isinstance(offset, list) else offset
    kw["key_lengths"] = dev(lengths)
    offsets = offset if isinstance(offset, list) else [offset] * B
    leaves = [t.detach().requires_grad_(train) for t in (q, k, v)]
    out, lse = tk.turbo_window_attention(*leaves, return_lse=True, **kw)
    assert out.dtype == q.dtype and out.shape == q.shape and out.is_contiguous()
    assert lse.dtype == torch.float32 and lse.shape == (B, H, N)
    d = _rn(*q.shape, seed=77, dtype=q.dtype)
    if lengths is not None:
        d[torch.arange(N, device="cuda")[None] >= torch.tensor(lengths, device="cuda")[:, None]] = 0
    ref = so.window_attention(q, k, v, window, sinks, offsets, lengths, scale, d if train else None)
    so.check(out, ref["out"], ref["out_off"], "out")
    empty = ref["lse"] == -math.inf
    assert torch.equal(lse == -math.inf, empty)
    assert (out.transpose(1, 2)[empty] == 0).all()
    so.check(lse[~empty], ref["lse"][~empty], ref["lse_off"][~empty], "lse")
    if train:
        grads = torch.autograd.grad(out, leaves, d)
        for n, g in zip(("dq", "dk", "dv"), grads):
            so.check(g, ref[n], ref[n + "_off"], n)
        assert (grads[0].transpose(1, 2)[empty] == 0).all()
    with torch.no_grad():
        assert torch.equal(tk.turbo_window_attention(*leaves, **kw), out)
    assert C.device_status() == 0
    return out


WINDOWS = [((None, 0), 0), ((0, 0), 0), ((5, 0), 2), ((63, 0), 0), ((64, 0), 1), ((100, 0), 4), ((16, 16), 0), ((0, 7), 3), ((70, 30), 64),
           ((None, None), 0), ((None, 5), 0), ((9, None), 5), ((200, 0), 17), ((130, 130), 33)]


# one sequence, and enough of them for the kernel of many queries
@pytest.mark.parametrize("window, sinks", WINDOWS)
@pytest.mark.parametrize("n", [1, 63, 64, 65, 130, 300])
@pytest.mark.parametrize("B, H", [(1, 2), (40, 6)])
def test_windows(window, sinks, n, B, H):
    _check(*_inputs(B, n, n, H, H // 2, 64, seed=n), window, sinks)


@pytest.mark.parametrize("D", [8, 16, 24, 32, 40, 64, 72, 80, 96, 104, 120, 128])
@pytest.mark.parametrize("dtype", [BF, FP16])
@pytest.mark.parametrize("B, n", [(2, 20), (2, 200), (40, 200)])
def test_head_sizes(D, dtype, B, n):
    _check(*_inputs(B, n, n, 4, 2, D, dtype, seed=D), (50, 0), 3)


@pytest.mark.parametrize("H, HK", [(1, 1), (3, 1), (4, 4), (8, 2), (16, 1), (24, 3), (40, 2)])
@pytest.mark.parametrize("B, n", [(2, 5), (2, 129), (40, 129)])
def test_shared_key_heads(H, HK, B, n):
    _check(*_inputs(B, n, n, H, HK, 32, seed=H), (40, 10), 2)


@pytest.mark.parametrize("n", [1, 2, 5, 17])
@pytest.mark.parametrize("M", [1, 15, 16, 17, 200, 1000, 5000])
def test_new_tokens_over_a_cache(n, M):
    """The last n tokens of sequences of different lengths."""
    lengths = [max(1, M - 3 * b) for b in range(3)]
    _check(*_inputs(3, n, M, 8, 2, 128, seed=M), (300, 0), 4, [x - n for x in lengths], lengths, train=False)


@pytest.mark.parametrize("B, H, HK, M", [(1, 8, 1, 20000), (2, 4, 4, 9000), (40, 16, 4, 700)])
def test_one_token(B, H, HK, M):
    lengths = [M - 7 * b for b in range(B)]
    for window in ((None, 0), (1023, 0)):
        _check(*_inputs(B, 1, M, H, HK, 64, seed=M), window, 4, [x - 1 for x in lengths], lengths, train=False)


@pytest.mark.parametrize("times, n", [(1, 3), (1, 100), (10, 100)])
def test_rows_that_see_nothing(times, n):
    """Empty sequences, queries before the first key and behind the window."""
    q, k, v = _inputs(5 * times, n, 150, 4, 2, 64)
    _check(q, k, v, (10, 0), 0, [0, -n, 400, -5, 149] * times, [0, 150, 150, 150, 150] * times)
    _check(q, k, v, (10, 0), 2, [0, -n, 400, -5, 149] * times, [0, 150, 150, 150, 1] * times)
    _check(q, k, v, (0, 3), 64, [-200, 2 ** 29, -2 ** 29, 60, 70] * times, [150, 150, 150, 64, 65] * times)


@pytest.mark.parametrize("times, n", [(1, 70), (1, 257), (8, 257)])
@pytest.mark.parametrize("window, sinks", [((30, 0), 1), ((64, 64), 0), ((None, 0), 0), ((128, 128), 20)])
def test_padded_batches(times, n, window, sinks):
    _check(*_inputs(4 * times, n, n, 4, 2, 64, seed=n), window, sinks, 0, [n, n - 1, 64, 1] * times)


@pytest.mark.parametrize("times, n", [(1, 1), (1, 90), (10, 90)])
@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_what_lies_behind_the_last_key_does_not_count(times, n, value):
    q, k, v = _inputs(3 * times, n, 200, 4, 2, 64)
    lengths = [200, 131, 7] * times
    for b, x in enumerate(lengths):
        k[b, x:] = value
        v[b, x:] = value
    _check(q, k, v, (60, 0), 3, [x - n for x in lengths], lengths)
    _check(q, k, v, (None, None), 0, 0, lengths)


@pytest.mark.parametrize("B, n", [(1, 4), (1, 200), (20, 200)])
def test_large_logits(B, n):
    """Maxima that rise from tile to tile, and a scale that makes them far apart."""
    q, k, v = _inputs(B, n, n, 2, 2, 64)
    k = (k.float() * torch.linspace(0.1, 8, n, device="cuda")[None, :, None, None]).to(BF)
    _check(q, k, v, (None, None), 0, scale=0.25)
    _check(q, (k.float() * 0).to(BF), v, (50, 50), 2)
    with torch.no_grad():
        big = tk.turbo_window_attention(q * 30, k * 30, v, window=(None, 0))
    assert torch.isfinite(big).all()


@pytest.mark.parametrize("n", [1, 33, 200, 500])
def test_strides(n):
    """Slices of a stacked projection, head-major tensors, expanded batches, odd pitches and starts."""
    s = _rn(2, n, 8 + 2 + 2, 64, seed=n)
    q, k, v = s[:, :, :8], s[:, :, 8:10], s[:, :, 10:]
    plain = _check(q.contiguous(), k.contiguous(), v.contiguous(), (40, 3), 2)
    assert torch.equal(_check(q, k, v, (40, 3), 2), plain)
    major = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)]
    assert torch.equal(_check(*major, (40, 3), 2), plain)
    odd = torch.zeros(2, n, 12 * 64 + 3, device="cuda", dtype=BF)
    odd[..., 1:-2] = s.flatten(-2)
    o = odd[..., 1:-2].unflatten(-1, (12, 64))
    assert torch.equal(_check(o[:, :, :8], o[:, :, 8:10], o[:, :, 10:], (40, 3), 2), plain)
    one = k[:1].expand(2, n, 2, 64)
    _check(q, one, one, (40, 3), 2)


def test_more_and_fewer_leading_dimensions():
    q, k, v = _inputs(6, 70, 70, 4, 2, 32)
    flat = tk.turbo_window_attention(q, k, v, window=(20, 0), key_lengths=torch.arange(65, 71, device="cuda"))
    deep = tk.turbo_window_attention(*(t.unflatten(0, (2, 3)) for t in (q, k, v)), window=(20, 0),
                                     key_lengths=torch.arange(65, 71, device="cuda").view(2, 3))
    assert torch.equal(deep.flatten(0, 1), flat)
    alone = tk.turbo_window_attention(q[1], k[1], v[1], window=(20, 0), key_lengths=torch.tensor(66, device="cuda"))
    assert torch.equal(alone, flat[1])


def test_nothing():
    for B, N, M in ((0, 5, 5), (2, 0, 5), (2, 5, 0), (2, 100, 0)):
        leaves = [t.requires_grad_(True) for t in _inputs(B, N, M, 4, 2, 64)]
        out = tk.turbo_window_attention(*leaves, window=(3, 0))
        assert out.shape == (B, N, 4, 64) and (out == 0).all()
        out.float().sum().backward()
        assert all((t.grad == 0).all() and t.grad.shape == t.shape for t in leaves)


@pytest.mark.parametrize("n, window, sinks", [(3000, (200, 0), 4), (2500, (100, 100), 64), (2000, (None, 0), 0), (1500, (700, 20), 9)])
def test_longer_sequences(n, window, sinks):
    _check(*_inputs(1, n, n, 4, 1, 128, seed=n), window, sinks)
    _check(*_inputs(2, n, n, 2, 2, 64, FP16, seed=n), window, sinks, [0, 40], [n, n - 77])


def test_equal_sequences_get_equal_bits():
    """64 equal planes, forward and backward: a race would show in some of them."""
    q, k, v = (t.expand(64, *t.shape[1:]).contiguous().requires_grad_(True) for t in _inputs(1, 700, 700, 4, 1, 128))
    d = _rn(1, 700, 4, 128, seed=9).expand(64, 700, 4, 128).contiguous()
    for _ in range(3):
        out = tk.turbo_window_attention(q, k, v, window=(150, 20), sinks=4)
        for t in (out, *torch.autograd.grad(out, [q, k, v], d)):
            assert (t == t[:1]).all()


def test_a_cache_beyond_2_31_elements():
    """Offsets of 64 bits: the last sequences of a cache of 2^31 + 2^29 elements."""
    B, M, HK, D = 40, 65536, 8, 128
    k = torch.zeros(B, M, HK, D, device="cuda", dtype=BF)
    v = torch.zeros(B, M, HK, D, device="cuda", dtype=BF)
    k[-1], v[-1] = _rn(M, HK, D, seed=1), _rn(M, HK, D, seed=2)
    for n in (1, 160):
        q = _rn(B, n, 16, D, seed=3)
        out = tk.turbo_window_attention(q, k, v, window=(500, 0), sinks=4, query_offset=M - n)
        ref = so.window_attention(q[-1:], k[-1:], v[-1:], (500, 0), 4, [M - n])
        so.check(out[-1:], ref["out"], ref["out_off"], "out")


def test_differences():
    """Directional differences of the computed function.  out is rounded to fp16 (2^-11) and the steps are 2^-4: with 64 x 2 x 64 outputs
    of size 1/2, the sum's rounding is below 2^-11 * sqrt(8192) = 0.045, over two steps of 2^-4 0.36; curvature adds 2^-8 of the third
    derivative, of the size of the slope's own terms."""
    q, k, v = (t.requires_grad_(True) for t in _inputs(1, 64, 64, 2, 1, 64, FP16))
    d = _rn(1, 64, 2, 64, seed=5, dtype=FP16)
    f = lambda: (tk.turbo_window_attention(q, k, v, window=(20, 5), sinks=2).double() * d.double()).sum()  # noqa: E731
    grads = torch.autograd.grad(f(), [q, k, v])
    for leaf, g in zip((q, k, v), grads):
        step = (_rn(*leaf.shape, seed=6, dtype=torch.float32) > 0).to(FP16) * 2 - 1
        keep = leaf.detach().clone()
        with torch.no_grad():
            leaf.copy_(keep + step * 2.0 ** -4)
            up, hi = f(), leaf.detach().clone()
            leaf.copy_(keep - step * 2.0 ** -4)
            down, lo = f(), leaf.detach().clone()
            leaf.copy_(keep)
        slope = (g.double() * (hi.double() - lo.double())).sum()
        assert abs((up - down) - slope) <= 0.1 + 0.05 * (g.double() * (hi.double() - lo.double())).norm() * 8


def test_captured_replays():
    q, k, v = (t.requires_grad_(True) for t in _inputs(2, 150, 150, 4, 2, 64))
    lengths = torch.tensor([150, 100], dtype=torch.int32, device="cuda")
    d = _rn(2, 150, 4, 64, seed=8)

    def step():
        out = tk.turbo_window_attention(q, k, v, window=(30, 0), sinks=3, key_lengths=lengths)
        return [out.detach(), *torch.autograd.grad(out, [q, k, v], d)]

    def token():
        with torch.no_grad():
            return tk.turbo_window_attention(q[:, :1], k, v, window=(30, 0), sinks=3, key_lengths=lengths, query_offset=lengths - 1)

    step(), token()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res, one = step(), token()
    for n in (150, 70, 3):
        lengths.copy_(torch.tensor([n, n // 2 + 1]))
        with torch.no_grad():
            k.mul_(1.25)
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(res, step())) and torch.equal(one, token())


def test_two_streams_at_once():
    ins = [_inputs(1, 600, 600, 4, 2, 128, seed=s) for s in (0, 10)]
    f = lambda t: tk.turbo_window_attention(*t, window=(100, 0), sinks=4)  # noqa: E731
    expected = [f(t) for t in ins]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in ins]
    outs = []
    for _ in range(10):
        for s, t in zip(streams, ins):
            with torch.cuda.stream(s):
                outs.append(f(t))
    torch.cuda.synchronize()
    assert all(torch.equal(o, expected[i % 2]) for i, o in enumerate(outs))


def test_traced_calls():
    torch.compiler.reset()
    f = lambda q, k, v, n: tk.turbo_window_attention(q, k, v, window=(30, 2), sinks=2, key_lengths=n)  # noqa: E731
    g = torch.compile(f, fullgraph=True, dynamic=True, backend="aot_eager")
    for n in (40, 100):
        q, k, v = (t.requires_grad_(True) for t in _inputs(2, n, n, 4, 2, 64))
        lengths = torch.tensor([n, n - 9], device="cuda")
        d = _rn(2, n, 4, 64, seed=3)
        a, b = f(q, k, v, lengths), g(q, k, v, lengths)
        assert torch.equal(a, b)
        assert all(torch.equal(x, y) for x, y in zip(torch.autograd.grad(a, [q, k, v], d), torch.autograd.grad(b, [q, k, v], d)))
    q, k, v = (t.requires_grad_(True) for t in _inputs(1, 20, 20, 2, 1, 64))
    torch.library.opcheck(torch.ops.tpf_b200.window_attn_fwd, (q, k, v, None, None, 0, 5, 0, 1, 0.125))


def test_some_gradients_only_and_no_second_ones():
    q, k, v = _inputs(1, 90, 90, 4, 2, 64)
    d = _rn(1, 90, 4, 64, seed=3)
    full = [t.clone().requires_grad_(True) for t in (q, k, v)]
    ref = torch.autograd.grad(tk.turbo_window_attention(*full, window=(20, 0)), full, d)
    for i in range(3):
        leaves = [t.clone().requires_grad_(i == j) for j, t in enumerate((q, k, v))]
        g, = torch.autograd.grad(tk.turbo_window_attention(*leaves, window=(20, 0)), leaves[i], d)
        assert torch.equal(g, ref[i])
    g, = torch.autograd.grad(tk.turbo_window_attention(*full, window=(20, 0)).float().sum(), full[0], create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        g.float().sum().backward()


@pytest.mark.parametrize("B, n, D, window, sinks", [(200, 4, 80, (800, 0), 0), (8, 300, 128, (1, 0), 0), (8, 300, 64, (3, 3), 1), (8, 300, 64, (8, 0), 0),
                                                    (4, 400, 128, (None, 0), 0), (300, 2, 32, (5, 0), 0), (3, 700, 96, (0, 40), 7)])
@pytest.mark.parametrize("dtype", [BF, FP16])
def test_few_keys_cost_no_precision(B, n, D, window, sinks, dtype):
    """dS and the result are rounded once each: in the norm 2 / sqrt(3) half steps at the most where the two never cancel, 1.5 with the
    spread of some hundred numbers.  Roundings of the output in delta would be beside a dS that is small where a query sees few keys."""
    q, k, v = (t.requires_grad_(True) for t in _inputs(B, n, n, 4, 2, D, dtype))
    d = _rn(B, n, 4, D, seed=8, dtype=dtype)
    ref = so.window_attention(q.detach(), k.detach(), v.detach(), window, sinks, d_out=d)
    grads = torch.autograd.grad(tk.turbo_window_attention(q, k, v, window=window, sinks=sinks), [q, k, v], d)
    for name, g in zip(("dq", "dk", "dv"), grads):
        assert (g.double() - ref[name]).norm() <= 1.5 * so.half_step(dtype) * ref[name].norm(), name


def test_gradients_from_packed_activations():
    """Inside `int8_activations` the backward pass runs on what the format holds of q, k, v and the output."""
    leaves = [t.requires_grad_(True) for t in _inputs(2, 300, 300, 8, 2, 64)]
    q, k, v = (t * 1 for t in leaves)
    d = _rn(2, 300, 8, 64, seed=3)
    with tk.int8_activations(min_elements=1):
        out, lse = tk.turbo_window_attention(q, k, v, window=(50, 0), sinks=2, return_lse=True)
    back = [tk.unpack_activation(*tk.pack_activation(t.detach().view(-1, 128)), t.dtype).view(t.shape) for t in (q, k, v, out)]
    got = torch.autograd.grad(out, leaves, d)
    want = torch.ops.tpf_b200.window_attn_bwd(d, *back, lse, None, None, 0, 50, 0, 2, 64 ** -0.5)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_saved_tensors_of_other_layouts():
    """A hook of the caller's may hand back any strides."""
    q, k, v = (t.requires_grad_(True) for t in _inputs(2, 100, 100, 4, 2, 64))
    d = _rn(2, 100, 4, 64, seed=3)
    ref = torch.autograd.grad(tk.turbo_window_attention(q, k, v, window=(50, 0)), [q, k, v], d)
    turned = lambda t: t.transpose(0, 1).contiguous().transpose(0, 1) if t.ndim > 1 else t  # noqa: E731
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach(), turned):
        out = tk.turbo_window_attention(q, k, v, window=(50, 0))
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(out, [q, k, v], d), ref))


def test_threads_at_once():
    import threading
    ins = [_inputs(2, 500, 500, 4, 2, 64, seed=s) for s in (0, 10)]
    d = _rn(2, 500, 4, 64, seed=3)

    def step(t):
        leaves = [x.detach().requires_grad_(True) for x in t]
        out = tk.turbo_window_attention(*leaves, window=(100, 0), sinks=4)
        return [out.detach(), *torch.autograd.grad(out, leaves, d)]

    expected = [step(t) for t in ins]
    torch.cuda.synchronize()
    results = [None, None]

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            results[i] = [step(ins[i]) for _ in range(20)]
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert all(torch.equal(a, b) for i in range(2) for r in results[i] for a, b in zip(r, expected[i]))


def test_a_layer_of_them():
    """What a sequence layer does: stacked projection, norm and rotation, attention, projection, dropout with the residual."""
    g = torch.Generator(device="cuda").manual_seed(0)
    C_, H, HK, D, N = 128, 8, 2, 32, 333
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    nw, nb = (1 + 0.1 * r(C_)).bfloat16().requires_grad_(True), (0.1 * r(C_)).bfloat16().requires_grad_(True)
    w = (r((H + 2 * HK) * D, C_) / math.sqrt(C_)).bfloat16().requires_grad_(True)
    wo = (r(C_, H * D) / math.sqrt(H * D)).bfloat16().requires_grad_(True)
    qw, kw = (1 + 0.1 * r(D)).requires_grad_(True), (1 + 0.1 * r(D)).requires_grad_(True)
    x = r(2, N, C_).bfloat16().requires_grad_(True)
    fr = tk.rotary_frequencies(D, device="cuda")
    lengths = [N, N - 50]
    d = r(2, N, C_).bfloat16()

    def layer():
        s = tk.turbo_norm_linear(x, nw, nb, w).unflatten(-1, (H + 2 * HK, D))
        q, k = tk.turbo_qk_norm_rotary(s[:, :, :H], s[:, :, H:H + HK], qw, kw, fr)
        o = tk.turbo_window_attention(q, k, s[:, :, H + HK:], window=(64, 64), sinks=1,
                                      key_lengths=torch.tensor(lengths, dtype=torch.int32, device="cuda"))
        return tk.turbo_dropout(o.flatten(-2) @ wo.t(), 0.25, 3, residual=x)

    def exact(x, nw, nb, w, wo, qw, kw):
        mu = x.mean(-1, keepdim=True)
        xn = (x - mu) / torch.sqrt(((x - mu) ** 2).mean(-1, keepdim=True) + 1e-5) * nw + nb
        s = (xn @ w.t()).unflatten(-1, (H + 2 * HK, D))
        f, pos = so.radians(D), torch.arange(N, device="cuda").expand(2, N)

        def turn(t, wt):
            t = t * torch.rsqrt((t ** 2).mean(-1, keepdim=True) + 1e-6) * wt
            a, b = t[..., :D // 2], t[..., D // 2:]
            ang = pos.double()[..., None, None] * f.cuda()
            return torch.cat([a * ang.cos() - b * ang.sin(), a * ang.sin() + b * ang.cos()], -1)

        q, k, v = turn(s[:, :, :H], qw), turn(s[:, :, H:H + HK], kw), s[:, :, H + HK:]
        k, v = (t.repeat_interleave(H // HK, 2) for t in (k, v))
        ok = torch.stack([so.seen(N, N, (64, 64), 1, 0, n, "cuda") for n in lengths])[:, None]
        a = torch.einsum("bihd,bjhd->bhij", q, k) * D ** -0.5
        p = torch.where(ok, torch.softmax(a.masked_fill(~ok, -1e300), -1), 0.0)
        o = torch.einsum("bhij,bjhd->bihd", p, v).flatten(-2) @ wo.t()
        return x + torch.where(so.dropout_mask((2, N, C_), 0.25, 3).cuda(), o / 0.75, 0.0)

    leaves = [x, nw, nb, w, wo, qw, kw]
    out = layer()
    grads = torch.autograd.grad(out, leaves, d)
    doubles = [t.detach().double().requires_grad_(True) for t in leaves]
    ref = exact(*doubles)
    want = torch.autograd.grad(ref, doubles, d.double())
    # six results in bf16 stand one behind the other, forward, and as many backward: half a step (2^-8) each, which add up as
    # independent errors do (sqrt(12)), with a factor of 2
    room = 2 * math.sqrt(12) * 2.0 ** -8
    assert (out.double() - ref).norm() <= room * ref.norm()
    for a, b in zip(grads, want):
        assert (a.double() - b).norm() <= room * b.norm()


def test_saved_offsets_and_lengths_of_other_layouts():
    """A hook of the caller's may hand back any strides of these, too: transposed, spread out, expanded."""
    q, k, v = (t.unflatten(0, (2, 3)).contiguous().requires_grad_(True) for t in _inputs(6, 40, 100, 4, 2, 64))
    d = _rn(2, 3, 40, 4, 64, seed=3)
    some = torch.tensor([[60, 10, 33]], dtype=torch.int32, device="cuda")
    offsets, lengths = torch.cat([some, some]), torch.cat([some + 40, some + 40])

    def call():
        return tk.turbo_window_attention(q, k, v, window=(20, 0), sinks=2, query_offset=offsets, key_lengths=lengths)

    want = torch.autograd.grad(call(), [q, k, v], d)
    turned = lambda t: t.transpose(0, 1).contiguous().transpose(0, 1)  # noqa: E731
    spread = lambda t: torch.stack([t, t + 1], -1)[..., 0]  # noqa: E731
    once = lambda t: t[:1].clone().expand(t.shape) if t.ndim == 2 else t  # noqa: E731
    for hook in (turned, spread, once):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach(), hook):
            out = call()
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(out, [q, k, v], d), want))


# Rounding to the nearest is off by up to half a step of a number's power of two, 1 / sqrt(3) of that in the mean square; over numbers of a
# normal distribution, whose mean square is 1.9 times that of their powers of two, 0.42 half steps of their norm.  Two such roundings,
# independent of one another, 0.42 sqrt(2).  A tenth on top for the spread (of some 70000 numbers: below a hundredth) and for what is in fp32.
ONE_ROUNDING = 1.1 * 0.42
TWO_ROUNDINGS = 1.1 * 0.42 * math.sqrt(2)


@pytest.mark.parametrize("B, n, D, window, sinks, bound", [
    (8, 300, 128, (1, 0), 0, TWO_ROUNDINGS), (8, 300, 64, (3, 3), 1, TWO_ROUNDINGS), (8, 300, 64, (8, 0), 0, TWO_ROUNDINGS),
    (16, 129, 64, (1, 0), 0, TWO_ROUNDINGS), (16, 128, 64, (1, 0), 0, ONE_ROUNDING), (200, 4, 80, (800, 0), 0, ONE_ROUNDING),
    (300, 2, 32, (5, 0), 0, ONE_ROUNDING)])
@pytest.mark.parametrize("dtype", [BF, FP16])
def test_roundings_of_gradients(B, n, D, window, sinks, bound, dtype):
    """dS and P are rounded once as operands (up to 128 tokens and keys in two parts: not at all, at this scale), and the results once.
    The roundings of the stored output in delta would make 0.72 to 1.15 half steps of these."""
    q, k, v = (t.requires_grad_(True) for t in _inputs(B, n, n, 4, 2, D, dtype))
    d = _rn(B, n, 4, D, seed=8, dtype=dtype)
    ref = so.window_attention(q.detach(), k.detach(), v.detach(), window, sinks, d_out=d)
    grads = torch.autograd.grad(tk.turbo_window_attention(q, k, v, window=window, sinks=sinks), [q, k, v], d)
    for name, g in zip(("dq", "dk", "dv"), grads):
        assert (g.double() - ref[name]).norm() <= bound * so.half_step(dtype) * ref[name].norm(), name


@pytest.mark.parametrize("B, n, M, bound", [(200, 1, 9, ONE_ROUNDING), (200, 1, 200, ONE_ROUNDING), (60, 3, 400, ONE_ROUNDING),
                                            (8, 300, 300, TWO_ROUNDINGS)])
@pytest.mark.parametrize("dtype", [BF, FP16])
def test_roundings_of_the_output(B, n, M, bound, dtype):
    """Few queries take P in two parts, many in one."""
    q, k, v = _inputs(B, n, M, 4, 2, 64, dtype)
    ref = so.window_attention(q, k, v, (None, 0), 0, [M - n] * B)
    out = tk.turbo_window_attention(q, k, v, window=(None, 0), query_offset=M - n)
    assert (out.double() - ref["out"]).norm() <= bound * so.half_step(dtype) * ref["out"].norm()

"""The triangle operators refuse wrong operands in a traced call too: in the fake kernels, in the operators that a graph
calls, and while a call is traced.  None of it needs a GPU."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import openfold3_triangle_kernel_b200 as tk

BF, F32 = torch.bfloat16, torch.float32
OPS = torch.ops.tpf_b200


def _attention(**kw):
    s = dict(q=(2, 5, 4, 40, 32), k=(2, 5, 4, 40, 32), v=(2, 5, 4, 40, 32), mask=(2, 5, 40), bias=(1, 4, 40, 40),
             d_out=(2, 5, 40, 4, 32), out=(2, 5, 40, 4, 32), lse=(2, 5, 4, 40))
    dt = dict(q=BF, k=BF, v=BF, mask=F32, bias=BF, d_out=BF, out=BF, lse=F32)
    for name, x in kw.items():
        (s if isinstance(x, tuple) else dt)[name] = x
    return {n: torch.empty(s[n], dtype=dt[n]) for n in s}


ATTENTION = [dict(q=(2, 5, 4, 40)), dict(k=(2, 5, 4, 24, 32)), dict(v=F32), dict(mask=(2, 5, 8)), dict(mask=torch.bool),
             dict(bias=(1, 4, 40, 16)), dict(bias=(3, 4, 40, 40)), dict(bias=torch.float16),
             dict(q=(2, 5, 4, 40, 24), k=(2, 5, 4, 40, 24), v=(2, 5, 4, 40, 24)),
             dict(q=(2, 0, 4, 40, 32), k=(2, 0, 4, 40, 32), v=(2, 0, 4, 40, 32), mask=(2, 0, 40))]


@pytest.mark.parametrize("wrong", ATTENTION + [dict(d_out=(2, 5, 40, 4, 16)), dict(d_out=F32), dict(out=(2, 5, 4, 40, 32)),
                                               dict(lse=(2, 5, 4, 8)), dict(lse=BF)])
@pytest.mark.parametrize("fake", [True, False])
def test_attention_operators_refuse(wrong, fake):
    import contextlib
    with FakeTensorMode() if fake else contextlib.nullcontext():
        a = _attention(**wrong)
        if not wrong.keys() & {"d_out", "out", "lse"}:
            with pytest.raises(ValueError, match="unsupported TurboPairFormer case"):
                OPS.attn_fwd(a["q"], a["k"], a["v"], a["mask"], a["bias"], 0.2)
        with pytest.raises(ValueError, match="unsupported TurboPairFormer case"):
            OPS.attn_bwd(a["q"], a["k"], a["v"], a["d_out"], a["out"], a["lse"], a["mask"], a["bias"], 0.2)


def _trimul(**kw):
    c, n = 64, 16
    s = dict(z=(2, n, n, c), mask=(2, n, n), p_in=(2 * c, c), g_in=(2 * c, c), p_out=(c, c), g_out=(c, c), nin_w=(c,),
             nin_b=(c,), nout_w=(c,), nout_b=(c,))
    s.update({k: x for k, x in kw.items() if isinstance(x, tuple)})
    return {k: torch.empty(x, dtype=kw[k] if isinstance(kw.get(k), torch.dtype) else BF if k == "z" else F32)
            for k, x in s.items()}


TRIMUL = [(dict(z=(2, 16, 16)), "z_shape"), (dict(z=(2, 16, 8, 64)), "z_shape"), (dict(z=(2, 12, 12, 64)), "z_shape"),
          (dict(z=F32), "z_dtype"), (dict(z=(2, 16, 16, 48)), "channels"), (dict(mask=(2, 16, 8)), "mask_shape"),
          (dict(mask=(1, 16, 16)), "mask_shape"), (dict(p_in=(64, 64)), "weight_shape"), (dict(g_out=(64, 8)), "weight_shape"),
          (dict(nin_w=(8,)), "weight_shape"), (dict(nout_w=torch.int64), "weight_dtype")]


@pytest.mark.parametrize("wrong, code", TRIMUL)
@pytest.mark.parametrize("fake", [True, False])
def test_trimul_operators_refuse(wrong, code, fake):
    import contextlib
    with FakeTensorMode() if fake else contextlib.nullcontext():
        t = _trimul(**wrong)
        with pytest.raises(ValueError, match=rf"unsupported \[{code}\]"):
            OPS.trimul_fwd(*t.values(), True)
        saved = [torch.empty(4)] * 11
        w = [t[n] for n in ("p_in", "g_in", "p_out", "g_out", "nin_w", "nout_w")]
        with pytest.raises(ValueError, match=rf"unsupported \[{code}\]"):
            OPS.trimul_bwd(t["z"], t["z"], t["mask"], *w, True, *saved)


def test_trimul_backward_operator_refuses_what_was_not_kept_for_it():
    with FakeTensorMode():
        t = _trimul()
        saved = OPS.trimul_fwd(*t.values(), False)
        w = [t[n] for n in ("p_in", "g_in", "p_out", "g_out", "nin_w", "nout_w")]
        assert len(OPS.trimul_bwd(t["z"], t["z"], t["mask"], *w, False, *saved)) == 9
        with pytest.raises(ValueError, match=r"unsupported \[d_out_shape\]"):
            OPS.trimul_bwd(t["z"][:1], t["z"], t["mask"], *w, False, *saved)
        for i in range(11):
            for bad in (saved[i][:1], saved[i].double()):
                with pytest.raises(ValueError, match=r"unsupported \[saved\]"):
                    OPS.trimul_bwd(t["z"], t["z"], t["mask"], *w, False, *saved[:i], bad, *saved[i + 1:])


def test_operands_of_two_devices_are_refused():
    with FakeTensorMode():
        a, t = _attention(), _trimul()
        a["q"] = a["q"].cuda()
        with pytest.raises(ValueError, match="one device"):
            OPS.attn_fwd(a["q"], a["k"], a["v"], a["mask"], a["bias"], 0.2)
        t["z"] = t["z"].cuda()
        with pytest.raises(ValueError, match="one device"):
            OPS.trimul_fwd(*t.values(), True)


def test_cpu_operands_are_refused_by_the_operators():
    a, t = _attention(), _trimul()
    with pytest.raises(ValueError, match="CUDA tensors"):
        OPS.attn_fwd(a["q"], a["k"], a["v"], a["mask"], a["bias"], 0.2)
    with pytest.raises(ValueError, match=r"\[device\]"):
        OPS.trimul_fwd(*t.values(), True)


def _att_call(**kw):
    a = _attention(**kw)
    return a["q"], a["bias"].unsqueeze(1), a["mask"][:, :, None, None]


def _tri_call(direction="outgoing", **kw):
    t = _trimul(**kw)
    names = ("p_in_weight", "g_in_weight", "p_out_weight", "g_out_weight", "norm_in_weight", "norm_in_bias",
             "norm_out_weight", "norm_out_bias")
    return t["z"], direction, t["mask"], dict(zip(names, list(t.values())[2:]))


CALLS = [(lambda q, b, m: tk.turbo_attention(q, q, q, pair_bias=b, res_mask=m), _att_call(bias=(1, 4, 40, 16)), "pair_bias tail"),
         (lambda q, b, m: tk.turbo_attention(q, q, q, pair_bias=b, res_mask=m), _att_call(mask=torch.bool), "additive mask"),
         (lambda q, b, m: tk.turbo_attention(q, q, q, pair_bias=b, res_mask=m.clone().requires_grad_(True)), _att_call(),
          "must not require gradients"),
         (lambda z, d, m, w: tk.turbo_trimul(z, d, m, **w), _tri_call("sideways"), r"\[direction\]"),
         (lambda z, d, m, w: tk.turbo_trimul(z, d, m, **w), _tri_call(p_in=(64, 64)), r"\[weight_shape\]"),
         (lambda z, d, m, w: tk.turbo_trimul(z, d, m, **w), _tri_call(mask=torch.int32), r"\[mask_dtype\]")]


@pytest.mark.parametrize("f, args, text", CALLS, ids=[c[2] for c in CALLS])
def test_tracing_refuses_what_an_eager_call_refuses(f, args, text):
    class M(torch.nn.Module):
        def forward(self, *a):
            return f(*a[:1], *rest, *a[1:]) if rest else f(*a)

    rest = [x for x in args if isinstance(x, str)]
    with pytest.raises(ValueError, match=text):
        torch.export.export(M(), tuple(x for x in args if not isinstance(x, str)), strict=False)
    torch.compiler.reset()
    with pytest.raises(Exception):
        torch.compile(f, backend="eager", fullgraph=True)(*args)


def test_right_calls_are_traced_whole():
    """On the CPU they fail where the graph would launch, not before."""
    torch.compiler.reset()
    with pytest.raises(ValueError, match="operands must be CUDA tensors"):
        torch.compile(CALLS[0][0], backend="eager", fullgraph=True)(*_att_call())
    with pytest.raises(ValueError, match=r"\[device\]"):
        torch.compile(CALLS[3][0], backend="eager", fullgraph=True)(*_tri_call())


@pytest.mark.gpu
@pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA device")
@pytest.mark.parametrize("checkpoint", [None, "int8"])
def test_dynamic_sizes_train_as_eager_ones(checkpoint):
    """The checks of the fake kernels meet free sizes, forward and backward."""
    g = torch.Generator(device="cuda").manual_seed(0)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    nw, nb = r(64).requires_grad_(True), r(64).requires_grad_(True)
    w = r(24, 64).requires_grad_(True)

    def f(x):
        y = tk.turbo_layer_norm(x, nw, nb, checkpoint=checkpoint)
        codes, scales = tk.pack_activation(x)
        return tk.turbo_norm_linear(y.bfloat16(), None, nb, w, checkpoint=checkpoint), tk.unpack_activation(codes, scales)

    torch.compiler.reset()
    compiled = torch.compile(f, fullgraph=True, dynamic=True, backend="aot_eager")
    for rows in (10, 33, 200):
        x, d = r(rows, 64).requires_grad_(True), r(rows, 24).bfloat16()
        res = []
        for call in (f, compiled):
            o, v = call(x)
            res.append([o, v, *torch.autograd.grad(o, (x, nw, nb, w), d)])
        assert all(torch.equal(a, b) for a, b in zip(*res))


@pytest.mark.gpu
@pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA device")
def test_triangle_operators_follow_dynamic_sizes():
    g = torch.Generator(device="cuda").manual_seed(0)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    from openfold3_triangle_kernel_b200.synthetic import trimul_weights
    tw = {n: t.cuda() for n, t in trimul_weights(32, 0).items()}
    torch.compiler.reset()
    att = lambda q, b: tk.turbo_attention(q, q, q, pair_bias=b)  # noqa: E731
    tri = lambda z, m: tk.turbo_trimul(z, "incoming", m, **tw)  # noqa: E731
    for n in (16, 24):
        q, b = r(1, n, 2, n, 32).bfloat16(), r(1, 1, 2, n, n)
        assert torch.equal(torch.compile(att, fullgraph=True, dynamic=True, backend="aot_eager")(q, b), att(q, b))
        z, m = r(1, n, n, 32).bfloat16(), (r(1, n, n) > 0).float()
        assert torch.equal(torch.compile(tri, fullgraph=True, dynamic=True, backend="aot_eager")(z, m), tri(z, m))

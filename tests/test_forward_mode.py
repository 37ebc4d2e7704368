"""No operator propagates a forward-mode tangent: a dual tensor is refused, it does not lose its tangent without a word."""
import pytest
import torch
from torch.autograd import forward_ad as fw

import openfold3_triangle_kernel_b200 as tk
from openfold3_triangle_kernel_b200._checks import has_tangent

BF = torch.bfloat16


def _dual(t):
    return fw.make_dual(t, torch.ones_like(t))


def test_tangents_are_seen_at_every_level():
    x = torch.randn(4)
    assert not has_tangent(x)
    with fw.dual_level():
        d = _dual(x)
        assert has_tangent(d) and has_tangent(d.view(2, 2)) and has_tangent(None, x, d) and not has_tangent(x)
    seen = []

    def f(y):
        seen.append(has_tangent(y))
        return (y * y).sum()

    torch.func.jvp(f, (x,), (x,))
    torch.func.jvp(torch.func.grad(f), (x,), (x,))
    torch.func.grad(lambda y: torch.func.jvp(f, (y,), (x,))[1])(x)
    torch.func.jvp(lambda y: torch.vmap(f)(y.view(2, 2)), (x,), (x,))
    torch.func.jacfwd(f)(x)
    assert seen == [True] * 5
    torch.func.grad(f)(x)
    torch.vmap(f)(x.view(2, 2))
    assert seen[5:] == [False, False]


def test_support_checks_name_the_tangent():
    with fw.dual_level():
        x, v, w = _dual(torch.zeros(4, 16)), _dual(torch.zeros(16)), _dual(torch.zeros(8, 16))
        p = lambda d: fw.unpack_dual(d).primal  # noqa: E731
        check = lambda *a: tk.check_layer_norm_support(*a, check_device=False)  # noqa: E731
        for a in ((x, None, None), (p(x), v, None), (p(x), None, v)):
            assert check(*a).code == "tangent"
        assert check(p(x), p(v), p(v)).supported
        b = p(x).bfloat16()
        check = lambda *a: tk.check_norm_linear_support(*a, check_device=False)  # noqa: E731
        for a in ((x.bfloat16(), None, None, p(w)), (b, v, None, p(w)), (b, None, v, p(w)), (b, None, None, w)):
            assert check(*a).code == "tangent"
        assert check(b, p(v), p(v), p(w)).supported
        z = _dual(torch.zeros(1, 8, 8, 32, dtype=BF))
        assert tk.check_trimul_support(z, "outgoing", None, {}, check_device=False).code == "tangent"
        nw = dict(norm_in_weight=_dual(torch.zeros(32)))
        assert tk.check_trimul_support(p(z), "outgoing", None, nw, check_device=False).code == "tangent"
        q = torch.zeros(1, 2, 2, 8, 16, dtype=BF)
        args = dict(q=q, k=q, v=q, res_mask=torch.zeros(1, 2, 1, 1, 8), pair_bias=torch.zeros(1, 1, 2, 8, 8))
        assert tk.is_turbo_attention_supported(**args, check_device=False)[0]
        for n in args:
            ok, reason = tk.is_turbo_attention_supported(**{**args, n: _dual(args[n])}, check_device=False)
            assert not ok and "forward-mode" in reason


@pytest.mark.gpu
@pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA device")
def test_dual_tensors_are_refused():
    r = lambda *s: torch.randn(*s, device="cuda")  # noqa: E731
    from openfold3_triangle_kernel_b200.synthetic import trimul_weights
    tw = {n: t.cuda() for n, t in trimul_weights(32, 0).items()}
    q, bias, z = r(1, 2, 2, 8, 16).bfloat16(), r(1, 1, 2, 8, 8), r(1, 8, 8, 32).bfloat16()
    x, v, w = r(6, 64), r(64), r(16, 64)
    calls = [(lambda t: tk.turbo_layer_norm(t, v), x), (lambda t: tk.turbo_layer_norm(x, t), v),
             (lambda t: tk.turbo_layer_norm(x, None, t, checkpoint="int8"), v),
             (lambda t: tk.turbo_norm_linear(t, v, v, w), x.bfloat16()),
             (lambda t: tk.turbo_norm_linear(x.bfloat16(), None, None, t), w),
             (lambda t: tk.turbo_norm_linear(x.bfloat16(), t, None, w), v),
             (lambda t: tk.turbo_attention(t, q, q, pair_bias=bias), q),
             (lambda t: tk.turbo_attention(q, q, q, pair_bias=t), bias),
             (lambda t: tk.turbo_trimul(t, "incoming", **tw), z),
             (lambda t: tk.turbo_trimul(z, "incoming", **{**tw, "p_in_weight": t}), tw["p_in_weight"])]
    for f, t in calls:
        for leaf in (t, t.clone().requires_grad_(True)):
            with fw.dual_level(), pytest.raises(ValueError, match="forward-mode"):
                f(_dual(leaf))
        with pytest.raises(ValueError, match="forward-mode"):
            torch.func.jvp(f, (t,), (t,))
        f(t)        # (afterwards as before)
    with fw.dual_level():       # put away without a derivative, as without a gradient
        codes, scales = tk.pack_activation(_dual(x))
        assert torch.equal(tk.unpack_activation(codes, scales), tk.unpack_activation(*tk.pack_activation(x)))


@pytest.mark.gpu
@pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA device")
def test_a_dual_gradient_is_refused():
    """The gradients are linear in the incoming one, whose tangent they would drop."""
    x = torch.randn(6, 64, device="cuda", requires_grad=True)
    w = torch.randn(16, 64, device="cuda")
    for y in (tk.turbo_layer_norm(x), tk.turbo_norm_linear(x.bfloat16(), None, None, w)):
        with fw.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
            torch.autograd.grad(y, x, _dual(torch.ones_like(y)), retain_graph=True)
        torch.autograd.grad(y, x, torch.ones_like(y))

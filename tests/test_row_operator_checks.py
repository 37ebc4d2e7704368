"""Refusals of the row-wise operators, none of which needs a GPU."""
import ctypes

import pytest
import torch

import openfold3_triangle_kernel_b200 as tk
from openfold3_triangle_kernel_b200 import _cabi as C
from openfold3_triangle_kernel_b200.activation_checkpoint import check_pack_support, check_unpack_support

ONE = ctypes.c_void_p(256)
NULL = ctypes.c_void_p(0)


def _codes(res):
    return res.supported, res.code


@pytest.mark.parametrize("kw, code", [
    (dict(x=[1.0]), "x_type"),
    (dict(x=torch.zeros(4, 8, dtype=torch.float64)), "x_dtype"),
    (dict(x=torch.zeros(())), "x_shape"),
    (dict(x=torch.zeros(4, 0)), "x_shape"),
    (dict(x=torch.zeros(1, 8193)), "columns"),
    (dict(x=torch.zeros(4, 8), weight=torch.zeros(7)), "weight_shape"),
    (dict(x=torch.zeros(4, 8), bias=torch.zeros(8, 1)), "weight_shape"),
    (dict(x=torch.zeros(4, 8), weight=torch.zeros(8, dtype=torch.float64)), "weight_dtype"),
    (dict(x=torch.zeros(4, 8), checkpoint="fp8"), "checkpoint"),
    (dict(x=torch.zeros(4, 8), eps=-1.0), "eps"),
    (dict(x=torch.zeros(4, 8), eps=float("nan")), "eps"),
])
def test_layer_norm_support(kw, code):
    assert _codes(tk.check_layer_norm_support(**kw, check_device=False)) == (False, code)


def test_layer_norm_support_accepts():
    for dt in (torch.bfloat16, torch.float16, torch.float32):
        x = torch.zeros(2, 3, 5, dtype=dt)
        assert tk.check_layer_norm_support(x, torch.ones(5), None, check_device=False).supported
    assert tk.check_layer_norm_support(torch.zeros(0, 8192), check_device=False).supported


@pytest.mark.parametrize("kw, code", [
    (dict(x=torch.zeros(4, 16)), "x_dtype"),
    (dict(x=torch.zeros(4, 12).bfloat16()), "columns"),
    (dict(weight=torch.zeros(16, 8)), "weight_shape"),
    (dict(weight=torch.zeros(16)), "weight_shape"),
    (dict(weight=torch.zeros(12, 16)), "outputs"),
    (dict(weight=torch.zeros(0, 16)), "outputs"),
    (dict(weight=torch.zeros(1).expand(2 ** 30 + 8, 16)), "extent"),
    (dict(x=torch.zeros(1).bfloat16().expand(2 ** 31 - 256, 16)), "extent"),
    (dict(weight=torch.zeros(8, 16, dtype=torch.int8)), "weight_dtype"),
    (dict(norm_weight=torch.zeros(8)), "weight_shape"),
    (dict(norm_bias=torch.zeros(16, dtype=torch.float64)), "weight_dtype"),
    (dict(checkpoint=True), "checkpoint"),
])
def test_norm_linear_support(kw, code):
    full = dict(x=torch.zeros(4, 16).bfloat16(), norm_weight=None, norm_bias=None, weight=torch.zeros(24, 16))
    full.update(kw)
    assert _codes(tk.check_norm_linear_support(**full, check_device=False)) == (False, code)


@pytest.mark.parametrize("x, code", [
    ("x", "x_type"), (torch.zeros(()), "x_shape"), (torch.zeros(4, dtype=torch.int8), "x_dtype"),
    (torch.zeros(1, 1).bfloat16().expand(2 ** 31, 1), "extent"),
    (torch.zeros(1).bfloat16().expand(2 ** 31), "extent"),
])
def test_pack_support(x, code):
    assert _codes(check_pack_support(x, check_device=False)) == (False, code)


@pytest.mark.parametrize("codes, scales, dtype, code", [
    (torch.zeros(4, 200), torch.zeros(4, 2), torch.float32, "x_dtype"),
    (torch.zeros(4, 200, dtype=torch.int8), torch.zeros(4, 2).half(), torch.float32, "x_dtype"),
    (torch.zeros(4, 200, dtype=torch.int8), torch.zeros(4, 1), torch.float32, "x_shape"),
    (torch.zeros(4, 200, dtype=torch.int8), torch.zeros(2), torch.float32, "x_shape"),
    (torch.zeros(4, 200, dtype=torch.int8), torch.zeros(4, 2), torch.float64, "dtype"),
])
def test_unpack_support(codes, scales, dtype, code):
    assert _codes(check_unpack_support(codes, scales, dtype, check_device=False)) == (False, code)


@pytest.mark.parametrize("eps", [float("inf"), 1e39, 10 ** 400, -1e-300], ids=["inf", "1e39", "1e400", "-1e-300"])
def test_eps_is_a_number_of_32_bits(eps):
    """A larger one became an infinity, and every row its bias."""
    x = torch.zeros(4, 16)
    assert tk.check_layer_norm_support(x, eps=torch.finfo(torch.float32).max, check_device=False).supported
    assert _codes(tk.check_layer_norm_support(x, eps=eps, check_device=False)) == (False, "eps")
    assert _codes(tk.check_norm_linear_support(x.bfloat16(), None, None, torch.zeros(8, 16), eps, check_device=False)) == (
        False, "eps")
    for f in (lambda: tk.turbo_layer_norm(x, eps=eps), lambda: tk.turbo_norm_linear(x.bfloat16(), None, None, x[:, :], eps=eps)):
        with pytest.raises(ValueError, match=r"unsupported \[eps\]"):
            f()


def test_operators_refuse_cpu_tensors():
    x = torch.zeros(4, 16)
    with pytest.raises(ValueError, match=r"turbo_layer_norm unsupported \[device\]"):
        tk.turbo_layer_norm(x)
    with pytest.raises(ValueError, match=r"turbo_norm_linear unsupported \[device\]"):
        tk.turbo_norm_linear(x.bfloat16(), None, None, torch.zeros(8, 16))
    with pytest.raises(ValueError, match=r"pack_activation unsupported \[device\]"):
        tk.pack_activation(x)
    with pytest.raises(ValueError, match=r"unpack_activation unsupported \[device\]"):
        tk.unpack_activation(x.to(torch.int8), torch.zeros(4, 1))


# ---- traced calls ---------------------------------------------------------------------------------
BF, I8 = torch.bfloat16, torch.int8
OPS = torch.ops.tpf_b200
E = lambda *s, dt=torch.float32: torch.empty(*s, dtype=dt)  # noqa: E731
# a call of an operator and the reason for its refusal; sizes are those of x [64, 128] unless they say otherwise
WRONG = [
    (lambda: OPS.layer_norm_fwd(E(64, 128), E(16), None, 1e-5, False), "weight_shape"),
    (lambda: OPS.layer_norm_fwd(E(64, 128), None, E(128, dt=torch.float64), 1e-5, True), "weight_dtype"),
    (lambda: OPS.layer_norm_fwd(E(64, 128, dt=I8), None, None, 1e-5, False), "x_dtype"),
    (lambda: OPS.layer_norm_fwd(E(4, 9000), None, None, 1e-5, False), "columns"),
    (lambda: OPS.layer_norm_fwd(E(64, 128), None, None, -1.0, False), "eps"),
    (lambda: OPS.layer_norm_bwd(E(64, 128), E(64, 64), E(2, 64), E(0, dt=I8), E(0), None, None), "x_shape"),
    (lambda: OPS.layer_norm_bwd(E(64, 128), E(64, 128, dt=BF), E(2, 64), E(0, dt=I8), E(0), None, None), "x_dtype"),
    (lambda: OPS.layer_norm_bwd(E(64, 128), E(64, 128), E(2, 32), E(0, dt=I8), E(0), None, None), "stats"),
    (lambda: OPS.layer_norm_bwd(E(64, 128), None, E(2, 64), E(0, dt=I8), E(64, 1), None, None), "codes"),
    (lambda: OPS.layer_norm_bwd(E(64, 120), None, E(2, 64), E(64, 120, dt=I8), E(64, 1), None, None), "codes"),
    (lambda: OPS.layer_norm_bwd(E(64, 128), None, E(2, 64), E(64, 128, dt=I8), E(1, 1), None, None), "scales"),
    (lambda: OPS.layer_norm_bwd(E(64, 128), E(64, 128), E(2, 64), E(0, dt=I8), E(0), E(8), None), "weight_shape"),
    (lambda: OPS.norm_linear_fwd(E(64, 128, dt=BF), None, None, E(64, 16), 1e-5, False), "weight_shape"),
    (lambda: OPS.norm_linear_fwd(E(64, 128, dt=BF), E(8), None, E(64, 128), 1e-5, False), "weight_shape"),
    (lambda: OPS.norm_linear_fwd(E(64, 128, dt=BF), None, None, E(12, 128), 1e-5, False), "outputs"),
    (lambda: OPS.norm_linear_fwd(E(64, 128), None, None, E(64, 128), 1e-5, False), "x_dtype"),
    (lambda: OPS.norm_linear_bwd(E(64, 8), E(64, 128, dt=BF), E(2, 64), E(0, dt=I8), E(0), None, None, E(16, 128)),
     "d_out_shape"),
    (lambda: OPS.norm_linear_bwd(E(64, 16), E(32, 128, dt=BF), E(2, 64), E(0, dt=I8), E(0), None, None, E(16, 128)),
     "d_out_shape"),
    (lambda: OPS.norm_linear_bwd(E(64, 16), E(64, 128, dt=BF), E(2, 63), E(0, dt=I8), E(0), None, None, E(16, 128)), "stats"),
    (lambda: OPS.norm_linear_bwd(E(64, 16), None, E(2, 64), E(64, 112, dt=I8), E(64, 1), None, None, E(16, 128)), "codes"),
    (lambda: OPS.norm_linear_bwd(E(64, 16), None, E(2, 64), E(64, 128, dt=I8), E(64, 2), None, None, E(16, 128)), "scales"),
    (lambda: OPS.int8_pack(E(64, 128, dt=torch.float64)), "x_dtype"),
    (lambda: OPS.int8_unpack(E(64, 128, dt=I8), E(1, 1), BF), "x_shape"),
    (lambda: OPS.int8_unpack(E(64, 128, dt=I8), E(64, 1, dt=torch.float16), BF), "x_dtype"),
    (lambda: OPS.int8_unpack(E(64, 128, dt=I8), E(64, 1), torch.float64), "dtype"),
]


@pytest.mark.parametrize("call, code", WRONG, ids=[f"{c}{n}" for n, (_, c) in enumerate(WRONG)])
def test_operators_of_a_traced_graph_refuse(call, code):
    """Where the fake kernels run and where the operator would launch."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode(), pytest.raises(ValueError, match=rf"unsupported \[{code}\]"):
        call()
    with pytest.raises(ValueError, match=r"unsupported \["):   # (on the CPU the device may be what it names)
        call()


def test_fake_tensors_of_two_devices_are_refused():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        x, w = torch.empty(64, 128, dtype=BF, device="cuda"), E(64, 128)
        codes = torch.empty(64, 128, dtype=I8, device="cuda")
        for call in (lambda: OPS.norm_linear_fwd(x, None, None, w, 1e-5, False),
                     lambda: OPS.layer_norm_fwd(x, E(128), None, 1e-5, False),
                     lambda: OPS.layer_norm_bwd(x, x, E(2, 64), codes, E(0), None, None),
                     lambda: OPS.int8_unpack(codes, E(64, 1), BF)):
            with pytest.raises(ValueError, match=r"unsupported \[(weight_)?device\]"):
                call()


@pytest.mark.parametrize("f, args, code", [
    (lambda x, w: tk.turbo_layer_norm(x, w), (E(64, 128), E(16)), "weight_shape"),
    (lambda x, w: tk.turbo_norm_linear(x, None, None, w), (E(64, 128, dt=BF), E(64, 16)), "weight_shape"),
    (lambda c, s: tk.unpack_activation(c, s), (E(64, 128, dt=I8), E(1, 1)), "x_shape"),
    (lambda x, w: tk.pack_activation(x), (E(64, 128, dt=I8), E(1)), "x_dtype"),
])
def test_tracing_refuses_wrong_shapes(f, args, code):
    torch.compiler.reset()
    with pytest.raises(Exception, match=rf"unsupported \[{code}\]"):
        torch.compile(f, backend="eager", fullgraph=True)(*args)


def test_free_sizes_stay_free():
    """The checks of a fake kernel pin no size of an exported graph."""
    from torch.export import Dim, export

    class M(torch.nn.Module):
        def forward(self, x, nw, w, keep):
            y = tk.turbo_layer_norm(x, nw, checkpoint="int8")
            codes, scales = tk.pack_activation(y)
            z = tk.unpack_activation(codes, scales)
            return tk.turbo_norm_linear(z, nw, None, w), tk.turbo_norm_linear(z[keep], None, None, w)

    rows, outs = Dim("rows"), Dim("outs")
    args = (E(10, 64), E(64), E(24, 64), torch.ones(10, dtype=torch.bool))
    exported = export(M(), args, dynamic_shapes=({0: rows}, None, {0: outs}, {0: rows}))
    assert sum("tpf_b200" in str(n.target) for n in exported.graph.nodes) == 5


def test_int8_activations_leaves_cpu_tensors_alone():
    x = torch.randn(300, 300, requires_grad=True)
    with tk.int8_activations(min_elements=1):
        y = (x.bfloat16() * 2).sin().sum()
    y.backward()
    x2 = x.detach().clone().requires_grad_(True)
    (x2.bfloat16() * 2).sin().sum().backward()
    assert torch.equal(x.grad, x2.grad)


def test_what_int8_activations_takes_for_a_parameter():
    from openfold3_triangle_kernel_b200.activation_checkpoint import _is_parameter
    lin = torch.nn.functional.linear
    h = torch.randn(3, 8, dtype=BF, requires_grad=True) * 2

    def kept(f, autocast=False):
        """(is a parameter, shape) of what f keeps."""
        seen = []
        hooks = torch.autograd.graph.saved_tensors_hooks(lambda t: seen.append((_is_parameter(t), tuple(t.shape))) or t,
                                                         lambda t: t)
        with torch.autocast("cpu", BF, enabled=autocast), hooks:
            f()
        assert seen
        return {s for p, s in seen if p}, {s for p, s in seen if not p}

    for grad in (True, False):
        w = torch.nn.Parameter(torch.randn(4, 8, dtype=BF), requires_grad=grad)
        acts = {(3, 8)} if grad else set()
        assert kept(lambda: lin(h, w)) == ({(8, 4)}, acts)
        assert kept(lambda: h @ w[:2].t()) == ({(8, 2)}, acts)
        assert kept(lambda: h * w[0]) == ({(8,)}, acts)
    m = torch.nn.Parameter(torch.randn(4, 8))
    assert kept(lambda: lin(h, m), autocast=True) == ({(8, 4)}, {(3, 8)})
    assert kept(lambda: lin(h, torch.cat([m, m * 1]).to(BF))) == (set(), {(8, 8), (3, 8)})
    assert kept(lambda: lin(h, torch.cat([m, m]).to(BF))) == ({(8, 8)}, {(3, 8)})
    assert kept(lambda: lin(h, m.to(BF).split([1, 3])[1])) == ({(8, 3)}, {(3, 8)})
    assert kept(lambda: lin(h, m.to(BF).unsqueeze(0).squeeze(0))) == ({(8, 4)}, {(3, 8)})
    doubled = m.to(BF)[:, :1]
    for _ in range(40):     # (a walk over every path would take 2^40 steps)
        doubled = torch.cat([doubled, doubled])[:4]
    assert kept(lambda: h[:, :1] @ doubled.t())[1] >= {(1, 4)}
    assert kept(lambda: h * h) == (set(), {(3, 8)})
    assert kept(lambda: torch.softmax(h, -1)) == (set(), {(3, 8)})
    x = torch.randn(3, 8, dtype=BF)     # data: an activation
    w = torch.nn.Parameter(torch.randn(4, 8, dtype=BF))
    assert kept(lambda: lin(x, w)) == (set(), {(3, 8)})


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_the_8_bit_format_is_as_near_as_the_documents_say(dtype):
    """Half a step of the codes alone (a / 254) is not the bound: values are rounded once more."""
    from oracle import rows_oracle as ro
    g = torch.Generator().manual_seed(1)
    x = (torch.randn(4000, 128, generator=g) * torch.exp(3 * torch.randn(4000, 1, generator=g))).to(dtype)
    x[::3, 0] = 1.0625
    x[1::3] = (torch.randint(-254, 255, (len(x[1::3]), 128), generator=g) / 254).to(dtype)      # (ties and near ties)
    x[7], x[8], x[9] = torch.finfo(dtype).max, torch.finfo(dtype).tiny, torch.finfo(dtype).tiny / 4
    off = (ro.pack(x)[2].float().to(dtype).double() - x.double()).abs()
    assert (off <= ro.pack_off(x, dtype)).all()
    assert (off > x.double().abs().amax(-1, keepdim=True) / 254).any()


# ---- the C entries -------------------------------------------------------------------------------
def _ln_fwd(**kw):
    a = dict(x=ONE, pitch=8, type=1, w=NULL, wt=0, b=NULL, bt=0, y=ONE, codes=NULL, scales=NULL, mean=NULL, rstd=NULL, rows=4,
             cols=8, eps=1e-5, stream=NULL)
    a.update(kw)
    return C.call("tpf_layer_norm_fwd", *a.values())


def _ln_bwd(**kw):
    a = dict(dy=ONE, x=ONE, pitch=8, codes=NULL, scales=NULL, type=1, mean=ONE, rstd=ONE, w=NULL, wt=0, dx=ONE, dw=NULL, dwt=0,
             db=NULL, dbt=0, ws=NULL, wsb=0, rows=4, cols=8, stream=NULL)
    a.update(kw)
    return C.call("tpf_layer_norm_bwd", *a.values())


@pytest.mark.parametrize("kw, text", [
    (dict(type=3), "unknown element type"), (dict(rows=-1), "rows must not be negative"), (dict(cols=0), "1 to 8192 columns"),
    (dict(cols=8193, pitch=8193), "1 to 8192 columns"), (dict(pitch=7), "rows overlap"), (dict(codes=ONE), "come together"),
    (dict(mean=ONE), "come together"), (dict(w=ONE, wt=5), "unknown parameter type"), (dict(x=NULL), "null pointer"),
    (dict(y=NULL), "null pointer"),
])
def test_layer_norm_forward_entry_refuses(kw, text):
    with pytest.raises(ValueError, match=text):
        _ln_fwd(**kw)


@pytest.mark.parametrize("kw, text", [
    (dict(x=NULL), "null pointer"), (dict(mean=NULL, rstd=NULL), "null pointer"), (dict(dy=NULL), "null pointer"),
    (dict(dw=ONE, dwt=9), "unknown parameter type"), (dict(cols=9000, pitch=9000), "1 to 8192 columns"),
    (dict(dw=ONE, ws=ctypes.c_void_p(260), wsb=1 << 20), "workspace must be 16-byte aligned"),
])
def test_layer_norm_backward_entry_refuses(kw, text):
    with pytest.raises(ValueError, match=text):
        _ln_bwd(**kw)


def test_layer_norm_backward_entry_wants_a_workspace():
    with pytest.raises(C.TpfError, match="workspace of"):
        _ln_bwd(dw=ONE)
    lib = C.load()
    assert lib.tpf_layer_norm_bwd_workspace_bytes(4, 8) == 4 * 2 * 8 * 4
    assert lib.tpf_layer_norm_bwd_workspace_bytes(0, 8) == 0
    assert lib.tpf_layer_norm_bwd_workspace_bytes(10 ** 6, 128) <= 8 * 160 * 2 * 128 * 4


def test_no_rows_is_no_launch():
    before = C.load().tpf_launch_count()
    _ln_fwd(rows=0, x=NULL, y=NULL)
    _ln_bwd(rows=0, x=NULL, dy=NULL, mean=NULL, rstd=NULL)
    C.call("tpf_int8_pack", NULL, 8, 1, NULL, NULL, 0, 8, NULL)
    C.call("tpf_int8_unpack", NULL, NULL, 1, NULL, 4, 0, NULL)
    assert C.load().tpf_launch_count() == before


@pytest.mark.parametrize("args, text", [
    ((ONE, 8, 7, ONE, ONE, 4, 8, NULL), "unknown element type"), ((NULL, 8, 1, ONE, ONE, 4, 8, NULL), "null pointer"),
    ((ONE, 7, 1, ONE, ONE, 4, 8, NULL), "rows overlap"), ((ONE, 8, 1, ONE, ONE, -4, 8, NULL), "must not be negative"),
    ((ONE, 8, 1, ONE, ONE, 1 << 31, 8, NULL), "2\\^31"), ((ONE, 1 << 31, 1, ONE, ONE, 1, 1 << 31, NULL), "2\\^31"),
])
def test_pack_entry_refuses(args, text):
    with pytest.raises(ValueError, match=text):
        C.call("tpf_int8_pack", *args)


def _nl_fwd(**kw):
    a = dict(x=ONE, pitch=16, nw=NULL, nwt=0, nb=NULL, nbt=0, w=ONE, out=ONE, codes=NULL, scales=NULL, mean=NULL, rstd=NULL,
             ws=ONE, wsb=1 << 20, rows=4, cols=16, outs=8, eps=1e-5, stream=NULL)
    a.update(kw)
    return C.call("tpf_norm_linear_fwd", *a.values())


@pytest.mark.parametrize("kw, text", [
    (dict(cols=12, pitch=12), "multiples of 8"), (dict(outs=12), "multiples of 8"), (dict(outs=0), "multiples of 8"),
    (dict(w=NULL), "null pointer"), (dict(x=NULL), "null pointer"), (dict(out=NULL), "null pointer"),
    (dict(w=ctypes.c_void_p(264)), "weight must be 16-byte aligned"), (dict(out=ctypes.c_void_p(264)), "out must be 16-byte"),
    (dict(x=ctypes.c_void_p(258)), "x must"), (dict(pitch=20), "x must"), (dict(rows=1 << 31), "too large"),
    (dict(outs=(1 << 30) + 8), "too large"),  # (a few rows: outputs are counted in 32 bits, up to a grid's more than there are)
])
def test_norm_linear_forward_entry_refuses(kw, text):
    with pytest.raises(ValueError, match=text):
        _nl_fwd(**kw)


def _nl_bwd(**kw):
    a = dict(d_out=ONE, x=ONE, pitch=16, codes=NULL, scales=NULL, mean=ONE, rstd=ONE, nw=NULL, nwt=0, nb=NULL, nbt=0, w=ONE,
             dx=ONE, dnw=NULL, dnwt=0, dnb=NULL, dnbt=0, dw=NULL, dwt=1, ws=ONE, wsb=1 << 30, rows=4, cols=16, outs=8,
             stream=NULL)
    a.update(kw)
    return C.call("tpf_norm_linear_bwd", *a.values())


@pytest.mark.parametrize("kw, text", [
    (dict(d_out=NULL), "null pointer"), (dict(x=NULL), "null pointer"), (dict(d_out=ctypes.c_void_p(264)), "16-byte aligned"),
    (dict(dx=ctypes.c_void_p(264)), "16-byte aligned"), (dict(dw=ONE, dwt=4), "unknown parameter type"),
    (dict(outs=4), "multiples of 8"), (dict(x=ctypes.c_void_p(258)), "x must"),
    (dict(codes=ctypes.c_void_p(260), scales=ONE), "codes must"),
    (dict(dw=ctypes.c_void_p(264)), "d_weight must be 16-byte aligned"),
    (dict(ws=ctypes.c_void_p(264)), "workspace must be 16-byte aligned"),
])
def test_norm_linear_backward_entry_refuses(kw, text):
    with pytest.raises(ValueError, match=text):
        _nl_bwd(**kw)


def test_norm_linear_entries_want_workspaces():
    with pytest.raises(C.TpfError, match="workspace of"):
        _nl_fwd(rows=1000, cols=256, pitch=256, wsb=0, ws=NULL)
    with pytest.raises(C.TpfError, match="workspace of"):
        _nl_bwd(wsb=8)
    lib = C.load()
    assert lib.tpf_norm_linear_fwd_workspace_bytes(0, 256, 8) == 0
    assert lib.tpf_norm_linear_fwd_workspace_bytes(1000, 256, 8) == 1000 * 256 * 2
    assert lib.tpf_norm_linear_fwd_workspace_bytes(1000, 128, 512) == 0     # y stays on the SM
    assert lib.tpf_norm_linear_bwd_workspace_bytes(1000, 16, 8) % 256 == 0


def test_norm_linear_entries_without_rows():
    lib = C.load()
    before = lib.tpf_launch_count()
    _nl_fwd(rows=0, x=NULL, out=NULL, ws=NULL, wsb=0)
    _nl_bwd(rows=0, x=NULL, d_out=NULL, mean=NULL, rstd=NULL, ws=NULL, wsb=0)
    assert lib.tpf_launch_count() == before

"""Refusals of dropout, rotation and window attention, the frequencies, and the oracle against plain forms; none of it needs a GPU."""
import contextlib
import ctypes
import math

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.autograd import forward_ad as fw

import openfold3_triangle_kernel_b200 as tk
from openfold3_triangle_kernel_b200 import _cabi as C
from oracle import sequence_oracle as so

OPS = torch.ops.tpf_b200
BF, F16, F32, F64, I32, I64 = torch.bfloat16, torch.float16, torch.float32, torch.float64, torch.int32, torch.int64
E = lambda *s, dt=F32: torch.empty(*s, dtype=dt)  # noqa: E731
NULL, ONE, MIS = ctypes.c_void_p(0), ctypes.c_void_p(256), ctypes.c_void_p(258)


def _fr(dim=32):
    return tk.rotary_frequencies(dim)


# ---- support predicates ----------------------------------------------------------------------------
@pytest.mark.parametrize("a, kw, code", [
    (([1.0], 0.5), {}, "x_type"), ((E(()), 0.5), {}, "x_shape"), ((E(4, dt=F64), 0.5), {}, "x_dtype"), ((E(4), 1.5), {}, "p"),
    ((E(4), -0.1), {}, "p"), ((E(4), math.nan), {}, "p"), ((E(4), "half"), {}, "p"), ((E(4), 0.5, 1.5), {}, "seed"),
    ((E(4), 0.5, (1, 2, 3)), {}, "seed"), ((E(4), 0.5, 2 ** 64), {}, "seed"), ((E(4), 0.5, True), {}, "seed"),
    ((E(4), 0.5, E(2)), {}, "seed"), ((E(4), 0.5, E(3, dt=I64)), {}, "seed"), ((E(4, 5), 0.5, 1), dict(shared_dim=-1), "shared_dim"),
    ((E(4, 5), 0.5, 1), dict(shared_dim=1), "shared_dim"), ((E(4, 5), 0.5, 1), dict(shared_dim=-3), "shared_dim"),
    ((E(4, 5), 0.5, 1), dict(shared_dim=0.0), "shared_dim"), ((E(4, 5), 0.5, 1), dict(residual=E(5)), "residual_shape"),
    ((E(4, 5), 0.5, 1), dict(residual=E(4, 5, dt=BF)), "residual_dtype")])
def test_dropout_support(a, kw, code):
    assert tk.check_dropout_support(*a, **kw, check_device=False).code == code
    with pytest.raises(ValueError, match=rf"turbo_dropout unsupported \[{code}\]"):
        tk.turbo_dropout(*a, **kw)


def test_dropout_support_accepts():
    ok = lambda *a, **kw: tk.check_dropout_support(*a, **kw, check_device=False).supported  # noqa: E731
    for dt in (BF, F16, F32):
        assert ok(E(3, 4, 5, dt=dt), 0, 2 ** 64 - 1, shared_dim=-2, residual=E(3, 4, 5, dt=dt))
    assert ok(E(4), 1.0, (-1, 5)) and ok(E(4), 0.5, E(2, dt=I64)) and ok(E(4), 0.5)
    x = E(4)
    assert tk.turbo_dropout.__doc__ and tk.check_dropout_support(x, 0.5, 1).code == "device"


@pytest.mark.parametrize("a, kw, code", [
    ((E(4, 8), None), {}, "x_shape"), ((E(3, 4, 32, dt=F64), None), {}, "x_dtype"), ((E(3, 4, 1), None), {}, "head_dim"),
    ((E(3, 4, 300), None), {}, "head_dim"), ((E(3, 4, 32), (E(16), 1.0)), {}, "frequencies"),
    ((E(3, 4, 32), (E(17, dt=I64), 1.0)), {}, "frequencies"), ((E(3, 4, 32), (E(0, dt=I64), 1.0)), {}, "frequencies"),
    ((E(3, 4, 32), (E(16, dt=I64), math.nan)), {}, "frequencies"), ((E(3, 4, 32), (E(16, dt=I64), math.inf)), {}, "frequencies"),
    ((E(3, 4, 32), "half"), {}, "frequencies"), ((E(3, 4, 32), _fr(), E(3)), {}, "positions"),
    ((E(3, 4, 32), _fr(), E(4, dt=I64)), {}, "positions"), ((E(3, 4, 32), _fr(), E(2, 3, dt=I64)), {}, "positions"),
    ((E(3, 4, 32), _fr(), 1.5), {}, "positions"), ((E(3, 4, 32), _fr(), 2 ** 63), {}, "positions"),
    ((E(3, 4, 32), _fr()), dict(layout="both"), "layout")])
def test_rotary_support(a, kw, code):
    assert tk.check_rotary_support(*a, **kw, check_device=False).code == code
    with pytest.raises(ValueError, match=rf"turbo_rotary unsupported \[{code}\]"):
        tk.turbo_rotary(*a, **kw)


@pytest.mark.parametrize("a, kw, code", [
    ((E(3, 4, 32), E(3, 32), None, None, _fr()), {}, "x_shape"), ((E(3, 4, 32), None, None, None, _fr()), {}, "x_shape"),
    ((E(3, 4, 32), E(4, 4, 32), None, None, _fr()), {}, "x_shape"), ((E(3, 4, 32), E(3, 4, 16), None, None, _fr()), {}, "x_shape"),
    ((E(3, 4, 32), E(3, 4, 32, dt=BF), None, None, _fr()), {}, "x_dtype"),
    ((E(3, 4, 32), E(3, 2, 32), E(16), None, _fr()), {}, "weight_shape"), ((E(3, 4, 32), E(3, 2, 32), None, E(32, dt=F64), _fr()), {}, "weight_dtype"),
    ((E(3, 4, 32), E(3, 2, 32), None, None, _fr()), dict(eps=-1.0), "eps"), ((E(3, 4, 32), E(3, 2, 32), None, None, _fr()), dict(eps=1e39), "eps"),
    ((E(3, 4, 32), E(3, 2, 32), None, None, _fr()), dict(eps=None), "eps")])
def test_qk_norm_rotary_support(a, kw, code):
    assert tk.check_qk_norm_rotary_support(*a, **kw, check_device=False).code == code
    with pytest.raises(ValueError, match=rf"turbo_qk_norm_rotary unsupported \[{code}\]"):
        tk.turbo_qk_norm_rotary(*a, **kw)


def test_rotary_support_accepts():
    f = _fr(16)
    for dt in (BF, F16, F32):
        assert tk.check_rotary_support(E(2, 3, 4, 24, dt=dt), f, E(3, dt=I32), layout="interleaved", check_device=False).supported
        assert tk.check_qk_norm_rotary_support(E(3, 4, 32, dt=dt), E(3, 1, 32, dt=dt), E(32, dt=BF), None, f, -5, check_device=False).supported
    assert tk.check_rotary_support(E(3, 4, 32), f).code == "device"


Q, K = E(2, 5, 4, 32, dt=BF), E(2, 7, 2, 32, dt=BF)


@pytest.mark.parametrize("qkv, kw, code", [
    ((E(5, 32, dt=BF), K, K), {}, "shape"), ((Q, K, None), {}, "shape"), ((Q.float(), K, K), {}, "dtype"), ((Q, K, K.half()), {}, "dtype"),
    ((Q, K, K[:, :6]), {}, "shape"), ((Q, K[:1], K[:1]), {}, "shape"), ((Q, K[..., :16], K[..., :16]), {}, "shape"),
    ((Q[..., :12], K[..., :12], K[..., :12]), {}, "head_dim"), ((E(1, 2, 2, 136, dt=BF),) * 3, {}, "head_dim"),
    ((Q, E(2, 7, 3, 32, dt=BF), E(2, 7, 3, 32, dt=BF)), {}, "heads"), ((Q, K[:, :, :0], K[:, :, :0]), {}, "heads"),
    ((Q, K, K), dict(window=5), "window"), ((Q, K, K), dict(window=(5,)), "window"), ((Q, K, K), dict(window=(-1, 0)), "window"),
    ((Q, K, K), dict(window=(2 ** 28, 0)), "window"), ((Q, K, K), dict(window=(1.0, 0)), "window"), ((Q, K, K), dict(window=(True, 0)), "window"),
    ((Q, K, K), dict(sinks=65), "sinks"), ((Q, K, K), dict(sinks=-1), "sinks"), ((Q, K, K), dict(sinks=None), "sinks"),
    ((Q, K, K), dict(query_offset=2 ** 28 + 1), "query_offset"), ((Q, K, K), dict(query_offset=None), "query_offset"),
    ((Q, K, K), dict(query_offset=E(2)), "query_offset"), ((Q, K, K), dict(query_offset=E(3, dt=I32)), "query_offset"),
    ((Q, K, K), dict(key_lengths=7), "key_lengths"), ((Q, K, K), dict(key_lengths=E(2, 1, dt=I32)), "key_lengths"),
    ((Q, K, K), dict(scale=0.0), "scale"), ((Q, K, K), dict(scale=-1.0), "scale"), ((Q, K, K), dict(scale=math.inf), "scale"),
    ((Q, K, K), dict(scale=math.nan), "scale")])
def test_window_attention_support(qkv, kw, code):
    kw = dict(window=(3, 0)) | kw
    assert tk.check_window_attention_support(*qkv, **kw, check_device=False).code == code
    with pytest.raises(ValueError, match=rf"turbo_window_attention unsupported \[{code}\]"):
        tk.turbo_window_attention(*qkv, **kw)


def test_window_attention_support_accepts():
    ok = lambda *a, **kw: tk.check_window_attention_support(*a, **kw, check_device=False).supported  # noqa: E731
    assert ok(Q, K, K, window=(None, None)) and ok(Q, K, K, window=[0, 0], sinks=64, query_offset=E(2, dt=I64), key_lengths=E(2, dt=I32))
    assert ok(Q[0], K[0], K[0], window=(2 ** 28 - 1, 0), scale=2.0, query_offset=-2 ** 28, key_lengths=torch.tensor(3))
    assert ok(Q[:0], K[:0], K[:0], window=(1, 1)) and ok(Q[:, :0], K, K, window=(1, 1)) and ok(Q, K[:, :0], K[:, :0], window=(1, 1))
    assert tk.check_window_attention_support(Q, K, K, window=(1, 1)).code == "device"


def test_dual_tensors_are_refused():
    dual = lambda t: fw.make_dual(t, torch.ones_like(t))  # noqa: E731
    with fw.dual_level():
        x, q, k, w = torch.zeros(4, 8), torch.zeros(3, 4, 32), torch.zeros(3, 2, 32), torch.zeros(32)
        assert tk.check_dropout_support(dual(x), 0.5, 1, check_device=False).code == "tangent"
        assert tk.check_dropout_support(x, 0.5, 1, residual=dual(x), check_device=False).code == "tangent"
        assert tk.check_rotary_support(dual(q), _fr(), check_device=False).code == "tangent"
        for a in ((dual(q), k, None, None), (q, dual(k), None, None), (q, k, dual(w), None), (q, k, None, dual(w))):
            assert tk.check_qk_norm_rotary_support(*a, _fr(), check_device=False).code == "tangent"
        b, c = q.bfloat16(), k.bfloat16()
        for a in ((dual(b), c, c), (b, dual(c), c), (b, c, dual(c))):
            assert tk.check_window_attention_support(*a, window=(1, 1), check_device=False).code == "tangent"


# ---- the operators of a traced graph ---------------------------------------------------------------
T16 = torch.zeros(16, dtype=I64)
WRONG = [
    (lambda: OPS.dropout(E(4, dt=I32), None, None, 1, 0, 5, -1), "x_dtype"), (lambda: OPS.dropout(E(4, 5), E(4), None, 1, 0, 5, -1), "residual_shape"),
    (lambda: OPS.dropout(E(4, 5), None, E(3, dt=I64), 1, 0, 5, -1), "seed"), (lambda: OPS.dropout(E(4, 5), None, None, 1, 0, 70000, -1), r"\[p"),
    (lambda: OPS.dropout(E(4, 5), None, None, 1, 0, 5, 1), "shared_dim"),
    (lambda: OPS.rotary_fwd(E(3, 4, 300), None, None, None, torch.zeros(16, dtype=I64), None, 0, 1.0, True, False, 0.0), "head_dim"),
    (lambda: OPS.rotary_fwd(E(3, 4, 32), E(3, 4, 16), None, None, torch.zeros(16, dtype=I64), None, 0, 1.0, True, True, 0.0), "x_shape"),
    (lambda: OPS.rotary_fwd(E(3, 4, 32), None, None, None, torch.zeros(16, dtype=I64), E(3, dt=I32), 0, 1.0, True, False, 0.0), "positions"),
    (lambda: OPS.rotary_fwd(E(3, 4, 32), None, None, None, torch.zeros(16, dtype=I64), E(1, dt=I64), 0, 1.0, True, False, 0.0), "positions"),
    (lambda: OPS.rotary_bwd(None, None, None, None, None, None, torch.zeros(16, dtype=I64), None, 0, 1.0, True, False, 0.0), "d_out"),
    (lambda: OPS.rotary_bwd(E(3, 4, 32), None, E(3, 4, 16), None, None, None, torch.zeros(16, dtype=I64), None, 0, 1.0, True, True, 0.0), "x_shape"),
    (lambda: OPS.rotary_bwd(E(3, 4, 32), None, None, None, None, None, torch.zeros(16, dtype=I64), None, 0, 1.0, True, True, 0.0), "x_shape"),
    (lambda: OPS.window_attn_fwd(E(1, 2, 2, 12, dt=BF), E(1, 2, 2, 12, dt=BF), E(1, 2, 2, 12, dt=BF), None, None, 0, 1, 1, 0, 1.0), "head_dim"),
    (lambda: OPS.window_attn_fwd(E(1, 2, 2, 16, dt=BF), E(1, 2, 2, 16, dt=BF), E(1, 2, 2, 16, dt=BF), E(1, dt=I64), None, 0, 1, 1, 0, 1.0), "key_lengths"),
    (lambda: OPS.window_attn_bwd(E(1, 2, 2, 8, dt=BF), *(E(1, 2, 2, 16, dt=BF),) * 4, E(1, 2, 2), None, None, 0, 1, 1, 0, 1.0), r"\[out"),
    (lambda: OPS.window_attn_bwd(*(E(1, 2, 2, 16, dt=BF),) * 5, E(1, 2, 3), None, None, 0, 1, 1, 0, 1.0), "lse"),
]


@pytest.mark.parametrize("fake", [True, False])
@pytest.mark.parametrize("call, code", WRONG)
def test_operators_refuse(call, code, fake):
    with FakeTensorMode() if fake else contextlib.nullcontext():
        with pytest.raises(ValueError, match=code):
            call()


def test_operators_refuse_cpu_tensors():
    for f in (lambda: OPS.dropout(E(4, 5), None, None, 1, 0, 5, -1),
              lambda: OPS.rotary_fwd(E(3, 4, 32), None, None, None, T16, None, 0, 1.0, True, False, 0.0),
              lambda: OPS.window_attn_fwd(*(E(1, 2, 2, 16, dt=BF),) * 3, None, None, 0, 1, 1, 0, 1.0)):
        with pytest.raises(ValueError, match=r"\[device\]"):
            f()


def test_traced_calls_meet_the_contract():
    torch.compiler.reset()
    f = torch.compile(lambda x: tk.turbo_dropout(x, 0.5, 3, shared_dim=-2), backend="eager", fullgraph=True)
    with pytest.raises(ValueError, match=r"\[device\]"):    # traced whole; refused where it would launch
        f(E(3, 4, 5))
    fr = _fr()
    g = torch.compile(lambda q, k: tk.turbo_qk_norm_rotary(q, k, None, None, fr, 7), backend="eager", fullgraph=True)
    with pytest.raises(ValueError, match=r"\[device\]"):
        g(E(3, 4, 32), E(3, 2, 32))
    h = torch.compile(lambda q, k: tk.turbo_window_attention(q, k, k, window=(3, None), sinks=2), backend="eager", fullgraph=True)
    with pytest.raises(ValueError, match=r"\[device\]"):
        h(Q, K)
    for call in (lambda: torch.compile(lambda x: tk.turbo_dropout(x, 2.0, 3), backend="eager", fullgraph=True)(E(4)),
                 lambda: torch.compile(lambda q: tk.turbo_rotary(q, fr), backend="eager", fullgraph=True)(E(3, 4, 16)),
                 lambda: torch.compile(lambda q: tk.turbo_window_attention(q, q, q, window=(3, 0)), backend="eager", fullgraph=True)(E(1, 2, 2, 12, dt=BF))):
        with pytest.raises(Exception):
            call()


# ---- the C entries, without a device ---------------------------------------------------------------
ST = C.i64_array([8, 8, 8])


def _dropout(**kw):
    a = dict(x=ONE, xs=ST, r=NULL, rs=None, out=ONE, os=ST, sizes=C.i64_array([1, 1, 4, 8]), type=1, shared=0, threshold=5, so=NULL,
             seed=1, offset=0, stream=NULL)
    a.update(kw)
    return C.call("tpf_dropout", *a.values())


@pytest.mark.parametrize("kw, text", [
    (dict(type=3), "unknown element type"), (dict(sizes=C.i64_array([1, -1, 4, 8])), "must not be negative"), (dict(threshold=65537), "threshold"),
    (dict(x=NULL), "null pointer"), (dict(out=NULL), "null pointer"), (dict(xs=None), "null pointer"), (dict(r=ONE), "null pointer"),
    (dict(sizes=C.i64_array([1 << 31, 1, 1, 8])), "too many rows"), (dict(sizes=C.i64_array([1 << 20, 1 << 20, 1, 8])), "too many rows"),
    (dict(sizes=C.i64_array([1, 1, 70000, 8])), "too long"), (dict(sizes=C.i64_array([1, 1, 1, 1 << 36])), "too many elements")])
def test_dropout_entry_refuses(kw, text):
    with pytest.raises(ValueError, match=text):
        _dropout(**kw)


def test_empty_calls_launch_nothing():
    _dropout(sizes=C.i64_array([0, 1, 4, 8]), x=NULL, out=NULL)
    _rotary(batch=0, turns=NULL)
    _window(B=0, q=NULL, k=NULL, v=NULL, out=NULL)
    _window(N=0, q=NULL, k=NULL, v=NULL, out=NULL)


def _rotary(**kw):
    a = dict(q=ONE, qs=ST, qh=2, qw=NULL, qwt=0, qo=ONE, k=NULL, ks=None, kh=0, kw=NULL, kwt=0, ko=NULL, type=1, batch=1, tokens=4, dim=32,
             rot=32, turns=ONE, m=1.0, pos=NULL, first=0, half=1, norm=0, eps=0.0, stream=NULL)
    a.update(kw)
    return C.call("tpf_rotary_fwd", *a.values())


def _rotary_bwd(**kw):
    a = dict(dqo=ONE, q=ONE, qs=ST, qh=2, qw=NULL, qwt=0, dq=ONE, dqw=NULL, dko=NULL, k=NULL, ks=None, kh=0, kw=NULL, kwt=0, dk=NULL, dkw=NULL,
             type=1, batch=1, tokens=4, dim=32, rot=32, turns=ONE, m=1.0, pos=NULL, first=0, half=1, norm=1, eps=0.0, ws=NULL, wsb=0, stream=NULL)
    a.update(kw)
    return C.call("tpf_rotary_bwd", *a.values())


@pytest.mark.parametrize("kw, text", [
    (dict(type=-1), "unknown element type"), (dict(tokens=-1), "must not be negative"), (dict(dim=257), "2 to 256"), (dict(dim=1), "2 to 256"),
    (dict(rot=31), "must be even"), (dict(rot=34), "must be even"), (dict(rot=0), "must be even"), (dict(q=NULL), "null pointer"),
    (dict(qo=NULL), "null pointer"), (dict(turns=NULL), "null pointer"), (dict(qs=None), "null pointer"), (dict(qw=ONE, qwt=7), "type of a weight"),
    (dict(batch=1 << 20, tokens=1 << 20), "too many tokens"), (dict(tokens=1 << 28, qh=16), "too many heads")])
def test_rotary_entry_refuses(kw, text):
    with pytest.raises(ValueError, match=text):
        _rotary(**kw)


def test_rotary_backward_entry_refuses():
    with pytest.raises(ValueError, match="without a norm"):
        _rotary_bwd(norm=0, dqw=ONE)
    with pytest.raises(ValueError, match="null pointer"):
        _rotary_bwd(q=NULL)
    with pytest.raises(ValueError, match="null pointer"):
        _rotary_bwd(dqo=NULL)
    with pytest.raises(C.TpfError, match="workspace"):
        _rotary_bwd(dqw=ONE, qw=ONE)
    lib = C.load()
    need = lib.tpf_rotary_bwd_workspace_bytes(32)
    assert need > 0 and lib.tpf_rotary_bwd_workspace_bytes(0) == 0 and lib.tpf_rotary_bwd_workspace_bytes(300) == 0
    with pytest.raises(ValueError, match="workspace must be 16-byte aligned"):
        _rotary_bwd(dqw=ONE, qw=ONE, ws=MIS, wsb=need)


def _window(**kw):
    a = dict(q=ONE, qs=ST, k=ONE, ks=ST, v=ONE, vs=ST, out=ONE, lse=ONE, type=1, B=2, N=4, M=4, H=2, HK=1, D=32, scale=1.0, left=3, right=0,
             sinks=0, offsets=NULL, offset=0, lengths=NULL, stream=NULL)
    a.update(kw)
    return C.call("tpf_window_attn_fwd", *a.values())


def _window_bwd(**kw):
    a = dict(d_out=ONE, q=ONE, qs=ST, k=ONE, ks=ST, v=ONE, vs=ST, out=ONE, lse=ONE, dq=ONE, dk=ONE, dv=ONE, type=1, B=2, N=4, M=4, H=2, HK=1,
             D=32, scale=1.0, left=3, right=0, sinks=0, offsets=NULL, offset=0, lengths=NULL, ws=NULL, wsb=0, stream=NULL)
    a.update(kw)
    return C.call("tpf_window_attn_bwd", *a.values())


@pytest.mark.parametrize("kw, text", [
    (dict(type=0), "must be BF16 or FP16"), (dict(N=-1), "must not be negative"), (dict(H=3, HK=2), "multiple of the key heads"), (dict(D=12), "multiple of 8"),
    (dict(D=136), "multiple of 8"), (dict(N=(1 << 28) + 1), "too large"), (dict(B=65536), "too large"), (dict(left=1 << 28), "reach"),
    (dict(right=1 << 40), "reach"), (dict(sinks=65), "sinks"), (dict(sinks=-2), "sinks"), (dict(offset=(1 << 28) + 1), "position"),
    (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"), (dict(scale=math.inf), "scale"), (dict(scale=math.nan), "scale"), (dict(q=NULL), "null pointer"),
    (dict(v=NULL), "null pointer"), (dict(q=MIS), "q must be 16-byte aligned"), (dict(out=MIS), "out must be 16-byte aligned"),
    (dict(ks=C.i64_array([8, 4, 8])), "strides of k"), (dict(qs=C.i64_array([0, 8, 8])), "strides of q"), (dict(vs=None), "null pointer")])
def test_window_entries_refuse(kw, text):
    with pytest.raises(ValueError, match=text):
        _window(**kw)
    with pytest.raises(ValueError, match=text):
        _window_bwd(**kw)


def test_window_backward_entry_refuses():
    with pytest.raises(ValueError, match="come together"):
        _window_bwd(dk=NULL)
    for name in ("d_out", "dq", "dk", "dv"):
        with pytest.raises(ValueError, match=f"{name} must be 16-byte aligned"):
            _window_bwd(**{name: MIS})
    for name in ("lse", "d_out"):
        with pytest.raises(ValueError, match="null pointer"):
            _window_bwd(**{name: NULL})
    with pytest.raises(C.TpfError, match="workspace"):
        _window_bwd()
    size = C.load().tpf_window_attn_bwd_workspace_bytes
    assert size(2, 4, 4, 2, 1, 32, 3, 0, 0) == 2 * 2 * 2 * 64 * 4
    assert size(0, 4, 4, 2, 1, 32, 3, 0, 0) == size(2, 0, 4, 2, 1, 32, 3, 0, 0) == size(2, 4, 0, 2, 1, 32, 3, 0, 0) == 0
    assert size(2, 4, 4, 2, 1, 32, -1, 0, 4) == size(2, 4, 4, 2, 1, 32, 3, 0, 0) < size(2, 4, 4, 2, 1, 32, 3, 0, 4)
    with pytest.raises(ValueError, match="256-byte aligned"):
        _window_bwd(ws=ctypes.c_void_p(64), wsb=1 << 20)


# ---- frequencies ------------------------------------------------------------------------------------
def test_frequencies():
    f = tk.rotary_frequencies(8, base=100.0)
    radians = (f.turns.double() % 2.0 ** 64) * (2 * math.pi / 2.0 ** 64)
    assert torch.allclose(radians, torch.tensor([100.0 ** (-i / 4) for i in range(4)], dtype=F64), rtol=1e-14, atol=0) and f.magnitude == 1.0
    half = tk.rotary_frequencies(8, base=100.0, scaling="linear", factor=2.0)
    assert torch.allclose(half.turns.double() * 2, f.turns.double() % 2.0 ** 64, rtol=1e-14, atol=0)
    ntk = tk.rotary_frequencies(8, base=100.0, scaling="ntk", factor=4.0)
    assert ntk.turns[0] == f.turns[0] and abs(ntk.turns[-1].item() * 4 / f.turns[-1].item() - 1) < 1e-12
    yarn = tk.rotary_frequencies(64, scaling="yarn", factor=8.0, original_length=4096)
    plain = tk.rotary_frequencies(64)
    ratio = plain.turns.double() / yarn.turns.double()
    assert ratio[0] == 1 and abs(ratio[-1] - 8) < 1e-12 and (ratio[1:] >= ratio[:-1] - 1e-12).all() and abs(yarn.magnitude - (0.1 * math.log(8) + 1)) < 1e-15
    assert tk.rotary_frequencies(64, scaling="yarn", factor=8.0, original_length=4096, magnitude=1.0).magnitude == 1.0


@pytest.mark.parametrize("a, kw", [
    ((7,), {}), ((0,), {}), ((8, 1.0), {}), ((8, math.nan), {}), ((8,), dict(scaling="quadratic")), ((8,), dict(factor=0.5)),
    ((8,), dict(scaling="yarn", factor=2.0)), ((8,), dict(scaling="yarn", factor=2.0, original_length=100, beta_fast=1.0, beta_slow=2.0)),
    ((8,), dict(magnitude=math.inf)), (("8",), {})])
def test_frequencies_refuse(a, kw):
    with pytest.raises(ValueError, match="rotary_frequencies"):
        tk.rotary_frequencies(*a, **kw)


# ---- the oracle --------------------------------------------------------------------------------------
def test_philox_against_the_published_answers():
    """The known answers of Philox 4x32-10 that were published with the generator: all zeros, all ones."""
    assert so.philox(0, 0, 0) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    assert so.philox(2 ** 64 - 1, 2 ** 64 - 1, 2 ** 64 - 1) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]
    kept = so.dropout_mask((3, 40), 0.4, 9, 2)
    halves = [h for g in range(15) for w in so.philox(9, 2, g) for h in (w & 0xFFFF, w >> 16)]
    assert kept.flatten().tolist() == [h >= round(0.4 * 65536) for h in halves[:120]]
    shared = so.dropout_mask((3, 5, 8), 0.4, 9, 2, -2)
    assert torch.equal(shared[:, 0], shared[:, 4]) and torch.equal(shared[:, 0], so.dropout_mask((3, 8), 0.4, 9, 2))


def test_oracle_gradients_by_autograd():
    g = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=g, dtype=F64)  # noqa: E731
    x, w, d = r(2, 5, 3, 12).requires_grad_(True), r(12).requires_grad_(True), r(2, 5, 3, 12)
    f, pos = so.radians(8), torch.arange(5).expand(2, 5)
    for half in (True, False):
        y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-3) * w
        a, b = so.pairs(8, half)
        t = pos.double()[..., None, None] * f
        z = y.clone()
        z = z.index_copy(-1, a, y[..., a] * t.cos() - y[..., b] * t.sin()).index_copy(-1, b, y[..., a] * t.sin() + y[..., b] * t.cos())
        assert torch.allclose(z, so.qk_norm_rotary(x.detach(), w.detach(), f, pos, half, 1e-3)[0])
        gx, gw = torch.autograd.grad(z, [x, w], d)
        back = so.qk_norm_rotary_backward(d, x.detach(), w.detach(), f, pos, half, 1e-3)
        assert torch.allclose(gx, back["dx"]) and torch.allclose(gw, back["dw"])


def test_window_oracle_gradients_by_autograd():
    g = torch.Generator().manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=g).bfloat16()  # noqa: E731
    q, k, v, d = r(2, 6, 4, 8), r(2, 9, 2, 8), r(2, 9, 2, 8), r(2, 6, 4, 8)
    offsets, lengths, window, sinks = [0, 4], [9, 7], (2, 1), 1
    ref = so.window_attention(q, k, v, window, sinks, offsets, lengths, None, d)
    ql, kl, vl = (t.double().requires_grad_(True) for t in (q, k, v))
    outs = []
    for b in range(2):
        rows = []
        for i in range(6):
            pos = offsets[b] + i
            keys = [j for j in range(9) if j < lengths[b] and j <= pos + 1 and (j >= pos - 2 or j < sinks)]
            heads = []
            for h in range(4):
                s = torch.stack([(ql[b, i, h] * kl[b, j, h // 2]).sum() for j in keys]) * 8 ** -0.5 if keys else None
                heads.append((torch.softmax(s, 0)[:, None] * vl[b, keys, h // 2]).sum(0) if keys else torch.zeros(8, dtype=F64))
            rows.append(torch.stack(heads))
        outs.append(torch.stack(rows))
    out = torch.stack(outs)
    assert torch.allclose(out, ref["out"])
    for n, t in zip(("dq", "dk", "dv"), torch.autograd.grad(out, [ql, kl, vl], d.double())):
        assert torch.allclose(t, ref[n])


def test_a_sharded_block_with_dropout_wants_a_seed():
    from openfold3_triangle_kernel_b200.pair_block import _site_seeds, pair_stack_block
    with pytest.raises(ValueError, match="a seed that all ranks share"):
        pair_stack_block(E(1, 4, 4, 32, dt=BF), E(1, 4, 4), {}, 2, group=object(), dropout=0.1)
    assert _site_seeds(7) == [(7, i) for i in range(4)] and _site_seeds((7, 3)) == [(7, 12 + i) for i in range(4)] and _site_seeds(None) == [None] * 4
    assert [t.tolist() for t in _site_seeds(torch.tensor([7, 3]))] == [[7, 12 + i] for i in range(4)]


def test_dropout_sizes():
    """What no launch takes is refused by the check.  (Expanded tensors of any size need no memory.)"""
    big = lambda *s: E(1, dt=BF).expand(*s)  # noqa: E731
    code = lambda x, **kw: tk.check_dropout_support(x, 0.5, 1, **kw, check_device=False).code  # noqa: E731
    assert code(big(2 ** 36 - 1)) == code(big(2 ** 31, 16)) == code(big(2 ** 31 - 1, 4), shared_dim=0) == "ok"
    assert code(big(2 ** 31 - 1, 4, 2), shared_dim=1) == code(big(200000, 64), shared_dim=0) == "ok"
    assert code(big(2 ** 36)) == code(big(2 ** 18, 2 ** 18)) == "x_shape"
    assert code(big(2 ** 31, 4), shared_dim=0) == code(big(2 ** 31, 2, 2), shared_dim=1) == "shared_dim"
    assert code(big(2 ** 16, 2 ** 15, 1, 2), shared_dim=-2) == "shared_dim"


@pytest.mark.parametrize("offset", [0, 3, -1, 2 ** 61, 2 ** 62, -2 ** 61 - 1, 2 ** 63 - 1, -2 ** 63, 2 ** 64 - 1])
def test_site_seeds_of_any_offset(offset):
    """Numbers and the tensor that holds them give the same seeds: four in a row, modulo 2^64."""
    from openfold3_triangle_kernel_b200.pair_block import _site_seeds
    signed = lambda n: (n + 2 ** 63) % 2 ** 64 - 2 ** 63  # noqa: E731
    expected = [(7, signed(4 * offset + i)) for i in range(4)]
    assert _site_seeds((7, offset)) == expected
    assert [tuple(t.tolist()) for t in _site_seeds(torch.tensor([7, signed(offset)]))] == expected
    assert all(tk.check_dropout_support(E(4), 0.5, s, check_device=False).supported for s in expected)


@pytest.mark.parametrize("seed", [(1, 2, 3), "seed", 1.5, (1, 2 ** 64), (1, None), E(2), E(3, dt=I64), E(2, dt=I32), True])
def test_a_block_refuses_a_bad_seed(seed):
    from openfold3_triangle_kernel_b200.pair_block import pair_stack_block
    with pytest.raises(ValueError, match=r"pair_stack_block unsupported \[seed\]"):
        pair_stack_block(E(1, 4, 4, 32, dt=BF), E(1, 4, 4), {}, 2, dropout=0.1, seed=seed)


def test_public_names():
    """What the documents call is there; blocks of a stack that share a seed and count their offsets share no mask."""
    from openfold3_triangle_kernel_b200 import pair_block
    assert all(hasattr(tk, name) for name in tk.__all__) and tk.pair_stack_block is pair_block.pair_stack_block
    assert "pair_stack_block" in tk.__all__
    assert len({s for n in range(48) for s in pair_block._site_seeds((5, n))}) == 4 * 48


def test_rotary_sizes():
    """What no launch takes is refused by the check.  (Expanded tensors of any size need no memory.)"""
    big = lambda *s: E(1, dt=BF).expand(*s)  # noqa: E731
    one = lambda *s: tk.check_rotary_support(big(*s), _fr(2), check_device=False).code  # noqa: E731
    both = lambda n, h, hk: tk.check_qk_norm_rotary_support(big(n, h, 2), big(n, hk, 2), None, None, _fr(2), check_device=False).code  # noqa: E731
    assert one(2 ** 24, 127, 2) == one(1, 2 ** 24 - 1, 2) == both(1, 2 ** 24 - 2, 1) == both(100, 8, 2) == "ok"
    assert one(2 ** 24, 128, 2) == one(1, 2 ** 24, 2) == both(1, 2 ** 23, 2 ** 23) == "tokens"

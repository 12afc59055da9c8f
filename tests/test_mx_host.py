"""The microscaled operators' host side, on the CPU: what the C ABI and the Python functions refuse before any device
work, and the sizes of workspaces."""
import ctypes

import pytest
import torch

import mlxq
from mlxq import _lib

P = 4096  # any aligned address: nothing below gets as far as reading it
R = lambda x: None if x is None else ctypes.byref(x)  # noqa: E731


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def _mx(K=128, format=1, **kw):
    f = dict(codes=P, scales=P, scale_stride=-(-K // 128) * 4, format=format)
    f.update(kw)
    return _lib.Mx(*(f[n] for n, _ in _lib.Mx._fields_))


def _heads(heads=1, D=128, **kw):
    f = dict(data=P, heads=heads, token_stride=heads * D, head_stride=D)
    f.update(kw)
    return _lib.Heads(*(f[n] for n, _ in _lib.Heads._fields_))


def _router(**kw):
    f = dict(scoring=0, top_k=2, bias=None, groups=1, kept_groups=1, group_best=1, normalize=1, scale=1.0)
    f.update(kw)
    return _lib.Router(*(f[n] for n, _ in _lib.Router._fields_))


def _routing(**kw):
    f = dict(ids=P, weights=P, starts=P, rows=P, tokens=4, top_k=2, experts=8)
    f.update(kw)
    return _lib.Routed(*(f[n] for n, _ in _lib.Routed._fields_))


def _refused(lib, msg, call, status=_lib.MLXQ_EINVAL):
    assert call() == status
    assert msg in lib.mlxq_last_error().decode()


@pytest.mark.parametrize("msg,kw", [
    ("dtype 7", dict(dtype=7)), ("rows=-1", dict(rows=-1)), ("K=0", dict(K=0)), ("K=48", dict(K=48)), ("out is null", dict(out=None)),
    ("format 2", dict(out=_mx(format=2))), ("out must be 16", dict(out=_mx(codes=P + 8))), ("scales of out", dict(out=_mx(scales=P + 2))),
    ("scale_stride", dict(out=_mx(scale_stride=3))), ("scale_stride", dict(out=_mx(scale_stride=6))), ("x is null", dict(x=None)),
    ("x must be 16", dict(x=P + 4)), ("rows of x", dict(stride=130)),
])
def test_quantize_refusals(lib, msg, kw):
    a = dict(x=P, dtype=1, rows=4, K=128, stride=128, out=_mx())
    a.update(kw)
    _refused(lib, msg, lambda: lib.mlxq_mx_quantize(a["x"], a["dtype"], a["rows"], a["K"], a["stride"], R(a["out"]), None))


@pytest.mark.parametrize("msg,status,kw", [
    ("M=-1", 1, dict(M=-1)), ("N=-3", 1, dict(N=-3)), ("K=33", 1, dict(K=33)), ("x is null", 1, dict(x=None)), ("w is null", 1, dict(w=None)),
    ("format -1", 1, dict(x=_mx(format=-1))), ("weights must be e2m1", 2, dict(w=_mx(format=1))), ("y_dtype 5", 1, dict(y_dtype=5)),
    ("bias_dtype 3", 1, dict(bias=P, bias_dtype=3)), ("bias must be 4", 1, dict(bias=P + 2, bias_dtype=0)), ("y is null", 1, dict(y=None)),
    ("y must be 2", 1, dict(y=P + 1)), ("scale_stride", 1, dict(w=_mx(format=0, scale_stride=2))),
])
def test_matmul_refusals(lib, msg, status, kw):
    a = dict(x=_mx(), M=4, K=128, w=_mx(format=0), N=16, bias=None, bias_dtype=0, y=P, y_dtype=1)
    a.update(kw)
    _refused(lib, msg, lambda: lib.mlxq_mx_matmul(R(a["x"]), a["M"], a["K"], R(a["w"]), a["N"], a["bias"], a["bias_dtype"], a["y"], a["y_dtype"],
                                                 None), status)


@pytest.mark.parametrize("msg,status,kw", [
    ("dtype 9", 1, dict(dtype=9)), ("x is null", 1, dict(x=None)), ("0 heads", 1, dict(x=_heads(0))), ("D=0", 1, dict(D=0)), ("past 32768", 2, dict(D=32800)),
    ("tokens", 1, dict(T=-1)), ("eps=-1", 1, dict(eps=-1.0)), ("eps=nan", 1, dict(eps=float("nan"))), ("weight_dtype 4", 1, dict(w=P, w_dtype=4)),
    ("weight must be 2", 1, dict(w=P + 1, w_dtype=1)), ("one of y and y_mx", 1, dict(y=None)), ("one of y and y_mx", 1, dict(mx=_mx())),
    ("come together", 1, dict(residual=_heads())), ("come together", 1, dict(total=_heads())), ("y has 2 heads", 1, dict(y=_heads(2))),
    ("x must be 2", 1, dict(x=_heads(data=P + 1))), ("overlap", 1, dict(y=_heads(token_stride=127, data=2 * P))),
    ("in place", 1, dict(y=_heads(token_stride=256))), ("in place", 1, dict(residual=_heads(data=2 * P), total=_heads(token_stride=256))),
    ("not the sum", 1, dict(residual=_heads(data=2 * P), total=_heads(data=3 * P), y=_heads(data=3 * P))),
    ("e4m3", 2, dict(y=None, mx=_mx(format=0))), ("multiple of 32", 1, dict(y=None, mx=_mx(), D=100)),
])
def test_norm_refusals(lib, msg, status, kw):
    a = dict(x=_heads(), dtype=1, T=4, D=128, residual=None, total=None, w=None, w_dtype=0, eps=1e-6, y=_heads(data=8 * P), mx=None)
    a.update(kw)
    if "in place" in msg and "y" in kw:
        a["y"].data = a["x"].data
    if "in place" in msg and "total" in kw:
        a["total"].data = a["x"].data
    _refused(lib, msg, lambda: lib.mlxq_rms_norm(R(a["x"]), a["dtype"], a["T"], a["D"], R(a["residual"]), R(a["total"]), a["w"], a["w_dtype"],
                                                a["eps"], R(a["y"]), R(a["mx"]), None), status)


@pytest.mark.parametrize("msg,kw", [
    ("come together", dict(w=P, dw=None)), ("come together", dict(w=None, dw=P)), ("dy is null", dict(dy=None)), ("dx is null", dict(dx=None)),
    ("workspace of 0", dict(ws=0)), ("workspace must be 16", dict(ws_at=P + 8)), ("dweight must be 2", dict(dw=P + 1)), ("is not x", dict(dx=_heads())),
    ("in place", dict(dx=_heads(data=2 * P, token_stride=200))), ("in place", dict(dsum=_heads(data=6 * P, token_stride=200), dx=_heads(data=6 * P))),
    ("overlap", dict(dx=_heads(data=7 * P, token_stride=64))),
])
def test_norm_gradient_refusals(lib, msg, kw):
    need = lib.mlxq_rms_norm_backward_workspace_size(4, 1, 128, 1)
    assert need > 0
    a = dict(dy=_heads(data=2 * P), x=_heads(), w=P, dsum=None, dx=_heads(data=3 * P), dw=P, ws=need, ws_at=P)
    a.update(kw)
    _refused(lib, msg, lambda: lib.mlxq_rms_norm_backward(R(a["dy"]), R(a["x"]), 1, 4, 128, a["w"], 1, R(a["dsum"]), 1e-6, R(a["dx"]), a["dw"],
                                                         a["ws_at"], a["ws"], None))


@pytest.mark.parametrize("msg,status,kw", [
    ("routing is null", 1, dict(out=None)), ("0 experts", 1, dict(out=_routing(experts=0))), ("1025 experts", 2, dict(out=_routing(experts=1025))),
    ("top_k=0", 1, dict(out=_routing(top_k=0))), ("top_k=65", 2, dict(out=_routing(top_k=65))), ("-1 tokens", 1, dict(out=_routing(tokens=-1))),
    ("ids is null", 1, dict(out=_routing(ids=None))), ("weights is null", 1, dict(out=_routing(weights=None))), ("starts is null", 1, dict(out=_routing(starts=None))),
    ("rows must be 4", 1, dict(out=_routing(rows=P + 2))), ("router is null", 1, dict(router=None)), ("scoring 2", 1, dict(router=_router(scoring=2))),
    ("scale=inf", 1, dict(router=_router(scale=float("inf")))), ("top_k of router", 1, dict(router=_router(top_k=3))),
    ("8 experts in 3 groups", 1, dict(router=_router(groups=3))), ("in 0 groups", 1, dict(router=_router(groups=0))),
    ("kept_groups=3", 1, dict(router=_router(groups=2, kept_groups=3))), ("group_best=3", 1, dict(router=_router(group_best=3))),
    ("in the kept groups", 1, dict(router=_router(groups=8))), ("bias must be 4", 1, dict(router=_router(bias=P + 1))), ("logits is null", 1, dict(logits=None)),
    ("dtype 8", 1, dict(dtype=8)), ("workspace of 0 bytes", 1, dict(out=_routing(tokens=100000))),
])
def test_route_refusals(lib, msg, status, kw):
    a = dict(logits=P, dtype=1, router=_router(), out=_routing())
    a.update(kw)
    _refused(lib, msg, lambda: lib.mlxq_route_experts(a["logits"], a["dtype"], 8, R(a["router"]), None, R(a["out"]), None, 0, None), status)


@pytest.mark.parametrize("msg,status,kw", [
    ("K=40", 1, dict(K=40)), ("N=-1", 1, dict(N=-1)), ("weights must be e2m1", 2, dict(w=_mx())), ("y is null", 1, dict(y=None)),
    ("weights is null", 1, dict(routing=_routing(weights=None), combine=1)), ("workspace of 0", 1, dict(combine=1)), ("starts is null", 1, dict(routing=_routing(starts=None))),
    ("bias_dtype 6", 1, dict(bias=P, bias_dtype=6)), ("y_dtype 4", 1, dict(y_dtype=4)),
])
def test_experts_refusals(lib, msg, status, kw):
    a = dict(x=_mx(), K=128, w=_mx(format=0), N=16, bias=None, bias_dtype=0, routing=_routing(), combine=0, y=P, y_dtype=1)
    a.update(kw)
    _refused(lib, msg, lambda: lib.mlxq_mx_experts(R(a["x"]), 0, a["K"], R(a["w"]), a["N"], a["bias"], a["bias_dtype"], R(a["routing"]), a["combine"],
                                                  a["y"], a["y_dtype"], None, 0, None), status)


def test_nothing_to_do_is_no_error(lib):
    """No rows, no tokens: MLXQ_OK without a pointer to follow (what would write a plan or a weight's gradient is not called)."""
    none = _mx(codes=None, scales=None)
    assert lib.mlxq_mx_quantize(None, 1, 0, 128, 128, R(none), None) == 0
    assert lib.mlxq_mx_dequantize(R(none), 0, 128, None, 1, None) == 0
    assert lib.mlxq_mx_matmul(R(none), 0, 128, R(_mx(format=0)), 16, None, 0, None, 1, None) == 0
    assert lib.mlxq_rms_norm(R(_heads(data=None)), 1, 0, 128, None, None, None, 0, 1e-6, R(_heads(data=None)), None, None) == 0
    assert lib.mlxq_route_experts_backward(None, None, 1, 8, R(_router()), R(_routing(tokens=0, ids=None)), None, None) == 0


def test_workspace_sizes(lib):
    """They follow sizes, saturate at 0 for what the call refuses, and hold what the kernels lay out in them."""
    assert lib.mlxq_route_workspace_size(2048, 128) == 0 and lib.mlxq_route_workspace_size(0, 8) == 0
    for n in (2049, 65536, 65537, 10 ** 6, 2 ** 31 - 2 ** 20 - 1):
        segments = lib.mlxq_route_workspace_size(n, 128) // (129 * 4)
        assert 0 < segments <= 256 and lib.mlxq_route_workspace_size(n, 128) == segments * 129 * 4
    assert lib.mlxq_route_workspace_size(5000, 2000) == 0
    assert lib.mlxq_mx_experts_workspace_size(10, 4, 100, 0, 1) == 0
    assert lib.mlxq_mx_experts_workspace_size(10, 4, 100, 1, 1) == 10 * 4 * 100 * 2
    assert lib.mlxq_mx_experts_workspace_size(10, 4, 100, 1, 0) == 10 * 4 * 100 * 4
    assert lib.mlxq_mx_experts_workspace_size(2 ** 20, 64, 2 ** 20, 1, 0) == 2 ** 48
    for args in ((0, 1, 64, 1), (4, 0, 64, 1), (4, 1, 0, 1), (4, 1, 40000, 1), (2 ** 40, 1, 64, 1)):
        assert lib.mlxq_rms_norm_backward_workspace_size(*args) == 0
    for rows, D in ((1, 64), (10 ** 6, 64), (10 ** 6, 5000)):
        need = lib.mlxq_rms_norm_backward_workspace_size(rows, 1, D, 1)
        assert need % (4 * D) == 0 and 1 <= need // (4 * D) <= min(rows, 1024)


def _bad(msg, f, *a, **kw):
    with pytest.raises((mlxq.MlxqError, ValueError), match=msg):
        f(*a, **kw)


def test_python_refusals():
    z = torch.zeros
    x = mlxq.Mx(z(3, 64, dtype=torch.float8_e4m3fn), z(3, 2, dtype=torch.uint8))
    w = mlxq.Mx(z(5, 32, dtype=torch.uint8), z(5, 2, dtype=torch.uint8))
    _bad("GPU tensors", mlxq.mx_quantize, z(3, 64))
    _bad("format must be", mlxq.mx_quantize, z(3, 64), "e5m2")
    _bad("multiple of 32", mlxq.mx_quantize, z(3, 40))
    _bad("must be bfloat16", mlxq.mx_quantize, z(3, 64, dtype=torch.float64))
    _bad("GPU tensors", mlxq.mx_dequantize, x)
    _bad("dtype must be", mlxq.mx_dequantize, x, torch.int32)
    _bad("do not belong", mlxq.mx_dequantize, mlxq.Mx(x.codes, x.scales[:2]))
    _bad("one is needed for 32", mlxq.mx_dequantize, mlxq.Mx(x.codes, z(3, 4, dtype=torch.uint8)))
    _bad("uint8 or float8", mlxq.mx_dequantize, mlxq.Mx(z(3, 64), x.scales))
    _bad("GPU tensors", mlxq.mx_matmul, x, w)
    _bad("w must be", mlxq.mx_matmul, x, mlxq.Mx(z(5, 16, dtype=torch.uint8), z(5, 1, dtype=torch.uint8)))
    _bad("w must be", mlxq.mx_matmul, x, mlxq.Mx(w.codes[None], w.scales[None]))
    _bad("bias must be", mlxq.mx_matmul, x, w, z(4))
    _bad("out_dtype must be", mlxq.mx_matmul, x, w, None, torch.float64)
    _bad("GPU tensors", mlxq.rms_norm, z(3, 64))
    _bad("weight must be", mlxq.rms_norm, z(3, 64), z(63))
    _bad("residual must be", mlxq.rms_norm, z(3, 64), None, z(2, 64))
    _bad("residual must be", mlxq.rms_norm, z(3, 64), None, z(3, 64, dtype=torch.bfloat16))
    _bad("multiple of 32", mlxq.rms_norm, z(3, 65), mx=True)
    _bad("x must be", mlxq.rms_norm, z(3, 64, dtype=torch.int32))
    _bad("must be positive", mlxq.rms_norm, z(3, 0))
    _bad("last dimension", mlxq.rms_norm, torch.tensor(1.0))
    _bad("dy must be", mlxq.rms_norm_backward, z(2, 64), z(3, 64))
    _bad("dsum must be", mlxq.rms_norm_backward, z(3, 64), z(3, 64), None, z(3, 32))
    _bad("scoring must be", mlxq.route_experts, z(3, 8), 2, "relu")
    _bad("logits must be", mlxq.route_experts, z(8), 2)
    _bad("bias must be", mlxq.route_experts, z(3, 8), 2, bias=z(7))
    _bad("active must be", mlxq.route_experts, z(3, 8), 2, active=z(3))
    _bad("top_k=0", mlxq.route_experts, z(3, 8), 0)
    _bad("GPU tensors", mlxq.route_experts, z(3, 8), 2)
    ids, wt = z(3, 2, dtype=torch.int32), z(3, 2)
    _bad("ids must be", mlxq.route_plan, ids.long(), wt, 8)
    _bad("weights must be", mlxq.route_plan, ids, wt[:2], 8)
    _bad("GPU tensors", mlxq.route_plan, ids, wt, 8)
    _bad("dweights must be", mlxq.route_experts_backward, wt[:, :1], z(3, 8), ids)
    _bad("do not fit", mlxq.route_experts_backward, wt, z(4, 8), ids)
    stack = mlxq.Mx(z(8, 5, 32, dtype=torch.uint8), z(8, 5, 2, dtype=torch.uint8))
    routing = mlxq.Routing(ids, wt, z(9, dtype=torch.int32), z(6, dtype=torch.int32))
    _bad("w must be", mlxq.mx_experts, x, w, routing)
    _bad("x must be", mlxq.mx_experts, mlxq.Mx(x.codes[:2], x.scales[:2]), stack, routing)
    _bad("starts must be", mlxq.mx_experts, x, stack, routing._replace(starts=z(8, dtype=torch.int32)))
    _bad("rows must be", mlxq.mx_experts, x, stack, routing._replace(rows=z(6)))
    _bad("bias must be", mlxq.mx_experts, x, stack, routing, z(8, 4))
    _bad("GPU tensors", mlxq.mx_experts, x, stack, routing)


def test_row_strides():
    """The one stride of a tensor's rows, where there is one."""
    from mlxq.mx import _row_stride
    t = torch.zeros(4, 6, 40)
    for x, want in ((t, 40), (t[0], 40), (t[:, 0], 240), (t[:, 1:3], None), (t[:, :, :8], 40), (t[::2], None), (t[::2, 0], 480), (t[0, 0], 40),
                    (t.transpose(0, 1), None), (t[:1, :1], 40), (t[..., ::2], None), (t[:, :1].expand(4, 3, 40), None), (t[0, :1].expand(5, 40), 0)):
        assert _row_stride(x) == want, (x.shape, x.stride())

"""A decoder block in microscaled types: quantisation and products, norms, the routing of tokens to
experts and the experts' products.

The block's operators beside its affine packed projections (ops.py) and its attention (paged.py): `rms_norm`
adds the residual and writes the norm in 16 bits or as 8-bit microscaled activations, `mx_matmul` multiplies
those with 4-bit microscaled weights, `route_experts` chooses each token's experts and `mx_experts` runs
them.  They follow no call of the reference (mlx-gen-sensenova/src/qwen3.rs:178-181,
mlx-gen-lens/src/text_encoder/gpt_oss.rs:396-440), whose microscaled experts become affine packs.  As with
the other operators autograd records nothing by itself: `rms_norm_backward` and `route_experts_backward`
are the gradients.  include/mlxq.h has every operator's definition.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch

from . import _lib
from ._lib import MLXQ_MX_E2M1, MLXQ_MX_E4M3, MLXQ_ROUTE_SIGMOID, MLXQ_ROUTE_SOFTMAX, Heads, Routed, Router, check
from .ops import _bad, _dt, _dt_of, _need_gpu, _ptr, _stream

_SCORING = {"softmax": MLXQ_ROUTE_SOFTMAX, "sigmoid": MLXQ_ROUTE_SIGMOID}


class Mx(NamedTuple):
    """A microscaled tensor [..., K]: codes, e2m1 as uint8 [..., K/2] (two to a byte, the first in the low half) or
    float8_e4m3fn [..., K], and scales, uint8 [..., K/32] (2^(b - 127); 255: NaN), one for 32 values.  Scales
    whose rows do not start at multiples of 4 bytes (a checkpoint's, where K / 32 is no multiple of 4) are copied by each
    call that reads them; mx_quantize's and rms_norm's do.  A program that keeps such scales pads them once:
    Mx(codes, F.pad(scales, (0, -n % 4))[..., :n]) for scales [..., n]."""
    codes: torch.Tensor
    scales: torch.Tensor


class Routing(NamedTuple):
    """Where tokens go: ids (int32) and weights (f32) [T, top_k], and the plan of the experts' products (int32):
    rows [T * top_k], the choices t * top_k + j by expert, and starts [experts + 1], where each expert's begin."""
    ids: torch.Tensor
    weights: torch.Tensor
    starts: torch.Tensor
    rows: torch.Tensor


def _float(op, what, dtype):
    if dtype not in (torch.bfloat16, torch.float32, torch.float16):
        _bad(op, f"{what} must be bfloat16, float32 or float16, got {dtype}")


def _dense(t, align=16):
    t = t.contiguous()
    return t if t.data_ptr() % align == 0 else t.clone()


def _scales(lead, blocks, device):
    """Scales [*lead, blocks] whose rows start at multiples of 4 bytes."""
    return torch.empty((*lead, -(-blocks // 4) * 4), dtype=torch.uint8, device=device)[..., :blocks]


def _empty_mx(lead, K, format, device):
    codes = torch.empty((*lead, K // 2), dtype=torch.uint8, device=device) if format == MLXQ_MX_E2M1 else \
        torch.empty((*lead, K), dtype=torch.float8_e4m3fn, device=device)
    return Mx(codes, _scales(lead, K // 32, device))


def _row_stride(t):
    """The stride between the rows (last dimension: contiguous) of t, if there is one for all of them."""
    if t.numel() == 0:
        return t.shape[-1]
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        return None
    stride = rows = None
    for n, s in zip(reversed(t.shape[:-1]), reversed(t.stride()[:-1])):
        if n == 1:
            continue
        if stride is None:
            stride, rows = s, n
        elif s != stride * rows:
            return None
        else:
            rows *= n
    return t.shape[-1] if stride is None else stride


def _view(op, what, x):
    """(the struct the library reads, K, tensors to keep) of a microscaled tensor."""
    codes, scales = x
    if codes.dtype not in (torch.uint8, torch.float8_e4m3fn) or scales.dtype != torch.uint8:
        _bad(op, f"{what} must be (codes, scales) of uint8 or float8_e4m3fn and uint8, got {codes.dtype} and {scales.dtype}")
    if codes.dim() < 1 or codes.shape[:-1] != scales.shape[:-1] or codes.device != scales.device:
        _bad(op, f"codes {tuple(codes.shape)} and scales {tuple(scales.shape)} of {what} do not belong together")
    K = codes.shape[-1] * (2 if codes.dtype == torch.uint8 else 1)
    if K % 32 or scales.shape[-1] * 32 != K or K == 0:
        _bad(op, f"{what} has {K} values and {scales.shape[-1]} scales a row: one is needed for 32")
    codes = _dense(codes)
    stride = _row_stride(scales)
    rows = codes.numel() // codes.shape[-1]
    if stride is None or scales.data_ptr() % 4 or (rows > 1 and (stride % 4 or stride < K // 32)):
        copy = _scales(scales.shape[:-1], K // 32, scales.device)
        copy.copy_(scales)
        scales, stride = copy, -(-(K // 32) // 4) * 4
    if rows <= 1:
        stride = -(-(K // 32) // 4) * 4
    return _lib.Mx(codes.data_ptr(), scales.data_ptr(), stride,
                   MLXQ_MX_E2M1 if codes.dtype == torch.uint8 else MLXQ_MX_E4M3), K, (codes, scales)


def _bias(op, bias, shape, device):
    if bias is None:
        return None, 0
    _float(op, "bias", bias.dtype)
    if tuple(bias.shape) != tuple(shape) or bias.device != device:
        _bad(op, f"bias must be {tuple(shape)} on {device}, got {tuple(bias.shape)} on {bias.device}")
    bias = bias.contiguous()
    return bias, _dt(bias)


def _workspace(need, device):
    return torch.empty((need,), dtype=torch.uint8, device=device) if need else None


def mx_quantize(x, format: str = "e2m1") -> Mx:
    """x [..., K] (bf16, f32 or fp16; K a multiple of 32) to microscaled "e2m1" or "e4m3": each 32 values are divided by
    the smallest power of two that leaves none past the code's largest, and rounded to nearest."""
    op = "mx_quantize"
    if format not in ("e2m1", "e4m3"):
        _bad(op, f"format must be 'e2m1' or 'e4m3', got {format!r}")
    _float(op, "x", x.dtype)
    K = x.shape[-1] if x.dim() else 0
    if K == 0 or K % 32:
        _bad(op, f"the last dimension of x, {K}, must be a positive multiple of 32")
    y = _lib.fast().mx_quantize(x, format == "e4m3")
    if y is not None:
        return Mx(*y)
    stride, C = _row_stride(x), 16 // x.element_size()
    if stride is None or stride % C or x.data_ptr() % 16:
        x, stride = _dense(x), K
    _need_gpu(x)
    fmt = MLXQ_MX_E2M1 if format == "e2m1" else MLXQ_MX_E4M3
    out = _empty_mx(x.shape[:-1], K, fmt, x.device)
    rows = x.numel() // K
    view = _lib.Mx(out.codes.data_ptr(), out.scales.data_ptr(), -(-(K // 32) // 4) * 4, fmt)
    check(_lib.load().mlxq_mx_quantize(_ptr(x), _dt(x), rows, K, stride, ctypes.byref(view), _stream(x.device)))
    return out


def mx_dequantize(x: Mx, dtype=torch.bfloat16):
    """What x stands for, [..., K] in dtype."""
    op = "mx_dequantize"
    _float(op, "dtype", dtype)
    y = _lib.fast().mx_dequantize(x, _dt_of(dtype))
    if y is not None:
        return y
    view, K, keep = _view(op, "x", x)
    _need_gpu(*keep)
    codes = keep[0]
    out = torch.empty((*codes.shape[:-1], K), dtype=dtype, device=codes.device)
    check(_lib.load().mlxq_mx_dequantize(ctypes.byref(view), out.numel() // K, K, _ptr(out), _dt(out), _stream(codes.device)))
    return out


def mx_matmul(x: Mx, w: Mx, bias=None, out_dtype=torch.bfloat16):
    """x [..., K] . w^T + bias for w [N, K] e2m1: [..., N] in out_dtype.  x in either format; bias [N] in any of the
    three dtypes.  Sums are f32, rounded once, but for e4m3 rows with a bf16 result: the matrix cores then lose up to
    7 2^-13 of the largest of every eight neighbouring products (less than half a rounding to bf16 of a result that does
    not cancel).  out_dtype float32 or float16 asks for f32 sums."""
    op = "mx_matmul"
    _float(op, "out_dtype", out_dtype)
    y = _lib.fast().mx_matmul(x, w, bias, _dt_of(out_dtype))
    if y is not None:
        return y
    xv, K, keep_x = _view(op, "x", x)
    wv, Kw, keep_w = _view(op, "w", w)
    codes, wcodes = keep_x[0], keep_w[0]
    if wcodes.dim() != 2 or Kw != K or wcodes.device != codes.device:
        _bad(op, f"w must be [N, {K}] on {codes.device}, got {tuple(wcodes.shape[:-1])} rows of {Kw} on {wcodes.device}")
    N = wcodes.shape[0]
    bias, bias_dt = _bias(op, bias, (N,), codes.device)
    _need_gpu(codes, wcodes)
    out = torch.empty((*codes.shape[:-1], N), dtype=out_dtype, device=codes.device)
    M = codes.numel() // codes.shape[-1]
    check(_lib.load().mlxq_mx_matmul(ctypes.byref(xv), M, K, ctypes.byref(wv), N, _ptr(bias), bias_dt, _ptr(out), _dt(out),
                                     _stream(codes.device)))
    del keep_x, keep_w
    return out


# ---- norms -----------------------------------------------------------------------------------------


def _rows(op, what, t, like=None):
    """A [..., D] tensor as [tokens, heads, D] with the library's two strides: as it lies where it can be, else a copy."""
    if t.dim() < 1:
        _bad(op, f"{what} must have a last dimension")
    if like is not None and (t.shape != like.shape or t.dtype != like.dtype or t.device != like.device):
        _bad(op, f"{what} must be {like.dtype} of {tuple(like.shape)} on {like.device}, got {t.dtype} of {tuple(t.shape)} on {t.device}")
    if t.numel() == 0:  # nothing is read, whichever dimension is empty
        return t, (0, t.shape[-2] if t.dim() > 2 else 1, 0, 0)
    for turn in range(2):
        if t.shape[-1] == 1 or t.stride(-1) == 1:
            if t.dim() <= 2:
                return t, (t.shape[0] if t.dim() == 2 else 1, 1, t.stride(0) if t.dim() == 2 else t.shape[-1], 0)
            stride = _row_stride(t[..., 0, :])
            if stride is not None:
                tokens = t.numel() // (t.shape[-1] * t.shape[-2])
                return t, (tokens, t.shape[-2], stride if t.dim() > 2 else 0, t.stride(-2))
        t = t.contiguous()
    raise AssertionError(f"{op}: no strides for {what}")


def _heads_of(t, shape):
    return Heads(t.data_ptr(), shape[1], shape[2], shape[3])


def _norm_weight(op, weight, x):
    if weight is None:
        return None, 0
    _float(op, "weight", weight.dtype)
    if tuple(weight.shape) != (x.shape[-1],) or weight.device != x.device:
        _bad(op, f"weight must be [{x.shape[-1]}] on {x.device}, got {tuple(weight.shape)} on {weight.device}")
    weight = weight.contiguous()
    return weight, _dt(weight)


def rms_norm(x, weight=None, residual=None, eps: float = 1e-6, mx: bool = False):
    """The root-mean-square norm of x [..., D] over its last dimension, times weight [D]: in x's dtype, or with mx as
    e4m3 microscaled activations (Mx; D a multiple of 32).  With a residual the norm is that of x + residual,
    rounded to x's dtype, and (norm, x + residual) is returned.  D up to 32768."""
    op = "rms_norm"
    y = _lib.fast().rms_norm(x, weight, residual, eps, mx)
    if y is not None:
        if mx:
            y = (Mx(*y[:2]), *y[2:]) if residual is not None else Mx(*y)
        return y
    _float(op, "x", x.dtype)
    x, xs = _rows(op, "x", x)
    D = x.shape[-1]
    weight, w_dt = _norm_weight(op, weight, x)
    r = rs = total = None
    if residual is not None:
        r, rs = _rows(op, "residual", residual, like=x)
        if rs[:2] != xs[:2]:
            r, rs = _rows(op, "residual", r.contiguous())
        total = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    if D == 0 or (mx and D % 32):
        _bad(op, f"the last dimension of x, {D}, must be positive" + (" and a multiple of 32" if mx else ""))
    _need_gpu(x, weight, r)
    T, H = xs[:2]
    plain = (T, H, H * D, D)
    out = _empty_mx(x.shape[:-1], D, MLXQ_MX_E4M3, x.device) if mx else torch.empty(x.shape, dtype=x.dtype, device=x.device)
    if x.numel():
        xv = _heads_of(x, xs)
        rv, tv = (_heads_of(r, rs), _heads_of(total, plain)) if r is not None else (None, None)
        yv = None if mx else _heads_of(out, plain)
        mv = _lib.Mx(out.codes.data_ptr(), out.scales.data_ptr(), -(-(D // 32) // 4) * 4, MLXQ_MX_E4M3) if mx else None
        at = lambda v: None if v is None else ctypes.byref(v)  # noqa: E731
        check(_lib.load().mlxq_rms_norm(at(xv), _dt(x), T, D, at(rv), at(tv), _ptr(weight), w_dt, eps, at(yv), at(mv),
                                        _stream(x.device)))
    return out if residual is None else (out, total)


def rms_norm_backward(dy, x, weight=None, dsum=None, eps: float = 1e-6):
    """(dx, dweight) from the gradient dy of rms_norm's result: x is what was normed (x + residual where there was one;
    dx is then the gradient of both), dsum the gradient that arrives at it from elsewhere.  dweight is None without a
    weight."""
    op = "rms_norm_backward"
    y = _lib.fast().rms_norm_backward(dy, x, weight, dsum, eps)
    if y is not None:
        return y
    _float(op, "x", x.dtype)
    x, xs = _rows(op, "x", x)
    D = x.shape[-1]
    if D == 0:
        _bad(op, "the last dimension of x must be positive")
    weight, w_dt = _norm_weight(op, weight, x)
    views = []
    for what, t in (("dy", dy), ("dsum", dsum)):
        if t is None:
            views.append((None, None))
            continue
        t, s = _rows(op, what, t, like=x)
        if s[:2] != xs[:2]:
            t, s = _rows(op, what, t.contiguous())
        views.append((t, s))
    (dy, ys), (dsum, ds) = views
    _need_gpu(x, dy, weight, dsum)
    T, H = xs[:2]
    dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    dw = None if weight is None else torch.empty_like(weight)
    if x.numel() == 0:
        return dx, None if dw is None else dw.zero_()
    lib = _lib.load()
    need = lib.mlxq_rms_norm_backward_workspace_size(T, H, D, _dt(x)) if weight is not None else 0
    ws = _workspace(need, x.device)
    dsv = None if dsum is None else _heads_of(dsum, ds)
    check(lib.mlxq_rms_norm_backward(ctypes.byref(_heads_of(dy, ys)), ctypes.byref(_heads_of(x, xs)), _dt(x), T, D, _ptr(weight), w_dt,
                                     None if dsv is None else ctypes.byref(dsv), eps,
                                     ctypes.byref(_heads_of(dx, (T, H, H * D, D))), _ptr(dw), _ptr(ws), need, _stream(x.device)))
    return dx, dw


# ---- experts ---------------------------------------------------------------------------------------


def _logits(op, logits):
    _float(op, "logits", logits.dtype)
    if logits.dim() != 2:
        _bad(op, f"logits must be [tokens, experts], got {tuple(logits.shape)}")
    if logits.numel() and logits.stride(1) != 1 and logits.shape[1] > 1:
        logits = logits.contiguous()
    return logits


def _router(op, scoring, top_k, normalize, scale):
    if scoring not in _SCORING:
        _bad(op, f"scoring must be 'softmax' or 'sigmoid', got {scoring!r}")
    return Router(_SCORING[scoring], top_k, None, 1, 1, 1, int(normalize), scale)


def _routed(routing, T, k, E):
    return Routed(*(None if t is None else t.data_ptr() for t in routing), T, k, E)


def route_experts(logits, top_k: int, scoring: str = "softmax", bias=None, groups: int = 1, kept_groups: int = 1,
                  group_best: int = 1, normalize: bool = True, scale: float = 1.0, active=None) -> Routing:
    """Each token's top_k experts by its logits [T, experts], and the plan of their products.

    Scores are softmax(logits) or sigmoid(logits); the experts with the largest score + bias [experts] (f32, for the
    choice only) are taken, best first, the lowest first among equal ones.  With groups (equal runs of experts) only
    those of the kept_groups best are, by the sum of a group's group_best (1 or 2) best.  Weights are the chosen scores,
    divided by their sum when normalize, times scale.  Tokens whose active [T] (bool) is False get ids -1 and weights 0.
    NaN logits come last; a softmax's row with NaN or +infinity is chosen by its logits alone and has NaN weights."""
    op = "route_experts"
    y = _lib.fast().route_experts(logits, top_k, scoring, bias, groups, kept_groups, group_best, normalize, scale, active)
    if y is not None:
        return Routing(*y)
    logits = _logits(op, logits)
    T, E = logits.shape
    router = _router(op, scoring, top_k, normalize, scale)
    router.groups, router.kept_groups, router.group_best = groups, kept_groups, group_best
    if bias is not None:
        if bias.dtype != torch.float32 or tuple(bias.shape) != (E,) or bias.device != logits.device:
            _bad(op, f"bias must be float32 [{E}] on {logits.device}, got {bias.dtype} {tuple(bias.shape)} on {bias.device}")
        bias = bias.contiguous()
        router.bias = bias.data_ptr()
    if active is not None:
        if active.dtype != torch.bool or tuple(active.shape) != (T,) or active.device != logits.device:
            _bad(op, f"active must be bool [{T}] on {logits.device}, got {active.dtype} {tuple(active.shape)} on {active.device}")
        active = active.contiguous()
    if top_k < 1 or E < 1:
        _bad(op, f"top_k={top_k} of {E} experts")
    _need_gpu(logits)
    d = logits.device
    ints = lambda *n: torch.empty(n, dtype=torch.int32, device=d)  # noqa: E731
    out = Routing(ints(T, top_k), torch.empty((T, top_k), dtype=torch.float32, device=d), ints(E + 1), ints(T * top_k))
    lib = _lib.load()
    need = lib.mlxq_route_workspace_size(T * top_k, E)
    ws = _workspace(need, d)
    check(lib.mlxq_route_experts(_ptr(logits), _dt(logits), logits.stride(0), ctypes.byref(router), _ptr(active),
                                 ctypes.byref(_routed(out, T, top_k, E)), _ptr(ws), need, _stream(d)))
    return out


def _ids(op, ids):
    if ids.dtype != torch.int32 or ids.dim() != 2:
        _bad(op, f"ids must be int32 [tokens, top_k], got {ids.dtype} {tuple(ids.shape)}")
    return ids.contiguous()


def route_plan(ids, weights, experts: int) -> Routing:
    """The Routing of ids [T, top_k] (int32; one outside [0, experts) has no expert) and weights [T, top_k] that a router of
    one's own made."""
    op = "route_plan"
    ids = _ids(op, ids)
    if weights.dtype != torch.float32 or weights.shape != ids.shape or weights.device != ids.device:
        _bad(op, f"weights must be float32 {tuple(ids.shape)} on {ids.device}, got {weights.dtype} {tuple(weights.shape)} on "
                 f"{weights.device}")
    T, k = ids.shape
    if experts < 1 or k < 1:
        _bad(op, f"{k} choices of {experts} experts")
    _need_gpu(ids)
    out = Routing(ids, weights.contiguous(), torch.empty((experts + 1,), dtype=torch.int32, device=ids.device),
                  torch.empty((T * k,), dtype=torch.int32, device=ids.device))
    lib = _lib.load()
    need = lib.mlxq_route_workspace_size(T * k, experts)
    ws = _workspace(need, ids.device)
    check(lib.mlxq_route_plan(ctypes.byref(_routed(out, T, k, experts)), _ptr(ws), need, _stream(ids.device)))
    return out


def route_experts_backward(dweights, logits, ids, scoring: str = "softmax", normalize: bool = True, scale: float = 1.0):
    """The gradient of the logits, in their dtype, from that of route_experts' weights [T, top_k] (f32), for the choice ids
    (no expert twice in a row; an id outside the experts passes nothing on, and a token without any has a gradient of 0)."""
    op = "route_experts_backward"
    y = _lib.fast().route_experts_backward(dweights, logits, ids, scoring, normalize, scale)
    if y is not None:
        return y
    logits, ids = _logits(op, logits), _ids(op, ids)
    (T, E), k = logits.shape, ids.shape[1]
    if ids.shape[0] != T or ids.device != logits.device or k < 1 or E < 1:
        _bad(op, f"ids {tuple(ids.shape)} on {ids.device} do not fit logits {tuple(logits.shape)} on {logits.device}")
    if dweights.dtype != torch.float32 or dweights.shape != ids.shape or dweights.device != ids.device:
        _bad(op, f"dweights must be float32 {tuple(ids.shape)} on {ids.device}, got {dweights.dtype} {tuple(dweights.shape)} on "
                 f"{dweights.device}")
    dweights = dweights.contiguous()
    _need_gpu(logits)
    out = torch.empty((T, E), dtype=logits.dtype, device=logits.device)
    router = _router(op, scoring, k, normalize, scale)
    check(_lib.load().mlxq_route_experts_backward(_ptr(dweights), _ptr(logits), _dt(logits), logits.stride(0), ctypes.byref(router),
                                                  ctypes.byref(_routed((ids, None, None, None), T, k, E)), _ptr(out),
                                                  _stream(logits.device)))
    return out


def mx_experts(x: Mx, w: Mx, routing: Routing, bias=None, combine: bool = False, out_dtype=torch.bfloat16):
    """The products of the experts that tokens were routed to: x[t] . w[ids[t, j]]^T + bias[ids[t, j]], [T, top_k, N] in
    out_dtype, zero where ids names no expert; with combine their sum over j with the routing's weights, [T, N], of
    products that are rounded to out_dtype first, as separate products would be (float32 keeps them in f32).

    x [T, K], or [T, top_k, K] with a row for each choice, in either format; w [experts, N, K] e2m1; bias [experts, N]."""
    op = "mx_experts"
    _float(op, "out_dtype", out_dtype)
    y = _lib.fast().mx_experts(x, w, routing, bias, combine, _dt_of(out_dtype))
    if y is not None:
        return y
    xv, K, keep_x = _view(op, "x", x)
    wv, Kw, keep_w = _view(op, "w", w)
    codes, wcodes = keep_x[0], keep_w[0]
    device = codes.device
    ids, weights, starts, rows = routing
    ids = _ids(op, ids)
    T, k = ids.shape
    if wcodes.dim() != 3 or Kw != K or wcodes.device != device:
        _bad(op, f"w must be [experts, N, {K}] on {device}, got {tuple(wcodes.shape[:-1])} rows of {Kw} on {wcodes.device}")
    E, N = wcodes.shape[:2]
    if tuple(codes.shape[:-1]) not in ((T,), (T, k)):
        _bad(op, f"x must be [{T}, {K}] or [{T}, {k}, {K}], got rows {tuple(codes.shape[:-1])}")
    for what, t, shape, dtype in (("ids", ids, (T, k), torch.int32), ("weights", weights, (T, k), torch.float32),
                                  ("starts", starts, (E + 1,), torch.int32), ("rows", rows, (T * k,), torch.int32)):
        if t.dtype != dtype or tuple(t.shape) != shape or t.device != device:
            _bad(op, f"the routing's {what} must be {dtype} {shape} on {device}, got {t.dtype} {tuple(t.shape)} on {t.device}")
    weights, starts, rows = weights.contiguous(), starts.contiguous(), rows.contiguous()
    bias, bias_dt = _bias(op, bias, (E, N), device)
    _need_gpu(codes, wcodes)
    out = torch.empty((T, N) if combine else (T, k, N), dtype=out_dtype, device=device)
    if T == 0:
        return out
    lib = _lib.load()
    need = lib.mlxq_mx_experts_workspace_size(T, k, N, int(combine), _dt(out))
    ws = _workspace(need, device)
    check(lib.mlxq_mx_experts(ctypes.byref(xv), int(codes.dim() == 3), K, ctypes.byref(wv), N, _ptr(bias), bias_dt,
                              ctypes.byref(_routed((ids, weights, starts, rows), T, k, E)), int(combine), _ptr(out), _dt(out), _ptr(ws),
                              need, _stream(device)))
    del keep_x, keep_w
    return out

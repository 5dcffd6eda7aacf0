"""Projections with what follows them in one kernel: the ops behind lightning attention in a model block.

    linear_fn         y = act(x weight^T + bias) + residual
    gated_linear_fn   h = act(x w_gate^T + b_gate) * (x w_up^T + b_up)

x (..., K), weights (N, K) as torch.nn.Linear keeps them.  Products are accumulated in fp32 and rounded once, after
bias, activation, product of the pair and residual.  Gradients for every tensor given.  fp32 runs on the CUDA cores in
fp32; bf16 and fp16 on the tensor cores.  (The reference has the second projection of the pair as gate_linear,
xopes/ops/gate_linear, outside the attention path this library mirrors.)
"""
from typing import Optional

import torch

from . import _lib

_ACTS = {"none": 0, "relu": 1, "sigmoid": 2, "silu": 3, "gelu": 4}


def _rows(t):
    """t with its rows (last dimension) next to each other element by element and a common stride from row to row, and
    that stride; a copy where there is none."""
    f = t.shape[-1]
    if t.is_contiguous():
        return t, f
    try:
        t2 = t.view(-1, f)
    except RuntimeError:
        t2 = t.reshape(-1, f)
    if (t2.stride(1) != 1 and f > 1) or t2.stride(0) < f:
        t2 = t2.contiguous()
    return t2, max(t2.stride(0), f)


def _scratch(nbytes, device):
    if nbytes <= 0:
        if nbytes < 0:
            _lib.check(nbytes, "workspace size")
        return None
    return torch.empty(nbytes, dtype=torch.uint8, device=device)


def _linear_forward(x, weight, bias, residual, act, keep):
    """y and, to be kept for the backward, the pre-activations."""
    lib = _lib.load()
    k, n = x.shape[-1], weight.shape[0]
    m = x.numel() // k
    y = torch.empty((*x.shape[:-1], n), dtype=x.dtype, device=x.device)
    if m == 0:
        return y, None
    x2, ldx = _rows(x)
    w2, ldw = _rows(weight)
    r2, ldr = (None, 0) if residual is None else _rows(residual)
    b = None if bias is None else bias.contiguous()
    code = _lib.dtype_code(x)
    xp, wp = x2.data_ptr(), w2.data_ptr()
    with _lib.device_of(x):
        z = _scratch(lib.la_linear_saved_bytes(m, n, code, 0), x.device) if keep and act else None
        need = lib.la_linear_fwd_workspace_bytes(xp, ldx, wp, ldw, None, 0, m, n, k, code)
        ws = _scratch(need, x.device) if need else None
        rc = lib.la_linear_fwd(xp, ldx, wp, ldw, _lib.ptr(b), _lib.ptr(r2), ldr, y.data_ptr(), _lib.ptr(z), _lib.ptr(ws),
                               need, m, n, k, code, act, _lib.stream_of(x))
    if rc:
        _lib.check(rc, "la_linear_fwd")
    return y, z


class LinearFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act):
        y, z = _linear_forward(x, weight, bias, residual, act, True)
        ctx.save_for_backward(x, weight, z)
        ctx.act = act
        return y

    @staticmethod
    def backward(ctx, dy):
        _lib.once_differentiable()
        lib = _lib.load()
        x, weight, z = ctx.saved_tensors
        need_x, need_w, need_b, need_r, _ = ctx.needs_input_grad
        n, k = weight.shape
        m = x.numel() // k
        dx = torch.empty(x.shape, dtype=x.dtype, device=x.device) if need_x else None
        new = torch.empty if m else torch.zeros
        dw = new((n, k), dtype=x.dtype, device=x.device) if need_w else None
        db = new((n,), dtype=x.dtype, device=x.device) if need_b else None
        if m and (need_x or need_w or need_b):
            dy2, ldy = _rows(dy)
            x2, ldx = _rows(x)
            w2, ldw = _rows(weight)
            code = _lib.dtype_code(x)
            xp, wp, dyp = x2.data_ptr(), w2.data_ptr(), dy2.data_ptr()
            with _lib.device_of(x):
                need = lib.la_linear_bwd_workspace_bytes(xp, ldx, wp, ldw, None, 0, dyp, ldy, m, n, k, code, ctx.act, need_x,
                                                         need_w, need_b)
                ws = _scratch(need, x.device) if need else None
                rc = lib.la_linear_bwd(xp, ldx, wp, ldw, _lib.ptr(z), dyp, ldy, _lib.ptr(dx), _lib.ptr(dw), _lib.ptr(db),
                                       _lib.ptr(ws), need, m, n, k, code, ctx.act, _lib.stream_of(x))
            if rc:
                _lib.check(rc, "la_linear_bwd")
        return dx, dw, db, dy if need_r else None, None


def _gated_forward(x, w_gate, w_up, b_gate, b_up, act, keep):
    """h and, to be kept for the backward, both projections."""
    lib = _lib.load()
    k, n = x.shape[-1], w_gate.shape[0]
    m = x.numel() // k
    h = torch.empty((*x.shape[:-1], n), dtype=x.dtype, device=x.device)
    if m == 0:
        return h, None
    x2, ldx = _rows(x)
    (wg, ldg), (wu, ldu) = _rows(w_gate), _rows(w_up)
    bg, bu = None if b_gate is None else b_gate.contiguous(), None if b_up is None else b_up.contiguous()
    code = _lib.dtype_code(x)
    xp, gp, up = x2.data_ptr(), wg.data_ptr(), wu.data_ptr()
    with _lib.device_of(x):
        gu = _scratch(lib.la_linear_saved_bytes(m, n, code, 1), x.device) if keep else None
        need = lib.la_linear_fwd_workspace_bytes(xp, ldx, gp, ldg, up, ldu, m, n, k, code)
        ws = _scratch(need, x.device) if need else None
        rc = lib.la_gated_linear_fwd(xp, ldx, gp, ldg, up, ldu, _lib.ptr(bg), _lib.ptr(bu), h.data_ptr(), _lib.ptr(gu),
                                     _lib.ptr(ws), need, m, n, k, code, act, _lib.stream_of(x))
    if rc:
        _lib.check(rc, "la_gated_linear_fwd")
    return h, gu


class GatedLinearFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, b_gate, b_up, act):
        h, gu = _gated_forward(x, w_gate, w_up, b_gate, b_up, act, True)
        ctx.save_for_backward(x, w_gate, w_up, gu)
        ctx.act = act
        return h

    @staticmethod
    def backward(ctx, dh):
        _lib.once_differentiable()
        lib = _lib.load()
        x, w_gate, w_up, gu = ctx.saved_tensors
        need_x, need_wg, need_wu, need_bg, need_bu, _ = ctx.needs_input_grad
        need_w, need_b = need_wg or need_wu, need_bg or need_bu
        n, k = w_gate.shape
        m = x.numel() // k
        new = torch.empty if m else torch.zeros
        dx = torch.empty(x.shape, dtype=x.dtype, device=x.device) if need_x else None
        dwg, dwu = (new((n, k), dtype=x.dtype, device=x.device) if need_w else None for _ in range(2))
        dbg, dbu = (new((n,), dtype=x.dtype, device=x.device) if need else None for need in (need_bg, need_bu))
        if m and (need_x or need_w or need_b):
            dh2, ldh = _rows(dh)
            x2, ldx = _rows(x)
            (wg, ldg), (wu, ldu) = _rows(w_gate), _rows(w_up)
            code = _lib.dtype_code(x)
            xp, gp, up, dhp = x2.data_ptr(), wg.data_ptr(), wu.data_ptr(), dh2.data_ptr()
            with _lib.device_of(x):
                need = lib.la_linear_bwd_workspace_bytes(xp, ldx, gp, ldg, up, ldu, dhp, ldh, m, n, k, code, ctx.act, need_x,
                                                         need_w, need_b)
                ws = _scratch(need, x.device) if need else None
                rc = lib.la_gated_linear_bwd(xp, ldx, gp, ldg, up, ldu, _lib.ptr(gu), dhp, ldh, _lib.ptr(dx), _lib.ptr(dwg),
                                             _lib.ptr(dwu), _lib.ptr(dbg), _lib.ptr(dbu), _lib.ptr(ws), need, m, n, k, code,
                                             ctx.act, _lib.stream_of(x))
            if rc:
                _lib.check(rc, "la_gated_linear_bwd")
        return dx, dwg if need_wg else None, dwu if need_wu else None, dbg, dbu, None


def _check(x, weights, others, act):
    """Types, devices and the weights' shapes; whether autograd needs what the backward reads."""
    if act not in _ACTS:
        raise AssertionError(f"act {act} not supported")
    k = x.shape[-1] if x.dim() else 0
    n = weights[0].shape[0] if weights[0].dim() == 2 else 0
    if n == 0 or k == 0:
        raise ValueError("x and weight must have at least one feature, weight as (N,K)")
    dtype, device, grad = x.dtype, x.device, x.requires_grad
    for w in weights:
        if w.shape != (n, k):
            raise ValueError(f"weight must have shape (N,{k}), the same for both of a pair, got {tuple(w.shape)}")
    for t in (*weights, *others):
        if t is None:
            continue
        if t.dtype != dtype:
            raise TypeError(f"all tensors must have x's dtype {dtype}, got {t.dtype}")
        if t.device != device:
            raise ValueError(f"all tensors must be on {device}, got one on {t.device}")
        grad = grad or t.requires_grad
    _lib.dtype_code(x)
    _lib.require_cuda(x)
    return grad and torch.is_grad_enabled()


def _check_bias(b, n):
    if b is not None and b.shape != (n,):
        raise ValueError(f"bias must have shape ({n},), got {tuple(b.shape)}")


def linear_fn(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
              residual: Optional[torch.Tensor] = None, act: str = "none") -> torch.Tensor:
    """y = act(x weight^T + bias) + residual, in one kernel.

    x (..., K), weight (N, K), bias (N), residual (..., N), all of one dtype; rows may be strided (slices need no copy; rows
    of 16-bit tensors that do not start on 16 bytes, as with odd widths, are copied first, and so is a tensor whose features
    are not next to each other, such as a transposed weight, forward and backward).
    act: "none", "relu", "sigmoid", "silu" or "gelu" (the exact one, by erf).  relu's derivative is 0 at 0 and 1 at NaN; in
    fp32 the exact sum decides which side of 0 a value is on, in 16-bit types the fp32 sum.  The backward keeps x, the weight
    and, with an activation, the pre-activation (24 bits a value, fp32: 32), and rounds its gradient to x's dtype.
    Differentiable once: create_graph=True raises RuntimeError."""
    _check_bias(bias, weight.shape[0])
    if residual is not None and residual.shape != (*x.shape[:-1], weight.shape[0]):
        raise ValueError(f"residual must have shape {(*x.shape[:-1], weight.shape[0])}, got {tuple(residual.shape)}")
    if _check(x, (weight,), (bias, residual), act):
        return LinearFunction.apply(x, weight, bias, residual, _ACTS[act])
    return _linear_forward(x, weight, bias, residual, _ACTS[act], False)[0]


def gated_linear_fn(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, b_gate: Optional[torch.Tensor] = None,
                    b_up: Optional[torch.Tensor] = None, act: str = "silu") -> torch.Tensor:
    """h = act(x w_gate^T + b_gate) * (x w_up^T + b_up): both projections of a gated feed-forward block, the activation
    and the product in one kernel.  The block's way down is linear_fn(h, w_down, residual=x).

    x (..., K), w_gate and w_up (N, K), biases (N), all of one dtype.  act as in linear_fn.  The backward keeps x, the
    weights and both projections (2 N values a token of 24 bits, fp32: 32)."""
    _check_bias(b_gate, w_gate.shape[0])
    _check_bias(b_up, w_gate.shape[0])
    if _check(x, (w_gate, w_up), (b_gate, b_up), act):
        return GatedLinearFunction.apply(x, w_gate, w_up, b_gate, b_up, _ACTS[act])
    return _gated_forward(x, w_gate, w_up, b_gate, b_up, _ACTS[act], False)[0]

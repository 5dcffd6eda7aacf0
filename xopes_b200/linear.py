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
    """(M, F) view of t, features next to each other, with its row stride; t is copied where there is none."""
    f = t.shape[-1]
    try:
        t2 = t.view(-1, f)
    except RuntimeError:
        t2 = t.reshape(-1, f)
    if (t2.stride(1) != 1 and f > 1) or t2.stride(0) < f:
        t2 = t2.contiguous()
    return t2, max(t2.stride(0), f)


def _scratch(nbytes, device):
    if nbytes < 0:
        _lib.check(nbytes, "workspace size")
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


class LinearFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act, keep):
        lib = _lib.load()
        x2, ldx = _rows(x)
        w2, ldw = _rows(weight)
        r2, ldr = (None, 0) if residual is None else _rows(residual)
        m, k = x2.shape
        n = w2.shape[0]
        b = None if bias is None else bias.contiguous()
        y = torch.empty(*x.shape[:-1], n, dtype=x.dtype, device=x.device)
        code = _lib.dtype_code(x)
        z = None
        if m:
            if keep and act:
                z = _scratch(lib.la_linear_saved_bytes(m, n, code, 0), x.device)
            with _lib.device_of(x):
                need = lib.la_linear_fwd_workspace_bytes(_lib.ptr(x2), ldx, _lib.ptr(w2), ldw, None, 0, m, n, k, code)
                ws = _scratch(need, x.device)
                rc = lib.la_linear_fwd(_lib.ptr(x2), ldx, _lib.ptr(w2), ldw, _lib.ptr(b), _lib.ptr(r2), ldr, _lib.ptr(y),
                                       _lib.ptr(z), _lib.ptr(ws), need, m, n, k, code, act, _lib.stream_of(x))
            _lib.check(rc, "la_linear_fwd")
        if keep:
            ctx.save_for_backward(x, weight, z)
            ctx.act = act
        return y

    @staticmethod
    def backward(ctx, dy):
        lib = _lib.load()
        x, weight, z = ctx.saved_tensors
        need_x, need_w, need_b, need_r = ctx.needs_input_grad[:4]
        dy2, ldy = _rows(dy)
        x2, ldx = _rows(x)
        w2, ldw = _rows(weight)
        m, k = x2.shape
        n = w2.shape[0]
        dx = torch.empty(x.shape, dtype=x.dtype, device=x.device) if need_x else None
        new = torch.empty if m else torch.zeros
        dw = new(n, k, dtype=x.dtype, device=x.device) if need_w else None
        db = new(n, dtype=x.dtype, device=x.device) if need_b else None
        if m and (need_x or need_w or need_b):
            code = _lib.dtype_code(x)
            with _lib.device_of(x):
                need = lib.la_linear_bwd_workspace_bytes(_lib.ptr(x2), ldx, _lib.ptr(w2), ldw, None, 0, _lib.ptr(dy2), ldy,
                                                         m, n, k, code, ctx.act, need_x, need_w, need_b)
                ws = _scratch(need, x.device)
                rc = lib.la_linear_bwd(_lib.ptr(x2), ldx, _lib.ptr(w2), ldw, _lib.ptr(z), _lib.ptr(dy2), ldy, _lib.ptr(dx),
                                       _lib.ptr(dw), _lib.ptr(db), _lib.ptr(ws), need, m, n, k, code, ctx.act,
                                       _lib.stream_of(x))
            _lib.check(rc, "la_linear_bwd")
        return dx, dw, db, dy if need_r else None, None, None


class GatedLinearFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, b_gate, b_up, act, keep):
        lib = _lib.load()
        x2, ldx = _rows(x)
        (wg, ldg), (wu, ldu) = _rows(w_gate), _rows(w_up)
        m, k = x2.shape
        n = wg.shape[0]
        bg, bu = (None if b is None else b.contiguous() for b in (b_gate, b_up))
        h = torch.empty(*x.shape[:-1], n, dtype=x.dtype, device=x.device)
        code = _lib.dtype_code(x)
        gu = None
        if m:
            if keep:
                gu = _scratch(lib.la_linear_saved_bytes(m, n, code, 1), x.device)
            with _lib.device_of(x):
                need = lib.la_linear_fwd_workspace_bytes(_lib.ptr(x2), ldx, _lib.ptr(wg), ldg, _lib.ptr(wu), ldu, m, n, k,
                                                         code)
                ws = _scratch(need, x.device)
                rc = lib.la_gated_linear_fwd(_lib.ptr(x2), ldx, _lib.ptr(wg), ldg, _lib.ptr(wu), ldu, _lib.ptr(bg),
                                             _lib.ptr(bu), _lib.ptr(h), _lib.ptr(gu), _lib.ptr(ws), need, m, n, k, code,
                                             act, _lib.stream_of(x))
            _lib.check(rc, "la_gated_linear_fwd")
        if keep:
            ctx.save_for_backward(x, w_gate, w_up, gu)
            ctx.act = act
        return h

    @staticmethod
    def backward(ctx, dh):
        lib = _lib.load()
        x, w_gate, w_up, gu = ctx.saved_tensors
        need_x = ctx.needs_input_grad[0]
        need_w = ctx.needs_input_grad[1] or ctx.needs_input_grad[2]
        need_bg, need_bu = ctx.needs_input_grad[3:5]
        dh2, ldh = _rows(dh)
        x2, ldx = _rows(x)
        (wg, ldg), (wu, ldu) = _rows(w_gate), _rows(w_up)
        m, k = x2.shape
        n = wg.shape[0]
        new = torch.empty if m else torch.zeros
        dx = torch.empty(x.shape, dtype=x.dtype, device=x.device) if need_x else None
        dwg, dwu = (new(n, k, dtype=x.dtype, device=x.device) if need_w else None for _ in range(2))
        dbg, dbu = (new(n, dtype=x.dtype, device=x.device) if need else None for need in (need_bg, need_bu))
        if m and (need_x or need_w or need_bg or need_bu):
            code = _lib.dtype_code(x)
            with _lib.device_of(x):
                need = lib.la_linear_bwd_workspace_bytes(_lib.ptr(x2), ldx, _lib.ptr(wg), ldg, _lib.ptr(wu), ldu,
                                                         _lib.ptr(dh2), ldh, m, n, k, code, ctx.act, need_x, need_w,
                                                         need_bg or need_bu)
                ws = _scratch(need, x.device)
                rc = lib.la_gated_linear_bwd(_lib.ptr(x2), ldx, _lib.ptr(wg), ldg, _lib.ptr(wu), ldu, _lib.ptr(gu),
                                             _lib.ptr(dh2), ldh, _lib.ptr(dx), _lib.ptr(dwg), _lib.ptr(dwu), _lib.ptr(dbg),
                                             _lib.ptr(dbu), _lib.ptr(ws), need, m, n, k, code, ctx.act, _lib.stream_of(x))
            _lib.check(rc, "la_gated_linear_bwd")
        return (dx, dwg if ctx.needs_input_grad[1] else None, dwu if ctx.needs_input_grad[2] else None, dbg, dbu, None,
                None)


def _check(x, weights, biases, residual, act):
    """Shapes, types and devices; whether autograd needs what the backward reads."""
    if act not in _ACTS:
        raise AssertionError(f"act {act} not supported")
    k = x.shape[-1] if x.dim() else 0
    n = weights[0].shape[0] if weights[0].dim() == 2 else 0
    for w in weights:
        if w.dim() != 2 or tuple(w.shape) != (n, k):
            raise ValueError(f"weight must have shape (N,{k}), the same for both of a pair, got {tuple(w.shape)}")
    if n == 0 or k == 0:
        raise ValueError("x and weight must have at least one feature")
    for b in biases:
        if b is not None and tuple(b.shape) != (n,):
            raise ValueError(f"bias must have shape ({n},), got {tuple(b.shape)}")
    if residual is not None and tuple(residual.shape) != (*x.shape[:-1], n):
        raise ValueError(f"residual must have shape {(*x.shape[:-1], n)}, got {tuple(residual.shape)}")
    given = [t for t in (x, *weights, *biases, residual) if t is not None]
    for t in given:
        if t.dtype != x.dtype:
            raise TypeError(f"all tensors must have x's dtype {x.dtype}, got {t.dtype}")
        if t.device != x.device:
            raise ValueError(f"all tensors must be on {x.device}, got one on {t.device}")
    _lib.dtype_code(x)
    _lib.require_cuda(x)
    return torch.is_grad_enabled() and any(t.requires_grad for t in given)


def linear_fn(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
              residual: Optional[torch.Tensor] = None, act: str = "none") -> torch.Tensor:
    """y = act(x weight^T + bias) + residual, in one kernel.

    x (..., K), weight (N, K), bias (N), residual (..., N), all of one dtype; rows may be strided (slices need no copy).
    act: "none", "relu", "sigmoid", "silu" or "gelu" (the exact one, by erf).  The backward keeps x, the weight and,
    with an activation, the pre-activation (24 bits a value, fp32: 32)."""
    keep = _check(x, [weight], [bias], residual, act)
    return LinearFunction.apply(x, weight, bias, residual, _ACTS[act], keep)


def gated_linear_fn(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, b_gate: Optional[torch.Tensor] = None,
                    b_up: Optional[torch.Tensor] = None, act: str = "silu") -> torch.Tensor:
    """h = act(x w_gate^T + b_gate) * (x w_up^T + b_up): both projections of a gated feed-forward block, the activation
    and the product in one kernel.  The block's way down is linear_fn(h, w_down, residual=x).

    x (..., K), w_gate and w_up (N, K), biases (N), all of one dtype.  act as in linear_fn.  The backward keeps x, the
    weights and both projections (2 N values a token of 24 bits, fp32: 32)."""
    keep = _check(x, [w_gate, w_up], [b_gate, b_up], None, act)
    return GatedLinearFunction.apply(x, w_gate, w_up, b_gate, b_up, _ACTS[act], keep)

"""Norms of queries and keys for each head with the position rotation in the same pass: the op in front of
lightning attention in a model block.

    y   = c * x / sqrt(sum(x^2) + eps) * weight        per row (token, head), as in normalize_gate_fn
    out = y with its first rotary_dim features rotated by position * inv_freq

One CUDA pass over q and k each way.  c = sqrt(D) with eps = D * 1e-6 is the RMS norm with 1e-6, c = 1 the
L2 norm.  The norm is normalize's without gate (xopes/ops/normalize/normalize/normalize_torch.py:9-111).
"""
import ctypes
import functools
from typing import Optional, Sequence, Tuple

import torch

from . import _lib


@functools.lru_cache(maxsize=64)
def _frequencies(base: float, rotary_dim: int):
    """base^(-2i / rotary_dim) as the host array of doubles the C entry takes."""
    n = rotary_dim // 2
    return (ctypes.c_double * max(n, 1))(*[base ** (-2.0 * i / rotary_dim) for i in range(n)])


def _forward(q, k, q_weight, k_weight, positions, offset, cu, freq, rotary_dim, interleaved, c, eps):
    """The outputs, and q and k as the kernel read them (features next to each other)."""
    lib = _lib.load()
    b, n, h, d = q.shape
    hk = k.shape[2]
    q_sb, q_sn, q_sh, one = q.stride()
    if one != 1 and d > 1:
        q = q.contiguous()
        q_sb, q_sn, q_sh, _ = q.stride()
    k_sb, k_sn, k_sh, one = k.stride()
    if one != 1 and d > 1:
        k = k.contiguous()
        k_sb, k_sn, k_sh, _ = k.stride()
    wq, wk, wcode = _weights(q, q_weight, k_weight)
    qo = torch.empty((b, n, h, d), dtype=q.dtype, device=q.device)
    ko = torch.empty((b, n, hk, d), dtype=q.dtype, device=q.device)
    pos, pos_sb, pos_sn = _positions(positions)
    with _lib.device_of(q):
        rc = lib.la_qk_norm_rope_fwd(
            q.data_ptr(), q_sb, q_sn, q_sh, k.data_ptr(), k_sb, k_sn, k_sh, _lib.ptr(wq), _lib.ptr(wk), wcode, pos, pos_sb,
            pos_sn, offset, _lib.ptr(cu), 0 if cu is None else cu.numel() - 1, freq, qo.data_ptr(), ko.data_ptr(), b, n, h, hk,
            d, rotary_dim, _lib.dtype_code(q), interleaved, c, eps, _lib.stream_of(q))
    if rc:
        _lib.check(rc, "la_qk_norm_rope_fwd")
    return qo, ko, q, k


def _positions(positions):
    if positions is None:
        return None, 0, 0
    return positions.data_ptr(), positions.stride(0) if positions.shape[0] > 1 else 0, positions.stride(1)


def _weights(q, q_weight, k_weight):
    """The weights in one type the kernel reads: both of q's type, or fp32."""
    dt = q.dtype
    if (q_weight is not None and q_weight.dtype != dt) or (k_weight is not None and k_weight.dtype != dt):
        dt = torch.float32
    return _as(q_weight, dt), _as(k_weight, dt), _lib.LA_F32 if dt == torch.float32 else _lib.dtype_code(q)


def _as(t, dt):
    """t contiguous and of type dt; the common case costs no call into torch's dispatcher."""
    if t is None:
        return None
    return (t if t.dtype == dt else t.to(dt)).contiguous()


class QkNormRopeFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, positions, offset, cu, freq, rotary_dim, interleaved, c, eps):
        qo, ko, q, k = _forward(q, k, q_weight, k_weight, positions, offset, cu, freq, rotary_dim, interleaved, c, eps)
        ctx.save_for_backward(q, k, q_weight, k_weight, positions, cu)
        ctx.cfg = (offset, freq, rotary_dim, interleaved, c, eps)
        ctx.set_materialize_grads(False)
        return qo, ko

    @staticmethod
    def backward(ctx, dqo, dko):
        _lib.once_differentiable()
        lib = _lib.load()
        q, k, q_weight, k_weight, positions, cu = ctx.saved_tensors
        offset, freq, rotary_dim, interleaved, c, eps = ctx.cfg
        pos, pos_sb, pos_sn = _positions(positions)
        b, n, h, d = q.shape
        hk = k.shape[2]
        dqo = torch.zeros((b, n, h, d), dtype=q.dtype, device=q.device) if dqo is None else _as(dqo, q.dtype)
        dko = torch.zeros((b, n, hk, d), dtype=q.dtype, device=q.device) if dko is None else _as(dko, q.dtype)
        wq, wk, wcode = _weights(q, q_weight, k_weight)
        dq, dk = torch.empty_like(dqo), torch.empty_like(dko)
        dwq = torch.empty_like(wq) if wq is not None and ctx.needs_input_grad[2] else None
        dwk = torch.empty_like(wk) if wk is not None and ctx.needs_input_grad[3] else None
        ws, ws_bytes = None, 0
        if dwq is not None or dwk is not None:
            ws_bytes = lib.la_qk_norm_rope_bwd_workspace_bytes(d)
            ws = torch.empty(ws_bytes, dtype=torch.uint8, device=q.device)
        m = 0 if cu is None else cu.numel() - 1
        with _lib.device_of(q):
            rc = lib.la_qk_norm_rope_bwd(
                _lib.ptr(q), *q.stride()[:3], _lib.ptr(k), *k.stride()[:3], _lib.ptr(wq), _lib.ptr(wk), wcode,
                pos, pos_sb, pos_sn, offset, _lib.ptr(cu), m, freq, _lib.ptr(dqo), _lib.ptr(dko),
                _lib.ptr(dq), _lib.ptr(dk), _lib.ptr(dwq), _lib.ptr(dwk), _lib.ptr(ws), ws_bytes,
                b, n, h, hk, d, rotary_dim, _lib.dtype_code(q), interleaved, c, eps, _lib.stream_of(q))
        _lib.check(rc, "la_qk_norm_rope_bwd")
        return (dq, dk, None if dwq is None else _as(dwq, q_weight.dtype), None if dwk is None else _as(dwk, k_weight.dtype),
                None, None, None, None, None, None, None, None)


def qk_norm_rope_fn(q: torch.Tensor, k: torch.Tensor, q_weight: Optional[torch.Tensor] = None,
                    k_weight: Optional[torch.Tensor] = None, positions: Optional[torch.Tensor] = None, offset: int = 0,
                    cu_seqlens: Optional[torch.LongTensor] = None, c: float = 1.0, eps: float = 1e-6,
                    base: float = 10000.0, rotary_dim: Optional[int] = None,
                    inv_freq: Optional[Sequence[float]] = None, interleaved: bool = False
                    ) -> Tuple[torch.Tensor, torch.Tensor]:
    """q (B,N,H,D), k (B,N,HK,D), HK any number of key heads; any strides with the features next to each other
    (slices of one projection need no copy).  Returns new contiguous tensors of the same shapes and type.
    Gradients for q, k and the weights.

    q_weight, k_weight: (D,), shared by the heads; None = 1.
    positions: int64 (B,N), (1,N) or (N,); None counts from 0 in every sequence, or in every document of
        cu_seqlens (M+1,) int64, batch 1 (tokens behind the last boundary count from it).  offset is added (a host number; under a captured graph give positions).
    rotary_dim: rotated features, the first of each head; even, D if None, 0 for the norm alone.
    inv_freq: rotary_dim / 2 host numbers, radians per position; base^(-2i / rotary_dim) if None.
    interleaved: pairs are features (2i, 2i+1) instead of (i, i + rotary_dim / 2).
    D up to 512."""
    if q.dim() != 4 or k.dim() != 4 or q.shape[:2] != k.shape[:2] or q.shape[-1] != k.shape[-1]:
        raise ValueError(f"q (B,N,H,D) and k (B,N,HK,D) expected, got {tuple(q.shape)} and {tuple(k.shape)}")
    if q.dtype != k.dtype:
        raise TypeError(f"q and k must have one dtype, got {q.dtype} and {k.dtype}")
    b, n, _, d = q.shape
    for w in (q_weight, k_weight):
        if w is not None and w.shape != (d,):
            raise ValueError(f"q_weight and k_weight must have shape ({d},), got {tuple(w.shape)}")
    r = d - d % 2 if rotary_dim is None else int(rotary_dim)
    if r < 0 or r > d or r % 2:
        raise ValueError(f"rotary_dim must be even and between 0 and {d}, got {rotary_dim}")
    if inv_freq is None:
        freq = _frequencies(float(base), r)
    else:
        if isinstance(inv_freq, torch.Tensor):
            if inv_freq.is_cuda:
                raise ValueError("inv_freq is read on the host: give numbers or a CPU tensor")
            inv_freq = inv_freq.tolist()
        if len(inv_freq) != r // 2:
            raise ValueError(f"inv_freq must have {r // 2} entries, got {len(inv_freq)}")
        freq = (ctypes.c_double * max(r // 2, 1))(*[float(f) for f in inv_freq])
    if positions is not None:
        if cu_seqlens is not None:
            raise ValueError("give positions or cu_seqlens, not both")
        if positions.dtype != torch.int64:
            raise TypeError(f"positions must be int64, got {positions.dtype}")
        if positions.dim() == 1:
            positions = positions[None]
        if positions.dim() != 2 or positions.shape[0] not in (1, b) or positions.shape[1] != n:
            raise ValueError(f"positions must have shape ({b},{n}), (1,{n}) or ({n},), got {tuple(positions.shape)}")
    device, grad = q.device, q.requires_grad
    for t in (k, q_weight, k_weight, positions, cu_seqlens):
        if t is not None:
            if t.device != device:
                raise ValueError(f"all tensors must be on {device}, got one on {t.device}")
            grad = grad or t.requires_grad
    _lib.require_cuda(q)
    cu = None
    if cu_seqlens is not None:
        if b != 1:
            raise AssertionError("cu_seqlens is only supported for batch size 1")
        cu = cu_seqlens.to(torch.int64).contiguous()
    _lib.dtype_code(q)
    if q.numel() == 0 or k.numel() == 0:
        raise ValueError("q and k must have at least one element")
    args = (q, k, q_weight, k_weight, positions, int(offset), cu, freq, r, 1 if interleaved else 0, float(c), float(eps))
    if grad and torch.is_grad_enabled():
        return QkNormRopeFunction.apply(*args)
    return _forward(*args)[:2]

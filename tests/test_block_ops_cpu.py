"""CPU: the checks of arguments of the operators around the attention (qk_norm_rope_fn) -- no kernel is
launched."""
import ctypes

import pytest
import torch

from xopes_b200 import _lib

ONE = ctypes.c_void_p(256)  # never dereferenced: the checks fail first


def test_qk_norm_refusals_in_python():
    from xopes_b200.qk_norm import qk_norm_rope_fn
    q, k = torch.randn(2, 4, 3, 16), torch.randn(2, 4, 1, 16)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        qk_norm_rope_fn(q, k)
    for bad in (dict(q=q[0]), dict(k=k[:, :3]), dict(k=torch.randn(2, 4, 1, 8)), dict(q_weight=torch.ones(3, 16)),
                dict(k_weight=torch.ones(8)), dict(rotary_dim=3), dict(rotary_dim=18), dict(rotary_dim=-2),
                dict(inv_freq=[1.0]), dict(positions=torch.zeros(3, 4, dtype=torch.int64)),
                dict(positions=torch.zeros(2, 3, dtype=torch.int64)),
                dict(positions=torch.zeros(2, 4, dtype=torch.int64), cu_seqlens=torch.tensor([0, 4]))):
        with pytest.raises(ValueError):
            qk_norm_rope_fn(**{**dict(q=q, k=k), **bad})
    for bad in (dict(k=k.half()), dict(positions=torch.zeros(2, 4, dtype=torch.int32)),):
        with pytest.raises(TypeError):
            qk_norm_rope_fn(**{**dict(q=q, k=k), **bad})


def qk_call(lib, **kw):
    a = dict(q=ONE, k=ONE, wdt=_lib.LA_F32, pos=None, cu=None, M=0, freq=(ctypes.c_double * 256)(), qo=ONE, ko=ONE, B=1, N=4,
             H=2, HK=2, D=16, R=16, dtype=_lib.LA_BF16)
    a.update(kw)
    return lib.la_qk_norm_rope_fwd(a["q"], 0, 0, 0, a["k"], 0, 0, 0, None, None, a["wdt"], a["pos"], 0, 0, 0, a["cu"],
                                   a["M"], a["freq"], a["qo"], a["ko"], a["B"], a["N"], a["H"], a["HK"], a["D"],
                                   a["R"], a["dtype"], 0, 1.0, 0.0, None)


@pytest.mark.parametrize("kw,rc", [
    (dict(q=None), -1), (dict(k=None), -1), (dict(freq=None), -1), (dict(qo=None), -1), (dict(ko=None), -1),
    (dict(B=0), -2), (dict(N=0), -2), (dict(H=0), -2), (dict(HK=0), -2), (dict(D=0), -2), (dict(R=-2), -2),
    (dict(R=18), -2), (dict(R=7), -2), (dict(cu=ONE, M=0), -2), (dict(cu=ONE, M=2, B=2), -2), (dict(M=1), -2),
    (dict(cu=ONE, M=1, pos=ONE), -2), (dict(dtype=7), -3), (dict(wdt=_lib.LA_F16), -3), (dict(D=514), -3),
    (dict(N=1 << 32), -5), (dict(H=1 << 21), -5)])
def test_qk_norm_status_codes(lib, kw, rc):
    assert qk_call(lib, **kw) == rc


def test_qk_norm_backward_status_codes(lib):
    freq = (ctypes.c_double * 8)()
    need = lib.la_qk_norm_rope_bwd_workspace_bytes(16)
    assert need > 0 and lib.la_qk_norm_rope_bwd_workspace_bytes(0) == 0

    def call(dwq=ONE, ws=ONE, nbytes=need, dq=ONE):
        return lib.la_qk_norm_rope_bwd(ONE, 0, 0, 0, ONE, 0, 0, 0, ONE, None, _lib.LA_F32, None, 0, 0, 0, None, 0, freq,
                                       ONE, ONE, dq, ONE, dwq, None, ws, nbytes, 1, 4, 2, 2, 16, 16, _lib.LA_BF16, 0,
                                       1.0, 0.0, None)
    assert call(dq=None) == -1
    assert call(ws=None) == -7
    assert call(nbytes=need - 1) == -7
    assert call(ws=ctypes.c_void_p(257)) == -6


def test_linear_refusals_in_python():
    from xopes_b200.linear import gated_linear_fn, linear_fn
    x, w = torch.randn(3, 4, 16), torch.randn(8, 16)
    for call in (lambda: linear_fn(x, w), lambda: gated_linear_fn(x, w, w)):
        with pytest.raises(RuntimeError, match="CUDA tensors only"):
            call()
    for bad in (dict(weight=w[:, :8]), dict(weight=w[0]), dict(bias=torch.zeros(9)), dict(residual=torch.zeros(4, 3, 8)),
                dict(residual=torch.zeros(8)), dict(weight=torch.randn(0, 16)), dict(x=torch.randn(3, 0), weight=torch.randn(8, 0))):
        with pytest.raises(ValueError):
            linear_fn(**{**dict(x=x, weight=w), **bad})
    for bad in (dict(w_up=torch.randn(9, 16)), dict(b_up=torch.zeros(7)), dict(w_gate=torch.randn(9, 16))):
        with pytest.raises(ValueError):
            gated_linear_fn(**{**dict(x=x, w_gate=w, w_up=w), **bad})
    with pytest.raises(TypeError):
        linear_fn(x, w.half())
    with pytest.raises(TypeError):
        linear_fn(x, w, torch.zeros(8).double())
    with pytest.raises(TypeError):
        linear_fn(x.double(), w.double())
    with pytest.raises(AssertionError, match="not supported"):
        linear_fn(x, w, act="softmax")


@pytest.mark.parametrize("kw,rc", [
    (dict(x=None), -1), (dict(w=None), -1), (dict(y=None), -1), (dict(M=0), -2), (dict(N=0), -2), (dict(K=-1), -2),
    (dict(ldx=63), -2), (dict(ldw=8), -2), (dict(res=ONE, ldr=31), -2), (dict(dtype=5), -3), (dict(act=9), -3),
    (dict(act=-1), -3), (dict(M=1 << 40), -5), (dict(N=1 << 30), -5), (dict(K=1 << 30, ldx=1 << 30, ldw=1 << 30), -5)])
def test_linear_status_codes(lib, kw, rc):
    a = dict(x=ONE, w=ONE, y=ONE, res=None, ldx=64, ldw=64, ldr=0, M=8, N=32, K=64, dtype=_lib.LA_BF16, act=0)
    a.update(kw)
    got = lib.la_linear_fwd(a["x"], a["ldx"], a["w"], a["ldw"], None, a["res"], a["ldr"], a["y"], None, None, 0, a["M"],
                            a["N"], a["K"], a["dtype"], a["act"], None)
    assert got == rc
    if kw.keys() <= {"x", "w", "M", "N", "K", "ldx", "ldw", "dtype"}:
        assert lib.la_linear_fwd_workspace_bytes(a["x"], a["ldx"], a["w"], a["ldw"], None, 0, a["M"], a["N"], a["K"],
                                                 a["dtype"]) == rc


def test_linear_backward_status_codes(lib):
    def call(z=ONE, dy=ONE, ldy=32, dwg=ONE, dwu=ONE, ws=None, nbytes=0, pair=False, act=1):
        if pair:
            return lib.la_gated_linear_bwd(ONE, 64, ONE, 64, ONE, 64, z, dy, ldy, ONE, dwg, dwu, None, None, ws, nbytes, 8,
                                           32, 64, _lib.LA_BF16, act, None)
        return lib.la_linear_bwd(ONE, 64, ONE, 64, z, dy, ldy, ONE, dwg, None, ws, nbytes, 8, 32, 64, _lib.LA_BF16, act, None)
    assert call(z=None) == -1 and call(z=None, pair=True) == -1 and call(z=None, pair=True, act=0) == -1
    assert call(dy=None) == -1 and call(ldy=31) == -2
    assert call(dwu=None, pair=True) == -1
    assert call() == -7  # dz needs scratch
    need = lib.la_linear_bwd_workspace_bytes(ONE, 64, ONE, 64, None, 0, ONE, 32, 8, 32, 64, _lib.LA_BF16, 1, 1, 1, 0)
    assert need >= 8 * 32 * 2
    assert call(ws=ONE, nbytes=need - 1) == -7
    assert call(ws=ctypes.c_void_p(257), nbytes=need) == -6

"""GPU: norms of queries and keys with the position rotation (xopes_b200.qk_norm.qk_norm_rope_fn) against the
definition in 64 bits on the CPU.

Tolerances.  fp32: a row's arithmetic is a sum of D squares, a reciprocal root (2 ulp), a handful of products and an angle
known to 2^-24 turns, i.e. 4e-7 rad, with sincospi's 2 ulp: 1e-6 of the row's norm covers it.  The gradients are
differences and sums of such terms, and what cancels leaves the terms' errors behind: with terms t_r of relative
error d each, |error of sum t_r| <= d sum |t_r|, so the bound for dx = s (g - xh sum(g xh)) is 1e-6 of the norm of
s (|g| + |xh| sum |g xh|), and for dw = sum c xh dy it is 1e-6 of the norm of sum |c xh dy| (at D = 1, where g and
xh sum(g xh) are equal but for eps, and a sum of random signs, the gradients themselves are much smaller than that).
16-bit: half a step of the output, 2^-8 (bf16) or 2^-11 (fp16) relative to the value, comes on top."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
HALF_STEP = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def definition(x, w, pos, inv_freq, r, interleaved, c, eps):
    """x (B,N,H,D) in 64 bits; pos (B,N)."""
    y = c * x / (x.square().sum(-1, keepdim=True) + eps).sqrt()
    if w is not None:
        y = y * w
    return rotated(y, pos, inv_freq, r, interleaved)


def rotated(y, pos, inv_freq, r, interleaved):
    a = pos.double()[:, :, None, None] * inv_freq
    cos, sin = a.cos(), a.sin()
    if interleaved:
        lo, hi = y[..., 0:r:2], y[..., 1:r:2]
        rot = torch.stack([lo * cos - hi * sin, hi * cos + lo * sin], -1).flatten(-2)
    else:
        lo, hi = y[..., :r // 2], y[..., r // 2:r]
        rot = torch.cat([lo * cos - hi * sin, hi * cos + lo * sin], -1)
    return torch.cat([rot, y[..., r:]], -1)


def magnitudes(x, w, do, pos, inv_freq, r, interleaved, c, eps):
    """The sums of the absolute values of the terms of dx and of dw."""
    s = (x.square().sum(-1, keepdim=True) + eps).rsqrt()
    dy = rotated(do, pos, -inv_freq, r, interleaved)
    g = c * dy if w is None else c * w * dy
    xh = x * s
    return s * (g.abs() + xh.abs() * (g * xh).abs().sum(-1, keepdim=True)), (c * xh * dy).abs().sum((0, 1, 2))


def close(name, ref, got, dtype, terms=None):
    assert got.dtype == dtype and got.shape == ref.shape, name
    assert torch.isfinite(got.float()).all(), name
    ref = ref.detach()
    err = float((ref - got.detach().double().cpu()).norm())
    bound = HALF_STEP[dtype] * float(ref.norm()) + 1e-6 * float((ref if terms is None else terms).norm())
    assert err <= bound, f"{name}: {err:.2e} > {bound:.2e}"


def check(b, n, h, hk, d, r, dtype, interleaved=False, c=None, eps=1e-5, pos=None, cu=None, base=10000.0, inv_freq=None,
          weights=True, wdtype=None, offset=0, make=None, seed=0, train=True):
    from xopes_b200.qk_norm import qk_norm_rope_fn
    g = torch.Generator().manual_seed(seed * 1000 + d)
    c = math.sqrt(d) if c is None else c
    wdtype = dtype if wdtype is None else wdtype
    rand = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    q, k = rand(b, n, h, d).to(dtype), rand(b, n, hk, d).to(dtype)
    doq, dok = rand(b, n, h, d).to(dtype), rand(b, n, hk, d).to(dtype)
    wq, wk = ((1 + 0.1 * rand(d)).to(wdtype) for _ in range(2)) if weights else (None, None)
    make = make or (lambda t: t.cuda())
    args = [make(q).requires_grad_(train), make(k).requires_grad_(train)]
    ws = [None if w is None else w.cuda().requires_grad_(train) for w in (wq, wk)]
    out = qk_norm_rope_fn(*args, *ws, positions=None if pos is None else pos.cuda(), offset=offset,
                          cu_seqlens=None if cu is None else cu.cuda(), c=c, eps=eps, base=base, rotary_dim=r,
                          inv_freq=inv_freq, interleaved=interleaved)
    leaves = [t for t in args + ws if t is not None]
    grads = torch.autograd.grad(out, leaves, [doq.cuda(), dok.cuda()]) if train else []
    # the definition
    if cu is not None:
        t = torch.arange(n)
        start = torch.zeros(n, dtype=torch.int64)
        for a, e in zip(cu.tolist(), cu.tolist()[1:]):
            start[a:e] = a
        p = (t - start)[None]
    else:
        p = torch.arange(n)[None] if pos is None else pos
        p = p[None] if p.dim() == 1 else p
    p = (p + offset).expand(b, n)
    f = torch.tensor([base ** (-2.0 * i / max(r, 1)) for i in range(r // 2)] if inv_freq is None else list(inv_freq),
                     dtype=torch.float64)
    refs = [t.double().requires_grad_() for t in (q, k)]
    rws = [None if w is None else w.double().requires_grad_() for w in (wq, wk)]
    ro = [definition(x, w, p, f, r, interleaved, c, eps) for x, w in zip(refs, rws)]
    rl = [t for t in refs + rws if t is not None]
    rg = torch.autograd.grad(ro, rl, [doq.double(), dok.double()])
    for name, ref, got in zip(("q", "k"), ro, out):
        close(name, ref, got, dtype)
    if train:
        with torch.no_grad():
            parts = [magnitudes(x, w, do.double(), p, f, r, interleaved, c, eps)
                     for x, w, do in zip(refs, rws, (doq, dok))]
        terms = [m[0] for m in parts] + [m[1] for m, w in zip(parts, rws) if w is not None]
        for name, ref, got, leaf, term in zip(("dq", "dk", "dwq", "dwk"), rg, grads, leaves, terms):
            close(name, ref, got, leaf.dtype, term)
    return out


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,r", [(128, 128), (128, 64), (64, 64), (32, 32), (96, 24), (256, 256), (512, 128), (20, 12),
                                 (33, 32), (7, 4), (1, 0), (2, 2), (300, 300), (511, 510), (40, 0), (16, 16)])
def test_feature_widths(d, r, interleaved, dtype):
    check(2, 37, 5, 3, d, r, dtype, interleaved)


@pytest.mark.parametrize("b,n,h,hk", [(1, 1, 1, 1), (1, 1, 16, 16), (3, 1, 32, 4), (1, 2, 7, 1), (300, 1, 3, 3),
                                      (2, 1000, 12, 12), (1, 4099, 2, 1), (5, 129, 33, 9), (1, 3, 100, 40)])
def test_tokens_and_heads(b, n, h, hk):
    check(b, n, h, hk, 64, 64, torch.bfloat16)
    check(b, n, h, hk, 64, 64, torch.float32, interleaved=True)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("b,n,h,hk,d,r", [(3, 501, 16, 16, 128, 128), (1, 1777, 21, 9, 96, 64), (2, 2049, 13, 2, 64, 64),
                                          (1, 700, 40, 8, 256, 256), (2, 300, 17, 17, 512, 512), (1, 5000, 32, 32, 32, 16),
                                          (1, 60000, 1, 1, 64, 64)])
def test_large_calls(b, n, h, hk, d, r, dtype):
    check(b, n, h, hk, d, r, dtype, interleaved=bool(n % 2))

    def cut(t):  # heads cut from a projection: other strides for tokens than for heads
        buf = torch.zeros(b, n, t.shape[2] + 2, d, dtype=t.dtype)
        buf[:, :, 2:] = t
        return buf.cuda()[:, :, 2:].detach()
    check(b, n, h, hk, d, r, dtype, interleaved=not n % 2, make=cut, seed=1)


@pytest.mark.parametrize("where", ["packed", "transposed", "offset4", "offset1", "expanded"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strides_and_alignment(where, dtype):
    def make(t):
        b, n, h, d = t.shape
        if where == "packed":          # heads cut from the middle of a projection
            buf = torch.zeros(b, n, h + 4, d, dtype=t.dtype)
            buf[:, :, 3:3 + h] = t
            return buf.cuda()[:, :, 3:3 + h].detach()
        if where == "transposed":      # (B, H, N, D) in memory
            return t.transpose(1, 2).contiguous().cuda().transpose(1, 2).detach()
        if where == "expanded":        # features not next to each other
            return t.transpose(2, 3).contiguous().cuda().transpose(2, 3).detach()
        off = int(where[6:])           # starts that many elements off an aligned address
        buf = torch.zeros(t.numel() + off, dtype=t.dtype)
        buf[off:] = t.reshape(-1)
        return buf.cuda()[off:].view(t.shape).detach()
    check(2, 45, 6, 2, 64, 32, dtype, make=make)
    check(2, 45, 6, 2, 64, 32, dtype, interleaved=True, make=make)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_positions(dtype):
    g = torch.Generator().manual_seed(1)
    far = torch.randint(0, 1 << 28, (3, 50), generator=g)
    check(3, 50, 4, 2, 64, 64, dtype, pos=far)                       # far apart, exact angles
    check(3, 50, 4, 2, 64, 64, dtype, pos=far[:1])                   # one row for all
    check(3, 50, 4, 2, 64, 64, dtype, pos=far[0], interleaved=True)  # without a batch dimension
    check(3, 50, 4, 2, 64, 64, dtype, pos=-far)                      # before the origin
    check(3, 50, 4, 2, 64, 64, dtype, pos=far[:, :25].repeat_interleave(2, 1))
    check(1, 50, 4, 2, 64, 64, dtype, pos=torch.randint(0, 99, (50, 2), generator=g)[:, 0])  # strided
    check(2, 50, 4, 2, 64, 64, dtype, offset=123456)
    check(2, 50, 4, 2, 64, 32, dtype, inv_freq=[0.5 ** i for i in range(16)])
    check(2, 50, 4, 2, 64, 32, dtype, inv_freq=torch.rand(16, dtype=torch.float64))
    check(2, 50, 4, 2, 64, 64, dtype, base=500000.0, pos=far[:2] % 5000)


@pytest.mark.parametrize("ends", [[0, 70], [0, 1, 70], [0, 0, 31, 31, 32, 70, 70], list(range(71))])
def test_packed_documents(ends):
    cu = torch.tensor(ends)
    check(1, 70, 4, 2, 64, 64, torch.bfloat16, cu=cu)
    check(1, 70, 4, 2, 64, 64, torch.float32, cu=cu, interleaved=True, offset=5)


def test_weights_and_norms():
    check(2, 30, 4, 4, 64, 64, torch.bfloat16, weights=False)
    check(2, 30, 4, 4, 64, 64, torch.bfloat16, wdtype=torch.float32)
    check(2, 30, 4, 4, 64, 64, torch.float32, wdtype=torch.float32, c=1.0, eps=1e-6)
    check(2, 30, 4, 4, 64, 64, torch.float16, wdtype=torch.float32, c=1.0, eps=0.0)
    # weights in two types; one weight alone; one gradient alone
    from xopes_b200.qk_norm import qk_norm_rope_fn
    q = torch.randn(2, 5, 3, 32, device="cuda", dtype=torch.bfloat16)
    w = torch.rand(32, device="cuda").requires_grad_()
    w16 = w.detach().bfloat16().requires_grad_()
    a, b = qk_norm_rope_fn(q, q, w, w16)
    c, _ = qk_norm_rope_fn(q, q, w, None)
    assert torch.equal(a, c)
    gw, g16 = torch.autograd.grad((a, b), (w, w16), (q, q))
    assert gw.dtype == torch.float32 and g16.dtype == torch.bfloat16
    only, = torch.autograd.grad(c, w, q)
    assert torch.equal(only, gw)


def test_rows_without_a_value():
    """A row of zeros (a padded token): zeros out at eps > 0, and its neighbours' gradients stay finite.  Infinity and NaN
    stay in their row, except in the weights' gradients, which sum over all rows."""
    from xopes_b200.qk_norm import qk_norm_rope_fn
    q = torch.randn(2, 9, 4, 64, device="cuda", dtype=torch.bfloat16)
    clean = qk_norm_rope_fn(q, q)[0]
    q[0, 3] = 0
    q[1, 5, 2] = float("inf")
    q[1, 6, 1, 7] = float("nan")
    leaf = q.clone().requires_grad_()
    out, _ = qk_norm_rope_fn(leaf, q)
    dx, = torch.autograd.grad(out, leaf, torch.ones_like(out))
    assert (out[0, 3] == 0).all()
    keep = torch.ones(2, 9, 4, dtype=torch.bool, device="cuda")
    keep[0, 3] = keep[1, 5, 2] = keep[1, 6, 1] = False
    assert torch.equal(out[keep], clean[keep])
    assert torch.isfinite(dx[keep]).all() and torch.isfinite(dx[0, 3]).all()
    assert torch.isnan(out[1, 6, 1]).all()


def test_same_bits_every_time_and_in_a_graph():
    from xopes_b200.qk_norm import qk_norm_rope_fn
    q = torch.randn(2, 700, 8, 128, device="cuda", dtype=torch.bfloat16).requires_grad_()
    k = torch.randn(2, 700, 2, 128, device="cuda", dtype=torch.bfloat16).requires_grad_()
    w = torch.rand(128, device="cuda").requires_grad_()
    pos = torch.arange(700, device="cuda")[None] + 5
    do = (torch.randn_like(q), torch.randn_like(k))

    def step():
        out = qk_norm_rope_fn(q, k, w, w, positions=pos)
        # detached: while an eager graph of the same leaves lives, no backward can be captured (torch's own rule)
        return [t.detach() for t in out + torch.autograd.grad(out, (q, k, w), do)]

    first = step()
    assert all(torch.equal(a, b) for a, b in zip(first, step()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(first, got))
    pos += 1000  # the graph reads the positions where they lie
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(step(), got))


def test_long_stream_of_bytes_past_32_bits():
    """More than 2^31 elements in one tensor: offsets past 32 bits.  The last tokens are checked."""
    from xopes_b200.qk_norm import qk_norm_rope_fn
    n, h, d = 70000, 256, 128
    q = torch.zeros(1, n, h, d, device="cuda", dtype=torch.bfloat16)
    q[:, -3:] = torch.randn(1, 3, h, d, device="cuda")
    k = q[:, :, :1]
    out, ko = qk_norm_rope_fn(q, k, c=math.sqrt(d))
    f = torch.tensor([10000.0 ** (-2.0 * i / d) for i in range(d // 2)], dtype=torch.float64)
    ref = definition(q[:, -3:].double().cpu(), None, torch.arange(n - 3, n)[None], f, d, False, math.sqrt(d), 1e-6)
    close("q", ref, out[:, -3:], torch.bfloat16)
    close("k", ref[:, :, :1], ko[:, -3:], torch.bfloat16)
    assert (out[:, :-3] == 0).all()

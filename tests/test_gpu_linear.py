"""GPU: projections with their epilogue (linear_fn) and the gated pair (gated_linear_fn) against their definitions in
64 bits.

Tolerances, all on L2 norms; h = half a step of the type (2^-24, bf16 2^-8, fp16 2^-11):
  results   h |y| for the last rounding, and 1e-6 of the norm of the sums of absolute values of the terms for the
            products (fp32 partial sums of random walks of K terms: their rounding errors add up to about 2^-24 of
            that sum; 1e-6 is 16 of those, and holds what the exponentials add).
  gradients dz is an operand and is rounded (h |dz|); it comes from pre-activations that were kept rounded (h |z|, which
            moves the activation by at most 1.2 h |z| and its derivative likewise, the first two derivatives of every
            activation here being at most 1.13).  So an element of dz is off by at most E as below, with signs that are
            independent of each other: over a sum with weights w the errors add up in quadrature, to
            sqrt(sum E^2 w^2) / sqrt(3) for errors uniform in their bounds; twice sqrt(sum E^2 w^2) is 3.5 of that."""
import math

import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu
HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
ACTS = {"none": lambda t: t, "relu": F.relu, "sigmoid": torch.sigmoid, "silu": F.silu, "gelu": F.gelu}
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def close(name, ref, got, dtype, terms, quad=0.0):
    assert got.dtype == dtype and got.shape == ref.shape, (name, got.dtype, got.shape)
    assert torch.isfinite(got.float()).all(), name
    ref = ref.detach()
    err = float((ref - got.detach().to(ref.device).double()).norm())
    bound = HALF_STEP[dtype] * float(ref.norm()) + 1e-6 * float(terms.norm()) + 2 * quad
    assert err <= bound, f"{name}: {err:.3e} > {bound:.3e} (norm {float(ref.norm()):.3e})"


def derivative(z, kind):
    z = z.detach().requires_grad_()
    d, = torch.autograd.grad(ACTS[kind](z).sum(), z)
    return d


def check(m, k, n, dtype, act="none", bias=False, residual=False, pair=False, train=True, make=None, lead=None, seed=0):
    from xopes_b200.linear import gated_linear_fn, linear_fn
    g = torch.Generator(device="cuda").manual_seed(seed * 7 + m + k + n)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    make = make or (lambda t: t)
    P = 2 if pair else 1
    x = rand(m, k).to(dtype)
    ws = [(rand(n, k) * k ** -0.5).to(dtype) for _ in range(P)]
    bs = [rand(n).to(dtype) if bias else None for _ in range(P)]
    r = rand(m, n).to(dtype) if residual else None
    dy = rand(m, n).to(dtype)
    leaf = lambda t: None if t is None else make(t).detach().requires_grad_(train)  # noqa: E731
    lx, lws, lbs, lr = leaf(x), [leaf(w) for w in ws], [None if b is None else b.clone().requires_grad_(train) for b in bs], leaf(r)
    xin = lx if lead is None else lx.view(*lead, k)
    rin = lr if lead is None or r is None else lr.view(*lead, n)
    y = gated_linear_fn(xin, *lws, *lbs, act=act) if pair else linear_fn(xin, lws[0], lbs[0], residual=rin, act=act)
    assert y.shape == ((m,) if lead is None else tuple(lead)) + (n,)
    y = y.reshape(m, n)
    # the definition
    X, W, B = x.double(), [w.double() for w in ws], [None if b is None else b.double() for b in bs]
    Z = [X @ w.t() if b is None else X @ w.t() + b for w, b in zip(W, B)]
    T = [X.abs() @ w.abs().t() + (0 if b is None else b.abs()) for w, b in zip(W, B)]  # sums of absolute values
    a, d = ACTS[act](Z[0]), derivative(Z[0], act)
    ref = a * Z[1] if pair else a
    terms = T[0] * Z[1].abs() * 1.2 + T[1] * a.abs() if pair else T[0] * 1.2
    if residual:
        ref, terms = ref + r.double(), terms + r.double().abs()
    close("y", ref, y, dtype, terms)
    if not train:
        return
    leaves = [t for t in [lx, *lws, *lbs, lr] if t is not None]
    grads = list(torch.autograd.grad(y, leaves, make(dy)))
    D, h = dy.double(), HALF_STEP[dtype]
    if pair:
        dz = [D * Z[1] * d, D * a]
        E = [h * (2 * dz[0].abs() + 1.2 * (D * Z[1] * Z[0]).abs()), h * (dz[1].abs() + 1.2 * (D * Z[0]).abs())]
    else:
        dz = [D * d]
        E = [h * (dz[0].abs() + 1.2 * (D * Z[0]).abs())] if act != "none" else [torch.zeros_like(D)]
    dx = sum(a_ @ w for a_, w in zip(dz, W))
    close("dx", dx, grads.pop(0), dtype, sum(a_.abs() @ w.abs() for a_, w in zip(dz, W)),
          float(sum(e.square() @ w.square() for e, w in zip(E, W)).sum().sqrt()))
    for i in range(P):
        close(f"dw{i}", dz[i].t() @ X, grads.pop(0), dtype, dz[i].abs().t() @ X.abs(),
              float((E[i].square().t() @ X.square()).sum().sqrt()))
    if bias:
        for i in range(P):
            close(f"db{i}", dz[i].sum(0), grads.pop(0), dtype, dz[i].abs().sum(0), float(E[i].square().sum().sqrt()))
    if residual:
        assert torch.equal(grads.pop(0), dy)
    assert not grads


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", sorted(ACTS))
@pytest.mark.parametrize("pair", [False, True])
def test_activations(act, pair, dtype):
    check(150, 96, 72, dtype, act, bias=True, residual=not pair, pair=pair)
    check(150, 96, 72, dtype, act, pair=pair)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,k,n", [(1, 1, 1), (1, 64, 64), (2, 7, 3), (3, 130, 9), (5, 16, 257), (64, 64, 64), (127, 65, 129),
                                   (129, 200, 520), (256, 256, 256), (257, 264, 264), (300, 1000, 40), (7, 2000, 1000),
                                   (1000, 24, 16), (33, 1, 50), (400, 50, 1)])
def test_sizes(m, k, n, dtype):
    check(m, k, n, dtype, "silu", bias=True, residual=True)
    check(m, k, n, dtype, "gelu", bias=True, pair=True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m", [1, 2, 3, 4, 5, 8, 9, 16, 17, 31, 32, 33, 64, 65, 128])
def test_few_tokens(m, dtype):
    check(m, 512, 320, dtype, "silu", bias=True, residual=True, train=False)
    check(m, 512, 320, dtype, "silu", bias=True, pair=True, train=False)
    check(m, 1037, 75, dtype, train=False)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,k,n", [(1, 4096, 4096), (8, 8192, 1000), (64, 4096, 1408), (128, 2048, 2048), (17, 11008, 512),
                                   (100, 768, 9472), (40, 192, 20000)])
def test_few_tokens_many_weights(m, k, n, dtype):
    """Every size of a cluster and of its ring."""
    check(m, k, n, dtype, "gelu", bias=True, residual=True, train=False)
    check(m, k, n, dtype, "silu", pair=True, train=False)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,k,n", [(2048, 512, 768), (3000, 768, 2048), (515, 4096, 1024), (5000, 128, 128)])
def test_larger(m, k, n, dtype):
    check(m, k, n, dtype, "silu", bias=True, residual=True)
    check(m, k, n, dtype, "silu", pair=True)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("where", ["columns", "offset8", "offset1", "transposed"])
def test_strides_and_alignment(where, dtype):
    def make(t):
        if where == "columns":                       # a slice of a wider tensor
            buf = torch.zeros(t.shape[0], t.shape[1] + 24, dtype=t.dtype, device="cuda")
            buf[:, 8:8 + t.shape[1]] = t
            return buf[:, 8:8 + t.shape[1]]
        if where == "transposed":                    # features not next to each other
            return t.t().contiguous().t()
        off = int(where[6:])                         # off an aligned address
        buf = torch.zeros(t.numel() + off, dtype=t.dtype, device="cuda")
        buf[off:] = t.reshape(-1)
        return buf[off:].view(t.shape)
    check(140, 136, 264, dtype, "silu", residual=True, make=make)
    check(140, 136, 264, dtype, "silu", pair=True, make=make)
    check(4, 136, 264, dtype, "silu", pair=True, make=make, train=False)


def test_leading_dimensions_and_no_tokens():
    from xopes_b200.linear import gated_linear_fn, linear_fn
    check(24, 64, 40, torch.bfloat16, lead=(2, 3, 4), residual=True)
    check(24, 64, 40, torch.bfloat16, "silu", pair=True, lead=(4, 6))
    w = torch.randn(16, 8, device="cuda").requires_grad_()
    assert linear_fn(torch.randn(8, device="cuda"), w).shape == (16,)
    x = torch.empty(0, 8, device="cuda").requires_grad_()
    for y in (linear_fn(x, w, act="relu"), gated_linear_fn(x, w, w)):
        assert y.shape == (0, 16)
        dx, dw = torch.autograd.grad(y.sum(), (x, w))
        assert dx.shape == x.shape and (dw == 0).all()


def test_gradients_that_are_not_asked_for():
    from xopes_b200.linear import gated_linear_fn, linear_fn
    x, w, v = (torch.randn(*s, device="cuda", dtype=torch.bfloat16) for s in ((40, 64), (48, 64), (48, 64)))
    b, r = torch.randn(48, device="cuda", dtype=torch.bfloat16), torch.randn(40, 48, device="cuda", dtype=torch.bfloat16)
    dy = torch.randn_like(r)
    full = [t.clone().requires_grad_() for t in (x, w, v, b, r)]
    a = torch.autograd.grad(linear_fn(full[0], full[1], full[3], full[4], act="silu"), (full[0], full[1], full[3], full[4]), dy)
    p = torch.autograd.grad(gated_linear_fn(full[0], full[1], full[2], full[3], full[3]), full[:4], dy)
    for i, ref in enumerate(a):
        t = [x, w, b, r]
        t[i] = t[i].clone().requires_grad_()
        assert torch.equal(torch.autograd.grad(linear_fn(*t, act="silu"), t[i], dy)[0], ref)
    for i, ref in enumerate(p[:3]):
        t = [x, w, v]
        t[i] = t[i].clone().requires_grad_()
        assert torch.equal(torch.autograd.grad(gated_linear_fn(*t, b, b), t[i], dy)[0], ref)


def test_expanded_gradient_and_shared_weight():
    """y.sum() hands an expanded gradient; the same weight for both projections gets both its gradients."""
    from xopes_b200.linear import gated_linear_fn
    x = torch.randn(70, 64, device="cuda").requires_grad_()
    w = (torch.randn(32, 64, device="cuda") / 8).requires_grad_()
    gx, gw = torch.autograd.grad(gated_linear_fn(x, w, w).sum(), (x, w))
    xd, wd = x.detach().double().requires_grad_(), w.detach().double().requires_grad_()
    z = xd @ wd.t()
    rx, rw = torch.autograd.grad((F.silu(z) * z).sum(), (xd, wd))
    assert float((gx - rx).norm()) <= 1e-5 * float(rx.norm()) and float((gw - rw).norm()) <= 1e-5 * float(rw.norm())


@pytest.mark.parametrize("pair", [False, True])
def test_against_differences(pair):
    """Gradients against central differences of the fp32 operator itself, in random directions.  The step e moves y by
    e; rounding puts 1e-6 |y| / e on the quotient and curvature e^2, so with e = 1e-2 both are below 1e-3 of its size."""
    from xopes_b200.linear import gated_linear_fn, linear_fn
    g = torch.Generator(device="cuda").manual_seed(5)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    t = [rand(20, 32), rand(24, 32) / 6, rand(24, 32) / 6, rand(24), rand(24)]
    fn = (lambda *a: gated_linear_fn(*a, act="gelu")) if pair else (lambda x, w, _, b, __: linear_fn(x, w, b, act="silu"))
    dy = rand(20, 24)
    used = [0, 1, 2, 3, 4] if pair else [0, 1, 3]
    leaves = [a.clone().requires_grad_() for a in t]
    grads = torch.autograd.grad(fn(*leaves), [leaves[i] for i in used], dy)
    for i, got in zip(used, grads):
        v = rand(*t[i].shape)
        v /= v.norm()
        e = 1e-2
        lo, hi = ([a + s * e * v if j == i else a for j, a in enumerate(t)] for s in (-1, 1))
        with torch.no_grad():
            num = float(((fn(*hi).double() - fn(*lo).double()) * dy.double()).sum()) / (2 * e)
        assert abs(num - float((got.double() * v.double()).sum())) <= 2e-3 * float(got.norm())


def test_not_a_number_stays_in_its_row():
    from xopes_b200.linear import gated_linear_fn, linear_fn
    for dtype in TYPES:
        x, w = torch.randn(300, 72, device="cuda", dtype=dtype), torch.randn(48, 72, device="cuda", dtype=dtype)
        clean = [linear_fn(x, w, act="silu"), gated_linear_fn(x, w, w)]
        x[17, 5], x[200, 71] = float("nan"), float("inf")
        keep = torch.ones(300, dtype=torch.bool, device="cuda")
        keep[17] = keep[200] = False
        for a, b in zip(clean, [linear_fn(x, w, act="silu"), gated_linear_fn(x, w, w)]):
            assert torch.equal(a[keep], b[keep]) and torch.isnan(b[17]).all()


@pytest.mark.parametrize("m,k,n", [(3, 512, 256), (100, 1024, 128), (700, 256, 512)])
def test_same_bits_every_time_and_in_a_graph(m, k, n):
    from xopes_b200.linear import gated_linear_fn, linear_fn
    x, w, v, b = (torch.randn(*s, device="cuda").mul(0.1).bfloat16().requires_grad_() for s in ((m, k), (n, k), (n, k), (n,)))
    dy = torch.randn(m, n, device="cuda").bfloat16()

    def step():
        y, h = linear_fn(x, w, b, act="gelu"), gated_linear_fn(x, w, v, b, b)
        return [t.detach() for t in (y, h) + torch.autograd.grad((y, h), (x, w, v, b), (dy, dy))]

    first = step()
    assert all(torch.equal(a, b_) for a, b_ in zip(first, step()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b_) for a, b_ in zip(first, other))
    graph, graph2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    with torch.cuda.graph(graph2):
        got2 = step()
    for _ in range(3):
        graph.replay()
        graph2.replay()
    assert all(torch.equal(a, b_) and torch.equal(a, c) for a, b_, c in zip(first, got, got2))


def test_two_streams_at_once():
    from xopes_b200.linear import gated_linear_fn
    torch.manual_seed(0)
    x, w, v = (torch.randn(*s, device="cuda").mul(0.1).bfloat16() for s in ((600, 512), (640, 512), (640, 512)))
    ref = gated_linear_fn(x, w, v)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for i in range(40):
        with torch.cuda.stream(streams[i % 2]):
            outs.append(gated_linear_fn(x, w, v))
    torch.cuda.synchronize()
    assert all(torch.equal(ref, o) for o in outs)


def test_offsets_past_32_bits():
    """More than 2^31 results: the last rows of the output and of the gradients' operands."""
    from xopes_b200.linear import linear_fn
    m, k, n = 70000, 64, 32768
    x = torch.zeros(m, k, device="cuda", dtype=torch.bfloat16)
    x[-3:] = torch.randn(3, k, device="cuda")
    w = (torch.randn(n, k, device="cuda") / 8).bfloat16()
    leaf = x.clone().requires_grad_()
    y = linear_fn(leaf, w, act="silu")
    z = x[-3:].double() @ w.double().t()
    close("y", F.silu(z), y[-3:], torch.bfloat16, x[-3:].double().abs() @ w.double().abs().t())
    assert (y[:-3] == 0).all()
    dy = torch.zeros(m, n, device="cuda", dtype=torch.bfloat16)
    dy[-2:] = torch.randn(2, n, device="cuda")
    dx, = torch.autograd.grad(y, leaf, dy)
    dz = dy[-3:].double() * derivative(z, "silu")
    e = HALF_STEP[torch.bfloat16] * (dz.abs() + 1.2 * (dy[-3:].double() * z).abs())
    close("dx", dz @ w.double(), dx[-3:], torch.bfloat16, dz.abs() @ w.double().abs(),
          float((e.square() @ w.double().square()).sum().sqrt()))
    assert (dx[:-3] == 0).all()


@pytest.mark.parametrize("m,k,n", [(64, 4096, 64), (65, 2050, 67), (200, 1030, 130), (9, 1024, 30), (130, 4096, 1100), (1500, 768, 2048)])
@pytest.mark.parametrize("pair", [False, True])
def test_fp32_contraction_shared_by_a_cluster(m, k, n, pair):
    """Splits of 2 to 16 (clusters above 8 among them), ragged tiles, both tile sizes."""
    check(m, k, n, torch.float32, "silu", bias=True, residual=not pair, pair=pair)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,k,n,pair", [(300, 2048, 10000, False), (300, 2050, 9992, False), (257, 1024, 10004, True), (1100, 4096, 4100, False)])
def test_last_round_of_tiles_split(m, k, n, pair, dtype):
    """A few tiles more than the GPU holds at once: those are split, the others whole."""
    check(m, k, n, dtype, "gelu", bias=True, residual=not pair, pair=pair)


@pytest.mark.parametrize("m,k,n,dtype", [(64, 4096, 64, torch.float32), (300, 2048, 10000, torch.bfloat16)])
def test_split_sums_repeat_and_replay(m, k, n, dtype):
    from xopes_b200.linear import linear_fn
    g = torch.Generator(device="cuda").manual_seed(3)
    x, w = (torch.randn(*s, generator=g, device="cuda").to(dtype) for s in ((m, k), (n, k)))
    want = linear_fn(x, w)
    assert torch.equal(want, linear_fn(x, w))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = linear_fn(x, w)
    for _ in range(3):
        got.zero_()
        graph.replay()
        assert torch.equal(want, got)

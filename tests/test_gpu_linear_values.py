"""GPU: linear_fn and gated_linear_fn value by value, where a norm over a whole tensor says nothing: pre-activations next
to relu's border.

An element of a result is off by at most half a step of its type (2^-24 in fp32) and what its fp32 sum is off: K roundings
of partial sums, each at most 2^-24 of the sum of the absolute values of the terms, with signs that are independent of each
other: 8 sqrt(K) 2^-24 of that sum is eight standard deviations of an upper bound."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def near(name, got, ref, terms, count, half=2.0 ** -24):
    """Every element of got within the bound above of ref (64 bits); terms: sums of absolute values of `count` terms."""
    off = (got.double() - ref).abs() - half * ref.abs() - 8 * count ** 0.5 * 2.0 ** -24 * terms
    worst = int(off.argmax())
    assert off.flatten()[worst] <= 0, (name, worst, float(got.flatten()[worst]), float(ref.flatten()[worst]))


@pytest.mark.parametrize("m,k,n", [(1, 64, 40), (7, 4096, 300), (8, 130, 33), (40, 2048, 100), (130, 516, 1100), (514, 512, 512)])
@pytest.mark.parametrize("pair", [False, True])
def test_relu_border_fp32(pair, m, k, n):
    """The bias takes back the fp32 rounding of one sum of each column, so that column n's pre-activation of token n mod m is
    within 2^-24 of that sum around zero, less than fp32 sums are off.  Which side it is on decides the derivative."""
    from xopes_b200.linear import gated_linear_fn, linear_fn
    g = torch.Generator(device="cuda").manual_seed(m + k + n)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    wide = rand(m, k + 3)
    x = wide[:, :k] if n % 2 else wide[:, :k].contiguous()  # rows that start anywhere, too
    w, dy = rand(n, k) * k ** -0.5, rand(m, n)
    X, W = x.double(), w.double()
    sums = X @ W.t()
    token = torch.arange(n, device="cuda") % m
    b = -sums[token, torch.arange(n, device="cuda")].float()
    z = sums + b.double()
    assert float(z[token, torch.arange(n, device="cuda")].abs().max()) < 1e-5
    x, w, b = (t.detach().requires_grad_() for t in (x, w, b))
    if pair:
        v = rand(n, k) * k ** -0.5
        u = X @ v.double().t()
        y = gated_linear_fn(x, w, v, b, act="relu")
        near("h", y, z.clamp(min=0) * u, (X.abs() @ W.abs().t() + b.double().abs()) * u.abs() + z.abs() * (X.abs() @ v.double().abs().t()), k)
        dz = dy.double() * u * (z > 0)
        more = dy.double().abs() * (X.abs() @ v.double().abs().t())  # u is a sum as well
    else:
        y = linear_fn(x, w, b, act="relu")
        near("y", y, z.clamp(min=0), X.abs() @ W.abs().t() + b.double().abs(), k)
        dz, more = dy.double() * (z > 0), dy.double().abs()
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    dx64 = dz @ W + ((dy.double() * z.clamp(min=0)) @ v.double() if pair else 0)
    up = dy.double().abs() * z.clamp(min=0) if pair else torch.zeros_like(z)
    size = dz.abs() + more
    near("dx", dx, dx64, size @ W.abs() + (up @ v.double().abs() + dy.double().abs() @ v.double().abs() if pair else 0), 2 * n + k)
    near("dw", dw, dz.t() @ X, size.t() @ X.abs(), m + k)
    near("db", db, dz.sum(0), size.sum(0), m + k)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m", [1, 8, 20, 200])
@pytest.mark.parametrize("pair", [False, True])
def test_relu_of_small_whole_numbers(pair, m, dtype):
    """Sums of small whole numbers are exact in fp32, so results and gradients are those in 64 bits, rounded once:
    many pre-activations are 0, where the derivative is 0, and those of one column are NaN, where the gradient passes."""
    import torch.nn.functional as F
    from xopes_b200.linear import gated_linear_fn, linear_fn
    k, n = 16, 24
    g = torch.Generator(device="cuda").manual_seed(m)
    whole = lambda *s: torch.randint(-1, 2, s, generator=g, device="cuda").to(dtype)  # noqa: E731
    x, w, v, dy, b = whole(m, k), whole(n, k), whole(n, k), whole(m, n), whole(n)
    b[5] = float("nan")
    leaves = [t.requires_grad_() for t in (x, w, b)]
    leaves64 = [t.detach().double().requires_grad_() for t in (x, w, b)]
    z = leaves64[0] @ leaves64[1].t() + leaves64[2]
    assert int((z == 0).sum()) > 0
    if pair:
        y = gated_linear_fn(x, w, v, b, act="relu")
        y64 = F.relu(z) * (x.detach().double() @ v.double().t())
        wanted = [1, 2]  # dx takes in du of the NaN column
    else:
        y, y64, wanted = linear_fn(x, w, b, act="relu"), F.relu(z), [0, 1, 2]
    assert torch.equal(torch.nan_to_num(y, nan=-99.0), torch.nan_to_num(y64.to(dtype), nan=-99.0))
    got, ref = torch.autograd.grad(y, leaves, dy), torch.autograd.grad(y64, leaves64, dy.double())
    for i in wanted:
        assert torch.equal(got[i], ref[i].to(dtype)), (i, got[i], ref[i])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m", [7, 100, 4000])
@pytest.mark.parametrize("act", ["gelu", "silu", "sigmoid"])
def test_activations_over_their_whole_range(act, m, dtype):
    """Pre-activations that are given (a product with one term, of weight 1), so that every result and gradient stands for one
    value of the activation or its derivative.  Half a step of the type (in the subnormal range of fp16 2^-25) for the
    rounding, and for the value 3e-5 of it: exponentials e^a with a rounded two or three times, 2^-24 |a| each, |a| below 90;
    the normal distribution's tail e^(-z^2 / 2) R(|z|) with R fitted to 5e-6; a few steps of 2^-23.  The derivative is a sum
    of two such values, and has 1 - s for a sigmoid s, which is off by 2^-24.  It is taken at what the forward kept of z: 24 of
    32 bits for 16-bit types, the others filled, so off by at most 2^-15 |z| (bits of z below the 15 of the mantissa), which
    moves the derivative by 2^-15 |z act''(z)|; bf16 has no such bits.  Below 2^-118 nothing is said (1 / x of the
    special function unit ends at 2^-126)."""
    import torch.nn.functional as F
    from xopes_b200.linear import linear_fn
    top = 13.0 if act == "gelu" else 80.0
    z = torch.linspace(-top, top, m * 16, device="cuda").to(dtype).view(m, 16).requires_grad_()
    y = linear_fn(z, torch.eye(16, device="cuda").to(dtype), act=act)
    dz, = torch.autograd.grad(y, z, torch.ones_like(y))
    t = z.detach().double()
    s, phi = torch.sigmoid(t), torch.exp(-0.5 * t * t) * 0.3989422804014327
    cdf = 0.5 * torch.special.erfc(-t * 0.5 ** 0.5)
    y64, parts = {"gelu": (t * cdf, (cdf, t * phi)), "silu": (t * s, (s, t * s * torch.sigmoid(-t))),
                  "sigmoid": (s, (s * torch.sigmoid(-t), 0 * s))}[act]
    assert torch.allclose(y64, {"gelu": F.gelu, "silu": F.silu, "sigmoid": torch.sigmoid}[act](t), rtol=0, atol=1e-14)
    floor = 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -118
    half = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}[dtype]
    more = {"gelu": (2 - t * t) * phi, "silu": s * torch.sigmoid(-t) * (2 + t * (1 - 2 * s)),
            "sigmoid": s * torch.sigmoid(-t) * (1 - 2 * s)}[act].abs() * t.abs() * (2.0 ** -15 if dtype == torch.float16 else 0.0)
    more = more + (2.0 ** -23 if act == "sigmoid" else 0.0)
    for name, got, ref, size, more in (("y", y, y64, y64.abs(), 0.0),
                                       ("dz", dz, parts[0] + parts[1], parts[0].abs() + parts[1].abs(), more)):
        off = (got.detach().double() - ref).abs() - half * ref.abs() - 3e-5 * size - floor - more
        worst = int(off.argmax())
        assert float(off.flatten()[worst]) <= 0, (name, *(float(v.detach().flatten()[worst]) for v in (z, got, ref)))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m", [1, 8, 100, 300])
@pytest.mark.parametrize("n", [24, 140, 204, 75])
def test_epilogue_access_widths(n, m, dtype):
    """Bias and residual on 16 bytes, on 8 and on neither, results of widths that are multiples of 8, of 4 and of neither; whole
    numbers, whose sums are exact in every type (at most 64 + 2), so that every element is known."""
    from xopes_b200.linear import gated_linear_fn, linear_fn
    g = torch.Generator(device="cuda").manual_seed(m + n)
    whole = lambda *s: torch.randint(-1, 2, s, generator=g, device="cuda").to(dtype)  # noqa: E731
    x, w, v = whole(m, 64), whole(n, 64), whole(n, 64)
    biases, wide = whole(n + 8), whole(m, n + 16)
    z, u = x.double() @ w.double().t(), x.double() @ v.double().t()
    for at in (0, 8, 4, 1):
        b, r = biases[at:at + n], wide[:, at:at + n]
        y = linear_fn(x, w, b, residual=r, act="relu")
        assert torch.equal(y, ((z + b.double()).clamp(min=0) + r.double()).to(dtype)), at
        y = linear_fn(x, w, residual=r)
        assert torch.equal(y, (z + r.double()).to(dtype)), at
        h = gated_linear_fn(x, w, v, b, biases[:n], act="relu")
        assert torch.equal(h, ((z + b.double()).clamp(min=0) * (u + biases[:n].double())).to(dtype)), at


def same_kind(name, got, ref, rows=slice(None)):
    """NaN where ref (64 bits) has NaN, the same infinities, and numbers elsewhere."""
    got, ref = got.double()[rows], ref[rows]
    for f in (torch.isnan, torch.isposinf, torch.isneginf):
        assert torch.equal(f(got), f(ref)), (name, f.__name__, (f(got) != f(ref)).nonzero()[:4].tolist())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m", [6, 70, 300])
@pytest.mark.parametrize("act", ["none", "relu", "sigmoid", "silu", "gelu"])
@pytest.mark.parametrize("pair", [False, True])
def test_infinities_and_not_a_number(pair, act, m, dtype):
    """A token with an infinity and one with NaN: what becomes of them is what the formulas in 64 bits make of them, forward and in
    the gradients, and the other tokens' results have the bits that they have without."""
    import torch.nn.functional as F
    from xopes_b200.linear import gated_linear_fn, linear_fn
    fn64 = {"none": lambda t: t, "relu": F.relu, "sigmoid": torch.sigmoid, "silu": lambda t: t * torch.sigmoid(t),
            "gelu": lambda t: t * 0.5 * torch.special.erfc(-t * 0.5 ** 0.5)}[act]
    torch.manual_seed(m)
    x, w, v, dy = (torch.randn(*s, device="cuda").to(dtype) for s in ((m, 72), (48, 72), (48, 72), (m, 48)))

    def run(x):
        leaves = [t.clone().requires_grad_() for t in (x, w)]
        y = gated_linear_fn(leaves[0], leaves[1], v, act=act) if pair else linear_fn(*leaves, act=act)
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]
    clean = run(x)
    x[2, 5], x[m - 2, 71] = float("inf"), float("nan")
    got = run(x)
    X, W = x.double().requires_grad_(), w.double().requires_grad_()
    z = X @ W.t()
    y64 = fn64(z) * (X @ v.double().t()) if pair else fn64(z)
    dx64, dw64 = torch.autograd.grad(y64, (X, W), dy.double())
    others = torch.ones(m, dtype=torch.bool, device="cuda")
    others[2] = others[m - 2] = False
    assert torch.equal(got[0][others], clean[0][others]) and torch.equal(got[1][others], clean[1][others])
    same_kind("y", got[0], y64.detach())
    same_kind("dx", got[1], dx64)
    same_kind("dw", got[2], dw64)


def test_relu_border_in_a_graph_and_on_two_streams():
    """What is near 0 is found anew in every replay, and calls side by side have room of their own for it."""
    from xopes_b200.linear import gated_linear_fn, linear_fn
    m, k, n = 90, 260, 130
    torch.manual_seed(0)

    def data():
        x, w = torch.randn(m, k, device="cuda"), torch.randn(n, k, device="cuda") * k ** -0.5
        z = x.double() @ w.double().t()
        return x, w, -z[torch.arange(n, device="cuda") % m, torch.arange(n, device="cuda")].float()

    def step(x, w, b, dy):
        x, w, b = (t.detach().requires_grad_() for t in (x, w, b))
        y, h = linear_fn(x, w, b, act="relu"), gated_linear_fn(x, w, w, b, act="relu")
        return [y.detach(), h.detach(), *torch.autograd.grad((y, h), (x, w, b), (dy, dy))]
    sets, dy = [data() for _ in range(3)], torch.randn(m, n, device="cuda")
    refs = [step(*s, dy) for s in sets]
    place = [torch.empty_like(t) for t in sets[0]]
    for p, t in zip(place, sets[0]):
        p.copy_(t)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(*place, dy)
    for s, ref in zip(sets, refs):
        for p, t in zip(place, s):
            p.copy_(t)
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(ref, got))
    streams, outs = [torch.cuda.Stream() for _ in range(2)], []
    torch.cuda.synchronize()
    for i in range(12):
        with torch.cuda.stream(streams[i % 2]):
            outs.append(step(*sets[i % 3], dy))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for i, out in enumerate(outs) for a, b in zip(refs[i % 3], out))

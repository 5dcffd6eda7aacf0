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

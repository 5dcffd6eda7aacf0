"""GPU: the operators around the attention together with it, as a block uses them: projection -> norms and rotation of q and k
-> attention -> norm + gate -> projection with the residual -> norm -> gated pair -> projection with the residual.

Tolerances.  fp32: about a dozen operators in a chain, each within 1e-5 of its terms (TOL_FP32) and none amplifying relative
errors by more than 2 (norms): 1e-4.  bf16: every operator rounds its output, 2^-8 of the value at most, about
twelve roundings on the way to the output, twice as many on the way to a gradient; independent roundings add in
quadrature, sqrt(24) 2^-8 = 1.9e-2, and the same factor of 2 gives 4e-2.  With a single token the attention's output is (q.k) v
and the norm behind it divides its length out, so that the gradients on the way of q and k vanish but for eps: what
the norm's backward leaves there is s (g - xh sum(g xh)) with two equal parts, and its error is relative to those.  They
are what the definition's gradient is with the norm's length held constant; errors are measured against that there."""
import math

import pytest
import torch
import torch.nn.functional as F

from util import assert_close

pytestmark = pytest.mark.gpu
TOL = {torch.float32: 1e-4, torch.bfloat16: 4e-2}
BASE, EPS = 10000.0, 1e-6


def weights(h, d, inner, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    c = h * d
    rand = lambda *s: torch.randn(*s, generator=g) * s[-1] ** -0.5  # noqa: E731
    w = dict(qkv=rand(3 * c, c), gate=rand(c, c), out=rand(c, c), w_gate=rand(inner, c), w_up=rand(inner, c),
             down=rand(c, inner), q_norm=1 + 0.1 * torch.randn(d, generator=g), k_norm=1 + 0.1 * torch.randn(d, generator=g))
    return {k: v.to(dtype) for k, v in w.items()}


def decays(h):
    return torch.log(1 - 2.0 ** (-3 - torch.arange(h, dtype=torch.float64) / 2))


def block(x, w, ld, h, d, positions=None, state=None, cu=None):
    """(y, final state); with a state and one token: a decode step that updates the state where it lies."""
    from xopes_b200 import lasd_decode_step, lightning_attn_func
    from xopes_b200.linear import gated_linear_fn, linear_fn
    from xopes_b200.normalize import normalize_gate_fn
    from xopes_b200.qk_norm import qk_norm_rope_fn
    b, n, c = x.shape
    qkv = linear_fn(x, w["qkv"]).view(b, n, 3 * h, d)
    q, k = qk_norm_rope_fn(qkv[:, :, :h], qkv[:, :, h:2 * h], w["q_norm"], w["k_norm"], positions=positions, cu_seqlens=cu)
    v = qkv[:, :, 2 * h:].contiguous()
    if state is not None:
        o, s = lasd_decode_step(q, k, v, ld, state)
    else:
        o, s = lightning_attn_func(q, k, v, ld=ld, cu_seqlens=cu, decay_type="scalar")
    o = normalize_gate_fn(o.reshape(b, n, c), gate=linear_fn(x, w["gate"]), num_groups=h, c=math.sqrt(d))
    x = linear_fn(o, w["out"], residual=x)
    m = gated_linear_fn(normalize_gate_fn(x, c=math.sqrt(c)), w["w_gate"], w["w_up"])
    return linear_fn(m, w["down"], residual=x), s


def definition(x, w, ld, h, d, cu=None, constant=False):
    """The block in 64 bits on the CPU; constant: with the length that the attention's norm divides by held constant."""
    b, n, c = x.shape
    qkv = (x @ w["qkv"].t()).view(b, n, 3 * h, d)
    q, k, v = qkv.split(h, 2)
    pos = torch.arange(n)
    same = torch.ones(n, n, dtype=torch.bool)
    if cu is not None:
        doc = torch.bucketize(pos, cu[1:-1], right=True)
        pos, same = pos - cu[doc], doc[:, None] == doc[None]
    a = pos.double()[:, None, None] * BASE ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)

    def turn(t, g):
        t = t / (t.square().sum(-1, keepdim=True) + EPS).sqrt() * g
        lo, hi = t.chunk(2, -1)
        return torch.cat([lo * a.cos() - hi * a.sin(), hi * a.cos() + lo * a.sin()], -1)

    def norm(t, size):
        return t / (t.square().sum(-1, keepdim=True) + EPS).sqrt() * math.sqrt(size)

    q, k = turn(q, w["q_norm"]), turn(k, w["k_norm"])
    t = torch.arange(n, dtype=torch.float64)
    weight = ((t[:, None] - t[None]).clamp(min=0)[None] * ld[:, None, None]).exp() * (same & (t[:, None] >= t[None]))
    o = torch.einsum("bihd,bjhd,hij,bjhe->bihe", q, k, weight, v)
    gate = torch.sigmoid(x @ w["gate"].t()).view(b, n, h, d)
    o = o * gate
    o = o / (o.square().sum(-1, keepdim=True) + EPS).sqrt().detach() * math.sqrt(d) if constant else norm(o, d)
    x = o.reshape(b, n, c) @ w["out"].t() + x
    y = norm(x, c)
    return (F.silu(y @ w["w_gate"].t()) * (y @ w["w_up"].t())) @ w["down"].t() + x


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("b,n,h,d,inner,docs", [(2, 150, 4, 64, 704, None), (1, 130, 3, 128, 250, None), (1, 200, 2, 64, 352, (70, 71, 200)),
                                                (3, 1, 4, 64, 128, None)])
def test_training_step(b, n, h, d, inner, docs, dtype):
    g = torch.Generator().manual_seed(n)
    x, dy = (torch.randn(b, n, h * d, generator=g).to(dtype) for _ in range(2))
    w, ld = weights(h, d, inner, dtype, 3), decays(h)
    cu = None if docs is None else torch.tensor((0,) + docs)
    leaves = {k: v.cuda().requires_grad_() for k, v in {"x": x, **w}.items()}
    y, _ = block(leaves["x"], leaves, ld.float().cuda(), h, d, cu=None if cu is None else cu.cuda())
    grads = torch.autograd.grad(y, list(leaves.values()), dy.cuda())
    refs = {k: v.double().requires_grad_() for k, v in {"x": x, **w}.items()}
    ry = definition(refs["x"], refs, ld, h, d, cu)
    rgrads = torch.autograd.grad(ry, list(refs.values()), dy.double())
    assert_close("y", ry.float(), y.float(), TOL[dtype])
    parts = rgrads
    if n == 1:
        parts = torch.autograd.grad(definition(refs["x"], refs, ld, h, d, cu, constant=True), list(refs.values()), dy.double())
    for name, ref, part, got in zip(refs, rgrads, parts, grads):
        assert torch.isfinite(got).all(), name
        err = float((ref - got.double().cpu()).norm())
        assert err <= TOL[dtype] * max(float(ref.norm()), float(part.norm())), f"{name}: {err:.2e}"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_prompt_then_tokens(dtype):
    """A prompt in one call, then tokens one by one with the state and positions, eagerly and as a replayed graph."""
    b, n, h, d, inner, steps = 2, 60, 4, 64, 352, 5
    g = torch.Generator().manual_seed(9)
    x = torch.randn(b, n + steps, h * d, generator=g).to(dtype)
    w, ld = weights(h, d, inner, dtype, 4), decays(h)
    ref = definition(x.double(), {k: v.double() for k, v in w.items()}, ld, h, d)
    wc, ldc, xc = {k: v.cuda() for k, v in w.items()}, ld.float().cuda(), x.cuda()
    with torch.no_grad():
        y, state = block(xc[:, :n], wc, ldc, h, d)
        assert_close("prompt", ref[:, :n].float(), y.float(), TOL[dtype])
        pos = torch.full((b, 1), n, device="cuda")
        first = state.clone()
        eager = []
        for i in range(steps):
            y, state = block(xc[:, n + i:n + i + 1], wc, ldc, h, d, positions=pos + i, state=state)
            eager.append(y)
            assert_close(f"token {i}", ref[:, n + i:n + i + 1].float(), y.float(), TOL[dtype])
        token, state = xc[:, n:n + 1].clone(), first.clone()
        block(token, wc, ldc, h, d, positions=pos, state=state.clone())  # first use outside the capture
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out, _ = block(token, wc, ldc, h, d, positions=pos, state=state)
        state.copy_(first)
        for i in range(steps):
            token.copy_(xc[:, n + i:n + i + 1])
            pos.fill_(n + i)
            graph.replay()
            assert torch.equal(out, eager[i]), i


def test_tensors_of_another_stream():
    """A block on a stream of its own, next to work on the default one."""
    w, ld = {k: v.cuda() for k, v in weights(4, 64, 352, torch.bfloat16, 5).items()}, decays(4).float().cuda()
    x = torch.randn(2, 300, 256, device="cuda", dtype=torch.bfloat16)
    with torch.no_grad():
        ref = block(x, w, ld, 4, 64)[0]
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        outs = []
        for _ in range(8):
            with torch.cuda.stream(side):
                outs.append(block(x, w, ld, 4, 64)[0])
            outs.append(block(x, w, ld, 4, 64)[0])
        torch.cuda.synchronize()
    assert all(torch.equal(ref, o) for o in outs)


FIRST = """
import torch
from xopes_b200.linear import gated_linear_fn, linear_fn
from xopes_b200.qk_norm import qk_norm_rope_fn
def rand(*s):
    return torch.randn(*s, device="cuda").mul(0.1).to(torch.%s)
torch.manual_seed(0)
m = %d
x, w, v, b, q = rand(m, 256), rand(320, 256), rand(320, 256), rand(320), rand(1, m, 16, 128)
def call():
    return [linear_fn(x, w, b, act="gelu"), gated_linear_fn(x, w, v, b), *qk_norm_rope_fn(q, q)]
torch.cuda.synchronize()
with torch.no_grad():
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    graph.replay()
    ref = call()
    torch.cuda.synchronize()
for o, r in zip(out, ref):
    assert torch.isfinite(o.float()).all() and torch.equal(o, r)
"""


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("m", [3, 600])
def test_first_use_under_capture(m, dtype):
    """What the kernels need once per device is found inside a capture too."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    run = subprocess.run([sys.executable, "-c", FIRST % (dtype, m)], cwd=root, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stderr[-2000:]


def test_second_derivatives_are_refused():
    from xopes_b200.linear import gated_linear_fn, linear_fn
    from xopes_b200.qk_norm import qk_norm_rope_fn
    x, w = (torch.randn(8, 8, device="cuda").requires_grad_() for _ in range(2))
    for y in (linear_fn(x, w), gated_linear_fn(x, w, w), qk_norm_rope_fn(x.view(1, 8, 1, 8), x.view(1, 8, 1, 8))[0]):
        with pytest.raises(RuntimeError, match="differentiable once"):
            torch.autograd.grad(y.sum(), x, create_graph=True)

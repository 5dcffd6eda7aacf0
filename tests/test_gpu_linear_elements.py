"""GPU: every element of linear_fn's and gated_linear_fn's results, through the C ABI, with workspaces, kept values and
results full of NaN before the call and room around the results.

Inputs are -1, 0 and 1.  Their sums are whole numbers far below 2^24, exact in fp32 in any order, so a result is the sum
in 64 bits rounded once to its type, and one element that is missing, doubled or in another's place shows.  dz, dg and du
are whole numbers up to 256 (checked), exact in every type."""
import pytest
import torch

pytestmark = pytest.mark.gpu
ROOM = 64  # elements before and behind each result


def whole(g, *s):
    """Every fourth element 1 or -1."""
    t = torch.randint(0, 8, s, generator=g, device="cuda")
    return (t == 1).float() - (t == 0).float()


class Room:
    """A contiguous result with room around it, all NaN."""

    def __init__(self, shape, dtype):
        n = 1
        for s in shape:
            n *= s
        self.all = torch.full((n + 2 * ROOM,), float("nan"), dtype=dtype, device="cuda")
        self.t = self.all[ROOM:ROOM + n].view(shape)

    def ptr(self):
        return self.t.data_ptr()

    def is_(self, ref, name):
        assert torch.isnan(self.all[:ROOM]).all() and torch.isnan(self.all[-ROOM:]).all(), name + ": written outside"
        wrong = (self.t != ref.to(self.t.dtype)).nonzero()
        assert len(wrong) == 0, (name, len(wrong), wrong[:4].tolist(), wrong[-4:].tolist())


def scratch(nbytes):
    assert nbytes >= 0
    return torch.full((max(nbytes, 1),), 255, dtype=torch.uint8, device="cuda")


SIZES = [(1, 64, 200), (7, 1024, 300), (64, 4096, 1408), (128, 130, 75),                   # few tokens
         (129, 200, 520), (129, 520, 200), (300, 1024, 96), (257, 4096, 512), (1000, 4096, 260),  # few tiles: all of them split
         (300, 2048, 10000), (257, 1024, 10004), (1100, 2048, 4100),                       # the last round's tiles split
         (130, 2048, 9992), (1100, 4096, 1024), (1100, 4096, 2048),
         (130, 2048, 64), (1100, 64, 64), (3000, 4096, 64), (2000, 130, 9992),             # a gradient's tiles split, narrow and wide
         (200, 1030, 130), (515, 513, 1023), (2000, 512, 768), (3000, 768, 2048)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,k,n", SIZES)
@pytest.mark.parametrize("pair", [False, True])
def test_every_element(lib, pair, m, k, n, dtype):
    from xopes_b200 import _lib
    g = torch.Generator(device="cuda").manual_seed(m + 3 * k + 5 * n)
    P = 2 if pair else 1
    x, dy = whole(g, m, k).to(dtype), whole(g, m, n).to(dtype)
    ws, bs = [whole(g, n, k).to(dtype) for _ in range(P)], [whole(g, n).to(dtype) for _ in range(P)]
    code, act = _lib.dtype_code(x), 1
    st = torch.cuda.current_stream().cuda_stream
    y, kept = Room((m, n), dtype), scratch(lib.la_linear_saved_bytes(m, n, code, pair))
    up, ldu = (ws[1].data_ptr(), k) if pair else (None, 0)
    need = lib.la_linear_fwd_workspace_bytes(x.data_ptr(), k, ws[0].data_ptr(), k, up, ldu, m, n, k, code)
    work = scratch(need)
    if pair:
        rc = lib.la_gated_linear_fwd(x.data_ptr(), k, ws[0].data_ptr(), k, up, k, bs[0].data_ptr(), bs[1].data_ptr(), y.ptr(),
                                     kept.data_ptr(), work.data_ptr(), need, m, n, k, code, act, st)
    else:
        rc = lib.la_linear_fwd(x.data_ptr(), k, ws[0].data_ptr(), k, bs[0].data_ptr(), None, 0, y.ptr(), kept.data_ptr(),
                               work.data_ptr(), need, m, n, k, code, act, st)
    assert rc == 0
    X, W, D = x.double(), [w.double() for w in ws], dy.double()
    Z = [X @ w.t() + b.double() for w, b in zip(W, bs)]
    a = Z[0].clamp(min=0)
    y.is_(a * Z[1] if pair else a, "y")
    dz = [D * Z[1] * (Z[0] > 0), D * a] if pair else [D * (Z[0] > 0)]
    assert all(float(d.abs().max()) <= 256 for d in dz)
    dx, dws, dbs = Room((m, k), dtype), [Room((n, k), dtype) for _ in range(P)], [Room((n,), dtype) for _ in range(P)]
    need = lib.la_linear_bwd_workspace_bytes(x.data_ptr(), k, ws[0].data_ptr(), k, up, ldu, dy.data_ptr(), n, m, n, k, code, act,
                                             1, 1, 1)
    work = scratch(need)
    if pair:
        rc = lib.la_gated_linear_bwd(x.data_ptr(), k, ws[0].data_ptr(), k, up, k, kept.data_ptr(), dy.data_ptr(), n, dx.ptr(),
                                     dws[0].ptr(), dws[1].ptr(), dbs[0].ptr(), dbs[1].ptr(), work.data_ptr(), need, m, n, k,
                                     code, act, st)
    else:
        rc = lib.la_linear_bwd(x.data_ptr(), k, ws[0].data_ptr(), k, kept.data_ptr(), dy.data_ptr(), n, dx.ptr(), dws[0].ptr(),
                               dbs[0].ptr(), work.data_ptr(), need, m, n, k, code, act, st)
    assert rc == 0
    dx.is_(sum(d @ w for d, w in zip(dz, W)), "dx")
    for i in range(P):
        dws[i].is_(dz[i].t() @ X, f"dw{i}")
        dbs[i].is_(dz[i].sum(0), f"db{i}")

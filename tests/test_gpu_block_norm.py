"""The norms between two blocks against their formula in 64 bits."""
import pytest
import torch

from gpu_util import announce, require_gpu

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
EPS = 1e-5


@pytest.fixture(scope="module")
def S():
    require_gpu()
    import syntropy_amd.gemv as S
    return S


def real(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


def rms(v, g):
    return v / torch.sqrt((v * v).mean(1, keepdim=True) + EPS) * g


# A sum of squares over a row is at most 64 additions deep (a lane's values in turn, the lanes by halves, the
# wavefronts in order), all of one sign: 64 steps of U, half of them behind the root; the square root, the quotient and
# the products by r and the weight are a step each.
NORM = U * (64 / 2 + 6)


def formula(x, branch, g, post=None, gate=None, scale=1.0):
    """(h, y, and what the F32 steps may move each by)"""
    x = x.double()
    h, eh = x, torch.zeros_like(x)
    if branch is not None:
        a = branch.double()
        ea = 0.0
        if post is not None:
            a = rms(a, post.double())
            ea = NORM * a.abs()
        if gate is not None:
            a = a * gate.double()
            ea = ea * gate.double().abs() + U * a.abs()
        scale = float(torch.tensor(scale, dtype=F32))
        h = x + scale * a
        eh = abs(scale) * ea + U * h.abs() + U * abs(scale) * a.abs()
    y = ey = None
    if g is not None:
        # y = h r g: h is off by eh, r by its own steps and what eh moves the mean's root by
        n = x.shape[1]
        r = 1 / torch.sqrt((h * h).mean(1, keepdim=True) + EPS)
        dr = (eh * h.abs()).sum(1, keepdim=True) / n * r ** 3
        y = h * r * g.double()
        ey = NORM * y.abs() + 1.01 * (eh * r + h.abs() * dr) * g.double().abs()
    return h, y, eh, ey


def near(got, want, err, what):
    t = got.dtype
    off = (got.double() - want).abs()
    tol = 1.01 * err + (torch.finfo(t).eps / 2) * (want.abs() + 1.01 * err) + torch.finfo(t).smallest_normal * torch.finfo(t).eps
    assert bool(torch.isfinite(got).all()), what
    assert bool((off <= tol).all()), f"{what}: off by {float((off / tol).max()):.3g} of what it may be"


WIDTHS = [1, 2, 7, 8, 63, 64, 511, 512, 513, 1000, 1024, 2011, 2048, 4096, 4100, 5120, 8192, 8200, 12000, 16384, 20001, 32768]


@pytest.mark.parametrize("n", WIDTHS)
def test_widths(S, n):
    announce(f"block_norm {n}")
    for rows in (1, 3, 300 if n <= 4096 else 20):
        x, b = 3 * real(1, rows, n), real(2, rows, n).to(BF16)
        g, post, gate = real(3, n), real(4, n), real(5, rows, n).to(BF16)
        for kw in (dict(), dict(post=post), dict(gate=gate, scale=0.3), dict(post=post, gate=gate[0], scale=-1.7)):
            h, y = S.block_norm(x, b, g, EPS, rows, **kw)
            assert h.dtype == F32 and y.dtype == BF16
            wh, wy, eh, ey = formula(x, b, g, **kw)
            near(h, wh, eh, f"h {rows} {kw.keys()}")
            near(y, wy, ey, f"y {rows} {kw.keys()}")


@pytest.mark.parametrize("tx", [F32, F16, BF16])
@pytest.mark.parametrize("tb", [F32, F16, BF16])
def test_types_strides_and_offsets(S, tx, tb):
    for n in (40, 1003, 4608):
        for rows in (2, 65):
            for off in (0, 1):
                def apart(seed, t, more):
                    v = torch.full((rows, n + more), float("nan"), dtype=t, device="cuda")
                    return v[:, off:off + n].copy_(real(seed, rows, n))
                x, b, gate = apart(1, tx, 3), apart(2, tb, 16), apart(3, tb, 5)
                g, post = real(4, n + 1)[1:].clone(), real(5, n + 1)[1:]
                post = real(5, n)
                for ty in (F32, F16, BF16):
                    hb = torch.full((rows + 1, n + 9), 77.0, dtype=tx, device="cuda")
                    yb = torch.full((rows + 1, n + 9), 77.0, dtype=ty, device="cuda")
                    h, y = hb[:rows, off + 1:off + 1 + n], yb[:rows, off + 2:off + 2 + n]
                    r = S.block_norm(x, b, g, EPS, rows, post=post, gate=gate, scale=0.5, h=h, y=y)
                    assert r.h is h and r.y is y
                    wh, wy, eh, ey = formula(x, b, g, post, gate, 0.5)
                    near(h, wh, eh, "h")
                    near(y, wy, ey, "y")
                    h.fill_(77.0), y.fill_(77.0)
                    assert bool((hb == 77.0).all()) and bool((yb == 77.0).all()), "written beside the outputs"


def test_in_place_and_parts(S):
    for n in (256, 4096, 10000):
        x, b, g = real(1, 33, n).to(BF16), real(2, 33, n).to(BF16), real(3, n)
        wh, wy, eh, ey = formula(x, b, g)
        keep = x.clone()
        r = S.block_norm(x, b, g, EPS, 33, h=x)
        assert r.h is x
        near(x, wh, eh, "h in place")
        near(r.y, wy, ey, "y in place")
        r = S.block_norm(keep, b, None, EPS, 33)             # no norm behind
        assert r.y is None
        near(r.h, wh, eh, "h alone")
        r = S.block_norm(keep, None, g, EPS, 33, dtype=F16)  # no branch before
        assert r.h is keep
        near(r.y, *formula(keep, None, g)[1::2], "y alone")
        part = S.block_norm(keep, b, g, EPS, 5)              # the first rows
        assert part.h.shape == part.y.shape == (5, n)
        near(part.h, wh[:5], eh[:5], "the first rows")


def test_special_values(S):
    n = 1000
    x, b, g = real(1, 6, n), real(2, 6, n), real(3, n)
    x[0], b[0] = 0.0, 0.0                      # a row of nothing: 0 / sqrt(eps)
    x[1, 3] = float("inf")
    b[2, 999] = float("nan")
    b[3] = 1e15
    b[4] = 1e-30
    h, y = S.block_norm(x, b, g, EPS, 6, post=g)
    wh, wy, eh, ey = formula(x, b, g, g)
    assert bool((y[0] == 0).all()) and bool((h[0] == 0).all())
    assert bool(torch.isnan(h[2]).all()) and bool(torch.isnan(y[2]).all())
    assert float(h[1, 3]) == float("inf") and bool(torch.isnan(y[1, 3]))
    rest = [i for i in range(n) if i != 3]
    assert bool((y[1, rest] == 0).all())
    for r in (3, 4, 5):
        near(h[r], wh[r], eh[r], f"h {r}")
        near(y[r], wy[r], ey[r], f"y {r}")
    assert S.block_norm(x[:0], b[:0], g, EPS, 0).y.shape == (0, n)


def test_captured_and_replayed_on_another_stream(S):
    x, b, g, post = real(1, 9, 4096).to(BF16), real(2, 9, 4096).to(BF16), real(3, 4096), real(4, 4096)
    h, y = torch.empty_like(x), torch.empty_like(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    S.block_norm(x, b, g, EPS, 9, post=post, h=h, y=y, stream=side)
    torch.cuda.synchronize()
    want = S.block_norm(x, b, g, EPS, 9, post=post)
    assert torch.equal(h, want.h) and torch.equal(y, want.y)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        S.block_norm(x, b, g, EPS, 9, post=post, h=h, y=y)
    for i in range(4):
        b.copy_(real(20 + i, 9, 4096))
        graph.replay()
        got = h.clone(), y.clone()
        torch.cuda.synchronize()
        want = S.block_norm(x, b, g, EPS, 9, post=post)
        assert torch.equal(got[0], want.h) and torch.equal(got[1], want.y), i

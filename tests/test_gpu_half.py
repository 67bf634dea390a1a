"""The half-precision product with its epilogue against its formula in 64 bits.  Over whole numbers the sums are
exact in F32 whatever their order, so that outputs are equal or off by the epilogue's roundings alone; over real ones
a sum of K products is within (K + 8) U of the sum of their magnitudes (the products of 8- and 11-bit significands
are exact in F32)."""
import numpy as np
import pytest
import torch

from gpu_util import announce, require_gpu

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.fixture(scope="module")
def H():
    require_gpu()
    import syntropy_amd.half as H
    return H


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def whole(seed, most, *shape):
    return torch.randint(-most, most + 1, shape, generator=gen(seed), device="cuda").float()


def real(seed, *shape):
    return torch.randn(*shape, generator=gen(seed), device="cuda")


def activation(act, v):
    return {"none": lambda: v, "relu": lambda: torch.where(v < 0, 0.0, v), "silu": lambda: v / (1 + torch.exp(-v)),
            "gelu": lambda: 0.5 * v * torch.special.erfc(-v / 2 ** 0.5),
            "gelu_tanh": lambda: v / (1 + torch.exp(-2 * (2 / np.pi) ** 0.5 * (v + 0.044715 * v ** 3)))}[act]()


def formula(w, x, bias=None, act="none", gate=None, residual=None):
    """(y in 64 bits, the sum of the magnitudes of a sum's products)"""
    x, w = x.double().cpu(), w.double().cpu()
    v = x @ w.T
    if bias is not None:
        v = v + bias.double().cpu()
    v = activation(act, v)
    if gate is not None:
        v = v * gate.double().cpu()
    if residual is not None:
        v = v + residual.double().cpu()
    return v, x.abs() @ w.abs().T


def same(got, want, what):
    """Equal to the 64-bit value rounded once."""
    g, w = got.cpu(), want.to(got.dtype)
    if not torch.equal(g, w):
        bad = torch.nonzero(g != w)
        i = tuple(bad[0].tolist())
        raise AssertionError(f"{what}: {len(bad)} of {g.numel()} differ; first at {i}: {g[i]} for {w[i]}")


def near(got, want, err, what):
    """Within err (of the F32 value) and half a step of the output's type, and the least step where it is subnormal."""
    t = got.dtype
    g = got.cpu().double()
    tol = err + (torch.finfo(t).eps / 2) * (want.abs() + err) + torch.finfo(t).smallest_normal * torch.finfo(t).eps
    off = (g - want).abs()
    assert bool(torch.isfinite(g).all()), f"{what}: {int((~torch.isfinite(g)).sum())} are not finite"
    assert bool((off <= tol).all()), f"{what}: off by {float((off / tol).max()):.3g} of what it may be"


# n, k, rows: one and few rows, the borders of what a tile, a line and a turn hold, odd ones, several tiles each way
SHAPES = [(1, 1, 1), (1, 64, 1), (7, 3, 2), (16, 64, 1), (33, 65, 3), (130, 640, 5), (64, 2048, 8), (257, 130, 9), (1000, 4096, 1),
          (96, 192, 16), (300, 1000, 17), (512, 1024, 31), (130, 8192, 33), (65, 63, 64), (1027, 320, 65), (256, 512, 128),
          (384, 257, 129), (520, 1344, 200), (1500, 704, 257), (72, 14336, 40), (2100, 448, 300), (4096, 192, 513)]
# each tile, over whole K and over many parts of it
SHAPES += [(12957, 81, 417), (6114, 6461, 129), (8306, 37, 132), (2754, 5090, 66), (8203, 36, 36), (76, 5898, 1370), (8776, 167, 33),
           (101, 5689, 1406), (8324, 52, 9), (34, 5633, 738), (2982, 5916, 30), (33, 2878, 14), (4096, 256, 7), (4096, 193, 5)]


@pytest.mark.parametrize("ty", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("n,k,rows", SHAPES)
def test_whole_numbers_are_exact(H, ty, n, k, rows):
    announce(f"half whole {n} {k} {rows} {ty}")
    w, x = whole(1, 3, n, k).to(ty), whole(2, 3, rows, k).to(ty)
    bias = whole(3, 9, n) / 4
    gate, res = whole(4, 3, rows, n).to(ty), whole(5, 20, rows, n)
    W = H.Weights(w, bias)
    for kw in (dict(dtype=F32), dict(gate=gate, residual=res, dtype=F32), dict(act="relu", residual=res.to(ty))):
        y = H.gemv(W, x, rows, **kw)
        want, _ = formula(w, x, bias, **{a: b for a, b in kw.items() if a != "dtype"})
        assert float(want.abs().max()) < 2 ** 21  # quarters below it are exact in F32
        same(y, want, f"{kw.keys()}")


@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("n,k,rows", [(300, 1000, 1), (130, 2048, 6), (300, 1000, 12), (500, 960, 40), (777, 1280, 270)])
def test_real_numbers(H, act, n, k, rows):
    announce(f"half real {act} {n} {k} {rows}")
    w, x = (0.05 * real(1, n, k)).to(BF16), real(2, rows, k).to(BF16)
    bias, gate, res = real(3, n), real(4, rows, n).to(F16), real(5, rows, n).to(BF16)
    y = H.gemv(H.Weights(w, bias), x, rows, act=act, gate=gate, residual=res, dtype=F32)
    want, mag = formula(w, x, bias, act, gate, res)
    v = formula(w, x, bias)[0]
    e = (k + 8) * U * mag + U * v.abs()          # of the sum and the bias
    f = activation(act, v).abs()
    slope = 1.2                                  # the steepest of the activations is 1.13
    e = slope * e + 2.0 ** -20 * f               # each within 2^-20
    near(y, want, gate.cpu().double().abs() * (e + U * f) + U * (want.abs() + 1), f"{act}")


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
def test_activations_far_and_near(H, act):
    """One weight of 1 a row: the activation of the bias (exact), from -100 to 100 and the smallest numbers."""
    v = torch.cat([torch.linspace(-100, 100, 4001), torch.linspace(-12.9, 6, 4001),
                   torch.tensor([0.0, 2.0 ** -126, -2.0 ** -100, 1e-20, -1e-10, 1e-5, 1e4, 1e30, -1e4, -1e30, -180.5, -300.0])]).cuda()
    W = H.Weights(torch.zeros(len(v), 64, dtype=BF16, device="cuda"), v)
    for rows in (1, 40):
        y = H.gemv(W, torch.ones(rows, 64, dtype=BF16, device="cuda"), rows, act=act, dtype=F32)
        want = activation(act, v.cpu().double())
        want = torch.where(torch.isnan(want), 0.0, want)  # (where the formula's exponential passes 64 bits)
        # within 2^-19.  An exponential's argument z is exact to 2^-24 of a part that is itself 2^-24 of z.
        near(y, want.expand(rows, -1), 2.0 ** -19 * want.abs().expand(rows, -1) + 2.0 ** -146, act)


def test_infinities_and_nans_stay_in_their_rows(H):
    n, k, rows = 200, 200, 50
    for ty in (BF16, F16):
        w, x = whole(1, 3, n, k).to(ty), whole(2, 3, rows, k).to(ty)
        w[5, 7], x[:, 7] = float("inf"), 1.0
        w[9, 199] = float("nan")
        x[3, 199], x[4, 0] = float("inf"), float("nan")
        w[:, 199] = torch.where(w[:, 199] == 0, 1.0, w[:, 199])
        for r in (3, 9, rows):
            y = H.gemv(H.Weights(w), x, r, dtype=F32).cpu().double()
            want = formula(w, x[:r])[0]
            assert torch.equal(torch.isnan(y), torch.isnan(want))
            y, want = torch.nan_to_num(y, 0.0), torch.nan_to_num(want, 0.0)
            assert torch.equal(y, want), (ty, r)


def test_strides_offsets_and_types(H):
    """Rows apart, at odd addresses, operands and outputs of each type; what lies between and behind stays."""
    n, k = 301, 192
    for rows in (2, 11, 70):
        w = whole(1, 3, n, k).to(F16)
        wide = torch.zeros(n, 320, dtype=F16, device="cuda")
        wide[:, 64:64 + k] = w
        for W in (H.Weights(w), H.Weights(wide[:, 64:64 + k]), H.Weights(w.t().contiguous().t())):
            for off in (0, 1, 8):
                xb = torch.full((rows, k + 77), float("nan"), dtype=F16, device="cuda")
                x = xb[:, off:off + k]
                x.copy_(whole(2, 3, rows, k))
                for i, t in enumerate((F32, F16, BF16)):
                    gt, rt = (F16, BF16, F32)[i], (BF16, F32, F16)[i]
                    gate = torch.zeros(rows, n + 5, dtype=gt, device="cuda")[:, 3:3 + n].copy_(whole(3, 2, rows, n))
                    res = torch.zeros(rows, n + 9, dtype=rt, device="cuda")[:, 1:1 + n].copy_(whole(4, 2, rows, n))
                    yb = torch.full((rows + 1, n + 13), 77.0, dtype=t, device="cuda")
                    y = yb[:rows, 5:5 + n]
                    assert H.gemv(W, x, rows, gate=gate, residual=res, y=y) is y
                    same(y, formula(w, x, None, "none", gate, res)[0], f"{rows} {off} {t}")
                    yb[:rows, 5:5 + n] = 77.0
                    assert bool((yb == 77.0).all()), "written beside y"


def test_the_residual_or_the_gate_may_be_the_output(H):
    for rows in (1, 7, 14, 40, 300):
        for n, k in ((256, 512), (130, 4096)):
            w, x, r = whole(1, 2, n, k).to(BF16), whole(2, 1, rows, k).to(BF16), whole(3, 9, rows, n)
            W, want, gated = H.Weights(w), formula(w, x, residual=r)[0], formula(w, x, gate=r)[0]
            y = r.clone()
            assert H.gemv(W, x, rows, residual=y, y=y) is y
            same(y, want, "residual")
            y = r.clone()
            H.gemv(W, x, rows, gate=y, y=y)
            same(y, gated, "gate")


def test_no_rows(H):
    W = H.Weights(torch.ones(8, 64, dtype=F16, device="cuda"))
    assert H.gemv(W, torch.ones(0, 64, dtype=F16, device="cuda"), 0).shape == (0, 8)
    none = H.Weights(torch.ones(0, 64, dtype=F16, device="cuda"))
    assert H.gemv(none, torch.ones(3, 64, dtype=F16, device="cuda"), 3).shape == (3, 0)


def test_equal_calls_give_equal_outputs(H):
    """Whatever else runs: the order of the sums is the call's alone."""
    for n, k, rows in ((512, 8192, 24), (1024, 4096, 5), (700, 1000, 300)):
        w, x = real(1, n, k).to(BF16), real(2, rows, k).to(BF16)
        W = H.Weights(w)
        first = H.gemv(W, x, rows)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        other = torch.empty_like(first)
        for _ in range(5):
            H.gemv(W, x, rows, y=other, stream=side)
            assert torch.equal(first, H.gemv(W, x, rows))
        side.synchronize()
        assert torch.equal(first, other)


def test_captured_and_replayed(H):
    n, k = 640, 4096
    W = H.Weights(real(1, n, k).to(BF16), real(2, n))
    for rows in (1, 6, 14, 40, 130):
        x, res = real(3, rows, k).to(BF16), real(4, rows, n).to(BF16)
        y = torch.empty_like(res)
        H.gemv(W, x, rows, act="gelu", residual=res, y=y)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            H.gemv(W, x, rows, act="gelu", residual=res, y=y)
        for i in range(4):
            x.copy_(real(10 + i, rows, k))
            g.replay()
            got = y.clone()
            torch.cuda.synchronize()
            assert torch.equal(got, H.gemv(W, x, rows, act="gelu", residual=res)), (rows, i)

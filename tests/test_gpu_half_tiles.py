"""The epilogue of the half-precision product on each of its tiles: every activation, operand and output of every type,
in place, captured; against its formula in 64 bits.  Which tile a case takes is checked on the CPU
(test_block_forms.py)."""
import pytest
import torch

from gpu_util import announce, require_gpu
from test_gpu_half import activation, real, whole

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPES = [F32, F16, BF16]
# n, k, rows of each tile, 256 x 256 first, K in one part: what is left of a row of y behind whole pieces of 4 and of 8
# values is 1 and 5, 2, 3, 0, 0 and 4 values
CASES = [(12957, 81, 417), (8306, 37, 132), (8203, 36, 36), (8776, 167, 33), (8324, 52, 9), (300, 128, 40)]
tiles = pytest.mark.parametrize("n,k,rows", CASES, ids=[f"tile{i}" for i in range(len(CASES))])
types = pytest.mark.parametrize("ty", [BF16, F16], ids=["bf16", "f16"])


@pytest.fixture(scope="module")
def H():
    require_gpu()
    import syntropy_amd.half as H
    return H


def apart(t, off, more):
    """t's values in rows with `off` NaN before them and further ones behind."""
    rows, n = t.shape
    wide = torch.full((rows, off + n + more), float("nan"), dtype=t.dtype, device="cuda")
    return wide[:, off:off + n].copy_(t)


def same(got, want, what):
    w = want.to(got.dtype)
    if not torch.equal(got, w):
        bad = torch.nonzero(got != w)
        i = tuple(bad[0].tolist())
        raise AssertionError(f"{what}: {len(bad)} of {got.numel()} differ; first at {i}: {got[i]} for {w[i]}")


@tiles
@types
@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu", "gelu_tanh"])
def test_activations(H, n, k, rows, ty, act):
    """Bounds: a sum of K products and its bias is within (K + 8) U of the sum of the magnitudes and U of itself; no
    activation is steeper than 1.13, and each is within 2^-20 of its value; the product and the residual's sum take a
    step of U each, the output half a step of its type."""
    announce(f"half tiles {n} {k} {rows} {ty} {act}")
    w, x = (real(1, n, k) / k ** 0.5).to(ty), (2 * real(2, rows, k)).to(ty)
    bias, gate, res = real(3, n), real(4, rows, n).to(ty), real(5, rows, n).to(ty)
    W = H.Weights(w, bias)
    mag = x.double().abs() @ w.double().abs().T + bias.double().abs()
    v = x.double() @ w.double().T + bias.double()
    f = activation(act, v)
    e = 1.14 * ((k + 8) * U * mag + U * v.abs()) + 2.0 ** -20 * f.abs()
    gated = f * gate.double()
    eg = gate.double().abs() * e + U * gated.abs()
    for out in (F32, ty):
        for kw, want, err in ((dict(), f, e), (dict(gate=gate), gated, eg),
                              (dict(gate=gate, residual=res), gated + res.double(), eg + U * (gated + res.double()).abs())):
            y = H.gemv(W, x, rows, act=act, dtype=out, **kw)
            err = 1.01 * err
            tol = err + torch.finfo(out).eps / 2 * (want.abs() + err) + torch.finfo(out).smallest_normal * torch.finfo(out).eps
            off = (y.double() - want).abs()
            assert bool((off <= tol).all()), f"{out} {kw.keys()}: off by {float((off / tol).max()):.3g} of what it may be"


@tiles
@types
def test_operand_and_output_types(H, n, k, rows, ty):
    """Over whole numbers: sums, products and residual sums are exact in F32 (below 9 K 3 + 9 < 2^13), so that an output
    is the formula's value rounded once.  Strided rows at odd addresses; nothing beside them is written."""
    w, x, bias = whole(1, 3, n, k).to(ty), whole(2, 3, rows, k).to(ty), whole(3, 9, n)
    gate, res = whole(4, 3, rows, n), whole(5, 9, rows, n)
    W, xs = H.Weights(w, bias), apart(x, 1, 6)
    v = x.double() @ w.double().T + bias.double()
    for out in TYPES:
        base = torch.full((rows + 1, n + 13), 77.0, dtype=out, device="cuda")
        y = base[:rows, 5:5 + n]
        for gt in [None, *TYPES]:
            for rt in [None, *TYPES]:
                announce(f"half tiles {n} {k} {rows} {ty} out {out} gate {gt} residual {rt}")
                g, r = None if gt is None else apart(gate.to(gt), 3, 2), None if rt is None else apart(res.to(rt), 1, 8)
                want = torch.relu(v)
                want = want if g is None else want * g.double()
                want = want if r is None else want + r.double()
                assert H.gemv(W, xs, rows, act="relu", gate=g, residual=r, y=y) is y
                same(y, want, f"out {out} gate {gt} residual {rt}")
                y.fill_(77.0)
                assert bool((base == 77.0).all()), "written beside y"


@tiles
@types
def test_in_place(H, n, k, rows, ty):
    w, x, r = whole(1, 2, n, k).to(ty), whole(2, 1, rows, k).to(ty), whole(3, 9, rows, n)
    W, v = H.Weights(w), x.double() @ w.double().T
    other = whole(4, 3, rows, n).to(ty)
    for out in TYPES:
        announce(f"half tiles in place {n} {k} {rows} {ty} {out}")
        fresh = lambda: apart(r.to(out), 3, 2)  # noqa: E731
        y = fresh()
        H.gemv(W, x, rows, gate=other, residual=y, y=y)
        same(y, v * other.double() + r.double(), f"residual {out}")
        y = fresh()
        H.gemv(W, x, rows, gate=y, residual=other, y=y)
        same(y, v * r.double() + other.double(), f"gate {out}")
        y = fresh()
        H.gemv(W, x, rows, gate=y, residual=y, y=y)
        same(y, v * r.double() + r.double(), f"both {out}")


@tiles
def test_captured_and_replayed(H, n, k, rows):
    W = H.Weights(real(1, n, k).to(BF16), real(2, n))
    x, gate, res = real(3, rows, k).to(BF16), real(4, rows, n).to(BF16), real(5, rows, n)
    y = H.gemv(W, x, rows, act="silu", gate=gate, residual=res)
    torch.cuda.synchronize()
    announce(f"half tiles captured {n} {k} {rows}")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        H.gemv(W, x, rows, act="silu", gate=gate, residual=res, y=y)
    for i in range(3):
        x.copy_(real(10 + i, rows, k))
        g.replay()
        got = y.clone()
        torch.cuda.synchronize()
        assert torch.equal(got, H.gemv(W, x, rows, act="silu", gate=gate, residual=res)), i

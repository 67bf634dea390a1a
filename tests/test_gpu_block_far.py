"""The half-precision product, the norms between blocks and sampling at the ends of what they take: rows that lie past 32
bits of offset, and the longest rows."""
import numpy as np
import pytest
import torch

from gpu_util import announce, require_gpu
from test_gpu_half import formula, same, whole
from test_gpu_sample import check, real, uniform

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
APART = (1 << 28) + 8  # values: the ninth row begins past 2^31 of them, and 2^32 bytes of 16-bit ones


@pytest.fixture(scope="module")
def ops():
    require_gpu()
    import syntropy_amd.gemv as S
    import syntropy_amd.half as H
    return S, H


def far(rows, n, dtype):
    return torch.empty((rows - 1) * APART + n, dtype=dtype, device="cuda").as_strided((rows, n), (APART, 1))


def test_products_of_rows_far_apart(ops):
    _, H = ops
    n, k, rows = 200, 256, 10
    w, x, gate, res = whole(1, 3, n, k).to(F16), whole(2, 3, rows, k).to(F16), whole(3, 3, rows, n).to(F16), whole(4, 9, rows, n).to(F16)
    W, want = H.Weights(w), formula(w, x, None, "relu", gate, res)[0]
    xf, yf, gf, rf = far(rows, k, F16).copy_(x), far(rows, n, F16), far(rows, n, F16).copy_(gate), far(rows, n, F16).copy_(res)
    for xs in (x, xf):
        announce(f"half far {xs.stride()}")
        yf.fill_(-1.0)
        H.gemv(W, xs, rows, act="relu", gate=gf, residual=rf, y=yf)
        same(yf, want, "far")
    y = H.gemv(W, xf, 3, act="relu", gate=gate, residual=res)
    same(y, want[:3], "few")
    wide = far(n // 20, k, F16).copy_(w[:n // 20])     # weight rows as far apart
    y = H.gemv(H.Weights(wide), x, rows, dtype=F32)
    same(y, formula(w[:n // 20], x)[0], "weights")


def test_norms_of_rows_far_apart(ops):
    S, _ = ops
    rows, n = 9, 600
    x, b, gate, g = real(1, rows, n).to(F16), real(2, rows, n).to(F16), real(3, rows, n).to(F16), real(4, n)
    want = S.block_norm(x, b, g, 1e-5, rows, gate=gate)
    hf, yf = far(rows, n, F16), far(rows, n, F16)
    got = S.block_norm(far(rows, n, F16).copy_(x), far(rows, n, F16).copy_(b), g, 1e-5, rows, gate=far(rows, n, F16).copy_(gate), h=hf, y=yf)
    assert torch.equal(got.h, want.h) and torch.equal(got.y, want.y)


@pytest.mark.parametrize("n", [3000, 70000])
def test_samples_of_rows_far_apart(ops, n):
    S, _ = ops
    x = (2 * real(1, 9, n)).to(F16)
    for kw in (dict(top_p=0.9), dict(top_k=30)):
        want, got = S.sample_tokens(x, uniform(2, 9), **kw), S.sample_tokens(far(9, n, F16).copy_(x), uniform(2, 9), **kw)
        assert all(torch.equal(a, b) for a, b in zip(got, want)), kw


def test_the_longest_sums(ops):
    _, H = ops
    n, k = 70, 1 << 20
    w = whole(1, 1, n, k).to(BF16)
    W = H.Weights(w)
    for rows in (3, 40):
        announce(f"half longest {rows}")
        x = whole(2, 1, rows, k).to(BF16)
        same(H.gemv(W, x, rows, dtype=F32), formula(w, x)[0], f"{rows}")  # (below 2^20: exact in F32 in any order)


def test_the_longest_logits(ops):
    S, _ = ops
    x = 2 * real(1, 1, 1 << 24)
    x[0, np.random.default_rng(0).integers(0, 1 << 24, 9)] = 13.0
    for kw in (dict(top_k=40, top_p=0.9), dict(top_p=0.8), dict(temperature=0.3)):
        announce(f"sample longest {kw}")
        check(S, x, uniform(3, 1), what=f"{kw}", **kw)

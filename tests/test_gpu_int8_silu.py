"""The gate of the int8 products over all of F32: gate_up_act's silu(g) u at given g and u against the
formula in 64 bits.  A scale of 0 and a bias make a channel's value the bias whatever its codes, so that every
gate here is chosen.

What the steps of silu(g) = g / (1 + exp(-g)) may move it, U half a step of F32 relative to the value: the
exponential two U (an instruction within a step), the factor beside it and their product one each, the sum
one, the reciprocal two, the product one: 8 U = 2^-21, the stated bound.  A subnormal result is rounded once more, by 2^-150.  The
product with u adds its own rounding."""
import numpy as np
import pytest
import torch

from gpu_util import announce, require_gpu

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.fixture(scope="module")
def I():
    require_gpu()
    import syntropy_amd.int8 as I
    return I


def gates():
    rng = np.random.default_rng(3)
    near = [c + d for c in (-110, -104, -103.5, -96, -91.9, -88.73, -88, -87.4, -64, -17, 0, 17, 64, 88, 100)
            for d in np.linspace(-0.6, 0.6, 41)]
    some = np.concatenate([np.linspace(-125, 110, 1400), rng.normal(0, 4, 300), -np.exp(rng.uniform(-100, 88, 80)), near])
    ends = [0.0, -0.0, np.inf, -np.inf, np.nan, 3e38, -3e38, 1e-45, -1e-45, 1.2e-38, -1.2e-38, -2.0 ** 64]
    g = np.concatenate([some, ends]).astype(np.float32)
    return g[rng.permutation(len(g))]


# (gates apart, values of K, rows): rows quantized in the product's workgroups, ready rows, tiles, K in parts
@pytest.mark.parametrize("every,k,rows", [(1, 64, 1), (1, 64, 12), (1, 100, 40), (1, 64, 300), (5, 8192, 100)])
@pytest.mark.parametrize("up", [1.0, -1.5 * 2.0 ** 60])
def test_silu_of_any_gate(I, every, k, rows, up):
    g = gates()[::every]
    u = np.full_like(g, up)
    gen = torch.Generator().manual_seed(k)
    codes = torch.randint(-127, 128, (2 * len(g), -(-k // 16) * 16), generator=gen, dtype=torch.int8).cuda()[:, :k]
    W = I.Weights(codes, torch.zeros(2 * len(g), device="cuda"), torch.from_numpy(np.concatenate([g, u])).cuda())
    x = torch.randn(rows, k, generator=gen).cuda()
    announce(f"silu of {len(g)} gates, {rows} rows of {k}, up {up}")
    got = I.gate_up_act(W, x, rows).double().cpu().numpy()
    with np.errstate(all="ignore"):
        gd = g.astype(np.float64)
        s = gd / (1 + np.exp(-gd))  # (-infinity: a NaN, as the formula)
        want = s * up
        tol = (8 * U * np.abs(s) + 2.0 ** -150) * abs(up) * (1 + 2 * U) + U * np.abs(want) + 2.0 ** -150
        ok = (np.abs(got - want) <= tol) | (got == want) | (np.isnan(got) & np.isnan(want))
        ok |= (np.abs(want) + tol >= 2.0 ** 128 * (1 - U)) & np.isinf(got) & (np.sign(got) == np.sign(want))
    assert ok.all(), (f"{int((~ok).sum())} of {ok.size} out of tolerance: gates {np.unique(np.broadcast_to(g, ok.shape)[~ok])[:8]} "
                      f"{got[~ok][:4]} for {np.broadcast_to(want, ok.shape)[~ok][:4]}")

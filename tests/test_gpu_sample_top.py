"""The lists of a short top-k that are longer than a wavefront: near its greatest number, and where what is visible lies
in fewer groups of a row than k, so that the bound lets all of it pass."""
import pytest
import torch

from gpu_util import announce
from test_gpu_sample import F16, F32, BF16, S, check, real, uniform  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("ty", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,vocab", [(5, 1500), (5, 32064), (5, 128256)])
def test_top_k_near_a_wavefront(S, rows, vocab, ty):  # noqa: F811
    x = (2 * real(1, rows, vocab)).to(ty)
    x[1] -= 1000.0
    x[2, vocab // 2:] = 6.3
    for k in (60, 63, 64):
        for kw in (dict(), dict(temperature=0.02), dict(temperature=2.0 ** 40), dict(top_p=0.9), dict(min_p=0.2)):
            announce(f"sample top {rows} {vocab} {ty} {k} {kw}")
            check(S, x, uniform(k, rows), top_k=k, what=f"{k} {kw}", **kw)


@pytest.mark.parametrize("ty", [F32, F16], ids=["f32", "f16"])
@pytest.mark.parametrize("rows", [3, 140])
def test_few_groups(S, rows, ty):  # noqa: F811
    """What is visible every 256 pieces of 16 bytes: one group's, and all of it is listed."""
    vocab, per = 300001, 4 if ty == F32 else 8
    x = (2 * real(1, 3, vocab)).to(ty)
    x[1] = (x[1] / 512).to(ty)     # (near to one another)
    x[2] = 0.1                     # (equal)
    x[:, torch.arange(vocab, device="cuda") // per % 256 != 0] = -float("inf")
    u = uniform(2, 3)
    n = -(-rows // 3)
    for kw in (dict(top_k=64), dict(top_k=3), dict(top_k=50, top_p=0.47, temperature=0.01), dict(top_k=64, temperature=1e6)):
        announce(f"sample few groups {rows} {ty} {kw}")
        check(S, x, u, what=f"{kw}", **kw)
        few, many = S.sample_tokens(x, u, **kw), S.sample_tokens(x.repeat(n, 1), u.repeat(n), **kw)
        assert all(torch.equal(a.repeat(n), b) for a, b in zip(few, many)), kw

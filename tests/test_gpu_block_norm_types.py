"""The norms between two blocks by every pair of a stream's and a branch's type over every split of a row, against
their formula in 64 bits.  That these cases are every form of the kernel is checked on the CPU (test_block_forms.py)."""
import itertools

import pytest
import torch

from gpu_util import announce
from test_gpu_block_norm import BF16, EPS, F16, F32, S, formula, near, real  # noqa: F401

pytestmark = pytest.mark.gpu

TYPES = [F32, F16, BF16]
# (the stream's type, the branch's, a row's values): odd widths, up to what a form's wavefronts and pieces hold
CASES = list(itertools.product(TYPES, TYPES, [509, 1001, 2011, 4096, 8191, 12000, 32765]))


@pytest.mark.parametrize("tx,tb,n", CASES, ids=lambda v: str(v).replace("torch.", ""))
def test_types_of_every_split(S, tx, tb, n):  # noqa: F811
    rows = 7
    x, b = (3 * real(1, rows, n)).to(tx), real(2, rows, n).to(tb)
    g, post, gate = real(3, n), real(4, n), real(5, rows, n).to(tb)
    for i, kw in enumerate((dict(), dict(post=post, gate=gate, scale=0.3), dict(gate=gate[0], scale=-1.7))):
        ty = TYPES[i]
        announce(f"block_norm {tx} {tb} {n} {ty} {kw.keys()}")
        want = formula(x, b, g, **kw)
        h, y = S.block_norm(x, b, g, EPS, rows, dtype=ty, **kw)
        assert h.dtype == tx and y.dtype == ty
        near(h, want[0], want[2], f"h {kw.keys()}")
        near(y, want[1], want[3], f"y {kw.keys()}")
        own = x.clone()
        r = S.block_norm(own, b, g, EPS, rows, h=own, dtype=ty, **kw)
        assert r.h is own and torch.equal(own, h) and torch.equal(r.y, y), "in place"

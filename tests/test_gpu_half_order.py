"""The order of the half-precision product's sums, over real numbers, whose sums show it: the sizes' alone below strides of
2^22 values, and that of 8 rows where the rows of x or of the weights lie farther apart than a tile's offsets reach."""
import pytest
import torch

from gpu_util import announce, require_gpu
from test_gpu_half import formula, near, real

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture(scope="module")
def H():
    require_gpu()
    import syntropy_amd.half as H
    return H


def apart(t, stride):
    rows, n = t.shape
    return torch.empty((rows - 1) * stride + n, dtype=t.dtype, device="cuda").as_strided((rows, n), (stride, 1)).copy_(t)


@pytest.mark.parametrize("k", [256, 1024, 4096])
def test_rows_apart(H, k):
    n, rows = 40, 12
    w, x = real(1, n, k).to(BF16), real(2, rows, k).to(BF16)
    want, mag = formula(w, x)
    W = H.Weights(w)
    y = H.gemv(W, x, rows, dtype=F32)
    few = torch.cat([H.gemv(W, x[:6], 6, dtype=F32), H.gemv(W, x[6:], 6, dtype=F32)])
    for t in (y, few):
        near(t, want, (k + 8) * U * mag, "near rows")
    for stride in (k + 8, 1 << 20, (1 << 22) - 8):
        announce(f"half order {k} {stride}")
        assert torch.equal(H.gemv(W, apart(x, stride), rows, dtype=F32), y), stride
        assert torch.equal(H.gemv(H.Weights(apart(w, stride)), x, rows, dtype=F32), y), stride
    far = 1 << 25  # 2^31 bytes over the 32 rows of the smallest tile
    announce(f"half order {k} far")
    assert torch.equal(H.gemv(W, apart(x, far), rows, dtype=F32), few)
    assert torch.equal(H.gemv(H.Weights(apart(w, far)), x, rows, dtype=F32), few)
    # (x's rows are copied beside one another where they lie at odd places, however far apart)
    assert torch.equal(H.gemv(W, apart(x, far + 3), rows, dtype=F32), y)

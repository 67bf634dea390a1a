"""Matrices whose rows lie farther apart than the product's calls take them (2^30 values): copied, as others that do not
lie in whole lines."""
import pytest
import torch

from gpu_util import announce, require_gpu
from test_gpu_half import formula, same, whole

pytestmark = pytest.mark.gpu

F32, F16 = torch.float32, torch.float16


@pytest.mark.parametrize("n", [1, 2])
@pytest.mark.parametrize("stride", [1 << 30, (1 << 30) + 8])
def test_rows_very_far_apart(n, stride):
    require_gpu()
    import syntropy_amd.half as H
    k = 256
    w = whole(1, 3, n, k).to(F16)
    far = torch.empty((n - 1) * stride + k, dtype=F16, device="cuda").as_strided((n, k), (stride, 1)).copy_(w)
    W = H.Weights(far)
    assert W.matrix.stride(0) == (stride if stride == 1 << 30 else k)
    for rows in (1, 5, 20):
        announce(f"half weights {n} {stride} {rows}")
        x = whole(2, 3, rows, k).to(F16)
        same(H.gemv(W, x, rows, dtype=F32), formula(w, x)[0], f"{rows}")

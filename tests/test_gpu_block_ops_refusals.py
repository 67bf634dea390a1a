"""What the Python layer of the half-precision product, the norms between blocks and sampling refuses of device tensors."""
import pytest
import torch

from gpu_util import require_gpu

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def rows(n, k, t=torch.float32):
    return torch.zeros(n, k, dtype=t, device="cuda")


def test_refusals():
    require_gpu()
    import syntropy_amd.gemv as S
    import syntropy_amd.half as H
    w = H.Weights(rows(8, 64, F16))
    x, y = rows(4, 64, F16), rows(4, 8, F16)
    bad = [lambda: H.Weights(rows(8, 64)), lambda: H.Weights(rows(8, 64, F16)[0]), lambda: H.Weights(rows(8, 0, F16)),
           lambda: H.Weights(rows(8, 64, F16), rows(1, 8)[0].to(F16)), lambda: H.Weights(rows(8, 64, F16), rows(1, 9)[0]),
           lambda: H.gemv(w, x.to(BF16), 4), lambda: H.gemv(w, x.float(), 4), lambda: H.gemv(w, x, 5), lambda: H.gemv(w, x, -1),
           lambda: H.gemv(w, x[:, ::2], 4), lambda: H.gemv(w, x, 4, act="tanh"), lambda: H.gemv(w, x, 4, gate=y[:3]),
           lambda: H.gemv(w, x, 4, gate=y[:, :4]), lambda: H.gemv(w, x, 4, residual=y.to(torch.float64)),
           lambda: H.gemv(w, x, 4, y=y[:2]), lambda: H.gemv(w, x, 4, y=y, dtype=BF16), lambda: H.gemv(w, x, 4, dtype=torch.int8),
           lambda: H.gemv(w, x, 4, ws=torch.zeros(64, device="cuda")), lambda: H.gemv(w, x, 4, residual=y.cpu())]
    a, g = rows(4, 64), rows(1, 64)[0]
    bad += [lambda: S.block_norm(a, a[:3], g, 1e-5, 4), lambda: S.block_norm(a, a, g[:63], 1e-5, 4),
            lambda: S.block_norm(a, a, g.to(F16), 1e-5, 4), lambda: S.block_norm(a, a, g, 1e-5, 4, post=g[:63]),
            lambda: S.block_norm(a, a, g, 1e-5, 4, gate=a.to(F16)), lambda: S.block_norm(a, a, g, 1e-5, 4, gate=a[:2]),
            lambda: S.block_norm(a, a, g, 1e-5, 4, gate=g[:63]), lambda: S.block_norm(a, None, g, 1e-5, 4, post=g),
            lambda: S.block_norm(a, None, g, 1e-5, 4, gate=g), lambda: S.block_norm(a, None, None, 1e-5, 4),
            lambda: S.block_norm(a, a, g, 1e-5, 4, h=a.to(F16)), lambda: S.block_norm(a, a, g, 1e-5, 4, y=a, dtype=F16),
            lambda: S.block_norm(a, a, g, 1e-5, 5), lambda: S.block_norm(a, a.double(), g, 1e-5, 4),
            lambda: S.block_norm(a, a, g.cpu(), 1e-5, 4), lambda: S.block_norm(a, a.cpu(), g, 1e-5, 4)]
    u = torch.zeros(4, device="cuda")
    bad += [lambda: S.sample_tokens(a, u[:3]), lambda: S.sample_tokens(a, u.double()), lambda: S.sample_tokens(a.double(), u),
            lambda: S.sample_tokens(a, u.cpu()), lambda: S.sample_tokens(a, u, temperature=u[:2]), lambda: S.sample_tokens(a, u, top_k=u),
            lambda: S.sample_tokens(a, u, top_k=-1), lambda: S.sample_tokens(a, u, top_p=u.half()), lambda: S.sample_tokens(a[:, ::2], u),
            lambda: S.sample_tokens(a, u, min_p=u.cpu())]
    for i, call in enumerate(bad):
        with pytest.raises(S.GemvError):
            call()
            print("not refused:", i)
    worse = [dict(temperature=-1.0), dict(temperature=1e-30), dict(temperature=float("nan")), dict(top_p=0.0), dict(top_p=1.5),
             dict(min_p=-0.5), dict(min_p=2.0)]
    for kw in worse:
        with pytest.raises(S.SynError):
            S.sample_tokens(a, u, **kw)
    with pytest.raises(S.SynError):
        S.block_norm(rows(1, 40000), None, rows(1, 40000)[0], 1e-5, 1)
    torch.cuda.synchronize()

"""What the half-precision product, the norms between blocks and sampling refuse, through the C ABI and the Python
layer.  CPU only: a refused call reads no operand and enqueues nothing, so the pointers here are only numbers."""
import ctypes as C
import os

import pytest
import torch

from syntropy_amd import _lib

pytestmark = pytest.mark.skipif(not os.path.exists(_lib.LIB_PATH), reason="the library is not built")

INVALID, UNSUPPORTED, WORKSPACE = 1, 2, 3
F32, F16, BF16 = 0, 1, 30
A = 1 << 20  # an address on every alignment that is asked for
INF, NAN = float("inf"), float("nan")


def rc(name, *args):
    return getattr(_lib.lib(), name)(*args)


def message():
    return _lib.lib().syn_last_error().decode()


def name_of(b):
    return "-".join(f"{k}={v}" for k, v in b.items()) if isinstance(b, dict) else str(b)


def half(**o):
    d = dict(wtype=BF16, w=A, w_bytes=1 << 30, w_stride=256, bias=A, n=8, k=200, x=A, xs=200, rows=40, act=2, gtype=F16, gate=A,
             gs=8, rtype=F32, res=A, rs=8, ytype=F32, y=A, ys=8, ws=A, ws_bytes=1 << 24)
    assert set(o) <= set(d)
    return rc("syn_half_gemv", *{**d, **o}.values(), None)


@pytest.mark.parametrize("bad,code", [
    (dict(wtype=F32), UNSUPPORTED), (dict(wtype=8), UNSUPPORTED), (dict(w=0), INVALID), (dict(w=A + 8), INVALID),
    (dict(w_stride=255), INVALID), (dict(w_stride=252), INVALID), (dict(w_stride=200), INVALID), (dict(w_stride=248), INVALID),
    (dict(w_stride=1 << 31), INVALID), (dict(w_bytes=2 * 8 * 256 - 1), INVALID), (dict(bias=A + 2), INVALID), (dict(k=0), UNSUPPORTED),
    (dict(k=(1 << 20) + 1, w_stride=1 << 21), UNSUPPORTED), (dict(n=1 << 24), UNSUPPORTED), (dict(rows=2097121), UNSUPPORTED),
    (dict(x=0), INVALID), (dict(x=A + 1), INVALID), (dict(xs=199), INVALID), (dict(xs=1 << 41), INVALID), (dict(act=5), UNSUPPORTED),
    (dict(act=-1), UNSUPPORTED), (dict(gtype=12), UNSUPPORTED), (dict(gate=A + 1), INVALID), (dict(gs=7), INVALID),
    (dict(rtype=-1), UNSUPPORTED), (dict(res=A + 2), INVALID), (dict(rs=0), INVALID), (dict(ytype=2), UNSUPPORTED), (dict(y=0), INVALID),
    (dict(y=A + 2), INVALID), (dict(ys=7), INVALID)], ids=name_of)
def test_product_refuses(bad, code):
    assert half(**bad) == code, message()
    assert "syn_half_gemv" in message()


@pytest.mark.parametrize("rows", [1, 8, 40, 1000])
def test_product_workspaces(rows):
    """A copy of x's rows where they are not whole lines; a workspace that is too small or not there is refused."""
    out = C.c_uint64()
    query = lambda *a: rc("syn_half_gemv_workspace_bytes", *a, C.byref(out))  # noqa: E731
    assert query(8, 200, rows, 0) == 0
    need = out.value
    if need:
        assert half(rows=rows, ws=0) == INVALID and half(rows=rows, ws=A + 128) == INVALID
        assert half(rows=rows, ws_bytes=need - 1) == WORKSPACE
    assert query(8, 200, rows, 1) == 0 and out.value == need  # (200 values are no whole lines)
    assert query(8, 256, rows, 0) == 0
    apart = out.value
    assert query(8, 256, rows, 1) == 0 and out.value <= apart
    assert query(8, 0, rows, 0) == UNSUPPORTED and query(1 << 24, 64, rows, 0) == UNSUPPORTED
    assert rc("syn_half_gemv_workspace_bytes", 8, 64, rows, 0, None) == INVALID
    assert query(8, 64, 0, 0) == 0 and out.value == 0
    assert query(0, 64, rows, 0) == 0 and out.value == 0


def norm(**o):
    d = dict(xtype=BF16, x=A, xs=100, btype=F16, branch=A, bs=100, post=A, gate=A, gs=100, scale=0.5, g=A, eps=1e-5, rows=3, n=100, h=A,
             hs=100, ytype=F32, y=A, ys=100)
    assert set(o) <= set(d)
    return rc("syn_block_norm", *{**d, **o}.values(), None)


@pytest.mark.parametrize("bad,code", [
    (dict(n=0), UNSUPPORTED), (dict(n=32769), UNSUPPORTED), (dict(rows=1 << 24), UNSUPPORTED), (dict(xtype=8), UNSUPPORTED),
    (dict(x=0), INVALID), (dict(x=A + 1), INVALID), (dict(xs=99), INVALID), (dict(btype=2), UNSUPPORTED), (dict(branch=A + 1), INVALID),
    (dict(bs=99), INVALID), (dict(post=A + 2), INVALID), (dict(gate=A + 1), INVALID), (dict(gs=99), INVALID), (dict(g=A + 1), INVALID),
    (dict(h=0), INVALID), (dict(h=A + 1), INVALID), (dict(hs=99), INVALID), (dict(ytype=-1), UNSUPPORTED), (dict(y=0), INVALID),
    (dict(y=A + 2), INVALID), (dict(ys=99), INVALID), (dict(branch=0), INVALID), (dict(branch=0, post=0), INVALID),
    (dict(branch=0, post=0, gate=0, g=0), INVALID), (dict(branch=0, gate=0), INVALID)], ids=name_of)
def test_norm_refuses(bad, code):
    assert norm(**bad) == code, message()
    assert "syn_block_norm" in message()


def sample(**o):
    d = dict(xtype=F32, x=A, xs=50, rows=3, vocab=50, u=A, ts=0, ks=0, ps=0, ms=0, t=1.0, k=0, p=1.0, m=0.0, token=A, logprob=A, kept=A,
             ws=A, ws_bytes=1 << 30)
    assert set(o) <= set(d)
    return rc("syn_sample_tokens", *{**d, **o}.values(), None)


@pytest.mark.parametrize("bad,code", [
    (dict(xtype=2), UNSUPPORTED), (dict(vocab=0), INVALID), (dict(vocab=(1 << 24) + 1), UNSUPPORTED), (dict(rows=1 << 24), UNSUPPORTED),
    (dict(x=0), INVALID), (dict(x=A + 2), INVALID), (dict(xs=49), INVALID), (dict(u=0), INVALID), (dict(u=A + 2), INVALID),
    (dict(ts=A + 1), INVALID), (dict(ks=A + 2), INVALID), (dict(ps=A + 2), INVALID), (dict(ms=A + 2), INVALID), (dict(t=-1.0), INVALID),
    (dict(t=1e-30), INVALID), (dict(t=1e30), INVALID), (dict(t=NAN), INVALID), (dict(t=INF), INVALID), (dict(k=-1), INVALID),
    (dict(p=0.0), INVALID), (dict(p=1.5), INVALID), (dict(p=NAN), INVALID), (dict(m=-0.1), INVALID), (dict(m=1.5), INVALID),
    (dict(m=NAN), INVALID), (dict(token=0), INVALID), (dict(logprob=0), INVALID), (dict(kept=0), INVALID), (dict(token=A + 2), INVALID),
    (dict(logprob=A + 1), INVALID), (dict(kept=A + 2), INVALID)], ids=name_of)
def test_sampling_refuses(bad, code):
    assert sample(**bad) == code, message()
    assert "syn_sample_tokens" in message()


def test_sampling_workspaces():
    out = C.c_uint64()
    for ty in (F32, F16, BF16):
        for rows, vocab in ((1, 128256), (24, 128256), (300, 1 << 24), (3, 50)):
            assert rc("syn_sample_tokens_workspace_bytes", ty, rows, vocab, C.byref(out)) == 0
            if out.value:
                o = dict(xtype=ty, rows=rows, vocab=vocab, xs=vocab)
                assert sample(**o, ws=0) == INVALID and sample(**o, ws=A + 16) == INVALID
                assert sample(**o, ws_bytes=out.value - 1) == WORKSPACE
    assert rc("syn_sample_tokens_workspace_bytes", F32, 0, 50, C.byref(out)) == 0 and out.value == 0
    assert rc("syn_sample_tokens_workspace_bytes", F32, 3, 0, C.byref(out)) == INVALID
    assert rc("syn_sample_tokens_workspace_bytes", 12, 3, 50, C.byref(out)) == UNSUPPORTED
    assert rc("syn_sample_tokens_workspace_bytes", F32, 3, 50, None) == INVALID


def test_nothing_to_do_is_no_error():
    assert half(rows=0, ws=0) == 0 and half(n=0, ws=0) == 0 and norm(rows=0) == 0 and sample(rows=0, u=0) == 0


def test_the_python_layer_refuses():
    import syntropy_amd.gemv as S
    import syntropy_amd.half as H
    x = torch.zeros(4, 64)
    with pytest.raises(S.GemvError):
        H.Weights(torch.zeros(8, 64, dtype=torch.float16))          # not on a device
    with pytest.raises(S.GemvError):
        S.block_norm(x, x, torch.ones(64), 1e-5, 4)
    with pytest.raises(S.GemvError):
        S.block_norm(x, None, None, 1e-5, 4)
    with pytest.raises(S.GemvError):
        S.sample_tokens(x, torch.zeros(4))
    with pytest.raises(S.GemvError):
        S.sample_tokens(x, torch.zeros(3))
    with pytest.raises(S.GemvError):
        S.sample_tokens(x[0], torch.zeros(64))

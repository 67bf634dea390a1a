"""What the int8 products and the log probabilities refuse, through the C ABI and the Python layer.  CPU only: a
refused call reads no operand and enqueues nothing, so the pointers here are only numbers."""
import ctypes as C
import os

import pytest
import torch

from syntropy_amd import _lib

pytestmark = pytest.mark.skipif(not os.path.exists(_lib.LIB_PATH), reason="the library is not built")

INVALID, UNSUPPORTED, WORKSPACE = 1, 2, 3
F32, F16, BF16 = 0, 1, 30
A = 1 << 20  # an address on every alignment that is asked for


def rc(name, *args):
    return getattr(_lib.lib(), name)(*args)


def message():
    return _lib.lib().syn_last_error().decode()


def gemv(name="syn_i8_gemv", **o):
    d = dict(w=A, w_bytes=1 << 30, w_stride=256, scales=A, bias=0, n=8, k=256, xtype=F32, x=A, xs=256, rows=40, ytype=F32,
             y=A, ys=8, ws=A, ws_bytes=1 << 20)
    assert set(o) <= set(d)
    return rc(name, *{**d, **o}.values(), None)


BAD = [
    (dict(w=0), INVALID), (dict(w=A + 8), INVALID), (dict(w_stride=255), INVALID), (dict(w_stride=240), INVALID),
    (dict(w_stride=264), INVALID), (dict(w_stride=1 << 31), INVALID), (dict(scales=0), INVALID),
    (dict(scales=A + 2), INVALID), (dict(bias=A + 1), INVALID), (dict(k=0), UNSUPPORTED),
    (dict(k=131073, w_stride=131088), UNSUPPORTED), (dict(xtype=8), UNSUPPORTED), (dict(xtype=-1), UNSUPPORTED),
    (dict(ytype=12), UNSUPPORTED), (dict(x=0), INVALID), (dict(x=A + 2), INVALID), (dict(x=A + 1, xtype=F16), INVALID),
    (dict(xs=255), INVALID), (dict(xs=1 << 41), INVALID), (dict(y=0), INVALID), (dict(y=A + 1, ytype=BF16), INVALID),
    (dict(ys=7), INVALID), (dict(ws=0), INVALID), (dict(ws=A + 128), INVALID), (dict(ws_bytes=100), WORKSPACE),
    (dict(rows=2097121), UNSUPPORTED), (dict(n=1 << 24), UNSUPPORTED),
]


@pytest.mark.parametrize("bad,code", BAD, ids=lambda b: "-".join(f"{k}={v}" for k, v in b.items()) if isinstance(b, dict) else str(b))
@pytest.mark.parametrize("name", ["syn_i8_gemv", "syn_i8_gate_up_act"])
def test_products_refuse(name, bad, code):
    assert gemv(name, **bad) == code, message()
    assert name in message()


def test_views_that_end_before_the_last_code():
    assert gemv(w_bytes=7 * 256 + 255) == INVALID and "view" in message()
    assert gemv("syn_i8_gate_up_act", w_bytes=15 * 256 + 255) == INVALID
    assert gemv(w_stride=272, w_bytes=7 * 272 + 255) == INVALID


def test_nothing_to_do_is_no_error():
    assert gemv(rows=0) == 0 and gemv(n=0) == 0
    assert rc("syn_i8_quantize", F32, A, 64, 0, 64, A, 128, A, None) == 0
    assert rc("syn_token_logprobs", F32, A, 50, 0, 50, A, 4, 1.0, 0, A, A, A, 0, 0, 0, 0, None) == 0


def test_workspace_queries():
    out = C.c_uint64()
    assert rc("syn_i8_gemv_workspace_bytes", 4096, 2011, 50, 0, C.byref(out)) == 0 and out.value >= 50 * 2048 + 200
    assert rc("syn_i8_gemv_quantized_workspace_bytes", 4096, 2011, 1, C.byref(out)) == 0 and out.value >= 2048 + 4
    assert rc("syn_i8_gemv_workspace_bytes", 4096, 2011, 1, 0, C.byref(out)) == 0 and out.value == 0
    assert rc("syn_i8_gemv_quantized_workspace_bytes", 4096, 131073, 1, C.byref(out)) == UNSUPPORTED
    assert rc("syn_i8_gemv_workspace_bytes", 4096, 0, 5, 0, C.byref(out)) == UNSUPPORTED
    assert rc("syn_i8_gemv_workspace_bytes", 4096, 2011, 5, 0, None) == INVALID
    assert rc("syn_i8_gemv_workspace_bytes", 1 << 23, 64, 5, 1, C.byref(out)) == UNSUPPORTED
    assert rc("syn_token_logprobs_workspace_bytes", F32, 4, 50, 65, C.byref(out)) == UNSUPPORTED
    assert rc("syn_token_logprobs_workspace_bytes", F32, 4, 0, 0, C.byref(out)) == INVALID
    assert rc("syn_token_logprobs_workspace_bytes", 2, 4, 50, 0, C.byref(out)) == UNSUPPORTED


@pytest.mark.parametrize("o,code", [(dict(codes=0), INVALID), (dict(codes=A + 8), INVALID), (dict(cs=264), INVALID),
                                    (dict(cs=240), INVALID), (dict(scales=0), INVALID), (dict(x=0), INVALID),
                                    (dict(xs=10), INVALID), (dict(ty=3), UNSUPPORTED), (dict(k=0), UNSUPPORTED),
                                    (dict(k=200000, cs=200000, xs=200000), UNSUPPORTED)])
def test_quantize_refuses(o, code):
    d = {**dict(ty=F32, x=A, xs=256, rows=2, k=256, codes=A, cs=256, scales=A), **o}
    assert rc("syn_i8_quantize", *d.values(), None) == code, message()


def test_the_halves_refuse():
    assert rc("syn_i8_act_quantize", F32, A, 256, 3, 256, A, 100, None) == WORKSPACE
    assert rc("syn_i8_act_quantize", F32, A, 256, 3, 256, A + 8, 1 << 20, None) == INVALID
    assert rc("syn_i8_gemv_quantized", A, 1 << 20, 256, A, 0, 8, 256, 3, F32, A, 8, A, 100, None) == WORKSPACE
    assert rc("syn_i8_gemv_quantized", A, 1 << 20, 250, A, 0, 8, 256, 3, F32, A, 8, A, 1 << 20, None) == INVALID


@pytest.mark.parametrize("o,code", [(dict(head=A + 4), INVALID), (dict(bytes=7 * 256), INVALID), (dict(stride=100), INVALID),
                                    (dict(g=0), INVALID), (dict(x=0), INVALID), (dict(y=0), INVALID),
                                    (dict(hidden=16400, stride=16400), UNSUPPORTED), (dict(wsb=256), WORKSPACE)])
def test_logits_refuse(o, code):
    d = {**dict(head=A, bytes=1 << 20, stride=256, scales=A, vocab=8, hidden=256, g=A, eps=1e-5, x=A, rows=2, y=A, ws=A,
                wsb=1 << 20), **o}
    assert rc("syn_i8_logits", *d.values(), None) == code, message()


@pytest.mark.parametrize("o,code", [
    (dict(ty=2), UNSUPPORTED), (dict(x=0), INVALID), (dict(x=A + 2), INVALID), (dict(xs=49), INVALID),
    (dict(tokens=0), INVALID), (dict(tokens=A + 4), INVALID), (dict(tb=2), UNSUPPORTED), (dict(scale=0.0), INVALID),
    (dict(scale=-1.0), INVALID), (dict(scale=float("nan")), INVALID), (dict(scale=float("inf")), INVALID),
    (dict(scale=2.0 ** -65), INVALID), (dict(scale=2.0 ** 65), INVALID), (dict(scale=3e38), INVALID),
    (dict(top=51), UNSUPPORTED), (dict(vocab=100, xs=100, top=65), UNSUPPORTED), (dict(vocab=0), INVALID), (dict(vocab=(1 << 30) + 1, xs=1 << 31), UNSUPPORTED), (dict(rows=1 << 24), UNSUPPORTED),
    (dict(ids=0), INVALID), (dict(lps=0), INVALID), (dict(lps=A + 2), INVALID), (dict(lp=0), INVALID),
    (dict(rank=0), INVALID), (dict(ent=0), INVALID)])
def test_logprobs_refuse(o, code):
    d = {**dict(ty=F32, x=A, xs=50, rows=3, vocab=50, tokens=A, tb=8, scale=1.0, top=5, lp=A, rank=A, ent=A, ids=A, lps=A,
                ws=A, wsb=1 << 20), **o}
    assert rc("syn_token_logprobs", *d.values(), None) == code, message()


def test_python_refuses_what_is_not_on_the_device():
    import syntropy_amd.gemv as S
    import syntropy_amd.int8 as I
    with pytest.raises(S.GemvError):
        I.Weights(torch.zeros(4, 16, dtype=torch.int8), torch.zeros(4))
    with pytest.raises(S.GemvError):
        I.quantize_rows(torch.zeros(4, 16))
    with pytest.raises(S.GemvError):
        I.quantize_rows(torch.zeros(16))
    with pytest.raises(S.GemvError):
        S.token_logprobs(torch.zeros(4, 16), torch.zeros(4, dtype=torch.int64))
    for bad in (torch.zeros(3, dtype=torch.int64), torch.zeros(4), torch.zeros(4, 1, dtype=torch.int64)):
        with pytest.raises(S.GemvError):
            S.token_logprobs(torch.zeros(4, 16), bad)
    for top in (-1, 17, 65):
        with pytest.raises(S.GemvError):
            S.token_logprobs(torch.zeros(4, 16), torch.zeros(4, dtype=torch.int64), top=top)
    with pytest.raises(S.GemvError):
        S.token_logprobs(torch.zeros(4, 16, dtype=torch.float64), torch.zeros(4, dtype=torch.int64))

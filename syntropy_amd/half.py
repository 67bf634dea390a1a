"""Products over F16 or BF16 weights with an epilogue on the MI355X: activations of the weights' type, sums in F32,
then bias, activation, gate and residual before the one rounding.  Beside `gemv` (F32 activations, the reference's
order of sums, no epilogue) and `int8` (quantized inside); the reference has no such op.

    w = half.Weights(matrix, bias)                                # [n_out, k_in], bias F32 [n_out] or None
    h = half.gemv(w, x, rows, act="gelu")                         # act(x W^T + bias)
    y = half.gemv(up_gate, x, rows, act="silu", gate=up)          # silu(x W^T) * up, a gated feed-forward block
    x = half.gemv(down, h, rows, residual=x, y=x)                 # x + h W^T, in place

Every call runs the HIP kernels through the C ABI; there is no CPU path.
"""
from __future__ import annotations

from dataclasses import dataclass

import torch

from ._lib import SynError, call
from .gemv import GemvError, _current_device, _current_stream, _need, _on_stream, _ptr_width, _value_type

MAX_K = 1 << 20
ACTS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3, "gelu_tanh": 4}
_PAIR = 128  # values of two 128-byte lines
_MAX_STRIDE = 1 << 30


@dataclass(frozen=True, eq=False)
class Weights:
    """`matrix` F16 or BF16 [n_out, k_in] with an optional F32 `bias` [n_out], device tensors.  A matrix whose rows are
    whole pairs of 128-byte lines (k_in a multiple of 128) on 16 bytes, at most 2^30 values apart, is kept as it is; any
    other is copied once, here, into such rows with zeros behind the values."""

    matrix: torch.Tensor
    bias: torch.Tensor | None = None

    def __post_init__(self):
        w, b = self.matrix, self.bias
        if not (w.is_cuda and w.dtype in (torch.float16, torch.bfloat16) and w.dim() == 2):
            raise GemvError("Len", "the matrix must be an F16 or BF16 device tensor of rows")
        n_out, k_in = w.shape
        if not 1 <= k_in <= MAX_K:
            raise GemvError("RowLength", f"rows of {k_in} values (1 to {MAX_K})")
        if b is not None and (b.device != w.device or b.dtype != torch.float32 or not b.is_contiguous() or b.shape != (n_out,)):
            raise GemvError("Len", f"bias must be a contiguous F32 tensor of {n_out} values beside the matrix")
        if k_in % _PAIR or w.stride(1) != 1 or not k_in <= w.stride(0) <= _MAX_STRIDE or w.stride(0) % 8 or w.data_ptr() % 16:
            rows = torch.zeros(n_out, -(-k_in // _PAIR) * _PAIR, dtype=w.dtype, device=w.device)[:, :k_in]
            w = rows.copy_(w)
        stride = w.stride(0)
        row = -(-k_in // _PAIR) * _PAIR
        # the C ABI's arguments: type, the matrix's view (address, bytes, stride), bias
        view = (_value_type(w, "matrix"), w.data_ptr(), 2 * ((n_out - 1) * stride + row) if n_out else 0, stride,
                0 if b is None else b.data_ptr())
        for name, v in (("matrix", w), ("n_out", n_out), ("k_in", k_in), ("device", w.get_device()), ("view", view)):
            object.__setattr__(self, name, v)


def workspace_bytes(n_out: int, k_in: int, rows: int, x_aligned: bool = False) -> int:
    """Scratch bytes of a call: partial sums where K is split, and a copy of x's rows unless they can be read as they
    lie (`x_aligned`: on 16 bytes, a stride of a multiple of 8 values, and k_in a multiple of 128)."""
    return _need("syn_half_gemv_workspace_bytes", n_out, k_in, rows, 1 if x_aligned else 0)


def _operand(t, rows, n, what, device):
    """(type, address, stride) of an optional operand of the epilogue."""
    if t is None:
        return 0, None, 0
    return _value_type(t, what), t.data_ptr(), _ptr_width(t, rows, n, what, device)


def gemv(w: Weights, x: torch.Tensor, rows: int, act: str = "none", gate: torch.Tensor | None = None,
         residual: torch.Tensor | None = None, y: torch.Tensor | None = None, ws: torch.Tensor | None = None,
         dtype: torch.dtype | None = None, stream=None) -> torch.Tensor:
    """y [rows, n_out] = act(x W^T + bias) * gate + residual for the first `rows` rows of x [., k_in], which is of the
    weights' type; y of its own type, `dtype` or x's (F32, F16 or BF16).  act is none, relu, silu, gelu (v Phi(v)) or
    gelu_tanh; gate and residual are rows of n_out values of any of the three types, or None.  Rows may be strided.
    residual or gate may be y itself; y overlaps no operand otherwise."""
    code = ACTS.get(act)
    if code is None:
        raise GemvError("Activations", f"the activation {act!r} is none of {', '.join(ACTS)}")
    if x.dtype != w.matrix.dtype:
        raise GemvError("Activations", f"x is of {x.dtype}, the weights of {w.matrix.dtype}")
    xs = _ptr_width(x, rows, w.k_in, "x", w.device)
    if stream is not None or w.device != _current_device():
        return _on_stream(x, stream, lambda handle: _launch(w, x, xs, rows, code, gate, residual, y, ws, dtype, handle))
    return _launch(w, x, xs, rows, code, gate, residual, y, ws, dtype, _current_stream(w.device))


def _launch(w, x, xs, rows, act, gate, residual, y, ws, dtype, handle):
    n = w.n_out
    gs, rs = _operand(gate, rows, n, "gate", w.device), _operand(residual, rows, n, "residual", w.device)
    if y is None:
        y = torch.empty(rows, n, dtype=x.dtype if dtype is None else dtype, device=x.device)
        yty, ys = _value_type(y, "y"), n
    else:
        if dtype is not None and dtype != y.dtype:
            raise GemvError("Len", f"`y` is of {y.dtype}, not {dtype}")
        yty, ys = _value_type(y, "y"), _ptr_width(y, rows, n, "y", w.device)
    xp = x.data_ptr()
    if ws is None:
        aligned = xp % 16 == 0 and (rows <= 1 or xs % 8 == 0)
        wp, wb = None, _need("syn_half_gemv_workspace_bytes", n, w.k_in, rows, 1 if aligned else 0)
        if wb:
            ws = torch.empty(wb, dtype=torch.uint8, device=x.device)
            wp = ws.data_ptr()
    else:
        if ws.get_device() != w.device or ws.dtype != torch.uint8 or not ws.is_contiguous():
            raise GemvError("Len", "`ws` must be a contiguous uint8 tensor on the operands' device")
        wp, wb = ws.data_ptr(), ws.numel()
    call("syn_half_gemv", *w.view, n, w.k_in, xp, xs, rows, act, *gs, *rs, yty, y.data_ptr(), ys, wp, wb, handle)
    return y


__all__ = ["Weights", "SynError", "GemvError", "ACTS", "workspace_bytes", "gemv"]

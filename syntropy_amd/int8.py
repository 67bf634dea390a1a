"""Products over int8 weights with a scale a channel (output row) on the MI355X: activations of F32, F16 or
BF16 are quantized inside the call to int8 with a scale a token, the sums are exact in I32.  Beside
`gemv` (scales a block of 32 or 256 weights, bit-identical to the reference's provider) these take one
scale a row, which leaves the matrix cores nothing but integers; the reference has no such type.

    w = int8.quantize_weights(matrix)            # or int8.Weights(codes, scales) of a checkpoint
    y = int8.gemv(w, x, rows)                    # x [rows, k_in] -> [rows, n_out] of x's type
    h = int8.gate_up_act(gate_up, x, rows)       # silu(gate x) * (up x) of a stacked matrix

Every call runs the HIP kernels through the C ABI; there is no CPU path.
"""
from __future__ import annotations

import ctypes as C
from dataclasses import dataclass

import torch

from ._lib import SynError, call
from .gemv import GemvError, _current_device, _current_stream, _need, _on_stream, _ptr_rows, _value_type

MAX_K = 131072


@dataclass(frozen=True, eq=False)
class Weights:
    """`codes` int8 [n_out, k_in] with F32 `scales` [n_out] and an optional F32 `bias` [n_out], device
    tensors: the row o stands for codes[o] * scales[o].  Rows lie side by side and start on 16 bytes: a
    codes tensor whose rows do not (k_in no multiple of 16, say) is copied once, here, into rows of whole
    128-byte lines; any other is kept as it is."""

    codes: torch.Tensor
    scales: torch.Tensor
    bias: torch.Tensor | None = None

    def __post_init__(self):
        c, s, b = self.codes, self.scales, self.bias
        if not (c.is_cuda and c.dtype == torch.int8 and c.dim() == 2):
            raise GemvError("Len", "codes must be an int8 device tensor of rows")
        n_out, k_in = c.shape
        if not 1 <= k_in <= MAX_K:
            raise GemvError("RowLength", f"rows of {k_in} codes (1 to {MAX_K})")
        for what, t in (("scales", s), ("bias", b)):
            if t is None and what == "bias":
                continue
            if not (t.device == c.device and t.dtype == torch.float32 and t.is_contiguous()) or t.shape != (n_out,):
                raise GemvError("Len", f"{what} must be a contiguous F32 tensor of {n_out} values beside the codes")
        if c.stride(1) != 1 or c.stride(0) < k_in or c.stride(0) % 16 or c.data_ptr() % 16:
            rows = torch.zeros(n_out, -(-k_in // 128) * 128, dtype=torch.int8, device=c.device)[:, :k_in]
            c = rows.copy_(c)
        stride = c.stride(0)
        # the C ABI's arguments: the codes' view (address, bytes, stride), scales, bias
        view = (c.data_ptr(), (n_out - 1) * stride + k_in if n_out else 0, stride, s.data_ptr(),
                0 if b is None else b.data_ptr())
        for name, v in (("codes", c), ("n_out", n_out), ("k_in", k_in), ("device", c.get_device()), ("view", view)):
            object.__setattr__(self, name, v)


def quantize_rows(x: torch.Tensor, stream=None) -> tuple[torch.Tensor, torch.Tensor]:
    """Each row of x [rows, k] (F32, F16 or BF16): int8 codes [rows, k] (in rows of whole 128-byte lines)
    and F32 scales [rows], code = rint(x / scale) with scale = max |x| / 127.  A row with a NaN or an
    infinity has the scale NaN and codes 0."""
    if x.dim() != 2:
        raise GemvError("Len", "x must be rows of values")
    rows, k = x.shape
    ty, stride = _value_type(x, "x"), _ptr_rows(x, rows, k, "x")

    def launch(handle):
        codes = torch.empty(rows, -(-k // 128) * 128, dtype=torch.int8, device=x.device)
        scales = torch.empty(rows, dtype=torch.float32, device=x.device)
        call("syn_i8_quantize", ty, x.data_ptr(), stride, rows, k, codes.data_ptr(), codes.shape[1], scales.data_ptr(), handle)
        return codes[:, :k], scales
    return _on_stream(x, stream, launch)


def quantize_weights(w: torch.Tensor, bias: torch.Tensor | None = None, stream=None) -> Weights:
    """A matrix [n_out, k_in] of F32, F16 or BF16 with a scale a channel (quantize_rows of its rows)."""
    codes, scales = quantize_rows(w, stream)
    return Weights(codes, scales, bias)


def workspace_bytes(n_out: int, k_in: int, rows: int, gated: bool = False) -> int:
    """Scratch bytes of a call: the quantized rows (none where the product's kernel quantizes them itself),
    and partial sums where K is split."""
    return _need("syn_i8_gemv_workspace_bytes", n_out, k_in, rows, 1 if gated else 0)


def _product(name, gated, w, n, x, rows, y, ws, dtype, stream):
    ty, xs = _value_type(x, "x"), _ptr_rows(x, rows, w.k_in, "x", w.device)
    if stream is not None or w.device != _current_device():
        return _on_stream(x, stream, lambda handle: _launch(name, gated, w, n, x, ty, xs, rows, y, ws, dtype, handle))
    return _launch(name, gated, w, n, x, ty, xs, rows, y, ws, dtype, _current_stream(w.device))


def _launch(name, gated, w, n, x, ty, xs, rows, y, ws, dtype, handle):
    if y is None:
        y = torch.empty(rows, n, dtype=x.dtype if dtype is None else dtype, device=x.device)
        yty, ys = _value_type(y, "y"), n
    else:
        if dtype is not None and dtype != y.dtype:
            raise GemvError("Len", f"`y` is of {y.dtype}, not {dtype}")
        yty, ys = _value_type(y, "y"), _ptr_rows(y, rows, n, "y", w.device)
    if ws is None:
        wp, wb = 0, _need("syn_i8_gemv_workspace_bytes", n, w.k_in, rows, gated)
        if wb:
            ws = torch.empty(wb, dtype=torch.uint8, device=x.device)
            wp = ws.data_ptr()
    else:
        if ws.get_device() != w.device or ws.dtype != torch.uint8 or not ws.is_contiguous():
            raise GemvError("Len", "`ws` must be a contiguous uint8 tensor on the operands' device")
        wp, wb = ws.data_ptr(), ws.numel()
    call(name, *w.view, n, w.k_in, ty, x.data_ptr(), xs, rows, yty, y.data_ptr(), ys, wp, wb, handle)
    return y


def gemv(w: Weights, x: torch.Tensor, rows: int, y: torch.Tensor | None = None, ws: torch.Tensor | None = None,
         dtype: torch.dtype | None = None, stream=None) -> torch.Tensor:
    """y [rows, n_out] = x W^T (+ bias) for the first `rows` rows of x [., k_in], of x's type, y's or
    `dtype` (F32, F16, BF16).  x and y may have strided rows; no value of y lies in x or another operand."""
    return _product("syn_i8_gemv", 0, w, w.n_out, x, rows, y, ws, dtype, stream)


def gate_up_act(w: Weights, x: torch.Tensor, rows: int, y: torch.Tensor | None = None, ws: torch.Tensor | None = None,
                dtype: torch.dtype | None = None, stream=None) -> torch.Tensor:
    """GateUpAct{Silu} over a stacked matrix (gate rows, then up rows: w.n_out = 2 n): y [rows, n] =
    silu(gate x) * (up x), both products the F32 values of gemv, silu(g) = g / (1 + exp(-g)) within 2^-21 of its
    value (a NaN at -infinity).  Operands as gemv's."""
    if w.n_out % 2:
        raise GemvError("Len", f"a stacked gate/up matrix has an even row count, not {w.n_out}")
    return _product("syn_i8_gate_up_act", 1, w, w.n_out // 2, x, rows, y, ws, dtype, stream)


class Rows:
    """Rows of x quantized once (quantize_into) for several matrices of the same k_in (gemv_quantized): a
    workspace for their codes and for the products of `n_outs` outputs each."""

    def __init__(self, rows: int, k_in: int, *n_outs: int, device="cuda"):
        self.rows, self.k_in = rows, k_in
        need = max(_need("syn_i8_gemv_quantized_workspace_bytes", n, k_in, rows) for n in n_outs or (1,))
        self.ws = torch.empty(max(need, 256), dtype=torch.uint8, device=device)


def quantize_into(x: torch.Tensor, r: Rows, stream=None) -> None:
    """The first r.rows rows of x into r."""
    ty, xs = _value_type(x, "x"), _ptr_rows(x, r.rows, r.k_in, "x", r.ws.get_device())
    _on_stream(x, stream, lambda handle: call("syn_i8_act_quantize", ty, x.data_ptr(), xs, r.rows, r.k_in, r.ws.data_ptr(),
                                              r.ws.numel(), handle))


def gemv_quantized(w: Weights, r: Rows, y: torch.Tensor, stream=None) -> torch.Tensor:
    """gemv over rows quantized before: the same values."""
    if w.k_in != r.k_in:
        raise GemvError("Len", f"the rows hold {r.k_in} codes, the weights {w.k_in}")
    if w.device != r.ws.get_device():
        raise GemvError("Len", f"the rows are on {r.ws.device}, the weights on cuda:{w.device}")
    yty, ys = _value_type(y, "y"), _ptr_rows(y, r.rows, w.n_out, "y", w.device)
    _on_stream(y, stream, lambda handle: call("syn_i8_gemv_quantized", *w.view, w.n_out, w.k_in, r.rows, yty, y.data_ptr(),
                                              ys, r.ws.data_ptr(), r.ws.numel(), handle))
    return y


def logits(head: Weights, g: torch.Tensor, eps: float, x: torch.Tensor, rows: int, y: torch.Tensor | None = None,
           stream=None) -> torch.Tensor:
    """Logits over an int8 head: each F32 row of x [., hidden] normalised by (g, eps) as gemv.rms_norm, then
    y F32 [rows, vocab] = head x as gemv.  x, g and y hold their values side by side."""
    if not (x.is_cuda and x.dtype == torch.float32 and x.is_contiguous() and x.numel() >= rows * head.k_in):
        raise GemvError("Len", f"x must be a contiguous F32 device tensor of {rows * head.k_in} values")
    if not (head.device == x.get_device() and g.device == x.device and g.dtype == torch.float32 and g.is_contiguous()
            and g.numel() == head.k_in):
        raise GemvError("Len", f"g must be a contiguous F32 tensor of {head.k_in} values beside x and the head")
    if head.bias is not None:
        raise GemvError("Activations", "a head has no bias")
    if y is not None and not (y.device == x.device and y.dtype == torch.float32 and y.is_contiguous()
                              and y.numel() >= rows * head.n_out):
        raise GemvError("Len", f"y must be a contiguous F32 device tensor of {rows * head.n_out} values")

    def launch(handle):
        out = torch.empty(rows, head.n_out, dtype=torch.float32, device=x.device) if y is None else y
        need = _need("syn_i8_logits_workspace_bytes", head.n_out, head.k_in, rows)
        ws = torch.empty(max(need, 256), dtype=torch.uint8, device=x.device)
        call("syn_i8_logits", *head.view[:4], head.n_out, head.k_in, g.data_ptr(), C.c_float(eps), x.data_ptr(), rows,
             out.data_ptr(), ws.data_ptr(), ws.numel(), handle)
        return out
    return _on_stream(x, stream, launch)


__all__ = ["Weights", "Rows", "SynError", "GemvError", "quantize_rows", "quantize_weights", "workspace_bytes", "gemv",
           "gate_up_act", "quantize_into", "gemv_quantized", "logits"]

"""Decode GEMV on the MI355X, mirroring the reference CPU provider's `gemv` module
(crates/kernels-cpu/src/gemv.rs, gemv/act.rs, gemv/entry.rs): the same names, argument
meaning and refusals, over device tensors.  Every call runs the HIP kernels through the C ABI;
there is no CPU path.
"""
from __future__ import annotations

import ctypes as C
import functools
from dataclasses import dataclass
from enum import IntEnum
from typing import NamedTuple

import torch

from ._lib import SynError, call, lib


class WeightType(IntEnum):
    """A weight type this module computes (gemv.rs:87-151), by ggml type id."""

    F16 = 1
    Q4_0 = 2
    Q8_0 = 8
    Q4K = 12
    BF16 = 30

    def block_elems(self) -> int:
        return {WeightType.F16: 1, WeightType.BF16: 1, WeightType.Q4K: 256}.get(self, 32)

    def block_bytes(self) -> int:
        return {WeightType.F16: 2, WeightType.BF16: 2, WeightType.Q4_0: 18, WeightType.Q8_0: 34,
                WeightType.Q4K: 144}[self]

    def act(self) -> str:
        """The activation block a product over this type quantizes to (gemv.rs:145-151); F16 and
        BF16 products take the F32 activations as they are."""
        if self in (WeightType.F16, WeightType.BF16):
            return "F32"
        return "Q8K" if self is WeightType.Q4K else "Q8_0"


class GemvError(ValueError):
    """Why a GEMV call refused its inputs (gemv.rs:226-279).  A refused call writes nothing."""

    def __init__(self, kind: str, msg: str):
        super().__init__(f"Gemv: {msg}")
        self.kind = kind


LAYOUT_SOURCE, LAYOUT_X8, LAYOUT_SPLIT = 0, 1, 2


@dataclass
class Weights:
    """`n_out` rows of `k_in` weights of type `ty` in GGUF block layout, in device memory
    (gemv.rs:157-224).  `bytes` is a uint8 device tensor holding exactly the matrix; `layout` is
    LAYOUT_SOURCE (the GGUF order), for Q4_K LAYOUT_X8, for Q8_0 and Q4_0 LAYOUT_SPLIT (see
    repack)."""

    ty: WeightType
    bytes: torch.Tensor
    n_out: int
    k_in: int
    layout: int = LAYOUT_SOURCE

    def __post_init__(self):
        self.ty = WeightType(self.ty)
        if self.k_in % self.ty.block_elems():
            raise GemvError("RowLength", f"a row of {self.k_in} weights is not whole "
                            f"{self.ty.block_elems()}-weight {self.ty.name} blocks")
        need = self.row_bytes() * self.n_out
        if self.bytes.dtype != torch.uint8 or self.bytes.numel() != need:
            raise GemvError("Len", f"`weights` holds {self.bytes.numel()} values, the op needs {need}")

    def row_bytes(self) -> int:
        return self.k_in // self.ty.block_elems() * self.ty.block_bytes()


def _ask(name: str, *shape: int) -> int:
    out = C.c_uint64()
    call(name, *shape, C.byref(out))
    return out.value


class _NotKept(Exception):
    pass


@functools.lru_cache(maxsize=1024, typed=True)
def _kept(name: str, *shape: int) -> int:
    if any(v.__class__ is not int for v in shape):
        raise _NotKept  # which the cache does not keep
    return _ask(name, *shape)


def _need(name: str, *shape: int) -> int:
    """What a workspace query of the C ABI answers: a function of its whole numbers alone, so a call
    that repeats a shape does not ask again (a one-row Gemv's host time 10 -> 7 us with the stream's
    handle taken directly).  Only plain whole numbers are kept: a float that equals one is refused as it
    is when asked, and a tensor of one value, which hashes by identity, may change."""
    try:
        return _kept(name, *shape)
    except _NotKept:
        return _ask(name, *shape)


def workspace_bytes(ty: WeightType, rows: int, k: int) -> int:
    """Scratch bytes of one call's quantized activations (act.rs:108-111; the provider's own
    layout: codes, scales, 32-value sums)."""
    return _need("syn_gemv_workspace_bytes", int(ty), rows, k)


def _stream(stream) -> int:
    if stream is None:  # the current stream's handle, without the Stream object around it
        return torch._C._cuda_getCurrentRawStream(torch.cuda.current_device())
    return getattr(stream, "cuda_stream", stream)


def _check_x(x: torch.Tensor, rows: int, k: int):
    if not (x.is_cuda and x.dtype == torch.float32 and x.is_contiguous()):
        raise GemvError("Len", "x must be a contiguous F32 device tensor")
    if x.numel() < rows * k:
        raise GemvError("Len", f"`x` holds {x.numel()} values, the op needs {rows * k}")


def new_workspace(ty: WeightType, rows: int, k: int, device="cuda") -> torch.Tensor:
    return torch.empty(max(workspace_bytes(ty, rows, k), 256), dtype=torch.uint8, device=device)


def quantize_into(ty: WeightType, x: torch.Tensor, rows: int, k: int, ws: torch.Tensor,
                  stream=None) -> None:
    """Quantizes the first `rows` rows of x (k values each) into `ws` (act.rs:122-167)."""
    ty = WeightType(ty)
    if k % ty.block_elems():
        raise GemvError("Activations", "k is not whole activation blocks")
    _check_x(x, rows, k)
    call("syn_act_quantize", int(ty), x.data_ptr(), rows, k, ws.data_ptr(), ws.numel(), _stream(stream))


def gemv_quantized(w: Weights, ws: torch.Tensor, rows: int, y: torch.Tensor, stream=None) -> None:
    """y[r][o] for every row r < rows and every output o (gemv.rs:435-492)."""
    need = rows * w.n_out
    if y.numel() < need:
        raise GemvError("Len", f"`y` holds {y.numel()} values, the op needs {need}")
    call("syn_gemv_quantized_layout", w.layout, int(w.ty), w.bytes.data_ptr(), w.bytes.numel(), w.n_out,
         w.k_in, ws.data_ptr(), ws.numel(), rows, y.data_ptr(), _stream(stream))


def repack(w: Weights, layout: int | None = None, stream=None) -> Weights:
    """The matrix in another layout (a permutation of its bytes, crates/kernels/src/provider.rs:
    326-336 repack): LAYOUT_X8 stores each run of eight Q4_K super-blocks chunk-major, so the
    decode kernel reads whole 128-byte lines; LAYOUT_SPLIT stores every Q8_0 / Q4_0 block's codes
    first and every block's F16 scale after them, so the codes stream in 16-byte loads."""
    if layout is None:
        layout = LAYOUT_X8 if w.ty is WeightType.Q4K else LAYOUT_SPLIT
    if w.layout != LAYOUT_SOURCE:
        raise GemvError("Activations", "repack takes weights in the source layout")
    out = torch.empty_like(w.bytes)
    if w.ty is WeightType.Q4K and layout == LAYOUT_X8:
        call("syn_q4k_repack", layout, w.bytes.data_ptr(), out.data_ptr(), w.bytes.numel(), 0, _stream(stream))
    elif w.ty in (WeightType.Q8_0, WeightType.Q4_0) and layout == LAYOUT_SPLIT:
        call("syn_split_repack", layout, int(w.ty), w.bytes.data_ptr(), out.data_ptr(), w.bytes.numel(), 0,
             _stream(stream))
    else:
        raise GemvError("Activations", "repack takes Q4_K to LAYOUT_X8 and Q8_0 / Q4_0 to LAYOUT_SPLIT")
    return Weights(w.ty, out, w.n_out, w.k_in, layout)


def gemv(w: Weights, x: torch.Tensor, rows: int, y: torch.Tensor | None = None,
         ws: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """The Gemv op (gemv/entry.rs:167-247): quantize x F32 [rows, k_in], then
    y F32 [rows, n_out] = W x, bit-identical to the reference CPU provider."""
    _check_x(x, rows, w.k_in)
    if y is None:
        y = torch.empty(rows, w.n_out, dtype=torch.float32, device=x.device)
    elif y.numel() < rows * w.n_out:
        raise GemvError("Len", f"`y` holds {y.numel()} values, the op needs {rows * w.n_out}")
    ty, wb = int(w.ty), w.bytes
    if w.layout != LAYOUT_SOURCE:
        if ws is None:
            need = _need("syn_gemv_layout_workspace_bytes", w.layout, ty, rows, w.k_in)
            ws = torch.empty(max(need, 256), dtype=torch.uint8, device=x.device)
        call("syn_gemv_layout", w.layout, ty, wb.data_ptr(), wb.numel(), w.n_out, w.k_in,
             x.data_ptr(), rows, y.data_ptr(), ws.data_ptr(), ws.numel(), _stream(stream))
        return y
    if ws is None:
        ws = new_workspace(w.ty, rows, w.k_in, x.device)
    call("syn_gemv", ty, wb.data_ptr(), wb.numel(), w.n_out, w.k_in,
         x.data_ptr(), rows, y.data_ptr(), ws.data_ptr(), ws.numel(), _stream(stream))
    return y


def gate_up_act(w: Weights, x: torch.Tensor, rows: int, y: torch.Tensor | None = None,
                stream=None) -> torch.Tensor:
    """GateUpAct{Silu} (crates/kernels/src/reference/linear.rs:75-112): `w` stacks the gate rows
    then the up rows (w.n_out = 2 n), y F32 [rows, n] = silu(gate x) * (up x), each dot the
    Gemv value, silu with the reference's software exp, the product rounded once."""
    if w.n_out % 2:
        raise GemvError("Len", f"a stacked gate/up matrix has an even row count, not {w.n_out}")
    n = w.n_out // 2
    _check_x(x, rows, w.k_in)
    if y is None:
        y = torch.empty(rows, n, dtype=torch.float32, device=x.device)
    elif y.numel() < rows * n:
        raise GemvError("Len", f"`y` holds {y.numel()} values, the op needs {rows * n}")
    need = _need("syn_gate_up_act_workspace_bytes", w.layout, int(w.ty), rows, n, w.k_in)
    ws = torch.empty(max(need, 256), dtype=torch.uint8, device=x.device)
    call("syn_gate_up_act", w.layout, int(w.ty), w.bytes.data_ptr(), w.bytes.numel(), n, w.k_in,
         x.data_ptr(), rows, y.data_ptr(), ws.data_ptr(), ws.numel(), _stream(stream))
    return y


def rms_norm(x: torch.Tensor, g: torch.Tensor, eps: float, rows: int, y: torch.Tensor | None = None,
             stream=None) -> torch.Tensor:
    """RmsNorm of each row of x F32 [rows, n] (crates/kernels/src/reference/norm.rs:39-47)."""
    n = g.numel()
    _check_x(x, rows, n)
    if y is None:
        y = torch.empty(rows, n, dtype=torch.float32, device=x.device)
    call("syn_rms_norm", x.data_ptr(), g.data_ptr(), rows, n, C.c_float(eps), y.data_ptr(), _stream(stream))
    return y


def logits(head: Weights, g: torch.Tensor, eps: float, x: torch.Tensor, rows: int,
           y: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """Logits (crates/kernels/src/reference/linear.rs:118-161): each row of x [rows, hidden]
    normalised by (g, eps), then y F32 [rows, vocab] = head x as the Gemv op computes it."""
    _check_x(x, rows, head.k_in)
    if y is None:
        y = torch.empty(rows, head.n_out, dtype=torch.float32, device=x.device)
    need = _need("syn_logits_workspace_bytes", head.layout, int(head.ty), rows, head.n_out, head.k_in)
    ws = torch.empty(max(need, 256), dtype=torch.uint8, device=x.device)
    call("syn_logits", head.layout, int(head.ty), head.bytes.data_ptr(), head.bytes.numel(), head.n_out,
         head.k_in, g.data_ptr(), C.c_float(eps), x.data_ptr(), rows, y.data_ptr(), ws.data_ptr(), ws.numel(),
         _stream(stream))
    return y


_VALUE_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 30}


def _value_type(t: torch.Tensor, what: str) -> int:
    ty = _VALUE_TYPES.get(t.dtype)
    if ty is None:
        raise GemvError("Activations", f"`{what}` is of {t.dtype}, not float32, float16 or bfloat16")
    return ty


def _ptr_rows(t: torch.Tensor, rows: int, n: int, what: str, device=None) -> int:
    """The row stride, in values, of a device tensor of at least `rows` rows of n values side by side: one
    of two dimensions with any row stride, or a contiguous one of enough values."""
    if not t.is_cuda or (device is not None and t.get_device() != device):
        raise GemvError("Len", f"`{what}` must be on the operands' device")
    shape = t.shape
    if len(shape) == 2 and shape[1] == n and 0 <= rows <= shape[0]:
        step, inner = t.stride()
        if (inner == 1 or n == 1) and (step >= n or rows <= 1):
            return step if step > n else n
    if rows < 0:
        raise GemvError("Len", f"{rows} rows")
    if not t.is_contiguous() or t.numel() < rows * n:
        raise GemvError("Len", f"`{what}` holds {t.numel()} values, the op needs {rows} rows of {n} side by side")
    return n


def _ptr_width(t: torch.Tensor, rows: int, n: int, what: str, device=None) -> int:
    """_ptr_rows of a tensor whose rows, where it has two dimensions, are n values wide."""
    if t.dim() == 2 and t.shape[1] != n:
        raise GemvError("Len", f"`{what}` has rows of {t.shape[1]} values, not {n}")
    return _ptr_rows(t, rows, n, what, device)


_current_device, _current_stream = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream


def _on_stream(t: torch.Tensor, stream, body):
    """body(handle) on `stream` (a torch stream or a handle), or on the current one of t's device, with that
    device current, and what torch allocates meanwhile belonging to that stream."""
    device = t.get_device()
    if stream is None:
        if device == _current_device():
            return body(_current_stream(device))
        with torch.cuda.device(device):
            return body(_current_stream(device))
    if not hasattr(stream, "cuda_stream"):
        stream = torch.cuda.ExternalStream(int(stream), device=device)
    if stream.device.index != device:
        raise GemvError("Len", f"the stream is of {stream.device}, the operands of cuda:{device}")
    with torch.cuda.stream(stream):
        return body(stream.cuda_stream)


class TokenLogprobs(NamedTuple):
    """What token_logprobs gives, a row each: the token's log probability F32 and rank I32, the entropy F32,
    the greatest logits' indices I32 [rows, top] and their log probabilities F32 [rows, top]; all of one
    allocation."""

    logprob: torch.Tensor
    rank: torch.Tensor
    entropy: torch.Tensor
    top_ids: torch.Tensor
    top_logprobs: torch.Tensor


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, top: int = 0, scale: float = 1.0,
                   stream=None) -> TokenLogprobs:
    """Of each row of logits [rows, vocab] (F32, F16 or BF16; strided rows; -infinity hides a token), with z =
    logits * scale (the inverse of a sampling temperature, 2^-64 to 2^64): log softmax(z) at tokens[row] (int32 or int64), the
    number of logits greater than that token's, the entropy of softmax(z) in nats, and the `top` (0 to 64)
    greatest logits' indices, the lower one first among equals, with their log probabilities.

    A negative token asks for none (logprob 0, rank -1); one of vocab or more gives NaN and -1.  A row whose
    every logit is -infinity has log probabilities of -infinity and the entropy 0; one with a NaN or +infinity
    has NaN for both."""
    shape = logits.shape
    if len(shape) != 2 or tokens.shape != shape[:1]:
        raise GemvError("Len", "logits must be rows of values, with a token each")
    rows, vocab = shape
    if not 0 <= top <= min(vocab, 64):
        raise GemvError("Len", f"the {top} greatest of {vocab} logits (0 to 64)")
    device = logits.get_device()
    if tokens.dtype not in _TOKEN_TYPES or not tokens.is_contiguous() or tokens.get_device() != device:
        raise GemvError("Len", "tokens must be contiguous int32 or int64 values beside the logits")
    ty, stride = _value_type(logits, "logits"), _ptr_rows(logits, rows, vocab, "logits")
    if stream is None and device == _current_device():
        return _logprobs(logits, ty, stride, rows, vocab, tokens, top, scale, _current_stream(device))
    return _on_stream(logits, stream, lambda handle: _logprobs(logits, ty, stride, rows, vocab, tokens, top, scale, handle))


_TOKEN_TYPES = (torch.int32, torch.int64)


def _logprobs(logits, ty, stride, rows, vocab, tokens, top, scale, handle) -> TokenLogprobs:
    # the five outputs side by side in one allocation: a call's host time 13.2 -> 12.2 us, of two launches 18.0 -> 16.7
    dev, f32, i32, n = logits.device, torch.float32, torch.int32, rows * top
    lp, entropy, lps, rank, ids = torch.split_with_sizes(torch.empty(3 * rows + 2 * n, dtype=f32, device=dev),
                                                         (rows, rows, n, rows, n))
    lps, rank, ids = lps.view(rows, top), rank.view(i32), ids.view(i32).view(rows, top)
    need = _need("syn_token_logprobs_workspace_bytes", ty, rows, vocab, top)
    ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    at = lp.data_ptr()
    call("syn_token_logprobs", ty, logits.data_ptr(), stride, rows, vocab, tokens.data_ptr(), tokens.element_size(), scale,
         top, at, at + 4 * (2 * rows + n), at + 4 * rows, at + 4 * (3 * rows + n), at + 4 * 2 * rows,
         ws.data_ptr() if need else None, need, handle)
    return TokenLogprobs(lp, rank, entropy, ids, lps)


class BlockNorm(NamedTuple):
    """What block_norm gives: the residual stream behind the block, and its norm (None where none is asked for)."""

    h: torch.Tensor
    y: torch.Tensor | None


def _f32_values(t: torch.Tensor, n: int, what: str, device: int) -> int:
    if t.get_device() != device or t.dtype != torch.float32 or not t.is_contiguous() or t.numel() != n:
        raise GemvError("Len", f"`{what}` must be a contiguous F32 tensor of {n} values beside the rows")
    return t.data_ptr()


def block_norm(x: torch.Tensor, branch: torch.Tensor | None, g: torch.Tensor | None, eps: float, rows: int,
               post: torch.Tensor | None = None, gate: torch.Tensor | None = None, scale: float = 1.0,
               h: torch.Tensor | None = None, y: torch.Tensor | None = None, dtype: torch.dtype | None = None,
               stream=None) -> BlockNorm:
    """The end of a block and the beginning of the next over the first `rows` rows: with rms(v; g) = v g /
    sqrt(mean v^2 + eps),

        h = x + scale * gate * a,  a = rms(branch; post) (branch itself without `post`);  y = rms(h; g)

    in F32, each rounded once, y from the h that is not rounded.  x [., n], the residual stream, and h are of one type,
    branch and gate of one, y of y's, `dtype` or branch's (F32, F16 or BF16 each); g and post are F32 [n]; gate is
    [n], [1, n] or rows as x.  Rows may be strided; h may be x itself, and no other output lies in an operand.  Without
    a branch h is x; without g there is no y.  (rms_norm has the reference's order of sums.)"""
    if g is None and x.dim() != 2:
        raise GemvError("Len", "x must be rows of values where no norm's weights say how many")
    device = x.get_device()
    if device < 0:
        raise GemvError("Len", "`x` must be on a device")
    if stream is None and device == _current_device():
        return _block_norm(x, branch, g, eps, rows, post, gate, scale, h, y, dtype, device, _current_stream(device))
    return _on_stream(x, stream, lambda handle: _block_norm(x, branch, g, eps, rows, post, gate, scale, h, y, dtype, device, handle))


def _block_norm(x, branch, g, eps, rows, post, gate, scale, h, y, dtype, device, handle) -> BlockNorm:
    n = g.numel() if g is not None else x.shape[1]
    ty, xs = _value_type(x, "x"), _ptr_width(x, rows, n, "x")
    like, whole = x, x.shape == (rows, n)  # y's type; whether empty_like gives the outputs' shape (less host time)
    bty = bs = gs = bp = sp = pp = gp = None
    if branch is not None:
        like, bp = branch, branch.data_ptr()
        bty, bs = ty if branch.dtype is x.dtype else _value_type(branch, "branch"), _ptr_width(branch, rows, n, "branch", device)
        if post is not None:
            pp = _f32_values(post, n, "post", device)
        if gate is not None:
            if gate.dtype != branch.dtype:
                raise GemvError("Activations", f"the gate is of {gate.dtype}, the branch of {branch.dtype}")
            sp = gate.data_ptr()
            if gate.dim() == 1 or (gate.shape == (1, n) and rows != 1):
                _ptr_rows(gate, 1, n, "gate", device)
                if gate.numel() != n:
                    raise GemvError("Len", f"a gate of {gate.numel()} values for rows of {n}")
            else:
                gs = _ptr_width(gate, rows, n, "gate", device)
        if h is None:
            h = torch.empty_like(x) if whole and x.is_contiguous() else torch.empty(rows, n, dtype=x.dtype, device=x.device)
            hs = n
        else:
            if h.dtype != x.dtype:
                raise GemvError("Len", f"`h` is of {h.dtype}, not {x.dtype}")
            hs = _ptr_width(h, rows, n, "h", device)
    else:
        if post is not None or gate is not None:
            raise GemvError("Activations", "post and gate belong to a branch")
        if g is None:
            raise GemvError("Activations", "neither a branch nor a norm")
        h, hs = x, xs
    yp, yty, ys = None, 0, 0
    if g is not None:
        gp = _f32_values(g, n, "g", device)
        if y is None:
            if whole and like.shape == (rows, n) and (dtype is None or dtype is like.dtype) and like.is_contiguous():
                y = torch.empty_like(like)
            else:
                y = torch.empty(rows, n, dtype=dtype or like.dtype, device=x.device)
            ys = n
        else:
            if dtype is not None and dtype != y.dtype:
                raise GemvError("Len", f"`y` is of {y.dtype}, not {dtype}")
            ys = _ptr_width(y, rows, n, "y", device)
        yp, yty = y.data_ptr(), _value_type(y, "y")
    else:
        y = None
    call("syn_block_norm", ty, x.data_ptr(), xs, bty or 0, bp, bs or 0, pp, sp, gs or 0, scale, gp, eps, rows, n, h.data_ptr(), hs,
         yty, yp, ys, handle)
    return BlockNorm(h, y)


class Sampled(NamedTuple):
    """What sample_tokens gives, a row each: the token I32, its log probability F32 among those that were kept, and
    how many were kept I32; all of one allocation."""

    token: torch.Tensor
    logprob: torch.Tensor
    kept: torch.Tensor


def _setting(v, dtype, rows: int, what: str, device: int):
    """(address, number) of a setting: a tensor of a value a row, or a number for all."""
    if not torch.is_tensor(v):
        return None, v
    if v.get_device() != device or v.dtype != dtype or not v.is_contiguous() or v.shape != (rows,):
        raise GemvError("Len", f"`{what}` must be a number or a contiguous {dtype} tensor of {rows} values beside the logits")
    return v.data_ptr(), 0


def sample_tokens(logits: torch.Tensor, u: torch.Tensor, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0,
                  stream=None) -> Sampled:
    """A token of each row of logits [rows, vocab] (F32, F16 or BF16; strided rows; -infinity hides a token) from a
    uniform random number u [rows] F32 in [0, 1).  A row's visible logits stand in order (descending, the lower index
    first among equals), w = exp((x - max x) / temperature): top_k keeps the first k (0: all), top_p of those the least
    number whose sum of w reaches p times the sum of them (1: all), min_p of those the ones with w >= min_p (0:
    all).  The token is the first whose running sum of w passes u times the kept ones' sum; a temperature of 0 takes
    the greatest logit.  Each setting is a number or a tensor of a value a row (F32, top_k int32).

    As numbers: temperature 0 or 2^-64 to 2^64, top_k from 0, top_p above 0 to 1, min_p 0 to 1.  In a tensor values
    outside top_k's, top_p's and min_p's ranges count as the nearest in them, as u does outside its own.  A row with a
    NaN or +infinity, without a visible logit, or with a NaN setting or a temperature outside its range has the token
    -1, the logprob NaN and kept 0.  Equal calls give equal tokens."""
    shape = logits.shape
    if len(shape) != 2 or u.shape != shape[:1]:
        raise GemvError("Len", "logits must be rows of values, with a random number each")
    rows, vocab = shape
    device = logits.get_device()
    if u.dtype != torch.float32 or not u.is_contiguous() or u.get_device() != device:
        raise GemvError("Len", "u must be contiguous float32 values beside the logits")
    ty, xs = _value_type(logits, "logits"), _ptr_rows(logits, rows, vocab, "logits")
    f32 = torch.float32
    tp, t = _setting(temperature, f32, rows, "temperature", device)
    kp, k = _setting(top_k, torch.int32, rows, "top_k", device)
    pp, p = _setting(top_p, f32, rows, "top_p", device)
    mp, m = _setting(min_p, f32, rows, "min_p", device)
    if not 0 <= k < 1 << 31:
        raise GemvError("Len", f"top_k {k}")

    if stream is None and device == _current_device():
        return _sample(logits, ty, xs, rows, vocab, u, (tp, kp, pp, mp, t, k, p, m), _current_stream(device))
    return _on_stream(logits, stream, lambda handle: _sample(logits, ty, xs, rows, vocab, u, (tp, kp, pp, mp, t, k, p, m), handle))


def _sample(logits, ty, xs, rows, vocab, u, settings, handle) -> Sampled:
    need = _need("syn_sample_tokens_workspace_bytes", ty, rows, vocab)
    out = torch.empty(3, rows, dtype=torch.float32, device=logits.device)
    ws = torch.empty(need, dtype=torch.uint8, device=logits.device) if need else None
    at = out.data_ptr()
    call("syn_sample_tokens", ty, logits.data_ptr(), xs, rows, vocab, u.data_ptr(), *settings, at + 4 * rows, at, at + 8 * rows,
         ws.data_ptr() if need else None, need, handle)
    lp, token, kept = out.unbind()
    return Sampled(token.view(torch.int32), lp, kept.view(torch.int32))


class GemvBatch:
    """Up to 8 independent single-row Q4_K Gemv ops launched together (one batched Q8_K
    quantization, one grouped GEMV): each y[i] equals gemv(ws[i], x[i], 1) bit for bit.  The
    argument arrays are built once; `__call__` launches."""

    def __init__(self, weights: list[Weights], xs: list[torch.Tensor], ys: list[torch.Tensor],
                 ws: torch.Tensor | None = None):
        n = len(weights)
        if not (n == len(xs) == len(ys)) or n > 8:
            raise GemvError("Len", "GemvBatch takes up to 8 (weights, x, y) triples")
        for w, x, y in zip(weights, xs, ys):
            if w.ty is not WeightType.Q4K:
                raise GemvError("Activations", "GemvBatch takes Q4_K weights")
            _check_x(x, 1, w.k_in)
            if y.numel() < w.n_out:
                raise GemvError("Len", f"`y` holds {y.numel()} values, the op needs {w.n_out}")
        layouts = {w.layout for w in weights}
        if len(layouts) > 1:
            raise GemvError("Activations", "GemvBatch takes weights of one layout")
        self.layout = layouts.pop() if layouts else LAYOUT_SOURCE
        self.n = n
        u32 = C.c_uint32 * n
        self.k = u32(*[w.k_in for w in weights])
        self.n_out = u32(*[w.n_out for w in weights])
        self.ty = (C.c_int32 * n)(*[int(w.ty) for w in weights])
        self.w = (C.c_void_p * n)(*[w.bytes.data_ptr() for w in weights])
        self.wb = (C.c_uint64 * n)(*[w.bytes.numel() for w in weights])
        self.x = (C.c_void_p * n)(*[x.data_ptr() for x in xs])
        self.y = (C.c_void_p * n)(*[y.data_ptr() for y in ys])
        need = C.c_uint64()
        call("syn_gemv_batch_workspace_bytes", n, self.k, C.byref(need))
        self.ws = ws if ws is not None else torch.empty(max(need.value, 256), dtype=torch.uint8,
                                                        device=xs[0].device)
        self._keep = (weights, xs, ys)

    def __call__(self, stream=None) -> None:
        call("syn_gemv_batch_layout", self.layout, self.n, self.ty, self.w, self.wb, self.n_out, self.k,
             self.x, self.y, self.ws.data_ptr(), self.ws.numel(), _stream(stream))

    def quantize(self, stream=None) -> None:
        """The first half of __call__: every x[i] to Q8_K in the held workspace."""
        call("syn_act_quantize_batch", self.n, self.k, self.x, self.ws.data_ptr(), self.ws.numel(),
             _stream(stream))

    def gemv_quantized(self, stream=None) -> None:
        """The second half: every y[i] from the workspace quantize() filled."""
        call("syn_gemv_batch_quantized_layout", self.layout, self.n, self.ty, self.w, self.wb, self.n_out,
             self.k, self.ws.data_ptr(), self.ws.numel(), self.y, _stream(stream))


def gemm_workspace(rows: int, k: int, device="cuda") -> torch.Tensor:
    """Workspace of the prefill GEMM's activations (rows x k, Q8_K in the GEMM layout)."""
    out = C.c_uint64()
    call("syn_gemm_workspace_bytes", rows, k, C.byref(out))
    return torch.empty(max(out.value, 256), dtype=torch.uint8, device=device)


def gemm_quantize_into(x: torch.Tensor, rows: int, k: int, ws: torch.Tensor, stream=None) -> None:
    """The first `rows` rows of x to Q8_K in the prefill GEMM's layout (act.rs:351-373 values)."""
    _check_x(x, rows, k)
    call("syn_gemm_act_quantize", x.data_ptr(), rows, k, ws.data_ptr(), ws.numel(), _stream(stream))


def gemm_quantized(w: Weights, ws: torch.Tensor, rows: int, y: torch.Tensor, stream=None) -> None:
    """y[r][o] for every row r < rows from a workspace gemm_quantize_into filled: the Q4_K
    matrix-core GEMM, every output the Gemv value (gemv.rs:435-547)."""
    if w.ty is not WeightType.Q4K:
        raise GemvError("Activations", "the prefill GEMM takes Q4_K weights")
    if y.numel() < rows * w.n_out:
        raise GemvError("Len", f"`y` holds {y.numel()} values, the op needs {rows * w.n_out}")
    call("syn_gemm_q4k_quantized", w.bytes.data_ptr(), w.bytes.numel(), w.n_out, w.k_in, ws.data_ptr(),
         ws.numel(), rows, y.data_ptr(), _stream(stream))


def quantize(ty: WeightType, x: torch.Tensor, stream=None) -> torch.Tensor:
    """F32 values -> GGUF blocks, byte-identical to ggml's reference quantizers
    (crates/kernels-ggml/src/lib.rs:268 quantize).  Like that wrapper, refuses non-finite
    values and magnitudes above 65504 (checked on the device, one reduction)."""
    ty = WeightType(ty)
    x = x.contiguous()
    if x.numel() % ty.block_elems():
        raise GemvError("RowLength", f"{x.numel()} values are not whole {ty.block_elems()}-value blocks")
    if x.numel() and not bool(torch.isfinite(x).all() and x.abs().max() <= 65504.0):
        raise GemvError("OutOfRange", "a value is not finite or is out of the type's range")
    out = torch.empty(x.numel() // ty.block_elems() * ty.block_bytes(), dtype=torch.uint8, device=x.device)
    call("syn_quantize", int(ty), x.data_ptr(), x.numel(), out.data_ptr(), out.numel(), _stream(stream))
    return out


def dequantize(ty: WeightType, src: torch.Tensor, stream=None) -> torch.Tensor:
    """GGUF blocks -> F32, exact (dequant.rs:195-229)."""
    ty = WeightType(ty)
    out = torch.empty(src.numel() // ty.block_bytes() * ty.block_elems(), dtype=torch.float32,
                      device=src.device)
    call("syn_dequantize", int(ty), src.data_ptr(), src.numel(), out.data_ptr(), _stream(stream))
    return out


__all__ = ["WeightType", "Weights", "GemvError", "SynError", "GemvBatch", "workspace_bytes", "quantize_into",
           "repack", "LAYOUT_SOURCE", "LAYOUT_X8", "LAYOUT_SPLIT",
           "gemv_quantized", "gemv", "quantize", "dequantize", "new_workspace", "gemm_workspace",
           "gemm_quantize_into", "gemm_quantized", "gate_up_act", "token_logprobs", "TokenLogprobs", "block_norm", "BlockNorm",
           "sample_tokens", "Sampled", "lib"]

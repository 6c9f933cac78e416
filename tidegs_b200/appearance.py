"""Learned appearance of the Gaussians: operators over rows of per-Gaussian
features that complement the SH colors where photographs of one scene differ
in exposure, weather or time of day. No counterpart in the reference.

    layer_norm           rows to zero mean and unit spread; weight and bias
                         may come from an image's embedding
    gated_feed_forward   (silu(x Wg^T) * (x Wu^T)) Wd^T in one kernel
    dropout              of features, or of whole Gaussians by their ids, with
                         a mask that is drawn again instead of stored
    appearance_colors    the three of them added to SH colors or coefficients

All are differentiable (first order, reverse mode; others are refused) and run
on the current stream of the tensors' device. Inputs are CUDA tensors [..., C];
columns of any stride are taken (those whose rows are not contiguous values are
copied first). Sums are in 32 bits, outputs are rounded once to their type.
Every kernel adds in a fixed order: the same call gives the same bits.

Kernels: tgs_layer_norm_fwd/bwd, tgs_ffn_fwd/bwd, tgs_dropout
(libtidegs_b200.so).
"""
from __future__ import annotations

import contextlib
import ctypes
import operator
import threading
from typing import Dict, Optional, Tuple, Union

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib

__all__ = ["appearance_colors", "check", "dropout", "gated_feed_forward", "layer_norm"]

MAX_NORM_WIDTH = 8192
MAX_FFN_WIDTH = 256
MAX_FFN_HIDDEN = 4096
MAX_DROPOUT_WIDTH = 65536


def _check(t: torch.Tensor, who: str, name: str, device: Optional[torch.device] = None) -> None:
    if not t.is_cuda:
        raise RuntimeError(f"{who}: {name} must be a CUDA tensor; tidegs_b200 has no CPU path")
    if device is not None and t.device != device:
        raise ValueError(f"{who}: {name} is on {t.device}, the input on {device}")


def _rows(t: torch.Tensor, width: int) -> torch.Tensor:
    """t as [n, width] rows of contiguous values (a copy where it has none)."""
    if t.is_contiguous():
        return t if t.dim() == 2 else t.view(-1, width)
    t = t if t.dim() == 2 else t.reshape(-1, width)
    if t.stride(1) == 1 or width == 1:
        if t.shape[0] <= 1 or t.stride(0) >= width:
            return t
    return t.contiguous()


def _row_stride(t: torch.Tensor) -> int:
    n, width = t.shape
    return t.stride(0) if n > 1 else width


_HERE = contextlib.nullcontext()


def _on(device: torch.device):
    """The device as the current one (no call where it is already)."""
    return _HERE if device.index == torch._C._cuda_getDevice() else torch.cuda.device(device)


def _stream(device: torch.device) -> int:
    return torch._C._cuda_getCurrentRawStream(device.index)


def _refuse_tangents(who: str, *ts: Optional[torch.Tensor]) -> None:
    if forward_ad._current_level >= 0 and any(
            t is not None and forward_ad.unpack_dual(t).tangent is not None for t in ts):
        raise RuntimeError(f"{who}: forward-mode derivatives are not supported")


def _wants_grad(who: str, *ts: Optional[torch.Tensor]) -> bool:
    _refuse_tangents(who, *ts)
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts)


# --- layer norm --------------------------------------------------------------

def _norm_args(x, weight, bias, eps) -> "_lib.LayerNormArgs":
    param = weight if weight is not None else bias
    a = _lib.LayerNormArgs()
    a.x, a.weight, a.bias = x.data_ptr(), _lib.ptr(weight), _lib.ptr(bias)
    a.n, a.c = x.shape
    a.x_stride = _row_stride(x)
    a.dtype = _lib.DTYPES[x.dtype]
    a.param_dtype = _lib.DTYPES[param.dtype if param is not None else x.dtype]
    a.eps = eps
    return a


def _norm_forward(x, weight, bias, eps):
    rows = _rows(x, x.shape[-1])
    weight = None if weight is None else weight.contiguous()
    bias = None if bias is None else bias.contiguous()
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    a = _norm_args(rows, weight, bias, eps)
    a.y = y.data_ptr()
    with _on(x.device):
        _lib.call("tgs_layer_norm_fwd", a, _stream(x.device))
    return y


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        ctx.save_for_backward(x, weight)
        ctx.eps = eps
        ctx.bias = None if bias is None else bias.dtype
        return _norm_forward(x, weight, bias, eps)

    @staticmethod
    @once_differentiable
    def backward(ctx, v_y):
        _refuse_tangents("layer_norm", v_y)
        x, weight = ctx.saved_tensors
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        c = x.shape[-1]
        rows, v_rows = _rows(x, c), _rows(v_y, c)
        weight = None if weight is None else weight.contiguous()
        ptype = weight.dtype if weight is not None else ctx.bias if ctx.bias else x.dtype
        v_x = torch.empty(x.shape, dtype=x.dtype, device=x.device) if need_x else None
        v_w = torch.empty(c, dtype=ptype, device=x.device) if need_w else None
        v_b = torch.empty(c, dtype=ptype, device=x.device) if need_b else None
        b = _lib.LayerNormBwdArgs()
        b.fwd = _norm_args(rows, weight, None, ctx.eps)
        b.fwd.param_dtype = _lib.DTYPES[ptype]
        b.v_y, b.v_y_stride = v_rows.data_ptr(), _row_stride(v_rows)
        b.v_x, b.v_weight, b.v_bias = _lib.ptr(v_x), _lib.ptr(v_w), _lib.ptr(v_b)
        with _on(x.device):
            if need_w or need_b:
                words = _lib.load().tgs_layer_norm_scratch_floats(rows.shape[0], c)
                scratch = torch.empty(words, dtype=torch.float32, device=x.device)
                b.scratch = scratch.data_ptr()
            _lib.call("tgs_layer_norm_bwd", b, _stream(x.device))
        return v_x, v_w, v_b, None


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None,
               bias: Optional[torch.Tensor] = None, eps: float = 1e-5) -> torch.Tensor:
    """(x - mean) / sqrt(var + eps) * weight + bias over the last dimension
    (1 to 8192 wide) of float32, bfloat16 or float16 rows; differentiable in
    x, weight and bias. weight and bias [C] share a type, x's or float32."""
    who = "layer_norm"
    if x.dim() < 1 or not 1 <= x.shape[-1] <= MAX_NORM_WIDTH:
        raise ValueError(f"{who}: x {tuple(x.shape)} needs a last dimension of 1 to "
                         f"{MAX_NORM_WIDTH}")
    if x.dtype not in _lib.DTYPES:
        raise ValueError(f"{who}: x is {x.dtype}; float32, bfloat16 and float16 are supported")
    if not eps >= 0:
        raise ValueError(f"{who}: eps {eps} is negative")
    for t, name in ((weight, "weight"), (bias, "bias")):
        if t is None:
            continue
        if tuple(t.shape) != (x.shape[-1],):
            raise ValueError(f"{who}: {name} {tuple(t.shape)} is not [{x.shape[-1]}]")
        if t.dtype not in (x.dtype, torch.float32):
            raise ValueError(f"{who}: {name} is {t.dtype}; x's type ({x.dtype}) or float32 are "
                             "supported")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise ValueError(f"{who}: weight is {weight.dtype}, bias {bias.dtype}")
    _check(x, who, "x")
    for t, name in ((weight, "weight"), (bias, "bias")):
        if t is not None:
            _check(t, who, name, x.device)
    if _wants_grad(who, x, weight, bias):
        return _LayerNorm.apply(x, weight, bias, float(eps))
    return _norm_forward(x, weight, bias, float(eps))


# --- gated feed-forward block --------------------------------------------------

# A device's error word, in page-locked memory: kernels write it, the host reads
# it without waiting for them.
_err_words: Dict[torch.device, torch.Tensor] = {}
_err_values: Dict[torch.device, ctypes.Array] = {}
_err_lock = threading.Lock()


def _err_word(device: torch.device) -> torch.Tensor:
    word = _err_words.get(device)
    if word is None:
        with _err_lock, torch.inference_mode(False):
            word = _err_words.get(device)
            if word is None:
                word = torch.zeros(4, dtype=torch.int32, device="cpu", pin_memory=True)
                _err_values[device] = (ctypes.c_int32 * 4).from_address(word.data_ptr())
                _err_words[device] = word
    return word


def _raise_recorded(device: torch.device) -> None:
    """Raises, once, what a kernel on `device` has recorded."""
    values = _err_values.get(device)
    if values is not None and values[0]:
        problem = _lib.decode_device_error(list(values))
        _err_words[device].zero_()
        raise RuntimeError(f"[gated_feed_forward] in an earlier call on {device}: {problem}")


def check(device=None) -> None:
    """Raises if a bounded wait inside an earlier gated_feed_forward kernel on
    `device` (default: the current one) ran out, which leaves that call's
    results undefined. Waits for the device. (A later gated_feed_forward call,
    or backward, raises too, without waiting: as soon as the host can know.
    Either tells once.)"""
    device = torch.device("cuda" if device is None else device)
    if device.index is None:
        device = torch.device("cuda", torch.cuda.current_device())
    if device in _err_words:
        torch.cuda.synchronize(device)
        _raise_recorded(device)


def _ffn_rows(t: torch.Tensor, width: int) -> torch.Tensor:
    """_rows, for bfloat16 with every row on a 16-byte boundary."""
    t = _rows(t, width)
    if t.dtype is not torch.bfloat16 or t.shape[0] == 0:
        return t
    if t.data_ptr() % 16 == 0 and (t.shape[0] == 1 or t.stride(0) % 8 == 0):
        return t
    out = torch.empty((t.shape[0], -(-width // 8) * 8), dtype=t.dtype, device=t.device)
    with _on(t.device):
        _lib.call("tgs_align_rows", t.data_ptr(), _row_stride(t), t.shape[0], width, out.data_ptr(),
                  _stream(t.device))
    return out[:, :width]


def _ffn_stride(t: torch.Tensor) -> int:
    n, width = t.shape
    return t.stride(0) if n > 1 else -(-width // 8) * 8


def _ffn_args(x, w_gate, w_up, w_down, backward: bool):
    """(arguments, scratch tensor or None); on the tensors' device."""
    _raise_recorded(x.device)
    a = _lib.FfnArgs()
    a.x, a.w_gate = x.data_ptr(), w_gate.data_ptr()
    a.w_up, a.w_down = w_up.data_ptr(), w_down.data_ptr()
    a.n, a.x_stride = x.shape[0], _ffn_stride(x)
    a.d, a.h, a.o = int(w_gate.shape[1]), int(w_gate.shape[0]), int(w_down.shape[0])
    a.dtype = _lib.DTYPES[x.dtype]
    a.err = _err_word(x.device).data_ptr()
    words = _lib.load().tgs_ffn_scratch_floats(a.n, a.d, a.h, a.o, a.dtype, int(backward))
    scratch = torch.empty(words, dtype=torch.float32, device=x.device) if words else None
    a.scratch = _lib.ptr(scratch)
    return a, scratch


def _ffn_forward(x, w_gate, w_up, w_down):
    rows = _ffn_rows(x, x.shape[-1])
    weights = [w.contiguous() for w in (w_gate, w_up, w_down)]
    y = torch.empty((*x.shape[:-1], w_down.shape[0]), dtype=x.dtype, device=x.device)
    with _on(x.device):
        a, _scratch = _ffn_args(rows, *weights, backward=False)
        a.y = y.data_ptr()
        _lib.call("tgs_ffn_fwd", a, _stream(x.device))
    return y


class _GatedFeedForward(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, w_down):
        ctx.save_for_backward(x, w_gate, w_up, w_down)
        return _ffn_forward(x, w_gate, w_up, w_down)

    @staticmethod
    @once_differentiable
    def backward(ctx, v_y):
        _refuse_tangents("gated_feed_forward", v_y)
        x, *weights = ctx.saved_tensors
        weights = [w.contiguous() for w in weights]
        need_x, *need_w = ctx.needs_input_grad
        d, o = x.shape[-1], weights[2].shape[0]
        rows, v_rows = _ffn_rows(x, d), _ffn_rows(v_y, o)
        v_x = torch.empty(x.shape, dtype=x.dtype, device=x.device) if need_x else None
        v_w = [torch.empty_like(w) for w in weights] if any(need_w) else [None] * 3
        b = _lib.FfnBwdArgs()
        b.v_y, b.v_y_stride, b.v_x = v_rows.data_ptr(), _ffn_stride(v_rows), _lib.ptr(v_x)
        b.v_w_gate, b.v_w_up, b.v_w_down = (_lib.ptr(v) for v in v_w)
        with _on(x.device):
            b.fwd, _scratch = _ffn_args(rows, *weights, backward=True)
            _lib.call("tgs_ffn_bwd", b, _stream(x.device))
        return (v_x, *(v if need else None for v, need in zip(v_w, need_w)))


def gated_feed_forward(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor,
                       w_down: torch.Tensor) -> torch.Tensor:
    """(silu(x w_gate^T) * (x w_up^T)) w_down^T for rows x [..., D]; w_gate
    and w_up [H, D], w_down [O, H]; D and O up to 256, H up to 4096; every
    tensor float32 or every tensor bfloat16. Differentiable in all four; the
    hidden values are not kept: the backward computes them again. Raises if an
    earlier call's kernel gave up waiting (see `check`).

    A row's output is the same in calls of any number of rows.

    bfloat16: the hidden values are kept in two bfloat16 parts, 16 bits, between
    the products (one past bfloat16's range gives NaN). The backward rounds
    them, and their gradients, to one part in calls of more than 18,944 rows.
    float16 is refused: the hidden products leave its range long before their
    inputs do. float32: products of 32 bits; blocks of 12,288 multiply-adds a row
    and more keep a batch's hidden values in scratch memory, take an infinity
    (or a value that rounds to one in bfloat16, from 3.396e38 on) for NaN, and
    lose bits of values below 2^-100."""
    who = "gated_feed_forward"
    if w_gate.dim() != 2 or w_up.shape != w_gate.shape or w_down.dim() != 2 \
            or w_down.shape[1] != w_gate.shape[0]:
        raise ValueError(f"{who}: weights {tuple(w_gate.shape)}, {tuple(w_up.shape)}, "
                         f"{tuple(w_down.shape)} are not [H, D], [H, D], [O, H]")
    h, d = w_gate.shape
    o = w_down.shape[0]
    if x.dim() < 1 or x.shape[-1] != d:
        raise ValueError(f"{who}: x {tuple(x.shape)} is not [..., {d}]")
    if not (1 <= d <= MAX_FFN_WIDTH and 1 <= o <= MAX_FFN_WIDTH and 1 <= h <= MAX_FFN_HIDDEN):
        raise ValueError(f"{who}: widths of 1 to {MAX_FFN_WIDTH} and 1 to {MAX_FFN_HIDDEN} hidden "
                         f"values are supported (got D {d}, H {h}, O {o})")
    if x.dtype not in (torch.float32, torch.bfloat16):
        raise ValueError(f"{who}: x is {x.dtype}; float32 and bfloat16 are supported")
    _check(x, who, "x")
    for w, name in ((w_gate, "w_gate"), (w_up, "w_up"), (w_down, "w_down")):
        if w.dtype != x.dtype:
            raise ValueError(f"{who}: {name} is {w.dtype}, x {x.dtype}")
        _check(w, who, name, x.device)
    if _wants_grad(who, x, w_gate, w_up, w_down):
        return _GatedFeedForward.apply(x, w_gate, w_up, w_down)
    return _ffn_forward(x, w_gate, w_up, w_down)


# --- dropout -------------------------------------------------------------------

def _dropout_run(x, p, seed, offset, ids, per_row):
    n = int(x.shape[0])
    c = x.numel() // n if n else 1
    rows = _rows(x.reshape(n, c) if x.dim() != 2 else x, c)
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    a = _lib.DropoutArgs()
    a.x, a.y, a.ids = rows.data_ptr(), y.data_ptr(), _lib.ptr(ids)
    a.n, a.c, a.x_stride = n, c, _row_stride(rows)
    a.seed, a.p, a.per_row, a.dtype = seed, p, int(per_row), _lib.DTYPES[x.dtype]
    if isinstance(offset, torch.Tensor):
        a.offset_dev = offset.data_ptr()
    else:
        a.offset = offset
    with _on(x.device):
        _lib.call("tgs_dropout", a, _stream(x.device))
    return y


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, p, seed, offset, ids, per_row):
        dev = isinstance(offset, torch.Tensor)
        ctx.save_for_backward(ids, offset if dev else None)
        ctx.args = (p, seed, None if dev else offset, per_row)
        return _dropout_run(x, p, seed, offset, ids, per_row)

    @staticmethod
    @once_differentiable
    def backward(ctx, v_y):
        _refuse_tangents("dropout", v_y)
        ids, offset_dev = ctx.saved_tensors
        p, seed, offset, per_row = ctx.args
        offset = offset_dev if offset is None else offset
        return _dropout_run(v_y, p, seed, offset, ids, per_row), None, None, None, None, None


def dropout(x: torch.Tensor, p: float, seed: int, offset: Union[int, torch.Tensor] = 0,
            ids: Optional[torch.Tensor] = None, per_row: bool = False) -> torch.Tensor:
    """x / (1 - p) where a draw keeps the value, else 0; differentiable in x.

    The draw of dimension 0's row r and column c (the other dimensions
    flattened, up to 65536) depends on nothing but (seed, ids[r], c, offset):
    word c % 4 of Philox4x32-10 with key `seed` (64 bits) and counter (id low,
    id high, c // 4, offset); it keeps the value iff it is at least
    floor(p 2^32). per_row=True takes column 0's draw for the whole row. With
    ids [n] (int64; default 0..n-1) a Gaussian is dropped alike in whichever
    slot, view or rank it appears. offset, below 2^32, is the step; as an
    int64 tensor of one value on x's device it is read when the kernel runs
    (its low 32 bits), so a captured CUDA graph can advance it between
    replays. It must not change between a call and its backward."""
    who = "dropout"
    if x.dim() < 1:
        raise ValueError(f"{who}: x needs at least one dimension")
    n = int(x.shape[0])
    c = x.numel() // n if n else 1
    if n and not 1 <= c <= MAX_DROPOUT_WIDTH:
        raise ValueError(f"{who}: rows of 1 to {MAX_DROPOUT_WIDTH} values are supported (got {c})")
    if x.dtype not in _lib.DTYPES:
        raise ValueError(f"{who}: x is {x.dtype}; float32, bfloat16 and float16 are supported")
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"{who}: p {p} is not in [0, 1]")
    seed = operator.index(seed)
    if not 0 <= seed < 2 ** 64:
        raise ValueError(f"{who}: seed {seed} is not a 64-bit unsigned number")
    if isinstance(offset, torch.Tensor):
        if offset.dtype != torch.int64 or offset.numel() != 1:
            raise ValueError(f"{who}: an offset tensor holds one int64")
    elif not 0 <= operator.index(offset) < 2 ** 32:
        raise ValueError(f"{who}: offset {offset} is not a 32-bit unsigned number")
    if ids is not None and (ids.dtype != torch.int64 or tuple(ids.shape) != (n,)):
        raise ValueError(f"{who}: ids {ids.dtype} {tuple(ids.shape)} are not int64 [{n}]")
    _check(x, who, "x")
    if isinstance(offset, torch.Tensor):
        _check(offset, who, "offset", x.device)
    else:
        offset = operator.index(offset)
    if ids is not None:
        _check(ids, who, "ids", x.device)
        ids = ids.contiguous()
    args = (float(p), seed, offset, ids, bool(per_row))
    if _wants_grad(who, x):
        return _Dropout.apply(x, *args)
    return _dropout_run(x, *args)


# --- together ------------------------------------------------------------------

def appearance_colors(base: torch.Tensor, features: torch.Tensor,
                      norm: Tuple[Optional[torch.Tensor], Optional[torch.Tensor]],
                      weights: Tuple[torch.Tensor, torch.Tensor, torch.Tensor], *,
                      eps: float = 1e-5, p: float = 0.0, seed: int = 0,
                      offset: Union[int, torch.Tensor] = 0,
                      ids: Optional[torch.Tensor] = None) -> torch.Tensor:
    """base + dropout(gated_feed_forward(layer_norm(features, *norm), *weights))
    in base's type and shape: base holds one row per Gaussian, colors [N, 3]
    for `rasterize_to_pixels` or coefficients [N, K, 3] for
    `spherical_harmonics`, and the block's output width is that row's size.
    features [N, D]; norm (weight, bias) may be an image's own. p > 0 drops
    values of the residual by the Gaussians' ids (see `dropout`)."""
    if base.dim() < 2 or features.dim() != 2 or base.shape[0] != features.shape[0]:
        raise ValueError(f"appearance_colors: base {tuple(base.shape)} and features "
                         f"{tuple(features.shape)} are not [N, ...] and [N, D]")
    if base.shape[0] and base.numel() // base.shape[0] != weights[2].shape[0]:
        raise ValueError(f"appearance_colors: w_down {tuple(weights[2].shape)} does not give base's "
                         f"rows {tuple(base.shape[1:])}")
    y = gated_feed_forward(layer_norm(features, *norm, eps), *weights)
    if p:
        y = dropout(y, p, seed, offset=offset, ids=ids)
    return base + y.reshape(base.shape).to(base.dtype)

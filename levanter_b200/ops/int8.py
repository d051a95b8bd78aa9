"""Layers in 8-bit integers (the reference's ``QuantizationConfig(int8=True)``: Haliax ``Int8DotGeneralOp``, reached through
src/levanter/trainer.py:648).

A row is held as int8 numbers ``q = round(127 y / max |y|)`` (ties to even) and one fp32 scale ``max |y| / 127``: a row of activations has one scale per
token, a row of a weight matrix ``[out, in]`` one per output channel (:class:`Int8Rows`).  Rows are quantised where they are made (``csrc/int8_rows.cu``):
:func:`rms_norm_int8` with the residual's addition, :func:`gated_activation_int8`, :func:`quantize_rows`.  :func:`int8_product` multiplies
quantised rows and weights on the tensor cores, in whole numbers, and applies both scales, bias and residual to the sums (``csrc/gemm_int8.cu``).

:func:`int8_linear_many` is the differentiable form, which :class:`Int8Linear` trains with: activations and weights are quantised, several projections of the
same rows share them, and the 8-bit rows of both are what is kept for the backward pass.  Its gradients are those of the product at
the values that the whole numbers stand for (the rounding counts as having slope one).  :class:`Int8ServingLinear` holds a layer's weights in
8 bits for serving.

A row whose largest magnitude is below 2^-100 is held as zeros; one with an infinity or a NaN has the scale NaN, and all that is made from it is NaN.
The PyTorch statements are the CPU path and the test oracle."""
from __future__ import annotations

from typing import List, NamedTuple, Optional, Sequence, Tuple, Union

import torch
import torch.nn as nn
import torch.nn.functional as F
from torch.autograd import forward_ad

from ..utils.activation import ActivationFunctionEnum
from . import lib
from .glu import _ACT, GatedActivation, gated_activation

TINY = 2.0 ** -100
MOST_SCALE = float.fromhex("0x1.020406p+121")  # the largest scale whose 127-fold is an fp32 number
MAX_COLS = 131071  # 128 * 128 * cols has to fit into the 32-bit sums
_FLOATS = (torch.bfloat16, torch.float32)
_f = {}


class Int8Rows(NamedTuple):
    """Rows in 8 bits: ``values`` int8 ``[..., cols]`` and ``scale`` fp32 ``[...]``; they stand for ``values * scale``.  The rows that this module makes
    start at multiples of 16 bytes, as the products want them; others are copied there by every product."""

    values: torch.Tensor
    scale: torch.Tensor

    @property
    def shape(self) -> torch.Size:
        return self.values.shape

    @property
    def device(self) -> torch.device:
        return self.values.device

    # what a layer asks of the rows that it is given, whichever they are: a serving step's rows are bf16 ones
    dtype = property(lambda self: torch.bfloat16)
    is_cuda = property(lambda self: self.values.is_cuda)
    requires_grad = property(lambda self: False)

    def dim(self) -> int:
        return self.values.dim()

    def dequantize(self, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
        """What the rows stand for, ``values * scale`` rounded once to ``dtype`` (bf16 or fp32)."""
        v, s = self
        _check_rows(v, s, "rows")
        if dtype not in _FLOATS:
            raise TypeError(f"rows come back as bf16 or fp32, not {dtype}")
        if torch.is_grad_enabled() or forward_ad._current_level >= 0:
            _no_gradient("dequantize", s)
        if not _kernels(v):
            return (v.float() * s.unsqueeze(-1)).to(dtype)
        out = torch.empty(*v.shape, dtype=dtype, device=v.device)
        if out.numel() == 0:
            return out
        cols = v.size(-1)
        v, ptr, rows, ld = _rows_of(v)
        s = _dense(s)
        _launch("lvb_int8_dequantize", v, ptr, ld, s.data_ptr(), rows, cols, out.data_ptr(), int(dtype is torch.float32))
        return out


# ------------------------------------------------------------------------------------------------ calls
# Arguments of the launchers by letter (p pointer, l long long, i int, f float); a stream follows.
_ARGS = {"lvb_int8_quantize": "pilliplp", "lvb_int8_rms_norm": "pppilllpiffliplp", "lvb_int8_glu": "ppilliliplp", "lvb_int8_dequantize": "plplipi",
         "lvb_int8_gemm": "pppppiiilllippliiiip", "lvb_int8_quantize_parts": "pppppiiiiiipp"}


def _launch(name: str, t: torch.Tensor, *args) -> None:
    """Launches on the device of ``t`` and its current stream.  (Steps of a few rows take less time on the device than these lines on the host: what
    follows reads the state itself and makes no objects.)"""
    f = _f.get(name)
    if f is None:
        f = _f[name] = lib.quick(name, _ARGS[name] + "p")
    lib.launch_count += 1
    dev = t.get_device()
    if dev == _current():
        rc = f(*args, _stream(dev))
    else:
        with torch.cuda.device(dev):
            rc = f(*args, _stream(dev))
    if rc:
        lib.check_rc(rc, name)


_current = torch._C._cuda_getDevice if hasattr(torch._C, "_cuda_getDevice") else lambda: -1
_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _kernels(t: torch.Tensor) -> bool:
    if not t.is_cuda:
        return False
    major = lib._major.get(t.get_device())  # known after the first call on a device
    return lib.available() if major is None else major == 10 and not getattr(lib._tls, "reference", 0)


def _dense(t: torch.Tensor) -> torch.Tensor:
    return t if t.is_contiguous() else t.contiguous()


def _check_rows(v: torch.Tensor, s: torch.Tensor, what: str) -> None:
    if v.dtype is torch.int8 and s.dtype is torch.float32 and v.dim() == 2 and s.dim() == 1 and len(v) == len(s) and s.get_device() == v.get_device():
        return
    if v.dtype is not torch.int8 or s.dtype is not torch.float32:
        raise TypeError(f"{what}: int8 values with fp32 scales expected, got {v.dtype} and {s.dtype}")
    if v.dim() == 0 or s.shape != v.shape[:-1]:
        raise ValueError(f"{what}: values {tuple(v.shape)} need one scale per row, got {tuple(s.shape)}")
    if s.get_device() != v.get_device():
        raise ValueError(f"{what}: values on {v.device}, scales on {s.device}")


def _check_floats(what: str, like: torch.Tensor, other: Optional[torch.Tensor] = None) -> None:
    if like.dtype not in _FLOATS:
        raise TypeError(f"{what}: rows in bf16 or fp32 expected, got {like.dtype}")
    shape = like.shape
    if not shape or shape[-1] == 0:
        raise ValueError(f"{what}: rows of at least one element expected, got {tuple(shape)}")
    if other is not None and (other.dtype is not like.dtype or other.shape != shape or other.get_device() != like.get_device()):
        raise ValueError(f"{what}: {tuple(other.shape)} {other.dtype} on {other.device} does not go with {tuple(shape)} {like.dtype} on {like.device}")
    if torch.is_grad_enabled() or forward_ad._current_level >= 0:
        _no_gradient(what, like, other)


def _no_gradient(what: str, *tensors: Optional[torch.Tensor]) -> None:
    """Refuses tensors whose derivative, backward or forward, would be lost."""
    for t in tensors:
        if t is not None and t.requires_grad and torch.is_grad_enabled():
            raise RuntimeError(f"{what} has no gradient of its own: train with int8_linear_many, or call it under torch.no_grad()")
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise RuntimeError(f"{what} has no forward-mode derivative: call it with the primal values")


def _rows_of(t: torch.Tensor, align: int = 1) -> Tuple[torch.Tensor, int, int, int]:
    """``(t, address, rows, row stride in elements)`` of ``t [..., cols]`` as rows; copied unless the elements of a row lie side by side, rows do not
    overlap and they start at multiples of ``align`` bytes."""
    cols = t.shape[-1]
    if t.is_contiguous():
        rows, ptr = t.numel() // cols, t.data_ptr()
        if ptr % align == 0 and cols % 16 == 0:
            return t, ptr, rows, cols
        ld, ok = cols, True
    else:
        t = t if t.dim() == 2 else t.reshape(-1, cols)  # the caller keeps what a copy is read from
        rows, ld = t.shape[0], t.stride(0)
        ok = (cols == 1 or t.stride(1) == 1) and ld >= cols
    if rows == 1 and ok:
        ld = -(-cols // 16) * 16
    ptr = t.data_ptr()
    if not ok or (align > 1 and (ptr % align or ld * t.element_size() % align)):
        t = _room(t.shape, t.dtype, t.device, max(1, align // t.element_size())).copy_(t)
        return t, t.data_ptr(), rows, t.stride(-2) if rows > 1 and t.dim() > 1 else -(-cols // 16) * 16
    return t, ptr, rows, ld


def _room(shape, dtype: torch.dtype, device, multiple: int = 16) -> torch.Tensor:
    """An empty tensor whose rows start at multiples of that many elements."""
    cols = shape[-1]
    if cols % multiple == 0:
        return torch.empty(*shape, dtype=dtype, device=device)  # (sizes one by one are read faster than as a tuple)
    return torch.empty((*shape[:-1], -(-cols // multiple) * multiple), dtype=dtype, device=device)[..., :cols]


def _empty_rows(shape, device) -> Int8Rows:
    values = _room(shape, torch.int8, device)
    if len(shape) == 2:
        return Int8Rows(values, torch.empty(shape[0], dtype=torch.float32, device=device))
    return Int8Rows(values, torch.empty(shape[:-1], dtype=torch.float32, device=device))


# ------------------------------------------------------------------------------------------------ rows
def quantize_reference(y: torch.Tensor, factor: Optional[torch.Tensor] = None) -> Int8Rows:
    """PyTorch statement: the rows of ``factor * y`` (a positive number per row, which leaves the whole numbers as they are)."""
    y = y.float()
    top = y.abs().amax(-1, keepdim=True)
    most = top if factor is None else torch.where(top == 0, top, top * factor)  # (a row of zeros without an eps has an infinite factor)
    live = (most >= TINY) & (top >= 2.0 ** -120)
    q = torch.where(live & torch.isfinite(top), torch.round(y.double() * 127.0 / top.double()).float(), torch.zeros_like(y))  # (fp32 would run over)
    scale = torch.where(live, (most / 127.0).clamp_max(MOST_SCALE), torch.zeros_like(most))
    ok = torch.isfinite(top) & ~torch.isnan(most)
    scale = torch.where(ok, scale, torch.full_like(scale, float("nan")))
    values = _room(y.shape, torch.int8, y.device)
    return Int8Rows(values.copy_(torch.where(ok, q, torch.zeros_like(q))), scale.squeeze(-1))


def quantize_rows(x: torch.Tensor) -> Int8Rows:
    """The rows of ``x [..., cols]`` (bf16 or fp32, any strides) in 8 bits."""
    _check_floats("quantize_rows", x)
    return _quantize(x)


def _quantize(x: torch.Tensor) -> Int8Rows:
    if not _kernels(x):
        return quantize_reference(x.detach())
    shape = x.shape
    cols = shape[-1]
    x, ptr, rows, ld = _rows_of(x)
    out = _empty_rows(shape, x.device)
    if rows:
        _launch("lvb_int8_quantize", x, ptr, int(x.dtype is torch.float32), ld, rows, cols, out[0].data_ptr(), -(-cols // 16) * 16, out[1].data_ptr())
    return out


def rms_norm_int8(x: torch.Tensor, weight: Optional[torch.Tensor], eps: float = 1e-6, *, w_offset: float = 0.0,
                  residual: Optional[torch.Tensor] = None) -> Tuple[Int8Rows, Optional[torch.Tensor]]:
    """``(rows, h)``: the RMS norm of ``h = x + residual`` (rounded to the type of ``x``; without a residual ``x`` itself, and the second item is None) times
    ``weight + w_offset``, in 8 bits.  ``x [..., cols]`` and ``residual`` in bf16 or fp32, ``weight [cols]`` in bf16 or fp32 or None."""
    _check_floats("rms_norm_int8", x, residual)
    shape = x.shape
    cols = shape[-1]
    if weight is not None:
        if weight.dim() != 1 or weight.shape[0] != cols or weight.dtype not in _FLOATS or weight.get_device() != x.get_device():
            raise ValueError(f"rms_norm_int8: weight [{cols}] in bf16 or fp32 on {x.device} expected, got {tuple(weight.shape)} {weight.dtype} on {weight.device}")
        if torch.is_grad_enabled() or forward_ad._current_level >= 0:
            _no_gradient("rms_norm_int8", weight)
    if not _kernels(x):
        x = x.detach()
        h = x if residual is None else (x.float() + residual.detach().float()).to(x.dtype)
        f = h.float()
        mean = f.square().mean(-1, keepdim=True) + eps
        # squares that leave the range of fp32: of the elements times 2^-80 or 2^80, a factor that cancels
        s = torch.where(mean > torch.finfo(torch.float32).max, 2.0 ** -80, torch.where(mean < 2.0 ** -90, 2.0 ** 80, 1.0))
        f = f * s
        y = f if weight is None else f * (weight.detach().float() + w_offset)
        return quantize_reference(y, torch.rsqrt(f.square().mean(-1, keepdim=True) + eps * s * s)), None if residual is None else h
    x, ptr, rows, ldx = _rows_of(x)
    dev = x.device
    h, rptr, hptr, ldr = None, 0, 0, 0
    if residual is not None:
        residual, rptr, _, ldr = _rows_of(residual)
        h = torch.empty(*shape, dtype=x.dtype, device=dev)
        hptr = h.data_ptr()
    wptr = w32 = 0
    if weight is not None:
        weight = _dense(weight)
        wptr, w32 = weight.data_ptr(), int(weight.dtype is torch.float32)
    out = _empty_rows(shape, dev)
    if rows:
        _launch("lvb_int8_rms_norm", x, ptr, rptr, hptr, int(x.dtype is torch.float32), ldx, ldr, cols, wptr, w32, w_offset, eps, rows, cols, out[0].data_ptr(),
                -(-cols // 16) * 16, out[1].data_ptr())
    return out, h


def gated_activation_int8(gate: torch.Tensor, up: torch.Tensor, act: GatedActivation) -> Int8Rows:
    """``act(gate) * up`` in 8 bits; ``gate`` and ``up [..., cols]`` in bf16 or fp32 may be the halves of a joint product's rows."""
    _check_floats("gated_activation_int8", gate, up)
    if isinstance(act, str) and not isinstance(act, ActivationFunctionEnum):
        act = ActivationFunctionEnum(act)
    if act not in _ACT:  # bounded gates and the like: quantised as they come
        return _quantize(gated_activation(gate.detach(), up.detach(), act))
    if not _kernels(gate):
        return quantize_reference(act.to_fn()(gate.detach().float()) * up.detach().float())
    shape = gate.shape
    cols = shape[-1]
    gate, gptr, rows, ldg = _rows_of(gate)
    up, uptr, _, ldu = _rows_of(up)
    out = _empty_rows(shape, gate.device)
    if rows:
        _launch("lvb_int8_glu", gate, gptr, uptr, int(gate.dtype is torch.float32), ldg, ldu, _ACT[act], rows, cols, out[0].data_ptr(), -(-cols // 16) * 16,
                out[1].data_ptr())
    return out


# ------------------------------------------------------------------------------------------------ products
F_OUT_F32, F_BIAS, F_BIAS_F32, F_RESIDUAL, F_RESIDUAL_F32 = 1, 2, 4, 8, 16


def int8_product(rows: Int8Rows, weight: Int8Rows, bias: Optional[torch.Tensor] = None, residual: Optional[torch.Tensor] = None,
                 out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``(values_x values_w^T) scale_x scale_w + bias + residual`` of ``rows [..., in]`` and ``weight [out, in]`` -> ``[..., out]`` in bf16 or fp32.

    The sums are exact whole numbers; scales, ``bias [out]`` and ``residual [..., out]`` (each in bf16 or fp32) are applied in fp32 and the result is
    rounded once.  ``in`` is at most 131071."""
    return _product(rows, weight, bias, residual, out_dtype)


def _product(rows: Int8Rows, weight: Int8Rows, bias=None, residual=None, out_dtype=torch.bfloat16, form: int = 0, splits: int = 0, stages: int = 0, tile: int = 0) -> torch.Tensor:
    v, sv = rows
    w, sw = weight
    _check_rows(v, sv, "int8_product: rows")
    _check_rows(w, sw, "int8_product: weight")
    shape = v.shape
    N, K = w.shape if w.dim() == 2 else (0, 0)
    if shape[-1] != K or w.get_device() != v.get_device():
        raise ValueError(f"int8_product: rows {tuple(shape)} on {v.device} and weight {tuple(w.shape)} on {w.device} do not go together")
    if not 0 < K <= MAX_COLS:
        raise ValueError(f"int8_product: rows of 1 to {MAX_COLS} elements expected, got {K}")
    if out_dtype not in _FLOATS:
        raise TypeError(f"int8_product: results in bf16 or fp32, not {out_dtype}")
    shape = (shape[0], N) if len(shape) == 2 else (*shape[:-1], N)
    if bias is not None or residual is not None:
        for t, want, what in ((bias, (N,), "bias"), (residual, shape, "residual")):
            if t is not None and (t.shape != want or t.dtype not in _FLOATS or t.get_device() != v.get_device()):
                raise ValueError(f"int8_product: {what} {want} in bf16 or fp32 on {v.device} expected, got {tuple(t.shape)} {t.dtype} on {t.device}")
    if torch.is_grad_enabled() or forward_ad._current_level >= 0:
        _no_gradient("int8_product", sv, sw, bias, residual)
    if not _kernels(v):
        sums, sv = torch.matmul(v.double(), w.double().t()).float(), sv.unsqueeze(-1)
        y = sums * sv * sw
        y = torch.where(torch.isfinite(y), y, sums * (sv * 2.0 ** -32) * sw * 2.0 ** 32)  # rows of very large numbers run over in the first product
        for t in (bias, residual):
            y = y if t is None else y + t.float()
        return y.to(out_dtype)
    out = torch.empty(*shape, dtype=out_dtype, device=v.device)
    v, a, M, lda = _rows_of(v, 16)
    w, b, _, ldb = _rows_of(w, 16)
    if M == 0 or N == 0:
        return out
    flags = F_OUT_F32 if out_dtype is torch.float32 else 0
    bptr = rptr = ldr = 0
    if bias is not None:
        flags |= F_BIAS | (F_BIAS_F32 if bias.dtype is torch.float32 else 0)
        bias = _dense(bias)
        bptr = bias.data_ptr()
    if residual is not None:
        flags |= F_RESIDUAL | (F_RESIDUAL_F32 if residual.dtype is torch.float32 else 0)
        residual, rptr, _, ldr = _rows_of(residual)
    if not (sv.is_contiguous() and sw.is_contiguous()):
        sv, sw = sv.contiguous(), sw.contiguous()
    _launch("lvb_int8_gemm", v, a, b, sv.data_ptr(), sw.data_ptr(), out.data_ptr(), M, N, K, lda, ldb, N, flags, bptr, rptr, ldr, form, tile, splits, stages,
            _status(v))
    return out


def _status(t: torch.Tensor) -> int:
    """Address of the status word on the device of ``t``."""
    buf = lib._status.get(t.get_device())
    if buf is None:
        with torch.cuda.device(t.device):
            buf = lib.status_buffer()
    return buf.data_ptr()


# ------------------------------------------------------------------------------------------------ training
def _straight_through(x: torch.Tensor) -> torch.Tensor:
    """What the 8-bit rows of ``x`` stand for, in fp32, with the gradient passed on as it is."""
    x = x.float()
    return x + (quantize_reference(x.detach()).dequantize(torch.float32) - x).detach()


# Up to so many rows the host's part bounds a layer: the projections of a layer without biases are one product, whose columns are their results.  Above it their
# results are tensors of their own, as their readers expect them.
MANY_ROWS = 2048


def _side_by_side(rows: int, cols: int, outs: int) -> bool:
    """Whether the output gradients of several projections, ``outs`` columns in all, are copied side by side for one product each way.  That moves 4 bytes
    per row and output; a sum over the projections in fp32 moves 18 or more per row and column.  Forward and backward, us side by side / in fp32: 8192 rows of
    4096 by 4096 + 1024 + 1024 868 / 1034, 16384 of 2048 by 2048 + 512 + 512 516 / 828, 4096 of 2048 by two of 8192 639 / 682.  From some 4 outputs per column on
    there is little between them: 8192 rows of 4096 by two of 8192 2126 / 2193, of 10240 2782 / 2910, of 11008 3026 / 3055, of 14336 4061 / 4029; 32768 rows by two of 8192 9249 / 9041, of
    11008 13409 / 12612; 32768 of 1024 by two of 4096 1515 / 1363."""
    return rows <= 4096 or outs <= 5 * cols


def _hold(x: torch.Tensor, weights: Sequence[torch.Tensor]) -> Tuple[torch.Tensor, torch.Tensor, int]:
    """``(values, scale, stride)``: the 8-bit rows of ``x`` and of the weights, one behind the other, and the bytes from one to the next."""
    cols = x.shape[-1]
    ld = -(-cols // 16) * 16
    parts = [x, *weights]
    counts = [x.numel() // cols, *[w.shape[0] for w in weights]]
    total = sum(counts)
    values = torch.empty(total, ld, dtype=torch.int8, device=x.device)
    scale = torch.empty(total, dtype=torch.float32, device=x.device)
    q, s = values.data_ptr(), scale.data_ptr()
    if len(parts) <= 5 and ld == cols and 512 < cols <= 16384 and all(p.is_contiguous() and p.data_ptr() % 32 == 0 for p in parts):
        pad = (0,) * (5 - len(parts))
        _launch("lvb_int8_quantize_parts", x, *[p.data_ptr() for p in parts], *pad, *counts, *pad, cols, q, s)
    else:
        for part, n in zip(parts, counts):
            part, ptr, _, stride = _rows_of(part)
            _launch("lvb_int8_quantize", part, ptr, 0, stride, n, cols, q, ld, s)
            q, s = q + n * ld, s + 4 * n
    return values, scale, ld


def _held_products(x: torch.Tensor, values: torch.Tensor, scale: torch.Tensor, ld: int, weights, biases) -> Tuple[torch.Tensor, ...]:
    """The products of what :func:`_hold` gives for ``x`` and the weights."""
    lead, cols, rows = x.shape[:-1], x.shape[-1], x.numel() // x.shape[-1]
    q, s, status = values.data_ptr(), scale.data_ptr(), _status(x)

    def product(first: int, outs: int, bias):
        y = torch.empty(*lead, outs, dtype=torch.bfloat16, device=x.device)
        flags = 0
        if bias is not None:
            flags, bias = F_BIAS | (F_BIAS_F32 if bias.dtype is torch.float32 else 0), _dense(bias)
        _launch("lvb_int8_gemm", y, q, q + first * ld, s, s + 4 * first, y.data_ptr(), rows, outs, cols, ld, ld, outs, flags, lib.ptr(bias), 0, 0, 0, 0, 0, 0, status)
        return y

    if len(weights) > 1 and rows <= MANY_ROWS and all(b is None for b in biases):
        sizes = [w.shape[0] for w in weights]
        return product(rows, sum(sizes), None).split(sizes, dim=-1)
    ys, first = [], rows
    for w, b in zip(weights, biases):
        ys.append(product(first, w.shape[0], b))
        first += w.shape[0]
    return tuple(ys)


class _WeightRef:
    """What the backward pass wants to know of a weight, without keeping a converted copy of it."""

    __slots__ = ("shape", "dtype", "parameter")

    def __init__(self, w: torch.Tensor):
        self.shape, self.dtype = w.shape, w.dtype
        p = getattr(w, "converted_from", w)
        named = getattr(p, "main_grad", None) is not None or getattr(p, "grad_sink", None) is not None
        self.parameter = p if p.requires_grad and (p.is_leaf or named) else None

    main_grad = property(lambda self: getattr(self.parameter, "main_grad", None))
    grad_sink = property(lambda self: getattr(self.parameter, "grad_sink", None))


def _gemm_rows(d: torch.Tensor) -> torch.Tensor:
    """``d [rows, cols]`` as bf16 rows that the GEMM reads where they lie."""
    cols = d.shape[1]
    if d.dtype is torch.bfloat16 and d.stride(1) == 1 and d.stride(0) >= cols and d.stride(0) % 8 == 0 and d.data_ptr() % 16 == 0:
        return d
    return _room(d.shape, torch.bfloat16, d.device, 8).copy_(d)


class _Int8ManyFn(torch.autograd.Function):
    """Projections of the same rows.  Kept for the backward pass: the rows and the weights in 8 bits, once for all projections.  bf16 layers keep 2 bytes per activation and
    the parameters, which are there anyhow; this is 1 per activation and 1 per weight, so less of it where there are more rows than outputs.

    ``dx = sum dy w'`` and ``dw = dy^T x'`` are bf16 products of what the whole numbers stand for, rounded to bf16 (2^-8 of each value at most, as any operand
    of a bf16 layer); output gradients are not quantised, their rows span too many magnitudes for one scale.  The sum over several projections is rounded
    once: their output gradients are laid side by side for one product each way (:func:`_side_by_side`), or it is formed in fp32 (8192 rows of 4096 by two of
    11008 1268 to 1313 us; rounding the first product ahead of the second 1158 to 1239, at the price of a second rounding)."""

    @staticmethod
    def forward(ctx, x, count, *tensors):
        weights, biases = tensors[:count], tensors[count:]
        values, scale, ld = _hold(x, weights)
        ctx.save_for_backward(values, scale)
        ctx.refs, ctx.bias_dtypes = [_WeightRef(w) for w in weights], [None if b is None else b.dtype for b in biases]
        ctx.x_shape, ctx.ld = x.shape, ld
        ctx.set_materialize_grads(False)  # a product that nothing uses has no gradient, and its weight none
        # (parts of one tensor, which autograd would take for views of each other and refuse to have written in place)
        return tuple(y.data for y in _held_products(x, values, scale, ld, weights, biases))

    @staticmethod
    def backward(ctx, *dys):
        from .gemm import _weight_grad, col_sum, gemm

        values, scale = ctx.saved_tensors
        refs, shape, ld = ctx.refs, ctx.x_shape, ctx.ld
        n, cols = len(refs), shape[-1]
        total, rows = values.shape[0], values.shape[0] - sum(w.shape[0] for w in refs)
        need = ctx.needs_input_grad
        live = [i for i in range(n) if dys[i] is not None]
        dws, dbs = [None] * n, [None] * n
        if not live:
            return (None, None, *dws, *dbs)
        d2 = [_gemm_rows(dys[i].reshape(rows, refs[i].shape[0])) for i in live]
        need_w = [i for i in live if need[2 + i]]
        # what the rows in question stand for, in one launch: x, the weights or both
        first, last = 0 if need_w else rows, total if need[0] else rows
        wide = -(-cols // 8) * 8  # (the GEMM's rows start on 16 bytes; what is held has room for as many columns)
        back = torch.empty(last - first, wide, dtype=torch.bfloat16, device=values.device) if last > first else None
        if back is not None:
            _launch("lvb_int8_dequantize", values, values.data_ptr() + first * ld, ld, scale.data_ptr() + 4 * first, last - first, wide, back.data_ptr(), 0)
        side = d2[0] if len(live) == 1 else _gemm_rows(torch.cat(d2, dim=1)) if _side_by_side(rows, cols, sum(d.shape[1] for d in d2)) else None
        dx = None
        if need[0]:
            w = back[rows - first:]
            if len(live) < n or side is None:
                ws = [p for i, p in enumerate(w.split([r.shape[0] for r in refs])) if i in live]
            if side is not None:
                dx = gemm(side, (w if len(live) == n else torch.cat(ws))[:, :cols], b_mn=True)
            else:
                for d, w in zip(d2, ws):
                    dx = gemm(d, w[:, :cols], b_mn=True, out=dx, accumulate=dx is not None, out_dtype=torch.float32)
                dx = dx.to(torch.bfloat16)
            dx = dx.view(shape)
        if need_w:
            x2 = back[:rows, :cols]
            own = all(getattr(refs[i], "main_grad", None) is None and getattr(refs[i], "grad_sink", None) is None and refs[i].dtype is torch.bfloat16 for i in live)
            if len(live) > 1 and side is not None and need_w == live and own:
                for i, dw in zip(live, gemm(side, x2, a_mn=True, b_mn=True).split([refs[i].shape[0] for i in live])):
                    dws[i] = dw
            else:
                for i, d in zip(live, d2):
                    if need[2 + i]:
                        dws[i] = _weight_grad(refs[i], d, x2)
        for i, d in zip(live, d2):
            if ctx.bias_dtypes[i] is not None and need[2 + n + i]:
                dbs[i] = col_sum(d, ctx.bias_dtypes[i])
        return (dx, None, *dws, *dbs)


def int8_linear_many(x: torch.Tensor, weights: Sequence[torch.Tensor], biases: Optional[Sequence[Optional[torch.Tensor]]] = None) -> Tuple[torch.Tensor, ...]:
    """``[x' w'^T + b for w, b in ...]`` with ``x [..., in]`` and the ``weights [out, in]`` held in 8 bits (``x'``, ``w'``: what their whole numbers stand for);
    differentiable in ``x``, weights and biases.  bf16 on a GPU runs on the kernels, everything else on PyTorch's operations in fp32, rounded once.  Of several
    projections without biases of up to ``MANY_ROWS`` rows the results are columns of one tensor: each has the others' columns between its rows."""
    weights = list(weights)
    biases = [None] * len(weights) if biases is None else list(biases)
    if not weights or len(biases) != len(weights):
        raise ValueError(f"int8_linear_many: one bias (or None) per weight expected, got {len(biases)} for {len(weights)}")
    if x.dtype not in _FLOATS:
        raise TypeError(f"int8_linear_many: rows in bf16 or fp32 expected, got {x.dtype}")
    for w, b in zip(weights, biases):
        if w.dim() != 2 or w.shape[1] != x.shape[-1] or not 0 < w.shape[1] <= MAX_COLS or w.device != x.device or w.dtype not in _FLOATS:
            raise ValueError(f"int8_linear_many: x {tuple(x.shape)} on {x.device} and a weight {tuple(w.shape)} {w.dtype} on {w.device} do not go together")
        if b is not None and (b.shape != (w.shape[0],) or b.device != x.device or b.dtype not in _FLOATS):
            raise ValueError(f"int8_linear_many: bias [{w.shape[0]}] on {x.device} expected, got {tuple(b.shape)} {b.dtype} on {b.device}")
    if _kernels(x) and x.dtype == torch.bfloat16 and x.numel() and all(w.dtype == torch.bfloat16 and w.shape[0] > 0 for w in weights):
        if lib.plain_call():
            return _held_products(x, *_hold(x, weights), weights, biases)
        return _Int8ManyFn.apply(x, len(weights), *weights, *biases)
    x8 = _straight_through(x)
    return tuple(F.linear(x8, _straight_through(w), None if b is None else b.float()).to(x.dtype) for w, b in zip(weights, biases))


def int8_linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """:func:`int8_linear_many` of one projection."""
    return int8_linear_many(x, [weight], [bias])[0]


# ------------------------------------------------------------------------------------------------ modules
class Int8Linear(nn.Module):
    """Drop-in for :class:`levanter_b200.nn.Linear` that trains on :func:`int8_linear`: it owns the same ``weight`` and ``bias`` parameters; master weights,
    optimizer state and checkpoints are unchanged."""

    def __init__(self, weight: nn.Parameter, bias: Optional[nn.Parameter]):
        super().__init__()
        self.weight, self.bias = weight, bias
        self.in_features, self.out_features = weight.shape[1], weight.shape[0]

    @staticmethod
    def from_linear(linear: nn.Module) -> "Int8Linear":
        return Int8Linear(linear.weight, getattr(linear, "bias", None))

    def operand(self, dtype: torch.dtype) -> torch.Tensor:
        """The weight in ``dtype``; the gradient of a converted one goes into the buffer that the weight names."""
        if self.weight.dtype == dtype:
            return self.weight
        w = self.weight.to(dtype)
        w.converted_from = self.weight
        return w

    def forward(self, x: torch.Tensor, *, skip_bias: bool = False) -> torch.Tensor:
        return int8_linear(x, self.operand(x.dtype), None if skip_bias else self.bias)

    def extra_repr(self):
        return f"in={self.in_features}, out={self.out_features}, bias={self.bias is not None}, int8"


class Int8ServingLinear(nn.Module):
    """A projection that serves: its weights are held in 8 bits (buffers ``weight`` int8 ``[out, in]`` and ``weight_scale`` fp32 ``[out]``) and have no gradient.
    A state with the weight in another type is quantised as it is loaded.
    It takes rows in bf16 or fp32, or :class:`Int8Rows` that several projections share, gives results of their type (of 8-bit rows: bf16) or in ``out_dtype``, and
    adds a ``residual`` in its product's epilogue."""

    def __init__(self, weight: torch.Tensor, bias: Optional[torch.Tensor]):
        super().__init__()
        self.check_weight(weight)
        self.out_features, self.in_features = weight.shape
        rows = _quantize(weight.detach())
        self.register_buffer("weight", rows.values)
        self.register_buffer("weight_scale", rows.scale)
        self.register_buffer("bias", None if bias is None else bias.detach())

    @staticmethod
    def check_weight(weight: torch.Tensor) -> None:
        if weight.dim() != 2 or weight.dtype not in _FLOATS or not 0 < weight.shape[1] <= MAX_COLS:
            raise ValueError(f"a weight [out, in] in bf16 or fp32 with up to {MAX_COLS} columns expected, got {tuple(weight.shape)} {weight.dtype}")

    @staticmethod
    def from_linear(linear: nn.Module) -> "Int8ServingLinear":
        return Int8ServingLinear(linear.weight, getattr(linear, "bias", None))

    @property
    def rows(self) -> Int8Rows:
        return Int8Rows(self.weight, self.weight_scale)

    def _apply(self, fn, recurse=True):
        scale = self.weight_scale
        super()._apply(fn, recurse)
        if self.weight_scale.dtype != torch.float32:  # a model's conversion to another type leaves the scales as they are
            self.weight_scale = scale.to(self.weight.device)
        self._keep_rows_apart()
        return self

    def _keep_rows_apart(self):
        """A move or a load may have packed rows of a width that is no multiple of 16: every product would copy them back to where it reads them."""
        w = self.weight
        if w.stride(0) % 16 and w.shape[0] > 1:
            self.weight = _room(w.shape, w.dtype, w.device).copy_(w)

    def _load_from_state_dict(self, state_dict, prefix, *args):
        w = state_dict.get(prefix + "weight")
        if w is not None and w.is_floating_point() and w.shape == self.weight.shape:  # of a model that was not quantised
            rows = _quantize(w.detach().to(self.weight.device, torch.bfloat16 if w.dtype is torch.bfloat16 else torch.float32))
            state_dict[prefix + "weight"], state_dict[prefix + "weight_scale"] = rows
        super()._load_from_state_dict(state_dict, prefix, *args)
        self._keep_rows_apart()

    def forward(self, x: Union[torch.Tensor, Int8Rows], *, skip_bias: bool = False, residual: Optional[torch.Tensor] = None,
                out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
        return int8_product(as_int8_rows(x), self.rows, None if skip_bias else self.bias, residual, out_dtype=x.dtype if out_dtype is None else out_dtype)

    def extra_repr(self):
        return f"in={self.in_features}, out={self.out_features}, bias={self.bias is not None}, int8 weights"


def as_int8_rows(x: Union[torch.Tensor, Int8Rows]) -> Int8Rows:
    return x if isinstance(x, Int8Rows) else quantize_rows(x)

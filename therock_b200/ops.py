"""Operators an expert layer is built from when it is not one fused call.

    grouped_matmul(x, weight, offsets)             rows grouped by expert times that expert's weight
    matmul_block128(a, a_scale, w, w_scale, quant) e4m3 matrices with a scale for each block of 128
    silu_mul(gu, row_weight)                       the gated activation, optionally times a weight per row
    silu_mul_quantise(gu, quant, row_weight)       the same as e4m3 rows with their scales

`grouped_matmul` and `silu_mul` have gradients (first order, through torch.autograd).  Every call
enqueues kernels of libfmoe_b200.so on `stream` (the tensors' current stream by default) and
returns: no host synchronisation, no atomics, so the same inputs give the same bits, and a call can
be captured in a CUDA graph (a forward and its backward pass in one graph; no earlier graph of the
same tensors that was recorded on the default stream may be alive).  Inputs are contiguous CUDA tensors on one device, which need not be
the current one; a call on another stream than the current one allocates its results for that
stream, and the caller orders the streams.  Bad arguments raise FmoeError before any launch, and so does a
call that a tracer records (torch.ops.therock_b200 has all of them but silu_mul_quantise for traced and
compiled programs)."""
from __future__ import annotations

import ctypes
from typing import Optional

import torch
from torch.autograd import forward_ad
from torch.autograd.graph import increment_version

from .api import QUANT, FmoeError, _check, lib

_current_raw_stream = torch._C._cuda_getCurrentRawStream
_DTYPE = {torch.bfloat16: 0, torch.float16: 2}
_E4M3 = (torch.float8_e4m3fn, torch.uint8)
_BLOCK_QUANT = ("block128", "block128_ue8m0")


def _bound():
    """The library with the signatures of these entry points set."""
    l = lib()
    if l.fmoe_grouped_matmul.argtypes is None:
        vp, i32, i64 = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64
        l.fmoe_operator_status.argtypes = [i32, ctypes.POINTER(i32)]
        l.fmoe_grouped_matmul_wgrad.argtypes = [vp, vp, vp, i64, i32, i32, i32, i32, vp, vp, vp]
        l.fmoe_matmul_block128.argtypes = [vp, vp, vp, vp, i64, i32, i32, i32, vp, vp, vp]
        l.fmoe_describe_matmul_block128.argtypes = [i64, i32, i32, i32, ctypes.POINTER(_MatmulInfo)]
        l.fmoe_silu_mul.argtypes = [vp, vp, i64, i32, i32, vp, vp]
        l.fmoe_silu_mul_quantise.argtypes = [vp, vp, i64, i32, i32, i32, vp, vp, vp]
        l.fmoe_silu_mul_backward.argtypes = [vp, vp, vp, i64, i32, i32, vp, vp, vp]
        l.fmoe_grouped_matmul.argtypes = [vp, vp, vp, i64, i32, i32, i32, i32, i32, vp, vp, vp]
    return l


class _MatmulInfo(ctypes.Structure):
    _fields_ = [("kernel", ctypes.c_int32), ("rows_per_tile", ctypes.c_int32), ("cols_per_tile", ctypes.c_int32),
                ("k_split", ctypes.c_int32), ("reserved", ctypes.c_int32 * 4)]


_MATMUL_KERNEL = {0: "none", 1: "few_rows", 2: "tiles", 3: "cta_pairs"}
_binding = None


def _native():
    """The CPython binding of the calls without `out` and `stream` (torch_binding.cpp), which also holds
    the autograd nodes; bound to the library that api.lib() loads."""
    global _binding
    if _binding is None:
        l = _bound()
        try:
            from . import _fmoe_torch as binding
        except ImportError as e:
            raise FmoeError(-100, f"the torch binding is missing or does not load ({e}): build it with "
                                  "`python -m therock_b200.build` under this interpreter and torch") from None
        binding.bind(FmoeError, *(ctypes.cast(getattr(l, n), ctypes.c_void_p).value for n in (
            "fmoe_grouped_matmul", "fmoe_grouped_matmul_wgrad", "fmoe_matmul_block128", "fmoe_silu_mul",
            "fmoe_silu_mul_quantise", "fmoe_silu_mul_backward", "fmoe_last_error")))
        _binding = binding
    return _binding


def operator_status(device=None) -> int:
    """Waits for the device and returns the code of the last bounded wait that ran out in one of this
    module's kernels (0: none did), and clears it."""
    index = torch.device("cuda" if device is None else device).index
    code = ctypes.c_int32(0)
    _check(_bound().fmoe_operator_status(torch.cuda.current_device() if index is None else index, ctypes.byref(code)))
    return int(code.value)


def _stream_of(t: torch.Tensor, stream) -> int:
    if stream is None:
        return _current_raw_stream(t.get_device())
    return int(stream.cuda_stream) if hasattr(stream, "cuda_stream") else int(stream)


def _empty(shape, dtype, like: torch.Tensor, stream) -> torch.Tensor:
    """A result, allocated for the stream that writes it."""
    if stream is None:
        return like.new_empty(shape) if dtype is like.dtype else like.new_empty(shape, dtype=dtype)
    if not hasattr(stream, "cuda_stream"):
        stream = torch.cuda.ExternalStream(int(stream), device=like.device)
    with torch.cuda.stream(stream):
        return torch.empty(shape, dtype=dtype, device=like.device)


def _dense(name: str, t, device: int = -1, align: int = 16) -> int:
    """Checks a tensor and returns its device index (`device`: the index it has to be on, if given)."""
    try:
        index = t.get_device()
        if index < 0 or not t.is_contiguous():
            raise FmoeError(-1, f"{name} must be a contiguous CUDA tensor")
    except AttributeError:
        raise FmoeError(-1, f"{name} must be a contiguous CUDA tensor") from None
    if t.data_ptr() % align:
        raise FmoeError(-1, f"{name} must be {align}-byte aligned")
    if device >= 0 and index != device:
        raise FmoeError(-1, f"{name} is on cuda:{index}, the other tensors on cuda:{device}")
    return index


def _sizes(*sizes) -> None:
    """The entry points take these as 32-bit numbers."""
    if max(sizes) > 0x7fffffff:
        raise FmoeError(-2, "problem too large: all sizes but the number of rows must fit 32 bits")


def _result(name: str, out, shape, dtype, like: torch.Tensor, stream, *apart) -> torch.Tensor:
    """The tensor that takes the result; `apart` are those it must not share memory with."""
    if out is None:
        return _empty(shape, dtype, like, stream)
    _dense(name, out, like.get_device())
    if tuple(out.shape) != tuple(shape) or out.dtype != dtype:
        raise FmoeError(-1, f"{name} must be {dtype} {tuple(shape)}")
    if torch.is_grad_enabled() and out.requires_grad:
        raise FmoeError(-1, f"{name} must not require a gradient")
    first, last = out.data_ptr(), out.data_ptr() + out.numel() * out.element_size()
    for t in apart:
        if t is not None and t.data_ptr() < last and first < t.data_ptr() + t.numel() * t.element_size():
            raise FmoeError(-1, f"{name} must not share memory with the other tensors")
    return out


def _filled(given, result):
    """`result`, with the tensor that the caller gave for it marked as written: a graph that had saved it
    says so instead of using its new values."""
    if given is not None:
        increment_version(given)
    return result


def _for_kernel(t: torch.Tensor) -> torch.Tensor:
    """A gradient that autograd may hand over with any strides (expanded, sliced) as the kernels read it."""
    t = t.contiguous()
    return t.clone() if t.data_ptr() & 15 else t


_PROXY = torch._C._TorchDispatchModeKey.PROXY
_TRACERS = [torch._C._dispatch_key_parse(k) for k in ("Tracer", "PreDispatch")]


def _refuse_tracers() -> None:
    """A tracer (make_fx, torch.jit.trace, export) would record the allocation of the result and not the
    call that fills it.  Inside a registered operator it is off."""
    if torch._C._get_dispatch_mode(_PROXY) is not None or any(
            torch._C._dispatch_tls_is_dispatch_key_included(k) and not torch._C._dispatch_tls_is_dispatch_key_excluded(k) for k in _TRACERS):
        raise FmoeError(-1, "a traced program cannot hold this call: use the operator of torch.ops.therock_b200 (import "
                            "therock_b200.torch_op), or leave the call out of the trace")


def _refuse_gradients(*tensors) -> None:
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise FmoeError(-1, "out and stream are for calls without gradients (use torch.no_grad or torch.cuda.stream)")
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise FmoeError(-1, "forward-mode derivatives are not supported")


# ----------------------------------------------------------------------------- products grouped by expert
def _check_grouped(x, weight, offsets):
    _refuse_tracers()
    index = _dense("x", x)
    _dense("weight", weight, index)
    _dense("offsets", offsets, index, 4)
    if x.dtype not in _DTYPE or weight.dtype is not x.dtype:
        raise FmoeError(-1, "x and weight must both be bfloat16 or both float16")
    xs, ws = x.shape, weight.shape
    if len(xs) != 2 or len(ws) != 3 or ws[2] != xs[1]:
        raise FmoeError(-1, "x must be [rows, k] and weight [groups, n, k]")
    if offsets.dtype is not torch.int32 or offsets.dim() != 1 or offsets.numel() != ws[0] + 1:
        raise FmoeError(-1, "offsets must be int32 [groups + 1]")


def _grouped(x, weight, offsets, transpose: bool, out, stream):
    groups, n, k = weight.shape
    rows = x.shape[0]
    _sizes(groups, n, k)
    y = _result("out", out, (rows, k if transpose else n), x.dtype, x, stream, x, weight, offsets)
    rc = _bound().fmoe_grouped_matmul(x.data_ptr(), weight.data_ptr(), offsets.data_ptr(), rows, groups, n, k, _DTYPE[x.dtype],
                                      transpose, y.data_ptr(), None, _stream_of(x, stream))
    if rc:
        _check(rc)
    return _filled(out, y)


def grouped_matmul_dgrad(dy: torch.Tensor, weight: torch.Tensor, offsets: torch.Tensor, out: Optional[torch.Tensor] = None,
                         stream=None) -> torch.Tensor:
    """dx [rows, k] with dx[r] = weight[g]^T dy[r] for the rows of group g, zeros for rows of none: the
    gradient of grouped_matmul with respect to x, from dy [rows, n].  No gradient of its own."""
    _refuse_tracers()
    index = _dense("dy", dy)
    _dense("weight", weight, index)
    _dense("offsets", offsets, index, 4)
    if dy.dtype not in _DTYPE or weight.dtype != dy.dtype:
        raise FmoeError(-1, "dy and weight must both be bfloat16 or both float16")
    if dy.dim() != 2 or weight.dim() != 3 or weight.shape[1] != dy.shape[1]:
        raise FmoeError(-1, "dy must be [rows, n] and weight [groups, n, k]")
    if offsets.dtype != torch.int32 or offsets.dim() != 1 or offsets.shape[0] != weight.shape[0] + 1:
        raise FmoeError(-1, "offsets must be int32 [groups + 1]")
    return _grouped(dy, weight, offsets, True, out, stream)


def grouped_matmul_wgrad(dy: torch.Tensor, x: torch.Tensor, offsets: torch.Tensor, out: Optional[torch.Tensor] = None,
                         stream=None) -> torch.Tensor:
    """dw [groups, n, k] with dw[g] = dy[rows of g]^T x[rows of g]; zeros for a group without rows.
    Rows of no group do not enter it, whatever they hold.  No gradient of its own."""
    _refuse_tracers()
    index = _dense("dy", dy)
    _dense("x", x, index)
    _dense("offsets", offsets, index, 4)
    if x.dtype not in _DTYPE or dy.dtype != x.dtype:
        raise FmoeError(-1, "dy and x must both be bfloat16 or both float16")
    if x.dim() != 2 or dy.dim() != 2 or x.shape[0] != dy.shape[0]:
        raise FmoeError(-1, "dy must be [rows, n] and x [rows, k]")
    if offsets.dtype != torch.int32 or offsets.dim() != 1 or offsets.shape[0] < 2:
        raise FmoeError(-1, "offsets must be int32 [groups + 1]")
    groups, n, k = offsets.shape[0] - 1, dy.shape[1], x.shape[1]
    _sizes(groups, n, k)
    dw = _result("out", out, (groups, n, k), x.dtype, x, stream, dy, x, offsets)
    _check(_bound().fmoe_grouped_matmul_wgrad(dy.data_ptr(), x.data_ptr(), offsets.data_ptr(), x.shape[0], groups, n, k,
                                              _DTYPE[x.dtype], dw.data_ptr(), None, _stream_of(x, stream)))
    return _filled(out, dw)


def grouped_matmul(x: torch.Tensor, weight: torch.Tensor, offsets: torch.Tensor, out: Optional[torch.Tensor] = None,
                   stream=None) -> torch.Tensor:
    """y[r] = weight[g] @ x[r] for the rows offsets[g] <= r < offsets[g + 1] of group g.

    x [rows, k] and weight [groups, n, k] (the library's order: output channels, then k contiguous),
    both bfloat16 or both float16; offsets int32 [groups + 1] on the device, so routing needs no host
    step.  Sums are 32-bit, rounded once.  Groups may be empty; rows of no group (before offsets[0],
    from offsets[-1] on) give zero rows and zero gradients.  Offsets are read as a running maximum
    clamped to [0, rows].  n and k are multiples of 8, at most 1024 groups.  Differentiable in x and
    weight; `out` and `stream` are for calls without gradients."""
    if out is None and stream is None:
        y = (_binding or _native()).grouped_matmul(x, weight, offsets)
        if y is not None:
            return y
    _check_grouped(x, weight, offsets)
    _refuse_gradients(x, weight)
    return _grouped(x, weight, offsets, False, out, stream)


# ----------------------------------------------------------------------------- e4m3 products with block scales
def matmul_block128(a: torch.Tensor, a_scale: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor, quant: str = "block128",
                    out: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """bf16 [m, n] = (a * its scales) @ (w * its scales)^T, one scale per 128 of k.

    a [m, k] e4m3 (float8_e4m3fn, or its bytes as uint8) and a_scale as `quantise_rows(x, quant)`
    returns them, or a_scale as float32 [m, k/128] for "block128"; w [n, k] e4m3 and w_scale float32
    [ceil(n/128), k/128] (powers of two for "block128_ue8m0").  Each block's products are summed in 32
    bits and scaled by both scales before blocks are added, in 32 bits; one rounding.  k is a multiple
    of 128, m and n are any.  No gradient."""
    if quant not in _BLOCK_QUANT:
        raise FmoeError(-1, f"quant must be one of {_BLOCK_QUANT}")
    if out is None and stream is None:
        y = (_binding or _native()).matmul_block128(a, a_scale, w, w_scale, QUANT[quant])
        if y is not None:
            return y
    _refuse_tracers()
    index = _dense("a", a)
    _dense("w", w, index)
    if a.dtype not in _E4M3 or w.dtype not in _E4M3:
        raise FmoeError(-1, "a and w must be float8_e4m3fn (or uint8 holding it)")
    if a.dim() != 2 or w.dim() != 2:
        raise FmoeError(-1, "a must be [m, k] and w [n, k]")
    (m, k), (n, wk) = a.shape, w.shape
    if wk != k:
        raise FmoeError(-1, "a must be [m, k] and w [n, k]")
    if k % 128:
        raise FmoeError(-2, "k must be a multiple of 128")
    blocks = k // 128
    row_bytes = 4 * blocks if quant == "block128" else (blocks + 3) // 4 * 4
    _dense("a_scale", a_scale, index, 4)
    _dense("w_scale", w_scale, index, 4)
    if not (a_scale.dtype is torch.uint8 or (a_scale.dtype is torch.float32 and quant == "block128")) or \
            a_scale.shape != (m, row_bytes // a_scale.element_size()):
        raise FmoeError(-1, f"a_scale must hold {row_bytes} bytes for each of the {m} rows, as quantise_rows returns them")
    if w_scale.dtype is not torch.float32 or w_scale.shape != ((n + 127) // 128, blocks):
        raise FmoeError(-1, f"w_scale must be float32 [{(n + 127) // 128}, {blocks}]")
    _sizes(n, k)
    y = _result("out", out, (m, n), torch.bfloat16, a, stream, a, a_scale, w, w_scale)
    _check(_bound().fmoe_matmul_block128(a.data_ptr(), a_scale.data_ptr(), w.data_ptr(), w_scale.data_ptr(), m, n, k,
                                         QUANT[quant], y.data_ptr(), None, _stream_of(a, stream)))
    return _filled(out, y)


def describe_matmul_block128(m: int, n: int, k: int, quant: str = "block128") -> dict:
    """What matmul_block128 runs on for these sizes on the current device: the kernel ("few_rows", "tiles"
    or "cta_pairs"), the rows and columns of its tiles, and how many CTAs share a tile's blocks of k."""
    if quant not in _BLOCK_QUANT:
        raise FmoeError(-1, f"quant must be one of {_BLOCK_QUANT}")
    _sizes(n, k)
    info = _MatmulInfo()
    _check(_bound().fmoe_describe_matmul_block128(m, n, k, QUANT[quant], ctypes.byref(info)))
    return {"kernel": _MATMUL_KERNEL[info.kernel], **{f: int(getattr(info, f)) for f in ("rows_per_tile", "cols_per_tile", "k_split")}}


# ----------------------------------------------------------------------------- the gated activation
def _check_silu(gu, row_weight):
    _refuse_tracers()
    index = _dense("gu", gu)
    if gu.dtype not in _DTYPE:
        raise FmoeError(-1, "gu must be bfloat16 or float16")
    if gu.dim() != 2 or gu.shape[1] % 2:
        raise FmoeError(-1, "gu must be [rows, 2 * width]")
    if row_weight is not None:
        _dense("row_weight", row_weight, index, 4)
        if row_weight.dtype is not torch.float32 or row_weight.shape != gu.shape[:1]:
            raise FmoeError(-1, "row_weight must be float32 [rows]")
    _sizes(gu.shape[1])
    return gu.shape[0], gu.shape[1] // 2


def _silu(gu, row_weight, out, stream):
    rows, width = gu.shape[0], gu.shape[1] // 2
    y = _result("out", out, (rows, width), gu.dtype, gu, stream, gu, row_weight)
    _check(_bound().fmoe_silu_mul(gu.data_ptr(), None if row_weight is None else row_weight.data_ptr(), rows, width,
                                  _DTYPE[gu.dtype], y.data_ptr(), _stream_of(gu, stream)))
    return _filled(out, y)


def silu_mul_backward(gu: torch.Tensor, dy: torch.Tensor, row_weight: Optional[torch.Tensor] = None, stream=None):
    """Gradients of silu_mul: (dgu [rows, 2 * width], dweight float32 [rows] or None).  No gradients of their own."""
    rows, width = _check_silu(gu, row_weight)
    _dense("dy", dy, gu.get_device())
    if dy.dtype != gu.dtype or tuple(dy.shape) != (rows, width):
        raise FmoeError(-1, "dy must be [rows, width] of gu's type")
    dgu = _empty((rows, 2 * width), gu.dtype, gu, stream)
    dweight = None if row_weight is None else _empty((rows,), torch.float32, gu, stream)
    _check(_bound().fmoe_silu_mul_backward(gu.data_ptr(), None if row_weight is None else row_weight.data_ptr(), dy.data_ptr(),
                                           rows, width, _DTYPE[gu.dtype], dgu.data_ptr(),
                                           None if dweight is None else dweight.data_ptr(), _stream_of(gu, stream)))
    return dgu, dweight


def silu_mul(gu: torch.Tensor, row_weight: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
             stream=None) -> torch.Tensor:
    """out[r, i] = row_weight[r] * SiLU(gu[r, i]) * gu[r, width + i] for gu [rows, 2 * width] in
    bfloat16 or float16 (gate columns, then up columns), row_weight float32 [rows] or none.  32-bit
    arithmetic, one rounding; width is a multiple of 8.  Differentiable in gu and row_weight; `out`
    and `stream` are for calls without gradients."""
    if out is None and stream is None:
        y = (_binding or _native()).silu_mul(gu, row_weight)
        if y is not None:
            return y
    _check_silu(gu, row_weight)
    _refuse_gradients(gu, row_weight)
    return _silu(gu, row_weight, out, stream)


def silu_mul_quantise(gu: torch.Tensor, quant: str, row_weight: Optional[torch.Tensor] = None,
                      q: Optional[torch.Tensor] = None, scales: Optional[torch.Tensor] = None, stream=None):
    """quantise_rows(silu_mul(gu, row_weight), quant) in one pass, bit for bit, for the block modes:
    (q uint8 [rows, width], scales uint8 [rows, bytes]); from float16 by the same rule.  width is a multiple
    of 128.  A result that is infinite in gu's type spoils its group of 128.  No gradient."""
    if quant not in _BLOCK_QUANT:
        raise FmoeError(-1, f"quant must be one of {_BLOCK_QUANT}")
    if q is None and scales is None and stream is None:
        both = (_binding or _native()).silu_mul_quantise(gu, QUANT[quant], row_weight)
        if both is not None:
            return both
    rows, width = _check_silu(gu, row_weight)
    if width % 128:
        raise FmoeError(-2, "width must be a multiple of 128")
    groups = width // 128
    row_bytes = 4 * groups if quant == "block128" else (groups + 3) // 4 * 4
    to = _result("q", q, (rows, width), torch.uint8, gu, stream, gu, row_weight)
    s = _result("scales", scales, (rows, row_bytes), torch.uint8, gu, stream, gu, row_weight, to)
    _check(_bound().fmoe_silu_mul_quantise(gu.data_ptr(), None if row_weight is None else row_weight.data_ptr(), rows, width,
                                           _DTYPE[gu.dtype], QUANT[quant], to.data_ptr(), s.data_ptr(),
                                           _stream_of(gu, stream)))
    return _filled(q, to), _filled(scales, s)

"""The 8-bit float operators on torch tensors.

A thin layer over the entry points of include/futon_cuda.h (rms_norm_f8,
quantize_f8, matmul_t_f8, matmul_t_grouped): it checks types, shapes and
layouts, allocates what the caller did not pass, and queues the work on
torch's current stream of the tensors' device. Nothing is copied, converted
or kept; a tensor whose layout an operator does not take is refused.

  q, s      = quantize_f8(w, block_rows=128)               # weights, once
  q, s, h   = rms_norm_f8(x, gamma, eps, residual=r)       # next product's input
  y         = matmul_t_f8(q, s, wq, ws)                    # q · wᵀ
  q, s      = quantize_f8(y, activation="swiglu")          # between fc1‖gate and fc2
  y         = matmul_t_grouped(q, wq, offsets, a_scales=s, b_scales=ws)   # experts

Codes are torch.float8_e4m3fn, scales float32: code · scale is the value.
These operators have no backward pass: tensors that require a gradient are
refused while gradients are recorded.
"""
from __future__ import annotations

import ctypes as C
import threading
from typing import Optional, Tuple

from . import _lib
from ._lib import FutonError

BLOCK = 128  # columns of one scale (and rows, for weights)

_local = threading.local()
_T = None  # torch, and what is looked up in it on every call


class _Torch:
    def __init__(self) -> None:
        import torch
        self.torch = torch
        self.f8 = torch.float8_e4m3fn
        self.f32 = torch.float32
        self.codes = {torch.float32: _lib.DTYPE_F32, torch.float16: _lib.DTYPE_F16,
                      torch.bfloat16: _lib.DTYPE_BF16}
        self.grad = torch.is_grad_enabled
        # The raw handle of torch's current stream, without building a
        # torch.cuda.Stream object per call where torch offers that.
        self.stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
            lambda dev: torch.cuda.current_stream(dev).cuda_stream)
        L = _lib.lib()
        self.quantize = L.futon_cuda_quantize_f8
        self.norm = L.futon_cuda_rms_norm_f8
        self.matmul = L.futon_cuda_matmul_t_f8
        self.grouped = L.futon_cuda_matmul_t_grouped


def _torch() -> _Torch:
    global _T
    if _T is None:
        _T = _Torch()
    return _T


def _bad(msg: str) -> FutonError:
    return FutonError(_lib.FUTON_EINVAL, f"native: {msg}")


def _err():
    buf = getattr(_local, "err", None)
    if buf is None:
        buf = _local.err = C.create_string_buffer(512)
    return buf


def _run(fn, *args) -> None:
    buf = _err()
    rc = fn(*args, buf, 512)
    if rc:
        raise FutonError(rc, buf.value.decode("utf-8", "replace") or f"failed with code {rc}")


def _matrix(name: str, t, ndim: int = 2) -> int:
    """Row stride of a matrix (or a stack of matrices) whose columns are
    contiguous; refuses anything else."""
    if t.dim() != ndim:
        raise _bad(f"{name} has {t.dim()} dimensions, not {ndim}")
    st = t.stride()
    if t.shape[-1] > 1 and st[-1] != 1:
        raise _bad(f"{name}: the columns of a row must be contiguous")
    rows, k, ld = t.shape[-2], t.shape[-1], st[-2]
    if rows == 1:
        # One row has no row stride of its own.
        unit = max(1, 16 // t.element_size())
        ld = max(1, -(-k // unit)) * unit
    elif ld < k:
        raise _bad(f"{name}: rows overlap (stride {ld}, {k} columns)")
    return ld


def _dense(name: str, t, shape, dtype) -> None:
    if t.dtype != dtype or tuple(t.shape) != tuple(shape) or not t.is_contiguous():
        raise _bad(f"{name} must be a contiguous {dtype} tensor of shape {tuple(shape)}, "
                   f"got {t.dtype} {tuple(t.shape)}")


def _device(T: _Torch, *tensors) -> int:
    first = tensors[0].device
    if first.type != "cuda":
        raise _bad(f"tensors must be on a CUDA device, got {first}")
    grad = T.grad()
    for t in tensors:
        if t is None:
            continue
        if t.device != first:
            raise _bad(f"tensors on different devices: {first} and {t.device}")
        if grad and t.requires_grad:
            raise _bad("the 8-bit float operators have no backward pass: "
                       "call them under torch.no_grad() or on detached tensors")
    return first.index


def _pitched(T: _Torch, rows: int, k: int, device):
    """Codes [rows, k] whose rows start at multiples of 16 bytes, as the
    products take them."""
    wide = -(-k // 16) * 16
    q = T.torch.empty((rows, wide), dtype=T.f8, device=device)
    return q if wide == k else q[:, :k]


def _codes(T: _Torch, out, rows: int, k: int, scale_rows: int, device) -> Tuple:
    """(q, ldq, scales) of a quantiser's output."""
    nb = -(-k // BLOCK)
    if out is None:
        q = _pitched(T, rows, k, device)
        return q, q.stride(0), T.torch.empty((scale_rows, nb), dtype=T.f32, device=device)
    q, scales = out
    if q.dtype != T.f8 or tuple(q.shape) != (rows, k):
        raise _bad(f"out: codes must be float8_e4m3fn of shape {(rows, k)}, "
                   f"got {q.dtype} {tuple(q.shape)}")
    _dense("out: scales", scales, (scale_rows, nb), T.f32)
    return q, _matrix("out: codes", q), scales


_ACTS = {"none": _lib.QUANT_NONE, "gelu": _lib.QUANT_GELU, "swiglu": _lib.QUANT_SWIGLU}


def quantize_f8(src, activation: str = "none", block_rows: int = 1, out: Optional[Tuple] = None):
    """(codes, scales) of src [rows, k] after the activation.

    "swiglu" takes rows [fc1 | gate] of 2·k columns and gives
    fc1 · silu(gate); "gelu" is the exact-erf GELU. block_rows=1 gives every
    row and 128 columns a scale ([rows, ceil(k/128)]), block_rows=128 every
    128 × 128 block of a weight matrix."""
    T = _torch()
    if activation not in _ACTS:
        raise _bad(f"quantize_f8 activation {activation!r} (one of {', '.join(_ACTS)})")
    if block_rows not in (1, BLOCK):
        raise _bad(f"quantize_f8 block_rows={block_rows} (1 or {BLOCK})")
    dtype = T.codes.get(src.dtype)
    if dtype is None:
        raise _bad(f"quantize_f8 takes float32, float16 or bfloat16, got {src.dtype}")
    lds = _matrix("src", src)
    rows, k = src.shape
    if activation == "swiglu":
        if k % 2:
            raise _bad(f"quantize_f8: swiglu rows are [fc1 | gate], got {k} columns")
        k //= 2
    if k == 0:
        raise _bad(f"quantize_f8 shape rows={rows} k=0")
    q, ldq, scales = _codes(T, out, rows, k, rows if block_rows == 1 else -(-rows // BLOCK),
                            src.device)
    dev = _device(T, src, q, scales)
    _run(T.quantize, dev, q.data_ptr(), ldq, scales.data_ptr(), src.data_ptr(), lds, dtype, rows, k,
         _ACTS[activation], block_rows, T.stream(dev))
    return q, scales


def rms_norm_f8(x, weight, eps: float, residual=None, residual_out=None,
                out: Optional[Tuple] = None):
    """(codes, scales, h): h = x + residual, and the quantised rows of
    h / sqrt(mean(h²) + eps) · weight.

    h has x's type; it is written to residual_out where that is given (it
    may be the residual or x), to a new tensor where only residual is, and
    is None without a residual."""
    T = _torch()
    dtype = T.codes.get(x.dtype)
    if dtype is None:
        raise _bad(f"rms_norm_f8 takes float32, float16 or bfloat16, got {x.dtype}")
    ldx = _matrix("x", x)
    rows, k = x.shape
    if k == 0:
        raise _bad(f"rms_norm_f8 shape rows={rows} k=0")
    _dense("weight", weight, (k,), T.f32)
    if residual is not None and residual_out is None:
        residual_out = T.torch.empty((rows, k), dtype=x.dtype, device=x.device)
    ldr = ldo = 0
    for name, t in (("residual", residual), ("residual_out", residual_out)):
        if t is not None and (t.dtype != x.dtype or t.shape != x.shape):
            raise _bad(f"{name} must be {x.dtype} of shape {tuple(x.shape)}, "
                       f"got {t.dtype} {tuple(t.shape)}")
    if residual is not None:
        ldr = _matrix("residual", residual)
    if residual_out is not None:
        ldo = _matrix("residual_out", residual_out)
    q, ldq, scales = _codes(T, out, rows, k, rows, x.device)
    dev = _device(T, x, weight, residual, residual_out, q, scales)
    _run(T.norm, dev, q.data_ptr(), ldq, scales.data_ptr(),
         None if residual_out is None else residual_out.data_ptr(), ldo, x.data_ptr(), ldx,
         None if residual is None else residual.data_ptr(), ldr, weight.data_ptr(), dtype, rows, k,
         eps, T.stream(dev))
    return q, scales, residual_out


def _output(T: _Torch, out, out_dtype, m: int, n: int, device):
    """(out, its dtype code, its row stride)."""
    if out is None:
        out = T.torch.empty((m, n), dtype=out_dtype or T.torch.bfloat16, device=device)
    elif out_dtype is not None and out.dtype != out_dtype:
        raise _bad(f"out is {out.dtype}, out_dtype {out_dtype}")
    code = T.codes.get(out.dtype)
    if code is None:
        raise _bad(f"out must be float32, float16 or bfloat16, got {out.dtype}")
    if tuple(out.shape) != (m, n):
        raise _bad(f"out must have shape {(m, n)}, got {tuple(out.shape)}")
    return out, code, _matrix("out", out)


def matmul_t_f8(a, a_scales, b, b_scales, bias=None, out=None, out_dtype=None):
    """out [m, n] = values(a) [m, k] · values(b) [n, k]ᵀ (+ bias [n] float32).

    a_scales [m, ceil(k/128)], b_scales [ceil(n/128), ceil(k/128)]. Rows of a
    and b start at multiples of 16 bytes. out is float32, float16 or (the
    default) bfloat16."""
    T = _torch()
    if a.dtype != T.f8 or b.dtype != T.f8:
        raise _bad(f"matmul_t_f8 takes float8_e4m3fn operands, got {a.dtype} and {b.dtype}")
    lda, ldb = _matrix("a", a), _matrix("b", b)
    m, k = a.shape
    n = b.shape[0]
    if b.shape[1] != k or n == 0 or k == 0:
        raise _bad(f"matmul_t_f8 shapes {tuple(a.shape)} and {tuple(b.shape)}")
    nkb = -(-k // BLOCK)
    _dense("a_scales", a_scales, (m, nkb), T.f32)
    _dense("b_scales", b_scales, (-(-n // BLOCK), nkb), T.f32)
    if bias is not None:
        _dense("bias", bias, (n,), T.f32)
    out, code, ldd = _output(T, out, out_dtype, m, n, a.device)
    dev = _device(T, a, a_scales, b, b_scales, bias, out)
    _run(T.matmul, dev, out.data_ptr(), code, ldd, a.data_ptr(), lda, a_scales.data_ptr(),
         b.data_ptr(), ldb, b_scales.data_ptr(), m, n, k,
         None if bias is None else bias.data_ptr(), T.stream(dev))
    return out


def matmul_t_grouped(a, b, offsets, a_scales=None, b_scales=None, bias=None, out=None,
                     out_dtype=None):
    """out[i] = a[i] · b[g]ᵀ (+ bias[g]) for the rows offsets[g] ≤ i < offsets[g+1].

    a [m, k], b [groups, n, k], offsets int32 [groups + 1] on the device,
    non-decreasing within [0, m]. Both operands are float16, bfloat16 or
    float8_e4m3fn with a_scales [m, ceil(k/128)] and b_scales
    [groups, ceil(n/128), ceil(k/128)]. Rows of out in no group are left as
    they were (undefined in a new out). Offsets are read on the device: bad
    ones are clamped, and reported by f8_sync."""
    T = _torch()
    if a.dtype != b.dtype:
        raise _bad(f"matmul_t_grouped operands differ: {a.dtype} and {b.dtype}")
    f8 = a.dtype == T.f8
    dtype = _lib.DTYPE_E4M3 if f8 else T.codes.get(a.dtype)
    if dtype is None or dtype == _lib.DTYPE_F32:
        raise _bad(f"matmul_t_grouped takes float8_e4m3fn, float16 or bfloat16, got {a.dtype}")
    lda, ldb = _matrix("a", a), _matrix("b", b, 3)
    m, k = a.shape
    groups, n = b.shape[:2]
    if b.shape[2] != k or n == 0 or k == 0 or groups == 0:
        raise _bad(f"matmul_t_grouped shapes {tuple(a.shape)} and {tuple(b.shape)}")
    if groups > 1:
        # With one row per matrix the row stride is the matrices' distance.
        if n == 1:
            ldb = b.stride(0)
        if b.stride(0) != n * ldb or ldb < k:
            raise _bad(f"b: its matrices must lie {n * ldb} elements apart, not {b.stride(0)}")
    _dense("offsets", offsets, (groups + 1,), T.torch.int32)
    if f8:
        if a_scales is None or b_scales is None:
            raise _bad("matmul_t_grouped: float8_e4m3fn operands need a_scales and b_scales")
        nkb = -(-k // BLOCK)
        _dense("a_scales", a_scales, (m, nkb), T.f32)
        _dense("b_scales", b_scales, (groups, -(-n // BLOCK), nkb), T.f32)
    elif a_scales is not None or b_scales is not None:
        raise _bad(f"matmul_t_grouped: {a.dtype} operands take no scales")
    if bias is not None:
        _dense("bias", bias, (groups, n), T.f32)
    out, code, ldd = _output(T, out, out_dtype, m, n, a.device)
    dev = _device(T, a, b, offsets, a_scales, b_scales, bias, out)
    _run(T.grouped, dev, out.data_ptr(), code, ldd, a.data_ptr(), lda,
         a_scales.data_ptr() if f8 else None, b.data_ptr(), ldb,
         b_scales.data_ptr() if f8 else None, dtype, offsets.data_ptr(), groups, m, n, k,
         None if bias is None else bias.data_ptr(), T.stream(dev))
    return out


def f8_sync(device=None) -> None:
    """Waits for torch's current stream of `device` (default: the current
    device) and raises what the device found in these operators since the
    last call: offsets out of order, a wait that ran out."""
    T = _torch()
    dev = T.torch.device("cuda" if device is None else device)
    idx = T.torch.cuda.current_device() if dev.index is None else dev.index
    _lib.call("futon_cuda_f8_sync", idx, T.stream(idx))

"""Group norm and the fused matrix products (csrc/kernels/group_norm.hip, product.hip).

Channels last like every op here: the last dimension is contiguous, the leading ones may be a slice of a
wider (concat) buffer. Forward only, on the tensors' device and its current stream; a call allocates its
output and nothing that outlives it, so it can be captured into a graph. Weight and bias of a norm and bias of a
product are read in fp32: in x's type, each costs a conversion per call. Wrong arguments raise TypeError
or ValueError before anything is launched, a failure of the library raises ``NativeError``.
"""
from __future__ import annotations

import ctypes as C
import math
import struct
from typing import Optional, Tuple

import torch
from torch.autograd import forward_ad
from torch.autograd.graph import increment_version

from .. import _native as N

ACTIVATIONS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3, "gelu_tanh": 4}  # DML_ACT_*
_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}  # DML_BF16, DML_F16, DML_F32
_INT = 2 ** 31 - 1
# N.GroupNormArgs and N.ProductArgs as packed bytes: a call of small tensors is bound by the host, and filling the
# ctypes structures took a microsecond more
_NORM, _PROD = struct.Struct("@4P4qPq6if4x"), struct.Struct("@6P6q10i")
assert (_NORM.size, _PROD.size) == (C.sizeof(N.GroupNormArgs), C.sizeof(N.ProductArgs))


def _act(act: str) -> int:
    code = ACTIVATIONS.get(act)
    if code is None:
        raise ValueError(f"act is one of {', '.join(ACTIVATIONS)}: got {act!r}")
    return code


def _pitch(t: torch.Tensor, first: int, what: str) -> Tuple[int, int]:
    """(rows, elements from one row to the next) of dimensions first .. -2 of t seen as rows of its last one."""
    shape = t.shape
    if t.is_contiguous():
        if len(shape) == first + 2:
            return shape[first], shape[first + 1]
        return math.prod(shape[first:-1]), shape[-1]
    stride = t.stride()
    if shape[-1] > 1 and stride[-1] != 1:
        raise ValueError(f"{what}: the last dimension must be contiguous, got strides {stride}")
    rows, pitch = 1, None
    for d in range(t.dim() - 2, first - 1, -1):
        n = shape[d]
        if n != 1:
            if pitch is None:
                pitch = stride[d]
            elif stride[d] != pitch * rows and rows:
                raise ValueError(f"{what}: dimensions {first} to {t.dim() - 2} must step as one, got shape "
                                 f"{tuple(shape)} with strides {stride}")
            rows *= n
    return rows, shape[-1] if pitch is None else pitch


def _span(t: torch.Tensor) -> Tuple[int, int]:
    """First byte and the one behind the last of what t may touch."""
    p = t.data_ptr()
    if t.is_contiguous():
        return p, p + t.numel() * t.element_size()
    return p, p + t.element_size() * (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride())))


def _apart(out: torch.Tensor, same: str, **others: Optional[torch.Tensor]) -> None:
    """out must share no memory with the others unless they are other columns of one buffer. It may be the one named
    `same` itself (each workgroup reads its part before it writes there), but not where that is passed as another one too."""
    if not out.numel():
        return
    a, b = _span(out)
    for what, t in others.items():
        if t is None or not t.numel():
            continue
        c, d = _span(t)
        if b <= c or d <= a:
            continue
        if what == same and a == c and out.shape == t.shape and out.stride() == t.stride() and out.dtype == t.dtype:
            continue
        size = out.element_size()
        if size == t.element_size() and out.stride() == t.stride() and out.shape[:-1] == t.shape[:-1]:
            a1, c1 = a + out.shape[-1] * size, c + t.shape[-1] * size  # behind the first rows
            span = max(a1, c1) - min(a, c)
            fits = a1 <= c or c1 <= a
            for step, n in sorted((s * size, n) for s, n in zip(out.stride()[:-1], out.shape[:-1]) if n > 1):
                fits = fits and step >= span  # what both cover so far repeats without meeting itself
                span += (n - 1) * step
            if fits:
                continue
        raise ValueError(f"out overlaps {what}")


def _vector(v: torch.Tensor, shape: Tuple[int, ...], dtype: torch.dtype, what: str) -> None:
    if v.shape != shape:
        raise ValueError(f"{what}: expected shape {shape}, got {tuple(v.shape)}")
    if v.dtype is not torch.float32 and v.dtype is not dtype:
        raise TypeError(f"{what}: expected float32 or {dtype}, got {v.dtype}")


def _ready(x: torch.Tensor, *others: Optional[torch.Tensor]) -> int:
    """x's device number: all are on one HIP device, and none is one that autograd would expect a derivative for."""
    dev = x.get_device()
    grad = torch.is_grad_enabled()
    if grad and x.requires_grad:
        raise ValueError("this operator has no backward: call it under torch.no_grad()")
    for t in others:
        if t is not None:
            if t.get_device() != dev or (dev < 0 and t.device != x.device):
                raise ValueError(f"tensors on different devices: {x.device} and {t.device}")
            if grad and t.requires_grad:
                raise ValueError("this operator has no backward: call it under torch.no_grad()")
    if forward_ad._current_level >= 0:  # inside a dual_level; no_grad does not stop tangents
        for t in (x, *others):
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise ValueError("this operator has no derivative: call it on unpack_dual(t).primal")
    if dev < 0:
        raise ValueError(f"expected tensors on a HIP device, got {x.device}")
    return dev


def _launch(fn, args: bytes, device: int, what: str) -> int:
    """fn(args, the current stream of device), with device current."""
    if device == torch._C._cuda_getDevice():
        rc = fn(args, torch._C._cuda_getCurrentRawStream(device))
    else:
        with torch.cuda.device(device):
            rc = fn(args, torch._C._cuda_getCurrentRawStream(device))
    return N.check(rc, what) if rc else 0


def _f32(v: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    """v as contiguous fp32; v itself where it is that."""
    return v if v is None or v.dtype is torch.float32 and v.is_contiguous() else v.float().contiguous()


def group_norm(x: torch.Tensor, groups: int, weight: Optional[torch.Tensor] = None,
               bias: Optional[torch.Tensor] = None, eps: float = 1e-5, act: str = "none",
               out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Group norm, affine map and activation of channels-last features.

    x: [N, ..., C] bf16, fp16 or fp32; the dimensions between step as one (NHWC maps, [N, L, C] tokens, a
    channel slice of a concat buffer), any pitch between samples. Mean and variance (biased) go over all
    positions and the C / groups channels of a group, in fp32. weight, bias: [C], fp32 or x's type, or None.
    act: "none", "relu", "silu", "gelu" or "gelu_tanh". out: x's shape and type; may be x itself.
    """
    code = _act(act)
    dtype = _DTYPES.get(x.dtype)
    if dtype is None:
        raise TypeError(f"x: expected bfloat16, float16 or float32, got {x.dtype}")
    shape = x.shape
    if len(shape) < 2:
        raise ValueError(f"x: expected [N, ..., C], got shape {tuple(shape)}")
    n, c = shape[0], shape[-1]
    if isinstance(groups, bool) or not isinstance(groups, int) or groups < 1 or c < 1 or c % groups:
        raise ValueError(f"groups must divide the {c} channels, got {groups!r}")
    if not 0 <= eps <= 3e38:
        raise ValueError(f"eps must be a number from 0 to 3e38, got {eps}")
    if weight is not None:
        _vector(weight, (c,), x.dtype, "weight")
    if bias is not None:
        _vector(bias, (c,), x.dtype, "bias")
    rows, ldx = _pitch(x, 1, "x")
    if out is None:
        ldy = c
    else:
        if out.shape != x.shape or out.dtype is not x.dtype:
            raise ValueError(f"out: expected {x.dtype} of shape {tuple(x.shape)}, got {out.dtype} of {tuple(out.shape)}")
        _, ldy = _pitch(out, 1, "out")
        # positions apart, and samples behind each other ([N, L, C]) or between the positions of one ([L, N, C] seen so)
        step = out.stride(0) if n > 1 else _INT
        if rows > 1 and ldy < c or step < c or step < (rows - 1) * ldy + c and ldy < (n - 1) * step + c:
            raise ValueError("out: its positions overlap each other")
        _apart(out, "x", x=x, weight=weight, bias=bias)
    if max(n, rows, c, n * groups) > _INT - 4096:
        raise ValueError("x: over 2^31 - 4097 samples, positions, channels or groups")
    device = _ready(x, weight, bias, out)
    if out is None:
        out = x.new_empty(shape)
    else:
        increment_version(out)  # a backward pass that saved out's old values refuses instead of reading the new ones
    if not (n and rows):
        return out
    weight, bias = _f32(weight), _f32(bias)
    ws, need, fn = None, 0, N.lib().dml_group_norm
    while True:
        need = _launch(fn, _NORM.pack(
            x.data_ptr(), out.data_ptr(), 0 if weight is None else weight.data_ptr(),
            0 if bias is None else bias.data_ptr(), x.stride(0), out.stride(0), ldx, ldy,
            0 if ws is None else ws.data_ptr(), need, n, rows, c, groups, dtype, code, eps), device, "dml_group_norm")
        if not need:
            return out
        ws = torch.empty(need, device=x.device, dtype=torch.uint8)


def _product(x, weight, ends, bias, act, residual, act_last, out, out_dtype, what):
    code = _act(act)
    dtype = x.dtype
    if dtype is not torch.bfloat16 and dtype is not torch.float16:
        raise TypeError(f"x: expected bfloat16 or float16, got {dtype}")
    if weight.dtype is not dtype:
        raise TypeError(f"weight: expected {dtype} like x, got {weight.dtype}")
    xs, wsh = x.shape, weight.shape
    wdim = 2 if ends is None else 3
    if len(wsh) != wdim or not xs or wsh[-1] != xs[-1]:
        raise ValueError(f"{what}: x {tuple(xs)} does not fit weight {tuple(wsh)}")
    n, k = wsh[-2:]
    e = 1 if ends is None else wsh[0]
    shape = (*xs[:-1], n)
    to = out.dtype if out is not None else out_dtype if out_dtype is not None else dtype
    if to is not dtype and to is not torch.float32:
        raise TypeError(f"out: expected {dtype} or float32, got {to}")
    if out_dtype is not None and out_dtype is not to:
        raise TypeError(f"out is {to}, out_dtype {out_dtype}")
    if bias is not None:
        _vector(bias, (n,) if ends is None else (e, n), dtype, "bias")
    m, ldx = _pitch(x, 0, "x")
    _, ldw = _pitch(weight, wdim - 2, "weight")
    ldr = 0
    if residual is not None:
        if residual.shape != shape or residual.dtype is not to:
            raise ValueError(f"residual: expected {to} of shape {shape}, got {residual.dtype} of "
                             f"{tuple(residual.shape)}")
        ldr = _pitch(residual, 0, "residual")[1]
    ldy = n
    if out is not None:
        if out.shape != shape:
            raise ValueError(f"out: expected shape {shape}, got {tuple(out.shape)}")
        ldy = _pitch(out, 0, "out")[1]
        if m > 1 and ldy < n:
            raise ValueError("out: its rows overlap each other")
        _apart(out, "residual", x=x, weight=weight, bias=bias, ends=ends, residual=residual)
    if max(m, n, e) > _INT - 512 or k > 2 ** 30:
        raise ValueError(f"{what}: a dimension over 2^31 - 513, or K over 2^30")
    device = _ready(x, weight, ends, bias, residual, out)
    fill = 0
    if out is None:
        out = x.new_empty(shape, dtype=to)
        fill = int(ends is not None)
    else:
        increment_version(out)  # as in group_norm
    if not (m and n):
        return out
    if e == 0:
        return out.zero_() if fill else out
    bias = _f32(bias)
    _launch(N.lib().dml_product, _PROD.pack(
        x.data_ptr(), weight.data_ptr(), 0 if bias is None else bias.data_ptr(),
        0 if residual is None else residual.data_ptr(), out.data_ptr(), 0 if ends is None else ends.data_ptr(),
        ldx, ldw, weight.stride(0) if wdim == 3 else 0, n, ldr, ldy, m, n, k, e, _DTYPES[dtype],
        to is torch.float32, code, bool(act_last), ends is not None and ends.dtype is torch.int64, fill), device, what)
    return out


def linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, act: str = "none",
           residual: Optional[torch.Tensor] = None, act_last: bool = False, out: Optional[torch.Tensor] = None,
           out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """act(x . weight^T + bias) + residual, or with act_last act(x . weight^T + bias + residual).

    x: [..., K] bf16 or fp16, the leading dimensions stepping as one; weight: [N, K] of x's type (rows may be
    padded); any sizes, a product over K = 0 is 0. bias: [N], fp32 or x's type. residual: [..., N] of the output's
    type (an expanded one is read where it lies). Output [..., N] of x's type, or fp32 with out_dtype; out may be
    the residual itself, or a column slice of a wider buffer. Sums in fp32, one rounding at the end.
    """
    return _product(x, weight, None, bias, act, residual, act_last, out, out_dtype, "linear")


def grouped_linear(x: torch.Tensor, weight: torch.Tensor, ends: torch.Tensor, bias: Optional[torch.Tensor] = None,
                   act: str = "none", residual: Optional[torch.Tensor] = None, act_last: bool = False,
                   out: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """linear() with a weight per group of rows: rows ends[e-1] (0 for the first group) to ends[e] - 1 of x go
    through weight[e] and bias[e].

    x: [T, K] with its rows in the groups' order; weight: [E, N, K]; bias: [E, N]; ends: [E] int32 or int64 on the
    device, ascending, at most T (the counts' cumulative sum). Groups may be empty. The ends stay on the device:
    the host does not wait for them, and a captured call follows them from replay to replay. Out-of-order or
    out-of-range ends are clamped to an ascending sequence in [0, T]. Rows behind the last group stay as they are
    in out; without out they are 0.
    """
    if ends.dtype is not torch.int32 and ends.dtype is not torch.int64:
        raise TypeError(f"ends: expected int32 or int64, got {ends.dtype}")
    if weight.dim() != 3 or x.dim() != 2 or tuple(ends.shape) != (weight.shape[0],) or not ends.is_contiguous():
        raise ValueError(f"grouped_linear: expected x [T, K], weight [E, N, K] and contiguous ends [E], got "
                         f"{tuple(x.shape)}, {tuple(weight.shape)} and {tuple(ends.shape)}")
    return _product(x, weight, ends, bias, act, residual, act_last, out, out_dtype, "grouped_linear")

"""Tensor-level entry points: validate, allocate outputs with torch, enqueue the
C-ABI kernels on the current CUDA stream. No arithmetic happens in Python and
there is no non-CUDA path: a CPU tensor raises.
"""

from __future__ import annotations

import ctypes
import functools
import math
from array import array

import torch

from . import _cabi
from ._cabi import EVG_BF16, EVG_F16, EVG_F32, EvgError, PackedView, RopePositionsTensor, RopeTensor, \
    call, lib

_DTYPES = {torch.float32: EVG_F32, torch.float16: EVG_F16, torch.bfloat16: EVG_BF16}


def _dtype_enum(t: torch.Tensor) -> int:
    try:
        return _DTYPES[t.dtype]
    except KeyError:
        raise TypeError(f"unsupported dtype {t.dtype}; expected float32/float16/bfloat16") from None


def _require_cuda(*tensors: torch.Tensor) -> torch.device:
    dev = None
    for t in tensors:
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"expected a tensor, got {type(t).__name__}")
        d = t.device
        if d != dev:
            if d.type != "cuda":
                raise RuntimeError(
                    "evograd_b200 kernels run on CUDA (sm_100a) tensors only; there is no CPU path"
                )
            if dev is not None:
                raise RuntimeError(f"tensors on different devices: {dev} and {d}")
            dev = d
    return dev


def _stream(dev: torch.device) -> int:
    # the current stream's handle without the Stream object around it, which costs more host
    # time than a short kernel runs
    return torch._C._cuda_getCurrentRawStream(dev.index)


def _enqueue(dev: torch.device, fn_name: str, *args) -> None:
    """``call(fn_name, *args, current stream of dev)`` with ``dev`` the current device."""
    index = dev.index
    if torch._C._cuda_getDevice() == index:
        call(fn_name, *args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(dev):
            call(fn_name, *args, torch._C._cuda_getCurrentRawStream(index))


def _p(t) -> int | None:
    return None if t is None else t.data_ptr()


def _same(name_a, a, name_b, b, *, shape=True, dtype=True):
    if shape and a.shape != b.shape:
        raise ValueError(f"{name_a} {tuple(a.shape)} and {name_b} {tuple(b.shape)} differ in shape")
    if dtype and a.dtype != b.dtype:
        raise ValueError(f"{name_a} is {a.dtype} but {name_b} is {b.dtype}")


def _rows_view(t: torch.Tensor, cols: int) -> torch.Tensor:
    return t.contiguous().view(-1, cols)


# ------------------------------------------------------------------ softmax
def softmax_fwd(x: torch.Tensor) -> torch.Tensor:
    dev = _require_cuda(x)
    if x.ndim < 1:
        raise ValueError("softmax needs at least one dimension")
    cols = x.shape[-1]
    x2 = _rows_view(x, cols)
    y = torch.empty_like(x2)
    if x2.numel() == 0:
        return y.view(x.shape)
    with torch.cuda.device(dev):
        call("evg_softmax_fwd", x2.data_ptr(), y.data_ptr(), x2.shape[0], cols, _dtype_enum(x),
             _stream(dev))
    return y.view(x.shape)


def softmax_bwd(y: torch.Tensor, dy: torch.Tensor) -> torch.Tensor:
    dev = _require_cuda(y, dy)
    _same("y", y, "dy", dy)
    cols = y.shape[-1]
    y2, g2 = _rows_view(y, cols), _rows_view(dy, cols)
    dx = torch.empty_like(y2)
    if y2.numel() == 0:
        return dx.view(y.shape)
    with torch.cuda.device(dev):
        call("evg_softmax_bwd", y2.data_ptr(), g2.data_ptr(), dx.data_ptr(), y2.shape[0], cols,
             _dtype_enum(y), _stream(dev))
    return dx.view(y.shape)


# ----------------------------------------------------------- layernorm / rmsnorm
def _check_param(name: str, p: torch.Tensor, x: torch.Tensor):
    if p.ndim != 1 or p.shape[0] != x.shape[-1]:
        raise ValueError(f"{name} must be 1-D of length {x.shape[-1]}, got {tuple(p.shape)}")
    if p.dtype != x.dtype:
        raise ValueError(f"{name} is {p.dtype} but x is {x.dtype}")


def layernorm_fwd(x, weight, bias, eps: float = 1e-5):
    """Returns ``(y, mean, rstd)``; mean and rstd are float32 ``[rows]``."""
    dev = _require_cuda(x, weight, bias)
    _check_param("weight", weight, x)
    _check_param("bias", bias, x)
    hidden = x.shape[-1]
    x2 = _rows_view(x, hidden)
    rows = x2.shape[0]
    y = torch.empty_like(x2)
    mean = torch.empty(rows, device=dev, dtype=torch.float32)
    rstd = torch.empty(rows, device=dev, dtype=torch.float32)
    if rows == 0:
        return y.view(x.shape), mean, rstd
    with torch.cuda.device(dev):
        call("evg_layernorm_fwd", x2.data_ptr(), weight.contiguous().data_ptr(),
             bias.contiguous().data_ptr(), y.data_ptr(), mean.data_ptr(), rstd.data_ptr(), rows,
             hidden, float(eps), _dtype_enum(x), _stream(dev))
    return y.view(x.shape), mean, rstd


def layernorm_bwd(dy, x, weight, mean, rstd, *, partials_f32: bool = False, exchange=None):
    """Returns ``(dx, dweight, dbias)``.

    With ``partials_f32`` the parameter gradients come back as ONE float32
    tensor ``[2, hidden]`` (row 0 dweight, row 1 dbias) instead of two tensors in
    the parameter dtype, for callers that sum them across ranks before rounding:
    ``(dx, dwdb_f32, None)``. With ``exchange`` (a connected
    :class:`evograd_b200.sharded.PeerExchange`; x and dy are this rank's row
    shard) dweight / dbias are the sums over ALL ranks' rows, formed inside the
    second stage of the column reduction, rounded once, identical on every rank.
    """
    dev = _require_cuda(dy, x, weight, mean, rstd)
    _same("dy", dy, "x", x)
    _check_param("weight", weight, x)
    hidden = x.shape[-1]
    x2, g2 = _rows_view(x, hidden), _rows_view(dy, hidden)
    rows = x2.shape[0]
    if mean.numel() != rows or rstd.numel() != rows or mean.dtype != torch.float32 \
            or rstd.dtype != torch.float32:
        raise ValueError("mean/rstd must be float32 with one entry per row")
    dx = torch.empty_like(x2)
    en = _dtype_enum(x)
    if rows == 0:
        z = torch.zeros(hidden, device=dev, dtype=x.dtype)
        if partials_f32:
            return dx.view(x.shape), torch.zeros(2, hidden, device=dev, dtype=torch.float32), None
        return dx.view(x.shape), z, z.clone()
    with torch.cuda.device(dev):
        ws_bytes = lib.evg_layernorm_bwd_workspace_bytes(rows, hidden, en)
        ws = torch.empty(ws_bytes, device=dev, dtype=torch.uint8)
        if exchange is not None and not partials_f32:
            dwdb2 = torch.empty(2, hidden, device=dev, dtype=x.dtype)
            call("evg_layernorm_bwd_exchange", g2.data_ptr(), x2.data_ptr(),
                 weight.contiguous().data_ptr(), mean.contiguous().data_ptr(),
                 rstd.contiguous().data_ptr(), dx.data_ptr(), dwdb2[0].data_ptr(),
                 dwdb2[1].data_ptr(), ws.data_ptr(), ws_bytes, rows, hidden, en, exchange.handle,
                 _stream(dev))
            return dx.view(x.shape), dwdb2[0], dwdb2[1]
        if partials_f32:
            dwdb = torch.empty(2, hidden, device=dev, dtype=torch.float32)
            dweight = dbias = None
        else:
            dwdb = None
            dweight = torch.empty(hidden, device=dev, dtype=x.dtype)
            dbias = torch.empty(hidden, device=dev, dtype=x.dtype)
        call("evg_layernorm_bwd", g2.data_ptr(), x2.data_ptr(), weight.contiguous().data_ptr(),
             mean.contiguous().data_ptr(), rstd.contiguous().data_ptr(), dx.data_ptr(),
             _p(dweight), _p(dbias), _p(dwdb), ws.data_ptr(), ws_bytes, rows, hidden, en,
             _stream(dev))
    if partials_f32:
        return dx.view(x.shape), dwdb, None
    return dx.view(x.shape), dweight, dbias


def rmsnorm_fwd(x, weight, eps: float = 1e-5):
    """Returns ``(y, rstd)``; rstd is float32 ``[rows]``."""
    dev = _require_cuda(x, weight)
    _check_param("weight", weight, x)
    hidden = x.shape[-1]
    x2 = _rows_view(x, hidden)
    rows = x2.shape[0]
    y = torch.empty_like(x2)
    rstd = torch.empty(rows, device=dev, dtype=torch.float32)
    if rows == 0:
        return y.view(x.shape), rstd
    with torch.cuda.device(dev):
        call("evg_rmsnorm_fwd", x2.data_ptr(), weight.contiguous().data_ptr(), y.data_ptr(),
             rstd.data_ptr(), rows, hidden, float(eps), _dtype_enum(x), _stream(dev))
    return y.view(x.shape), rstd


def rmsnorm_bwd(dy, x, weight, rstd, *, partials_f32: bool = False, exchange=None):
    """Returns ``(dx, dweight)``; ``dweight`` is float32 when ``partials_f32``. With
    ``exchange`` (see :func:`layernorm_bwd`) dweight is the sum over all ranks' rows."""
    dev = _require_cuda(dy, x, weight, rstd)
    _same("dy", dy, "x", x)
    _check_param("weight", weight, x)
    hidden = x.shape[-1]
    x2, g2 = _rows_view(x, hidden), _rows_view(dy, hidden)
    rows = x2.shape[0]
    if rstd.numel() != rows or rstd.dtype != torch.float32:
        raise ValueError("rstd must be float32 with one entry per row")
    dx = torch.empty_like(x2)
    en = _dtype_enum(x)
    out_dtype = torch.float32 if partials_f32 else x.dtype
    if rows == 0:
        return dx.view(x.shape), torch.zeros(hidden, device=dev, dtype=out_dtype)
    with torch.cuda.device(dev):
        ws_bytes = lib.evg_rmsnorm_bwd_workspace_bytes(rows, hidden, en)
        ws = torch.empty(ws_bytes, device=dev, dtype=torch.uint8)
        dweight = torch.empty(hidden, device=dev, dtype=out_dtype)
        if exchange is not None and not partials_f32:
            call("evg_rmsnorm_bwd_exchange", g2.data_ptr(), x2.data_ptr(),
                 weight.contiguous().data_ptr(), rstd.contiguous().data_ptr(), dx.data_ptr(),
                 dweight.data_ptr(), ws.data_ptr(), ws_bytes, rows, hidden, en, exchange.handle,
                 _stream(dev))
            return dx.view(x.shape), dweight
        call("evg_rmsnorm_bwd", g2.data_ptr(), x2.data_ptr(), weight.contiguous().data_ptr(),
             rstd.contiguous().data_ptr(), dx.data_ptr(),
             None if partials_f32 else dweight.data_ptr(),
             dweight.data_ptr() if partials_f32 else None, ws.data_ptr(), ws_bytes, rows, hidden,
             en, _stream(dev))
    return dx.view(x.shape), dweight


def fused_add_rmsnorm_fwd(x, residual, weight, eps: float = 1e-6):
    """``out = rmsnorm(x + residual) * weight`` with the reference's rounding points
    (ops/level2/fused_add_rms_norm/forward_ref.py:6-14). Returns ``(out, rstd)``;
    rstd is float32 ``[rows]``; the sum itself is not kept."""
    dev = _require_cuda(x, residual, weight)
    _same("x", x, "residual", residual)
    _check_param("weight", weight, x)
    hidden = x.shape[-1]
    x2, r2 = _rows_view(x, hidden), _rows_view(residual, hidden)
    rows = x2.shape[0]
    out = torch.empty_like(x2)
    rstd = torch.empty(rows, device=dev, dtype=torch.float32)
    if rows == 0:
        return out.view(x.shape), rstd
    with torch.cuda.device(dev):
        call("evg_fused_add_rmsnorm_fwd", x2.data_ptr(), r2.data_ptr(),
             weight.contiguous().data_ptr(), out.data_ptr(), rstd.data_ptr(), rows, hidden,
             float(eps), _dtype_enum(x), _stream(dev))
    return out.view(x.shape), rstd


def fused_add_rmsnorm_bwd(dout, x, residual, weight, rstd, *, partials_f32: bool = False):
    """Returns ``(dx, dweight)``; the gradient of ``residual`` equals ``dx``.
    ``dweight`` is float32 when ``partials_f32``."""
    dev = _require_cuda(dout, x, residual, weight, rstd)
    _same("dout", dout, "x", x)
    _same("x", x, "residual", residual)
    _check_param("weight", weight, x)
    hidden = x.shape[-1]
    x2, r2, g2 = _rows_view(x, hidden), _rows_view(residual, hidden), _rows_view(dout, hidden)
    rows = x2.shape[0]
    if rstd.numel() != rows or rstd.dtype != torch.float32:
        raise ValueError("rstd must be float32 with one entry per row")
    dx = torch.empty_like(x2)
    en = _dtype_enum(x)
    out_dtype = torch.float32 if partials_f32 else x.dtype
    if rows == 0:
        return dx.view(x.shape), torch.zeros(hidden, device=dev, dtype=out_dtype)
    with torch.cuda.device(dev):
        ws_bytes = lib.evg_fused_add_rmsnorm_bwd_workspace_bytes(rows, hidden, en)
        ws = torch.empty(ws_bytes, device=dev, dtype=torch.uint8)
        dweight = torch.empty(hidden, device=dev, dtype=out_dtype)
        call("evg_fused_add_rmsnorm_bwd", g2.data_ptr(), x2.data_ptr(), r2.data_ptr(),
             weight.contiguous().data_ptr(), rstd.contiguous().data_ptr(), dx.data_ptr(),
             None if partials_f32 else dweight.data_ptr(),
             dweight.data_ptr() if partials_f32 else None, ws.data_ptr(), ws_bytes, rows, hidden,
             en, _stream(dev))
    return dx.view(x.shape), dweight


def cast_from_f32(src: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """Round a float32 tensor to ``dtype`` (after an all-reduce of partial sums)."""
    dev = _require_cuda(src)
    if src.dtype != torch.float32:
        raise TypeError("cast_from_f32 expects float32")
    src = src.contiguous()
    dst = torch.empty(src.shape, device=dev, dtype=dtype)
    with torch.cuda.device(dev):
        call("evg_cast_from_f32", src.data_ptr(), dst.data_ptr(), src.numel(), _DTYPES[dtype],
             _stream(dev))
    return dst


# ------------------------------------------------------------ swiglu / geglu
def _glu_fwd(symbol, a, b):
    dev = _require_cuda(a, b)
    _same("a", a, "b", b)
    a2, b2 = a.contiguous(), b.contiguous()
    c = torch.empty_like(a2)
    if a2.numel() == 0:
        return c
    with torch.cuda.device(dev):
        call(symbol, a2.data_ptr(), b2.data_ptr(), c.data_ptr(), a2.numel(),
             _dtype_enum(a), _stream(dev))
    return c


def _glu_bwd(symbol, dc, a, b, in_place):
    dev = _require_cuda(dc, a, b)
    _same("a", a, "b", b)
    _same("dc", dc, "a", a)
    dc2 = dc.contiguous()
    if in_place:
        if not (a.is_contiguous() and b.is_contiguous()):
            raise ValueError("in_place backward needs contiguous a and b")
        a2, b2, da, db = a, b, a, b
    else:
        a2, b2 = a.contiguous(), b.contiguous()
        da, db = torch.empty_like(a2), torch.empty_like(b2)
    if a2.numel() == 0:
        return da, db
    with torch.cuda.device(dev):
        call(symbol, dc2.data_ptr(), a2.data_ptr(), b2.data_ptr(), da.data_ptr(),
             db.data_ptr(), a2.numel(), _dtype_enum(a), _stream(dev))
    return da, db


def swiglu_fwd(a, b):
    return _glu_fwd("evg_swiglu_fwd", a, b)


def swiglu_bwd(dc, a, b, *, in_place: bool = False):
    """Returns ``(da, db)``. ``in_place`` writes them over ``a`` and ``b`` (which
    must then be contiguous), as the swiglu declaration permits."""
    return _glu_bwd("evg_swiglu_bwd", dc, a, b, in_place)


def geglu_fwd(a, b):
    """c = gelu_tanh(a) * b (ops/level1/geglu/forward_ref.py:6-9)."""
    return _glu_fwd("evg_geglu_fwd", a, b)


def geglu_bwd(dc, a, b, *, in_place: bool = False):
    """Returns ``(da, db)`` of the geglu pair; ``in_place`` as for swiglu."""
    return _glu_bwd("evg_geglu_bwd", dc, a, b, in_place)


# --------------------------------------------------------------------- rope
def _rope_launch(xs, layout: str, cos, sin, inverse: bool, outs=None):
    """Rotate 1 or 2 tensors in one launch. ``layout`` is "bhtd" or "bthd" and names
    the axis order of the tensors' SHAPES; inputs and outputs may be strided views
    (last dimension contiguous), so a rotation can also change the memory layout
    (for example read [B, T, H, D] memory through a transposed view and write
    contiguous [B, H, T, D]). ``outs`` supplies the output tensors."""
    dev = _require_cuda(*xs, cos, sin)
    if layout not in ("bhtd", "bthd"):
        raise ValueError(f"layout must be 'bhtd' or 'bthd', got {layout!r}")
    x0 = xs[0]
    if any(x.ndim != 4 for x in xs):
        raise ValueError("rope expects 4-D tensors")
    t_axis, h_axis = (2, 1) if layout == "bhtd" else (1, 2)
    batch, tokens, head_dim = x0.shape[0], x0.shape[t_axis], x0.shape[3]
    if head_dim % 2:
        raise ValueError(f"rope needs an even head_dim, got {head_dim}")
    for x in xs[1:]:
        if x.shape[0] != batch or x.shape[t_axis] != tokens or x.shape[3] != head_dim \
                or x.dtype != x0.dtype:
            raise ValueError("tensors rotated together must share batch, tokens, head_dim, dtype")
    if cos.shape != sin.shape or cos.dtype != sin.dtype or cos.ndim != 2 or cos.shape[0] != tokens:
        raise ValueError(f"cos/sin must both be [tokens, head_dim or head_dim/2]; got "
                         f"{tuple(cos.shape)} and {tuple(sin.shape)}")
    if cos.shape[1] not in (head_dim, head_dim // 2):
        raise ValueError(f"table width {cos.shape[1]} is neither head_dim nor head_dim/2")
    cos, sin = cos.contiguous(), sin.contiguous()
    arr = (RopeTensor * len(xs))()
    given, outs = outs, []
    keep = []
    for i, x in enumerate(xs):
        if x.stride(3) != 1:
            x = x.contiguous()
        keep.append(x)
        if given is None:
            y = torch.empty(x.shape, device=dev, dtype=x.dtype)
        else:
            y = given[i]
            if tuple(y.shape) != tuple(x.shape) or y.dtype != x.dtype or y.stride(3) != 1 \
                    or y.device != x.device:
                raise ValueError("rope output must match the input's shape, dtype and device and "
                                 "have a contiguous last dimension")
        outs.append(y)
        arr[i] = RopeTensor(x.data_ptr(), y.data_ptr(), x.shape[h_axis], x.stride(0),
                            x.stride(h_axis), x.stride(t_axis), y.stride(0), y.stride(h_axis),
                            y.stride(t_axis))
    with torch.cuda.device(dev):
        call("evg_rope", arr, len(xs), cos.data_ptr(), sin.data_ptr(), batch, tokens, head_dim,
             cos.shape[1], _dtype_enum(cos), _dtype_enum(x0), 1 if inverse else 0, _stream(dev))
    return outs


def rope_fwd(x, cos, sin, *, layout: str = "bhtd", out=None):
    return _rope_launch([x], layout, cos, sin, False, None if out is None else [out])[0]


def rope_bwd(dy, cos, sin, *, layout: str = "bhtd", out=None):
    return _rope_launch([dy], layout, cos, sin, True, None if out is None else [out])[0]


def rope_qk_fwd(q, k, cos, sin, *, layout: str = "bthd", outs=None):
    """Rotate q and k (possibly different head counts) in one launch."""
    return tuple(_rope_launch([q, k], layout, cos, sin, False, outs))


def rope_qk_bwd(dq, dk, cos, sin, *, layout: str = "bthd", outs=None):
    return tuple(_rope_launch([dq, dk], layout, cos, sin, True, outs))


# --------------------------------------------------------- causal attention
def _check_qkv(q, k, v):
    if q.ndim != 4:
        raise ValueError(f"causal attention expects [B, H, S, D], got {tuple(q.shape)}")
    _same("q", q, "k", k)
    _same("q", q, "v", v)
    if q.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"causal attention runs in bfloat16/float16, got {q.dtype}")


def causal_attention_fwd(q, k, v, scale: float | None = None):
    """Returns ``(o, lse)`` with ``lse`` float32 ``[B, H, S]``."""
    dev = _require_cuda(q, k, v)
    _check_qkv(q, k, v)
    B, H, S, D = q.shape
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    q2, k2, v2 = q.contiguous(), k.contiguous(), v.contiguous()
    o = torch.empty_like(q2)
    lse = torch.empty(B, H, S, device=dev, dtype=torch.float32)
    with torch.cuda.device(dev):
        call("evg_causal_attention_fwd", q2.data_ptr(), k2.data_ptr(), v2.data_ptr(), o.data_ptr(),
             lse.data_ptr(), B, H, S, D, float(scale), _dtype_enum(q), _stream(dev))
    return o, lse


def causal_attention_bwd(do, q, k, v, o, lse, scale: float | None = None):
    """Returns ``(dq, dk, dv)``."""
    dev = _require_cuda(do, q, k, v, o, lse)
    _check_qkv(q, k, v)
    _same("do", do, "q", q)
    _same("o", o, "q", q)
    B, H, S, D = q.shape
    if lse.dtype != torch.float32 or tuple(lse.shape) != (B, H, S):
        raise ValueError("lse must be float32 [B, H, S]")
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    do2, q2, k2, v2, o2 = (t.contiguous() for t in (do, q, k, v, o))
    dq, dk, dv = torch.empty_like(q2), torch.empty_like(k2), torch.empty_like(v2)
    en = _dtype_enum(q)
    with torch.cuda.device(dev):
        ws_bytes = lib.evg_causal_attention_bwd_workspace_bytes(B, H, S, D, en)
        ws = torch.empty(max(ws_bytes, 16), device=dev, dtype=torch.uint8)
        call("evg_causal_attention_bwd", do2.data_ptr(), q2.data_ptr(), k2.data_ptr(),
             v2.data_ptr(), o2.data_ptr(), lse.contiguous().data_ptr(), dq.data_ptr(),
             dk.data_ptr(), dv.data_ptr(), ws.data_ptr(), ws_bytes, B, H, S, D, float(scale), en,
             _stream(dev))
    return dq, dk, dv


def _check_gqa(q, k, v):
    if q.ndim != 4 or k.ndim != 4:
        raise ValueError(f"attention expects [B, H, S, D], got {tuple(q.shape)} / {tuple(k.shape)}")
    _same("k", k, "v", v)
    if q.dtype != k.dtype or q.device != k.device:
        raise ValueError("q and k must share dtype and device")
    B, Hq, S, D = q.shape
    if k.shape[0] != B or k.shape[2] != S or k.shape[3] != D or Hq % k.shape[1] != 0:
        raise ValueError(f"q {tuple(q.shape)} and k/v {tuple(k.shape)} do not form grouped-query "
                         "attention (same B, S, D; query heads a multiple of k/v heads)")
    return B, Hq, k.shape[1], S, D


def causal_gqa_attention_fwd(q, k, v, scale: float | None = None):
    """Causal attention with ``Hq`` query heads sharing ``Hkv`` key/value heads:
    q ``[B, Hq, S, D]``, k/v ``[B, Hkv, S, D]`` (any of float32 / float16 / bfloat16,
    D <= 256; 16-bit with D in {64, 128} runs on the tensor cores). Returns
    ``(o, lse)`` with ``lse`` float32 ``[B, Hq, S]``."""
    dev = _require_cuda(q, k, v)
    B, Hq, Hkv, S, D = _check_gqa(q, k, v)
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    q2, k2, v2 = q.contiguous(), k.contiguous(), v.contiguous()
    o = torch.empty_like(q2)
    lse = torch.empty(B, Hq, S, device=dev, dtype=torch.float32)
    if q2.numel() == 0:
        return o, lse
    with torch.cuda.device(dev):
        call("evg_causal_gqa_attention_fwd", q2.data_ptr(), k2.data_ptr(), v2.data_ptr(),
             o.data_ptr(), lse.data_ptr(), B, Hq, Hkv, S, D, float(scale), _dtype_enum(q),
             _stream(dev))
    return o, lse


def causal_gqa_attention_bwd(do, q, k, v, o, lse, scale: float | None = None):
    """Returns ``(dq, dk, dv)``; dk/dv are summed over the query heads of each group."""
    dev = _require_cuda(do, q, k, v, o, lse)
    B, Hq, Hkv, S, D = _check_gqa(q, k, v)
    _same("do", do, "q", q)
    _same("o", o, "q", q)
    if lse.dtype != torch.float32 or tuple(lse.shape) != (B, Hq, S):
        raise ValueError("lse must be float32 [B, Hq, S]")
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    do2, q2, k2, v2, o2 = (t.contiguous() for t in (do, q, k, v, o))
    dq, dk, dv = torch.empty_like(q2), torch.empty_like(k2), torch.empty_like(v2)
    if q2.numel() == 0:
        return dq, dk, dv
    en = _dtype_enum(q)
    with torch.cuda.device(dev):
        ws_bytes = lib.evg_causal_gqa_attention_bwd_workspace_bytes(B, Hq, Hkv, S, D, en)
        ws = torch.empty(max(ws_bytes, 16), device=dev, dtype=torch.uint8)
        call("evg_causal_gqa_attention_bwd", do2.data_ptr(), q2.data_ptr(), k2.data_ptr(),
             v2.data_ptr(), o2.data_ptr(), lse.contiguous().data_ptr(), dq.data_ptr(),
             dk.data_ptr(), dv.data_ptr(), ws.data_ptr(), ws_bytes, B, Hq, Hkv, S, D, float(scale),
             en, _stream(dev))
    return dq, dk, dv


def _tensor_core_attention(q) -> bool:
    return q.dtype in (torch.float16, torch.bfloat16) and q.shape[-1] in (64, 128)


def causal_gqa_attention_fwd_tm(q, k, v_tm, scale: float | None = None):
    """:func:`causal_gqa_attention_fwd` for a decoder layer's layouts: ``v_tm`` is
    token-major ``[B, S, Hkv, D]`` (a view of its projection's output) and ``o`` comes
    back token-major ``[B, S, Hq, D]`` (what the output projection reads as
    ``[B*S, Hq*D]``); q and k are ``[B, H, S, D]``. The tensor-core kernels read and
    write those layouts directly; other shapes go through the head-major call and
    transposing copies."""
    dev = _require_cuda(q, k, v_tm)
    v = v_tm.transpose(1, 2)
    B, Hq, Hkv, S, D = _check_gqa(q, k, v)
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    if not _tensor_core_attention(q) or q.numel() == 0:
        o, lse = causal_gqa_attention_fwd(q, k, v, scale)
        return o.transpose(1, 2).contiguous(), lse
    q2, k2, v2 = q.contiguous(), k.contiguous(), v_tm.contiguous()
    o = torch.empty(B, S, Hq, D, device=dev, dtype=q.dtype)
    lse = torch.empty(B, Hq, S, device=dev, dtype=torch.float32)
    with torch.cuda.device(dev):
        call("evg_causal_gqa_attention_fwd_tm", q2.data_ptr(), k2.data_ptr(), v2.data_ptr(),
             o.data_ptr(), lse.data_ptr(), B, Hq, Hkv, S, D, float(scale), _dtype_enum(q),
             _stream(dev))
    return o, lse


def causal_gqa_attention_bwd_tm(do_tm, q, k, v_tm, o_tm, lse, scale: float | None = None):
    """Backward for token-major ``do_tm`` / ``o_tm`` ``[B, S, Hq, D]`` and ``v_tm``
    ``[B, S, Hkv, D]``; returns ``(dq, dk, dv_tm)`` with ``dv_tm`` token-major and dq, dk
    head-major."""
    dev = _require_cuda(do_tm, q, k, v_tm, o_tm, lse)
    v = v_tm.transpose(1, 2)
    B, Hq, Hkv, S, D = _check_gqa(q, k, v)
    for name, t in (("do_tm", do_tm), ("o_tm", o_tm)):
        if tuple(t.shape) != (B, S, Hq, D) or t.dtype != q.dtype:
            raise ValueError(f"{name} must be [B, S, Hq, D] in the dtype of q")
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    if not _tensor_core_attention(q) or q.numel() == 0:
        dq, dk, dv = causal_gqa_attention_bwd(do_tm.transpose(1, 2), q, k, v,
                                              o_tm.transpose(1, 2), lse, scale)
        return dq, dk, dv.transpose(1, 2).contiguous()
    do2, q2, k2, v2, o2 = (t.contiguous() for t in (do_tm, q, k, v_tm, o_tm))
    dq, dk = torch.empty_like(q2), torch.empty_like(k2)
    dv = torch.empty(B, S, Hkv, D, device=dev, dtype=q.dtype)
    en = _dtype_enum(q)
    with torch.cuda.device(dev):
        ws_bytes = lib.evg_causal_gqa_attention_bwd_workspace_bytes(B, Hq, Hkv, S, D, en)
        ws = torch.empty(max(ws_bytes, 16), device=dev, dtype=torch.uint8)
        call("evg_causal_gqa_attention_bwd_tm", do2.data_ptr(), q2.data_ptr(), k2.data_ptr(),
             v2.data_ptr(), o2.data_ptr(), lse.contiguous().data_ptr(), dq.data_ptr(),
             dk.data_ptr(), dv.data_ptr(), ws.data_ptr(), ws_bytes, B, Hq, Hkv, S, D, float(scale),
             en, _stream(dev))
    return dq, dk, dv


# ------------------------------------------------- packed causal attention
PACKED_MAX_TOKENS = 1 << 27


class PackedPlan:
    """Work plan of a packed batch, made by :func:`packed_plan` and read by every attention
    call on that batch (all layers, forward and backward). It lives on the device and
    follows the offsets it was made from, not their later values."""

    __slots__ = ("data", "tokens", "sequences")

    def __init__(self, data: torch.Tensor, tokens: int, sequences: int):
        self.data, self.tokens, self.sequences = data, tokens, sequences

    def check(self) -> None:
        """Synchronise and raise :class:`EvgError` if the offsets were not ``0 = cu[0] <=
        cu[1] <= ... <= tokens`` (such a plan has no sequences: every row is treated as
        lying behind the last one)."""
        status = int(self.data[0].item())
        if status:
            raise EvgError("evg_packed_plan", status,
                           "cu_seqlens must start at 0, never fall and end inside the token axis")


@functools.lru_cache(maxsize=1024)
def _plan_bytes(tokens: int, sequences: int) -> int:
    return lib.evg_packed_plan_bytes(tokens, sequences)


def packed_plan(cu_seqlens: torch.Tensor, tokens: int) -> PackedPlan:
    """Plan for ``n`` sequences packed into ``tokens`` rows: ``cu_seqlens`` is a device tensor
    of ``n + 1`` int32 (or int64) offsets, sequence ``s`` being rows ``cu[s] .. cu[s+1] - 1``.
    Lengths may be zero; rows behind ``cu[n]`` belong to no sequence. Nothing is read back:
    :meth:`PackedPlan.check` validates the offsets for a caller that wants to wait."""
    dev = _require_cuda(cu_seqlens)
    if cu_seqlens.ndim != 1 or cu_seqlens.shape[0] < 1:
        raise ValueError(f"cu_seqlens must be 1-D with at least one entry, got {tuple(cu_seqlens.shape)}")
    n, tokens = cu_seqlens.shape[0] - 1, int(tokens)
    if not 0 <= tokens <= PACKED_MAX_TOKENS or n > PACKED_MAX_TOKENS:
        raise ValueError(f"{tokens} tokens in {n} sequences: 0 .. {PACKED_MAX_TOKENS} each")
    if cu_seqlens.dtype != torch.int32:
        if cu_seqlens.dtype != torch.int64:
            raise TypeError(f"cu_seqlens must be int32 or int64, got {cu_seqlens.dtype}")
        # offsets that int32 cannot hold must stay invalid, not wrap around
        cu_seqlens = cu_seqlens.clamp(-1, PACKED_MAX_TOKENS + 1).to(torch.int32)
    cu = cu_seqlens.contiguous()
    nbytes = _plan_bytes(tokens, n)
    data = torch.empty(nbytes // 4, device=dev, dtype=torch.int32)
    _enqueue(dev, "evg_packed_plan", cu.data_ptr(), n, tokens, data.data_ptr(), nbytes)
    return PackedPlan(data, tokens, n)


def _check_packed(q, k, v, plan, dev):
    if not isinstance(plan, PackedPlan):
        raise TypeError("plan must come from packed_plan()")
    qs, ks = q.shape, k.shape
    if len(qs) != 3 or len(ks) != 3:
        raise ValueError(f"packed attention expects [T, H, D], got {tuple(qs)} / {tuple(ks)}")
    if v.shape != ks or v.dtype != k.dtype or k.dtype != q.dtype:
        raise ValueError(f"q {q.dtype}, k {tuple(ks)} {k.dtype}, v {tuple(v.shape)} {v.dtype}: k and v must "
                         "share their shape, all three their dtype")
    T, Hq, D = qs
    Hkv = ks[1]
    if ks[0] != T or ks[2] != D or Hkv == 0 or Hq == 0 or D == 0 or Hq % Hkv:
        raise ValueError(f"q {tuple(qs)} and k/v {tuple(ks)} do not form grouped-query "
                         "attention (same T, D; query heads a multiple of k/v heads)")
    if T != plan.tokens:
        raise ValueError(f"q has {T} rows but the plan was made for {plan.tokens}")
    if plan.data.device != dev:
        raise RuntimeError(f"tensors on different devices: {dev} and {plan.data.device}")
    return T, Hq, Hkv, D


def _packed_in(t):
    """An input as the kernels take it: last dimension contiguous, no repeated rows or heads,
    and 16-byte aligned for 16-bit tensors (a copy otherwise). Returns ``(tensor, view)``."""
    T, H, D = t.shape
    st, sh, sd = t.stride()
    p = t.data_ptr()
    if sd != 1 or (st <= 0 and T > 1) or (sh <= 0 and H > 1) or (
            D % 8 == 0 and t.element_size() == 2 and (p | st * 2 | sh * 2) & 15):
        t = t.contiguous()
        if t.data_ptr() & 15:  # contiguous already, off a 16-byte boundary
            t = t.clone()
        p, st, sh = t.data_ptr(), H * D, D
    return t, PackedView(p, st, sh)


def _packed_out(t):
    return PackedView(t.data_ptr(), t.stride(0), t.stride(1))


def _check_out(name, out, like):
    if not torch.is_tensor(out) or tuple(out.shape) != tuple(like.shape) or out.dtype != like.dtype \
            or out.device != like.device:
        raise ValueError(f"{name} must be a tensor of shape {tuple(like.shape)}, {like.dtype} on {like.device}")
    sizes_strides = sorted((st, n) for n, st in zip(out.shape, out.stride()) if n > 1)
    reach = 0  # elements the axes so far span; the next stride has to step over them
    for st, n in sizes_strides:
        if st <= reach:
            raise ValueError(f"{name} has overlapping rows (strides {tuple(out.stride())})")
        reach += st * (n - 1)
    if out.shape[-1] > 1 and out.stride(-1) != 1:
        raise ValueError(f"{name} must have a contiguous last dimension")
    return out


def packed_attention_fwd(q, k, v, plan: PackedPlan, scale: float | None = None, out=None):
    """Causal grouped-query attention over a packed batch: q ``[T, Hq, D]``, k / v
    ``[T, Hkv, D]`` (strided views such as the thirds of one projection are taken as they
    are), each token attending to its own sequence's tokens up to itself. Returns
    ``(o, lse)`` with o like q and ``lse`` float32 ``[Hq, T]``; rows behind the last
    sequence are 0 and ``-inf``. float16 / bfloat16 with D a multiple of 8 up to 128 run on
    the tensor cores, float32 and other D <= 256 on plain kernels for small shapes. ``out``
    receives o (it must not overlap an input; off a 16-byte boundary the plain kernels run)."""
    dev = _require_cuda(q, k, v)
    T, Hq, Hkv, D = _check_packed(q, k, v, plan, dev)
    en = _dtype_enum(q)
    o = torch.empty(T, Hq, D, device=dev, dtype=q.dtype) if out is None else _check_out("out", out, q)
    lse = torch.empty(Hq, T, device=dev, dtype=torch.float32)
    (q, vq), (k, vk), (v, vv) = _packed_in(q), _packed_in(k), _packed_in(v)
    _enqueue(dev, "evg_packed_attention_fwd", vq, vk, vv, _packed_out(o), lse.data_ptr(),
             plan.data.data_ptr(), T, plan.sequences, Hq, Hkv, D,
             1.0 / math.sqrt(D) if scale is None else float(scale), en)
    return o, lse


@functools.lru_cache(maxsize=1024)
def _packed_bwd_bytes(tokens: int, sequences: int, heads: int, head_dim: int) -> int:
    return max(lib.evg_packed_attention_bwd_workspace_bytes(tokens, sequences, heads, head_dim), 16)


def packed_attention_bwd(do, q, k, v, o, lse, plan: PackedPlan, scale: float | None = None, outs=None):
    """Returns ``(dq, dk, dv)`` of :func:`packed_attention_fwd`; dk / dv are summed over the
    query heads of each group, rows behind the last sequence are zero. ``outs`` supplies the
    three output tensors, which may be strided views (the thirds of one projection's
    gradient; off a 16-byte boundary the plain kernels run) but overlap neither an input nor
    one another. float16 gradients may be of any size that their type holds. dq of the tensor-core path can
    differ in the last bit from run to run (float32 global adds)."""
    dev = _require_cuda(do, q, k, v, o, lse)
    T, Hq, Hkv, D = _check_packed(q, k, v, plan, dev)
    _same("do", do, "q", q)
    _same("o", o, "q", q)
    en = _dtype_enum(q)
    if lse.dtype != torch.float32 or lse.shape != (Hq, T):
        raise ValueError("lse must be float32 [Hq, T]")
    if outs is None:
        dq = torch.empty(T, Hq, D, device=dev, dtype=q.dtype)
        dk = torch.empty(T, Hkv, D, device=dev, dtype=q.dtype)
        dv = torch.empty(T, Hkv, D, device=dev, dtype=q.dtype)
    else:
        if len(outs) != 3:
            raise ValueError("outs must hold dq, dk and dv")
        dq, dk, dv = (_check_out(n, t, like) for n, t, like in zip(("dq", "dk", "dv"), outs, (q, k, v)))
    (do, vdo), (q, vq), (k, vk), (v, vv), (o, vo) = (_packed_in(t) for t in (do, q, k, v, o))
    lse = lse.contiguous()
    ws_bytes = _packed_bwd_bytes(T, plan.sequences, Hq, D)
    ws = torch.empty(ws_bytes, device=dev, dtype=torch.uint8)
    _enqueue(dev, "evg_packed_attention_bwd", vdo, vq, vk, vv, vo, lse.data_ptr(), _packed_out(dq),
             _packed_out(dk), _packed_out(dv), ws.data_ptr(), ws_bytes, plan.data.data_ptr(), T,
             plan.sequences, Hq, Hkv, D, 1.0 / math.sqrt(D) if scale is None else float(scale), en)
    return dq, dk, dv


# ------------------------------------------- rotary from position numbers
def rope_inv_freq(rotary_dim: int, base: float = 10000.0, *, scaling: str | None = None,
                  factor: float = 1.0, original_context: int = 8192, slow: float = 1.0,
                  fast: float = 4.0, device=None):
    """Frequencies ``[rotary_dim/2]`` (float64) and the factor on cos / sin for
    :func:`rope_positions_fwd`: ``(inv_freq, mscale)``. ``scaling`` stretches the context by
    ``factor``: ``"linear"`` divides every frequency; ``"base"`` raises the base so that the
    slowest component is divided and the fastest kept; ``"wavelength"`` divides the
    components that turn less than ``slow`` times over ``original_context`` positions,
    keeps those above ``fast`` turns and blends linearly in the number of turns between;
    ``"ramp"`` blends linearly in the component's index between the indices that make ``fast``
    and ``slow`` turns (rounded outwards, limited to 0 .. rotary_dim - 1) and sets
    ``mscale = 0.1 ln(factor) + 1``."""
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be even and positive, got {rotary_dim}")
    if not base > 1.0 or not factor > 0.0 or original_context < 1 or not 0.0 < slow < fast:
        raise ValueError("need base > 1, factor > 0, original_context >= 1 and 0 < slow < fast")
    n = rotary_dim // 2
    i = torch.arange(n, dtype=torch.float64)
    mscale = 1.0
    if scaling == "base":
        base = base * factor ** (rotary_dim / max(rotary_dim - 2, 1))
    f = base ** (-2.0 * i / rotary_dim)
    if scaling == "linear":
        f = f / factor
    elif scaling == "wavelength":
        turns = original_context * f / (2.0 * math.pi)
        keep = ((turns - slow) / (fast - slow)).clamp(0.0, 1.0)
        f = f * (keep + (1.0 - keep) / factor)
    elif scaling == "ramp":
        def index_of(turns):
            return n * math.log(original_context / (turns * 2.0 * math.pi)) / math.log(base)

        # (not the number of pairs: over a long context `slow` turns lie behind the last one)
        lo, hi = max(math.floor(index_of(fast)), 0), min(math.ceil(index_of(slow)), rotary_dim - 1)
        keep = 1.0 - ((i - lo) / max(hi - lo, 1e-3)).clamp(0.0, 1.0)
        f = f * (keep + (1.0 - keep) / factor)
        mscale = 0.1 * math.log(factor) + 1.0 if factor > 1.0 else 1.0
    elif scaling not in (None, "base"):
        raise ValueError(f"unknown scaling {scaling!r}")
    return f.to(device), mscale


_ROPE_ROWS = (None, RopePositionsTensor * 1, RopePositionsTensor * 2)


def _rope_positions(xs, positions, inv_freq, interleaved, mscale, inverse, outs):
    xs = [x for x in xs if x is not None]
    dev = _require_cuda(*xs, positions, inv_freq)
    x0 = xs[0]
    for x in xs:
        if x.ndim != 3 or x.shape[0] != x0.shape[0] or x.shape[2] != x0.shape[2] or x.dtype != x0.dtype:
            raise ValueError("rope_positions expects [T, H, D] tensors that share T, D and dtype; got "
                             + ", ".join(f"{tuple(t.shape)} {t.dtype}" for t in xs))
    T, _, D = x0.shape
    en = _dtype_enum(x0)
    pdt, fdt, n = positions.dtype, inv_freq.dtype, inv_freq.numel()
    if (pdt != torch.int32 and pdt != torch.int64) or positions.shape != (T,):
        raise ValueError(f"positions must be int32 or int64 [{T}], got {pdt} {tuple(positions.shape)}")
    if (fdt != torch.float64 and fdt != torch.float32) or inv_freq.ndim != 1 or not 0 < 2 * n <= D:
        raise ValueError(f"inv_freq must be float32 or float64 with 1 .. {D // 2} entries, got "
                         f"{fdt} {tuple(inv_freq.shape)}")
    if outs is not None and len(outs) != len(xs):
        raise ValueError(f"outs must hold {len(xs)} tensors")
    positions, inv_freq = positions.contiguous(), inv_freq.contiguous()
    rows, keep, results = [], [], []
    for i, x in enumerate(xs):
        st, sh, sd = x.stride()
        if sd != 1:
            x = x.contiguous()
            st, sh, _ = x.stride()
        keep.append(x)
        if outs is None:
            H = x.shape[1]
            y = torch.empty(T, H, D, device=dev, dtype=x.dtype)
            yst, ysh = H * D, D
        else:
            y = _check_out("out", outs[i], x)
            yst, ysh, _ = y.stride()
        results.append(y)
        rows.append((x.data_ptr(), y.data_ptr(), x.shape[1], st, sh, yst, ysh))
    _enqueue(dev, "evg_rope_positions", _ROPE_ROWS[len(rows)](*rows), len(rows), positions.data_ptr(),
             4 if pdt == torch.int32 else 8, inv_freq.data_ptr(), 8 if fdt == torch.float64 else 4, T, D,
             2 * n, 1 if interleaved else 0, float(mscale), en, 1 if inverse else 0)
    return tuple(results)


def rope_positions_fwd(q, k, positions, inv_freq, *, interleaved: bool = False, mscale: float = 1.0,
                       outs=None):
    """Rotate q ``[T, Hq, D]`` and k ``[T, Hk, D]`` (or q alone, with k None) by
    ``positions[t] * inv_freq[i]`` in one launch. The first ``2 * len(inv_freq)`` columns
    rotate, in two halves or, ``interleaved``, in neighbouring pairs; the rest is copied.
    cos and sin are multiplied by ``mscale``. Strided views are taken as they are; ``outs``
    supplies the results: the inputs themselves (in place), or tensors that overlap neither an
    input nor one another. Returns a tuple with one tensor per input."""
    return _rope_positions((q, k), positions, inv_freq, interleaved, mscale, False, outs)


def rope_positions_bwd(dq, dk, positions, inv_freq, *, interleaved: bool = False, mscale: float = 1.0,
                       outs=None):
    """Gradients of the inputs of :func:`rope_positions_fwd` from those of its outputs."""
    return _rope_positions((dq, dk), positions, inv_freq, interleaved, mscale, True, outs)


# ------------------------------------------- norms after and before a block
def _gate_kind(gate, x) -> int:
    if gate is None:
        return 0
    if gate.dtype != x.dtype:
        raise ValueError(f"gate is {gate.dtype} but x is {x.dtype}")
    shape, want = tuple(gate.shape), tuple(x.shape)
    if shape == (want[-1],):
        return 1
    if shape == want:
        return 3
    if shape == want[:-1] + (1,):
        return 2
    raise ValueError(f"gate must be [{want[-1]}], {want[:-1] + (1,)} or {want}, got {shape}")


def _rows2(t, hidden):
    """``[rows, hidden]`` contiguous, the tensor itself where it is that already."""
    if t.ndim == 2 and t.is_contiguous():
        return t
    return t.contiguous().view(-1, hidden)


def post_pre_norm_fwd(x, residual, post_weight, pre_weight, gate=None, *, alpha: float = 1.0,
                      eps: float = 1e-6):
    """A block boundary in one pass: ``h = residual + alpha * gate * rmsnorm(x) * post_weight``,
    ``y = rmsnorm(h) * pre_weight`` (from h before its rounding). ``gate`` is None, ``[C]``,
    ``[..., 1]`` or shaped like x. Returns ``(h, y, rstd_post, rstd_pre)``; the rstd are
    float32 ``[rows]``, saved for the backward with x and h."""
    given = (x, residual, post_weight, pre_weight)
    dev = _require_cuda(*given) if gate is None else _require_cuda(*given, gate)
    shape = x.shape
    _same("x", x, "residual", residual)
    _check_param("post_weight", post_weight, x)
    _check_param("pre_weight", pre_weight, x)
    kind = 0 if gate is None else _gate_kind(gate, x)
    en = _dtype_enum(x)
    hidden = shape[-1]
    x2, r2 = _rows2(x, hidden), _rows2(residual, hidden)
    rows = x2.shape[0]
    h, y = torch.empty_like(x2), torch.empty_like(x2)
    rstd_post = torch.empty(rows, device=dev, dtype=torch.float32)
    rstd_pre = torch.empty(rows, device=dev, dtype=torch.float32)
    if rows and hidden:
        wp, wn = post_weight.contiguous(), pre_weight.contiguous()
        g = None if gate is None else gate.contiguous()
        _enqueue(dev, "evg_post_pre_norm_fwd", x2.data_ptr(), r2.data_ptr(), wp.data_ptr(), wn.data_ptr(),
                 None if g is None else g.data_ptr(), kind, h.data_ptr(), y.data_ptr(),
                 rstd_post.data_ptr(), rstd_pre.data_ptr(), rows, hidden, float(alpha), float(eps), en)
    if len(shape) != 2:
        h, y = h.view(shape), y.view(shape)
    return h, y, rstd_post, rstd_pre


@functools.lru_cache(maxsize=1024)
def _post_pre_bwd_bytes(device_index: int, rows: int, hidden: int) -> int:
    with torch.cuda.device(device_index):
        return lib.evg_post_pre_norm_bwd_workspace_bytes(rows, hidden)


def post_pre_norm_bwd(dy, dh, x, h, post_weight, pre_weight, gate, rstd_post, rstd_pre, *,
                      alpha: float = 1.0):
    """Gradients of :func:`post_pre_norm_fwd` from those of its y and h (x and its h as saved).
    Returns ``(dx, dresidual, dpost_weight, dpre_weight, dgate)``; dgate has the gate's
    shape, None without one. Column sums are float32 and bit-reproducible."""
    given = (dy, dh, x, h, post_weight, pre_weight, rstd_post, rstd_pre)
    dev = _require_cuda(*given) if gate is None else _require_cuda(*given, gate)
    shape = x.shape
    for name, t in (("dy", dy), ("dh", dh), ("h", h)):
        _same(name, t, "x", x)
    _check_param("post_weight", post_weight, x)
    _check_param("pre_weight", pre_weight, x)
    kind = 0 if gate is None else _gate_kind(gate, x)
    en = _dtype_enum(x)
    hidden = shape[-1]
    dy2, dh2, x2, h2 = _rows2(dy, hidden), _rows2(dh, hidden), _rows2(x, hidden), _rows2(h, hidden)
    rows = x2.shape[0]
    for name, t in (("rstd_post", rstd_post), ("rstd_pre", rstd_pre)):
        if t.dtype != torch.float32 or t.numel() != rows:
            raise ValueError(f"{name} must be float32 with one entry per row")
    dx, dres = torch.empty_like(x2), torch.empty_like(x2)
    g = None if gate is None else gate.contiguous()
    if not rows or not hidden:
        dgate = None if g is None else torch.zeros_like(g)
        return (dx.view(shape), dres.view(shape), torch.zeros_like(post_weight),
                torch.zeros_like(pre_weight), dgate)
    wp, wn = post_weight.contiguous(), pre_weight.contiguous()
    r1, r2 = rstd_post.contiguous(), rstd_pre.contiguous()
    dwp, dwn = torch.empty_like(wp), torch.empty_like(wn)
    dgate = None if g is None else torch.empty_like(g)
    ws_bytes = _post_pre_bwd_bytes(dev.index, rows, hidden)
    ws = torch.empty(ws_bytes, device=dev, dtype=torch.uint8)
    _enqueue(dev, "evg_post_pre_norm_bwd", dy2.data_ptr(), dh2.data_ptr(), x2.data_ptr(), h2.data_ptr(),
             wp.data_ptr(), wn.data_ptr(), None if g is None else g.data_ptr(), kind, r1.data_ptr(),
             r2.data_ptr(), dx.data_ptr(), dres.data_ptr(), dwp.data_ptr(), dwn.data_ptr(),
             None if dgate is None else dgate.data_ptr(), ws.data_ptr(), ws_bytes, rows, hidden,
             float(alpha), en)
    if len(shape) != 2:
        dx, dres = dx.view(shape), dres.view(shape)
    return dx, dres, dwp, dwn, dgate


# ---------------------------------------------- gradient norm and clipping
def _dense(t) -> bool:
    """Every element once, no gaps: any order of the dimensions."""
    if t.is_contiguous():
        return True
    reach = 1
    for st, n in sorted((st, n) for n, st in zip(t.shape, t.stride()) if n != 1):
        if st != reach:
            return False
        reach *= n
    return True


def _grad_list(grads, what):
    """The tensors as a list, their device, dtype enums, addresses and element counts. One
    pass per property over the whole list: a model has hundreds of tensors and the kernels
    take microseconds."""
    grads = list(grads)
    if not grads:
        raise ValueError(f"{what}: no tensors")
    dev = _require_cuda(*grads)
    try:
        codes = [_DTYPES[t.dtype] for t in grads]
    except KeyError as e:
        raise TypeError(f"unsupported dtype {e.args[0]}; expected float32/float16/bfloat16") from None
    plain = [t.is_contiguous() for t in grads]
    if not all(plain):
        for i, t in enumerate(grads):
            if not plain[i] and not _dense(t):
                raise ValueError(f"{what}: tensor {i} has gaps or repeated elements "
                                 f"(strides {tuple(t.stride())})")
    return grads, dev, codes, plain, [t.data_ptr() for t in grads], [t.numel() for t in grads]


@functools.lru_cache(maxsize=256)
def _clip_bytes(count: int) -> int:
    return lib.evg_clip_grads_workspace_bytes(count)


def _clip_call(dev, codes, ptrs, out_ptrs, numel, max_norm, clip):
    n = len(ptrs)
    norm = torch.empty((), device=dev, dtype=torch.float32)
    ws_bytes = _clip_bytes(n)
    ws = torch.empty(ws_bytes, device=dev, dtype=torch.uint8)
    # host arrays, read before the call returns
    aptr, asize, akind = array("Q", ptrs), array("q", numel), array("i", codes)
    aout = None if out_ptrs is None else array("Q", out_ptrs)
    _enqueue(dev, "evg_clip_grads", aptr.buffer_info()[0], None if aout is None else aout.buffer_info()[0],
             asize.buffer_info()[0], akind.buffer_info()[0], n, float(max_norm), 1 if clip else 0,
             norm.data_ptr(), ws.data_ptr(), ws_bytes)
    return norm


def grad_norm(grads) -> torch.Tensor:
    """2-norm over all elements of all tensors (float32 / float16 / bfloat16, mixed), as a
    float32 scalar on their device."""
    _, dev, codes, _, ptrs, numel = _grad_list(grads, "grad_norm")
    return _clip_call(dev, codes, ptrs, None, numel, 0.0, False)


def clip_grad_norm(grads, max_norm: float, outs=None) -> torch.Tensor:
    """Scale all tensors by ``min(1, max_norm / (norm + 1e-6))`` with ``norm`` their global
    2-norm, in place or into ``outs`` (per gradient a tensor of its type with as many
    elements in the same memory order, the gradient itself or other memory). Returns the norm before clipping, a float32 scalar on the device; nothing is
    read back. A norm that is not finite scales as the formula says (infinite: finite
    elements to zero; NaN: everything to NaN). Lists in which a tensor is there twice, or what
    is written overlaps another tensor, are refused."""
    grads, dev, codes, plain, ptrs, numel = _grad_list(grads, "clip_grad_norm")
    if not max_norm >= 0.0:
        raise ValueError(f"max_norm must not be negative, got {max_norm}")
    out_ptrs = None
    if outs is not None:
        outs, odev, ocodes, oplain, out_ptrs, onumel = _grad_list(outs, "clip_grad_norm outs")
        if odev != dev:
            raise RuntimeError(f"tensors on different devices: {dev} and {odev}")
        if ocodes != codes or onumel != numel or oplain != plain or (not all(plain) and any(
                not c and (o.shape != t.shape or o.stride() != t.stride())
                for o, t, c in zip(outs, grads, plain))):
            raise ValueError("outs must have the types, sizes and memory order of their gradients")
    written = out_ptrs or ptrs
    # (an empty tensor has no address of its own)
    if len(set(written)) != len(written) and \
            len({p for p, n in zip(written, numel) if n}) != sum(1 for n in numel if n):
        raise ValueError("clip_grad_norm: the same tensor is listed twice")
    return _clip_call(dev, codes, ptrs, out_ptrs, numel, max_norm, True)


# ------------------------------------------------------------- evoattention
def _check_evo(q, k, v, res_mask, pair_bias):
    if q.ndim != 5:
        raise ValueError(f"evoattention expects [B, S, N, H, D], got {tuple(q.shape)}")
    _same("q", q, "k", k)
    _same("q", q, "v", v)
    B, S, N, H, D = q.shape
    if res_mask.dtype != torch.float32 or res_mask.numel() != B * S * N:
        raise ValueError(f"res_mask must be float32 with B*S*N entries ([B, S, 1, 1, N]), got "
                         f"{res_mask.dtype} {tuple(res_mask.shape)}")
    if pair_bias.dtype != torch.float32 or pair_bias.numel() != B * H * N * N:
        raise ValueError(f"pair_bias must be float32 with B*H*N*N entries ([B, 1, H, N, N]), got "
                         f"{pair_bias.dtype} {tuple(pair_bias.shape)}")
    return B, S, N, H, D


def evoattention_fwd(q, k, v, res_mask, pair_bias, scale: float | None = None):
    """EvoformerAttention forward (ops/level1/evoattention/forward_ref.py:22-49).
    Returns ``(o, lse)``; ``lse`` is float32 ``[B, S, H, N]``."""
    dev = _require_cuda(q, k, v, res_mask, pair_bias)
    B, S, N, H, D = _check_evo(q, k, v, res_mask, pair_bias)
    if scale is None:
        scale = D ** -0.5
    q2, k2, v2 = q.contiguous(), k.contiguous(), v.contiguous()
    o = torch.empty_like(q2)
    lse = torch.empty(B, S, H, N, device=dev, dtype=torch.float32)
    if q2.numel() == 0:
        return o, lse
    with torch.cuda.device(dev):
        call("evg_evoattention_fwd", q2.data_ptr(), k2.data_ptr(), v2.data_ptr(),
             res_mask.contiguous().data_ptr(), pair_bias.contiguous().data_ptr(), o.data_ptr(),
             lse.data_ptr(), B, S, N, H, D, float(scale), _dtype_enum(q), _stream(dev))
    return o, lse


def evoattention_bwd(do, q, k, v, res_mask, pair_bias, o, lse, scale: float | None = None):
    """Returns ``(dq, dk, dv, d_pair_bias)``; d_pair_bias is float32, shaped like pair_bias."""
    dev = _require_cuda(do, q, k, v, res_mask, pair_bias, o, lse)
    B, S, N, H, D = _check_evo(q, k, v, res_mask, pair_bias)
    _same("do", do, "q", q)
    _same("o", o, "q", q)
    if lse.dtype != torch.float32 or lse.numel() != B * S * H * N:
        raise ValueError("lse must be float32 [B, S, H, N]")
    if scale is None:
        scale = D ** -0.5
    do2, q2, k2, v2, o2 = (t.contiguous() for t in (do, q, k, v, o))
    dq, dk, dv = torch.empty_like(q2), torch.empty_like(k2), torch.empty_like(v2)
    dbias = torch.empty(pair_bias.shape, device=dev, dtype=torch.float32)
    if q2.numel() == 0:
        return dq, dk, dv, dbias.zero_()
    en = _dtype_enum(q)
    with torch.cuda.device(dev):
        ws_bytes = lib.evg_evoattention_bwd_workspace_bytes(B, S, N, H, D, en)
        ws = torch.empty(max(ws_bytes, 16), device=dev, dtype=torch.uint8)
        call("evg_evoattention_bwd", do2.data_ptr(), q2.data_ptr(), k2.data_ptr(), v2.data_ptr(),
             res_mask.contiguous().data_ptr(), pair_bias.contiguous().data_ptr(), o2.data_ptr(),
             lse.contiguous().data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
             dbias.data_ptr(), ws.data_ptr(), ws_bytes, B, S, N, H, D, float(scale), en,
             _stream(dev))
    return dq, dk, dv, dbias


def device_status(reset: bool = True) -> None:
    """Synchronise and raise :class:`EvgError` (EVG_ETIMEOUT) if a bounded device-side
    wait (attention, norm backward rings, wide softmax) gave up since the last reset."""
    call("evg_device_status", 1 if reset else 0)


def selftest_bounded_wait(limit_cycles: int = 2_000_000, device=None) -> int:
    """Launch the bounded-wait self-test (a wait nothing satisfies, given up after
    ``limit_cycles``) and return the abort word the block recorded. The sticky
    status is left set: the next :func:`device_status` raises EVG_ETIMEOUT once."""
    dev = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    word = torch.zeros(1, device=dev, dtype=torch.int32)
    with torch.cuda.device(dev):
        call("evg_selftest_bounded_wait", int(limit_cycles), word.data_ptr(), _stream(dev))
    return int(word.item())


def flush_l2(buffer: torch.Tensor) -> None:
    """Overwrite ``buffer`` (larger than L2) so cached lines of other tensors are evicted."""
    dev = _require_cuda(buffer)
    with torch.cuda.device(dev):
        call("evg_flush_l2", buffer.data_ptr(), buffer.numel() * buffer.element_size(),
             _stream(dev))

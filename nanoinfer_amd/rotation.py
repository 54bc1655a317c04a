"""Rotary positions on the GPU (``ni_rotary_init``, ``ni_rotary_apply``).

:class:`Rotary` is a model's rotation, made once; :func:`rotary` rotates
contiguous rows of heads (what :func:`nanoinfer_amd.attention` then reads), and
``PagedKv.append_rotary`` rotates keys on their way into the cache.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional

from . import _abi
from .batch import KvError, _on, _stream_now, _torch

SCALINGS = {None: _abi.NI_ROTARY_PLAIN, "linear": _abi.NI_ROTARY_LINEAR, "ntk": _abi.NI_ROTARY_NTK,
            "yarn": _abi.NI_ROTARY_YARN}

_types = None  # torch dtype -> NI_F32, NI_F16, NI_BF16


def dtype_code(dtype):
    """NI_* of a torch dtype, or None."""
    global _types
    if _types is None:
        torch = _torch()
        _types = {torch.float32: _abi.NI_F32, torch.float16: _abi.NI_F16, torch.bfloat16: _abi.NI_BF16}
    return _types.get(dtype)


class Rotary:
    """A rotation of heads of ``head_dim`` by position: pair ``i`` of the first
    ``rot_dim`` dims (all by default) turns by ``pos * base**(-2i/rot_dim)``.
    Pairs are ``(x[i], x[i + rot_dim/2])``, or ``(x[2i], x[2i+1])`` if
    ``interleaved``.  ``scaling`` stretches a context by ``factor``: "linear"
    (every angle divided), "ntk" (a larger base) or "yarn" (by the turns a pair
    makes over ``orig_ctx``, between ``beta_fast`` and ``beta_slow``, with
    cosines and sines times ``0.1 ln(factor) + 1``).  ``attn_scale`` replaces
    that last number."""

    def __init__(self, head_dim: int, base: float = 10000.0, rot_dim: Optional[int] = None, interleaved: bool = False,
                 scaling: Optional[str] = None, factor: float = 1.0, orig_ctx: int = 0, beta_fast: float = 32.0,
                 beta_slow: float = 1.0, attn_scale: Optional[float] = None):
        if scaling not in SCALINGS:
            raise ValueError(f"unknown scaling {scaling!r} (one of {list(SCALINGS)})")
        for name, x in (("head_dim", head_dim), ("rot_dim", rot_dim or 0), ("orig_ctx", orig_ctx)):
            if not 0 <= x <= 0xffffffff:
                raise ValueError(f"{name} {x} out of range")
        if rot_dim == 0 or (attn_scale is not None and not attn_scale > 0) or beta_fast <= 0 or beta_slow <= 0:
            raise ValueError("rot_dim, attn_scale, beta_fast and beta_slow must be positive")
        o = _abi.ni_rotary_opts(base, rot_dim or 0, int(interleaved), SCALINGS[scaling], orig_ctx, factor, beta_fast,
                                beta_slow, attn_scale or 0.0)
        self._r = _abi.ni_rotary()
        L = _abi.lib()
        rc = L.ni_rotary_init(C.byref(self._r), head_dim, C.byref(o))
        if rc != 0:
            raise KvError(rc, (L.ni_kv_last_error(None) or b"").decode())
        self.head_dim, self.rot_dim, self.interleaved = head_dim, self._r.rot_dim, bool(interleaved)
        self.scale = float(self._r.scale)
        self.ref = C.pointer(self._r)


def rotary(x, rotary: Rotary, n_head: int, positions=None, pos0: int = 0, out=None, stream=None):
    """Rotate rows of ``n_head`` heads: ``x`` is a 2-D CUDA tensor (float32,
    float16 or bfloat16) whose rows are at least ``n_head * head_dim`` wide,
    any row stride (rows on 16-byte borders are fastest).  Row ``i`` is at
    ``positions[i]`` (an int32 CUDA tensor) or at ``pos0 + i``.  Returns
    ``out`` ([n, n_head * head_dim] of x's type, allocated if not given; it may
    be ``x``).  Computed in float32 and rounded once."""
    torch = _torch()
    # The quick form of the checks below, which say what is wrong: a launch
    # takes the device less time than they take the host (64 rows of 12 heads:
    # 2.5 us of kernel).
    if type(x) is torch.Tensor and type(out) is torch.Tensor and x.is_cuda and 0 <= pos0 <= 0xffffffff and n_head >= 0:
        device, dtype, width = x.get_device(), x.dtype, n_head * rotary.head_dim
        shape, stride, oshape, ostride = x.shape, x.stride(), out.shape, out.stride()
        s = _stream_now(device, stream)
        if (s is not None and len(shape) == 2 and len(oshape) == 2 and stride[1] == 1 and ostride[1] == 1
                and shape[1] >= width and oshape[1] >= width and oshape[0] >= shape[0] and out.dtype is dtype
                and dtype_code(dtype) is not None and out.get_device() == device
                and (positions is None or type(positions) is torch.Tensor and positions.dtype is torch.int32
                     and positions.dim() == 1 and positions.stride(0) == 1 and positions.shape[0] >= shape[0]
                     and positions.get_device() == device)):
            rc = _abi.lib().ni_rotary_apply(rotary.ref, _types[dtype], x.data_ptr(), stride[0], out.data_ptr(),
                                            ostride[0], shape[0], n_head,
                                            None if positions is None else positions.data_ptr(), pos0, s)
            if rc != 0:
                raise KvError(rc, (_abi.lib().ni_kv_last_error(None) or b"").decode())
            return out
    if not isinstance(x, torch.Tensor) or x.dim() != 2 or dtype_code(x.dtype) is None:
        raise TypeError("x must be a 2-D float32, float16 or bfloat16 tensor")
    n, width = x.shape[0], n_head * rotary.head_dim
    if n_head < 0 or x.stride(1) != 1 or x.shape[1] < width:
        raise ValueError(f"x is {tuple(x.shape)}: needs rows of at least {width} with unit stride")
    if positions is not None and (not isinstance(positions, torch.Tensor) or positions.dtype != torch.int32
                                  or positions.dim() != 1 or not positions.is_contiguous()):
        raise TypeError("positions must be a contiguous 1-D int32 tensor")
    if positions is not None and positions.shape[0] < n:
        raise ValueError(f"positions holds {positions.shape[0]} of {n} rows")
    if not 0 <= pos0 <= 0xffffffff:
        raise ValueError("pos0 must be in 0..2^32-1")
    if out is not None and (not isinstance(out, torch.Tensor) or out.dtype != x.dtype or out.dim() != 2
                            or out.stride(1) != 1 or out.shape[0] < n or out.shape[1] < width):
        raise ValueError(f"out must be a {x.dtype} [{n}][{width}] tensor with contiguous rows")
    if not x.is_cuda:
        raise TypeError("x must be a CUDA tensor")
    for name, t in (("positions", positions), ("out", out)):
        if t is not None and t.device != x.device:
            raise ValueError(f"{name} is on {t.device}, x on {x.device}")
    L = _abi.lib()
    with _on(x.get_device(), stream) as s:
        if out is None:
            out = torch.empty((n, width), dtype=x.dtype, device=x.device)
        rc = L.ni_rotary_apply(rotary.ref, dtype_code(x.dtype), x.data_ptr(), x.stride(0), out.data_ptr(),
                               out.stride(0), n, n_head, None if positions is None else positions.data_ptr(), pos0, s)
    if rc != 0:
        raise KvError(rc, (L.ni_kv_last_error(None) or b"").decode())
    return out

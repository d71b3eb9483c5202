"""Queries and keys of an attention layer, normalised per head and turned by the positions of their rows: the step in front of
``neighbor_attention``, in one pass, with gradients.

No counterpart in the reference: its model adapters leave this to their libraries (dynamis_model/src/dynamis_model/nnp/uma.py).

All work is enqueued on the current stream of the tensors' device.  Gradients are formed without atomics: the same inputs give the same bits.
They can be taken once; a gradient of a gradient raises, and so does a tangent of forward mode.
"""

from __future__ import annotations

import ctypes
import math
from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .message import _DTYPES, FLOAT_MAX, INT32_MAX, _differentiates, _heads_last, _pointer

_POSITIONS = {torch.float32: _lib.DYNB_F32, torch.float64: _lib.DYNB_F64}
MAX_DIM = 256        # DYNB_ROTARY_MAX_DIM
MAX_AXES = 3         # DYNB_ROTARY_MAX_AXES


def _rotary_args(q, k, pos, wave, q_weight, k_weight, eps, interleaved) -> "_lib.Rotary":
    a = _lib.Rotary()
    a.q_dev, a.k_dev, a.pos_dev, a.wave_dev = q.data_ptr(), k.data_ptr(), pos.data_ptr(), wave.data_ptr()
    a.q_row, a.q_head, a.k_row, a.k_head = q.stride(0), q.stride(1), k.stride(0), k.stride(1)
    a.q_weight_dev, a.k_weight_dev = _pointer(q_weight), _pointer(k_weight)
    a.n_q, a.n_k, a.heads, a.kv_heads, a.dim, a.axes = q.size(0), k.size(0), q.size(1), k.size(1), q.size(2), pos.size(1)
    a.dtype, a.pos_dtype, a.interleaved = _DTYPES[q.dtype], _POSITIONS[pos.dtype], interleaved
    a.norm, a.eps = int(eps is not None), 0.0 if eps is None else eps
    return a


class _RotaryHeads(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, pos, wave, q_weight, k_weight, eps, interleaved):   # ctx None: without gradients nothing is kept for them
        dev = q.device
        q, k = _heads_last(q), _heads_last(k)
        with _lib.on_device(dev):
            q_out, k_out = (torch.empty(t.shape, dtype=t.dtype, device=dev) for t in (q, k))
            args = _rotary_args(q, k, pos, wave, q_weight, k_weight, eps, interleaved)
            _lib.check(_lib.lib().dynb_rotary_heads(ctypes.byref(args), q_out.data_ptr(), k_out.data_ptr(), _lib.stream_of(dev)), "rotary_heads")
        if ctx is not None:
            ctx.save_for_backward(q, k, pos, wave, q_weight, k_weight)
            ctx.eps, ctx.interleaved = eps, interleaved
        return q_out, k_out

    @staticmethod
    @once_differentiable
    def backward(ctx, d_q_out, d_k_out):
        q, k, pos, wave, q_weight, k_weight = ctx.saved_tensors
        want_q, want_k, want_pos, _, want_qw, want_kw = ctx.needs_input_grad[:6]
        dev, L = q.device, _lib.lib()
        d_q_out, d_k_out = _heads_last(d_q_out), _heads_last(d_k_out)
        with _lib.on_device(dev):
            dq = torch.empty(q.shape, dtype=q.dtype, device=dev) if want_q else None
            dk = torch.empty(k.shape, dtype=k.dtype, device=dev) if want_k else None
            d_pos = torch.empty_like(pos) if want_pos else None
            d_qw = torch.empty_like(q_weight) if want_qw else None
            d_kw = torch.empty_like(k_weight) if want_kw else None
            args = _rotary_args(q, k, pos, wave, q_weight, k_weight, ctx.eps, ctx.interleaved)   # anew: hooks may have moved what was saved
            ws = None
            if want_qw or want_kw:
                nbytes = ctypes.c_int64()
                _lib.check(L.dynb_rotary_heads_workspace_bytes(ctypes.byref(args), ctypes.byref(nbytes)), "rotary_heads_workspace_bytes")
                ws = torch.empty(nbytes.value, dtype=torch.uint8, device=dev)
            _lib.check(L.dynb_rotary_heads_backward(ctypes.byref(args), d_q_out.data_ptr(), d_q_out.stride(0), d_q_out.stride(1), d_k_out.data_ptr(),
                                                    d_k_out.stride(0), d_k_out.stride(1), _pointer(dq), _pointer(dk), _pointer(d_pos), _pointer(d_qw),
                                                    _pointer(d_kw), _pointer(ws), 0 if ws is None else ws.numel(), _lib.stream_of(dev)),
                       "rotary_heads_backward")
        return dq, dk, d_pos, None, d_qw, d_kw, None, None


def rotary_heads(q: torch.Tensor, k: torch.Tensor, pos: torch.Tensor, wave: torch.Tensor, q_weight: Optional[torch.Tensor] = None,
                 k_weight: Optional[torch.Tensor] = None, eps: Optional[float] = 1e-6, interleaved: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """Queries and keys for ``neighbor_attention`` whose products depend on where their rows are.  Per head: ``n = x / sqrt(mean(x^2) + eps) * weight``
    (``eps=None``: n = x), then pair p of n turns by the angle ``2 pi wave[p] . pos[i]``: ``(a, b)`` becomes ``(a cos - b sin, a sin + b cos)``.

    q [targets, heads, dim], k [sources, kv_heads, dim]; float32, float16 or bfloat16, both alike; dim even and at most 256.  Rows and heads may have any
    strides.  Row i of both is at ``pos[i]``: targets are the first of the rows [owned | ghost], pos [rows, axes] float32 or float64 has as many rows as the
    longer of q and k, and one to three axes.  wave [dim / 2, axes] float32: turns per unit of each axis.  Waves along one axis each are rotary positions with
    several axes; whole waves on fractional coordinates (``pos @ inv(cell)``) are the same in every image of a periodic box; pairs of zero waves stay
    unturned.  On Cartesian
    coordinates products of q and k depend on how the system is turned.  Pair p is elements (p, p + dim / 2), or (2 p, 2 p + 1) with ``interleaved``.  q_weight, k_weight [dim] float32: ones unless given.

    Turns are formed in 64 bits and whole ones dropped, all else is in 32 bits and rounded once.  Gradients for q, k, pos (forces; formed in 32
    bits, also for float64) and the weights, whose sums over rows are joined in 64 bits; waves have none."""
    for name, t in (("q", q), ("k", k)):
        if not isinstance(t, torch.Tensor) or not t.is_cuda:
            raise RuntimeError(f"{name} must be a CUDA tensor")
        if t.dim() != 3:
            raise RuntimeError(f"{name} must have shape [rows, heads, dim], got {list(t.shape)}")
    if q.dtype not in _DTYPES or k.dtype is not q.dtype:
        raise RuntimeError(f"q and k must both be float32, float16 or bfloat16, got {q.dtype} and {k.dtype}")
    on, dim = q.get_device(), q.size(2)
    if k.get_device() != on:
        raise RuntimeError("q and k must be on the same device")
    if k.size(2) != dim or dim % 2 != 0 or not 2 <= dim <= MAX_DIM:
        raise RuntimeError(f"q and k must have the same even dim in [2, {MAX_DIM}], got {dim} and {k.size(2)}")
    if not (1 <= q.size(1) <= 65535 and 1 <= k.size(1) <= 65535):
        raise RuntimeError(f"q and k must have 1 to 65535 heads, got {q.size(1)} and {k.size(1)}")
    rows = max(q.size(0), k.size(0))
    if rows >= INT32_MAX:
        raise RuntimeError(f"q and k must have fewer than 2^31 - 1 rows, got {rows}")
    if not isinstance(pos, torch.Tensor) or pos.get_device() != on or pos.dtype not in _POSITIONS:
        raise RuntimeError("pos must be a float32 or float64 tensor on the device of q")
    if pos.dim() != 2 or pos.size(0) != rows or not 1 <= pos.size(1) <= MAX_AXES:
        raise RuntimeError(f"pos must have shape [{rows}, 1 to {MAX_AXES}], got {list(pos.shape)}")
    if not isinstance(wave, torch.Tensor) or wave.get_device() != on or wave.dtype is not torch.float32:
        raise RuntimeError("wave must be a float32 tensor on the device of q")
    if wave.shape != (dim // 2, pos.size(1)):
        raise RuntimeError(f"wave must have shape [{dim // 2}, {pos.size(1)}], got {list(wave.shape)}")
    if wave.requires_grad and torch.is_grad_enabled():
        raise RuntimeError("wave has no gradient: pass it detached")
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w is None:
            continue
        if eps is None:
            raise RuntimeError(f"{name} belongs to the norm: give eps")
        if not isinstance(w, torch.Tensor) or w.get_device() != on or w.dtype is not torch.float32 or w.shape != (dim,):
            raise RuntimeError(f"{name} must be a float32 tensor of shape [{dim}] on the device of q")
    if eps is not None:
        eps = float(eps)
        if not 0.0 <= eps <= FLOAT_MAX or math.isinf(ctypes.c_float(eps).value) or eps > 3e38:
            raise RuntimeError(f"eps must be finite and not negative, got {eps}")
    weights = (None if w is None else w.contiguous() for w in (q_weight, k_weight))
    args = (q, k, pos.contiguous(), wave.contiguous(), *weights, eps, int(bool(interleaved)))
    if _differentiates(q, k, pos, q_weight, k_weight):
        return _RotaryHeads.apply(*args)
    return _RotaryHeads.forward(None, *args)     # a third of a small call's time is autograd's

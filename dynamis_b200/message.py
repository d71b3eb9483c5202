"""The work of a message-passing layer between two halo exchanges, with gradients.

A model over [owned | ghost] rows takes its graph from ``owned_graph`` (or any graph call of this package), its ghosts' embeddings from
``FeaturePushToExchange``, and between two exchanges computes along the edges.  With gathers and scatters that keeps a tensor of
[edges, heads, dim] per step of the formula (27 GB each for a million atoms, 52 neighbours, 128 columns); the calls here keep nothing of
the size of the edges but biases:

* ``neighbor_index(edge_index, num_targets, num_sources)``: the graph's lists by target and by source, once per MD step;
* ``neighbor_attention(q, k, v, index, bias, scale)``: every target attends to its neighbours;
* ``distance_bias(dist, table, cutoff)``: a learned bias of the logits, smooth in the distance and at the cutoff;
* ``type_linear(x, weight, type_index(types, num_types), bias)``: rows times the matrix of their atom type.

No counterpart in the reference: its model adapters leave this to their libraries (dynamis_model/src/dynamis_model/nnp/mace.py:260-364).

All work is enqueued on the current stream of the tensors' device.  Gradients are formed without atomics: the same inputs give the same bits.
They can be taken once; a gradient of a gradient raises.
"""

from __future__ import annotations

import ctypes
import math
import threading
from dataclasses import dataclass
from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .graph import give_host_words, lose_host_words, take_host_words

_DTYPES = {torch.float32: _lib.DYNB_F32, torch.float16: _lib.DYNB_F16, torch.bfloat16: _lib.DYNB_BF16}
MAX_DIM = 256            # DYNB_ATTENTION_MAX_DIM
MAX_ROW = 1 << 30        # DYNB_ATTENTION_MAX_ROW
MAX_BUCKETS = 1024       # DYNB_DISTANCE_BIAS_MAX_BUCKETS
MAX_BIAS_HEADS = 1024    # DYNB_DISTANCE_BIAS_MAX_HEADS
MAX_TYPES = 4096         # DYNB_TYPE_LINEAR_MAX_TYPES
MAX_WIDTH = 16384        # DYNB_TYPE_LINEAR_MAX_WIDTH
LONGEST_LIST = 256       # NI_LONGEST (csrc/neighbors.cu): longer lists take a larger workspace
INT32_MAX = 2 ** 31 - 1
FLOAT_MAX = 3.4028234663852886e38
MAX_EDGES = 2 ** 31 - 2 ** 16   # DYNB_MAX_EDGES


def _lists(what: str, names, lists) -> None:
    on = -1
    for name, t in zip(names, lists):
        if not (isinstance(t, torch.Tensor) and t.is_cuda):
            raise RuntimeError(f"{what}: {name} must be a CUDA tensor")
        if t.dtype is not torch.int32 or t.dim() != 1 or not t.is_contiguous():
            raise RuntimeError(f"{what}: {name} must be a contiguous 1-D int32 tensor, got {t.dtype} {list(t.shape)}")
        at = t.get_device()
        if on >= 0 and at != on:
            raise RuntimeError(f"{what}: all lists must be on the same device")
        on = at


def _lists_refused(what: str, checks) -> None:
    """``checks``: pairs of a text and a function that says whether it holds, taken in turn (a later one may rely on the earlier ones)."""
    _not_capturing(what)
    for text, holds in checks:
        if not holds():
            raise RuntimeError(f"{what}: {text}")


def _each_once(t: torch.Tensor) -> bool:
    """Whether ``t`` [n] names every number below n once."""
    n = t.numel()
    return n == 0 or bool(((t >= 0) & (t < n)).all()) and bool((torch.bincount(t, minlength=n) == 1).all())


def _runs(start: torch.Tensor, n: int) -> bool:
    return int(start[0]) == 0 and int(start[-1]) == n and bool((start[1:] >= start[:-1]).all())


def _spread(t: torch.Tensor, start: torch.Tensor) -> torch.Tensor:
    """The entry of ``t`` that every place of its run belongs to."""
    return torch.repeat_interleave(t, (start[1:] - start[:-1]).long())


_NEIGHBOR_LISTS = ("rows", "row_start", "src", "cols", "col_start", "in_edge", "in_dst")


@dataclass(frozen=True)
class NeighborIndex:
    """Lists of a graph (int32).  The edges keep the numbers that they have in ``edge_index``.

    rows [T], row_start [T + 1]   targets in the order of their edges, those without edges behind them (ascending); the edges of
                                  ``rows[r]`` are ``row_start[r]`` to ``row_start[r + 1] - 1``
    src [E]                       sources of the edges
    cols [S], col_start [S + 1]   sources in the order of their first edge, those without edges behind them (ascending)
    in_edge [E], in_dst [E]       edges that leave ``cols[c]``, ascending, at ``col_start[c]`` and on, and their targets

    ``neighbor_index`` makes them.  Lists made by hand have to be as described: entries out of range are passed over, but results of rows that ``rows`` or ``cols``
    leave out or name twice, and of edges that no run holds, are not defined (memory may show that was not written).  ``check_lists`` looks.
    """

    rows: torch.Tensor
    row_start: torch.Tensor
    src: torch.Tensor
    cols: torch.Tensor
    col_start: torch.Tensor
    in_edge: torch.Tensor
    in_dst: torch.Tensor

    def __post_init__(self):
        _lists("NeighborIndex", _NEIGHBOR_LISTS, (self.rows, self.row_start, self.src, self.cols, self.col_start, self.in_edge, self.in_dst))
        E = self.src.numel()
        if self.row_start.numel() != self.rows.numel() + 1 or self.col_start.numel() != self.cols.numel() + 1:
            raise RuntimeError("NeighborIndex: row_start and col_start must have one entry more than rows and cols")
        if self.in_edge.numel() != E or self.in_dst.numel() != E:
            raise RuntimeError("NeighborIndex: src, in_edge and in_dst must have one entry per edge")

    def check_lists(self) -> None:
        """Waits and raises if the lists are not those of one graph: for lists that ``neighbor_index`` did not make."""
        E, S = self.num_edges, self.num_sources
        _lists_refused("NeighborIndex", (
            ("rows must name every target once", lambda: _each_once(self.rows)),
            ("cols must name every source once", lambda: _each_once(self.cols)),
            ("in_edge must name every edge once", lambda: _each_once(self.in_edge)),
            (f"row_start must rise from 0 to {E}", lambda: _runs(self.row_start, E)),
            (f"col_start must rise from 0 to {E}", lambda: _runs(self.col_start, E)),
            (f"src must lie in [0, {S})", lambda: bool(((self.src >= 0) & (self.src < S)).all())),
            ("in_edge must list the edges of cols", lambda: torch.equal(self.src[self.in_edge.long()], _spread(self.cols, self.col_start))),
            ("in_dst must hold the targets of in_edge", lambda: torch.equal(_spread(self.rows, self.row_start)[self.in_edge.long()], self.in_dst))))

    @property
    def num_targets(self) -> int:
        return self.rows.numel()

    @property
    def num_sources(self) -> int:
        return self.cols.numel()

    @property
    def num_edges(self) -> int:
        return self.src.numel()


@dataclass(frozen=True)
class TypeIndex:
    """Rows by type (int32): ``order`` [N] lists the rows of type 0, of type 1, ..., ascending inside a type, every row once;
    ``start`` [types + 1] is where every type begins, and N behind the last.

    ``type_index`` makes them.  Lists made by hand have to be as described: entries out of range are passed over, but results of rows that are left out or
    named twice are not defined (memory may show that was not written).  ``check_lists`` looks."""

    order: torch.Tensor
    start: torch.Tensor

    def __post_init__(self):
        _lists("TypeIndex", ("order", "start"), (self.order, self.start))
        if self.start.numel() < 2 or self.start.numel() > MAX_TYPES + 1:
            raise RuntimeError(f"TypeIndex: the number of types must lie in [1, {MAX_TYPES}], got {self.start.numel() - 1}")
        if self.order.get_device() not in _STATUS:
            _make_status_word(self.order.device)

    def check_lists(self) -> None:
        """Waits and raises if the lists do not give every row one type: for lists that ``type_index`` did not make."""
        N = self.order.numel()
        _lists_refused("TypeIndex", (("order must name every row once", lambda: _each_once(self.order)),
                                     (f"start must rise from 0 to {N}", lambda: _runs(self.start, N))))

    def check_status(self) -> None:
        """Synchronises and raises if a wait inside a kernel of a ``type_linear`` on this device ran out, whose results are not valid then.  ``type_linear``
        looks, without waiting, before it launches; behind the last call, or where a graph replays the calls, look here."""
        dev = self.order.device
        torch.cuda.synchronize(dev)
        with _lib.on_device(dev):
            _status_word(dev)

    @property
    def num_types(self) -> int:
        return self.start.numel() - 1


def _not_capturing(what: str) -> None:
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError(f"{what} waits for counts and cannot be captured into a graph: call it outside")


def neighbor_index(edge_index: torch.Tensor, num_targets: int, num_sources: int) -> NeighborIndex:
    """The lists of ``edge_index`` [2, E] int64 (sources, targets) that ``neighbor_attention`` and its gradients read.

    Targets are rows 0 .. num_targets - 1, sources rows 0 .. num_sources - 1 (of [owned | ghost]: ``num_local`` and all).  The edges of a target must
    stand behind one another, as every graph call of this package returns them.  Waits for the stream once; raises on an endpoint out of
    range and on targets whose edges are apart."""
    if not isinstance(edge_index, torch.Tensor) or not edge_index.is_cuda:
        raise RuntimeError("edge_index must be a CUDA tensor")
    if edge_index.dim() != 2 or edge_index.size(0) != 2:
        raise RuntimeError(f"edge_index must have shape [2, E], got {list(edge_index.shape)}")
    if edge_index.dtype != torch.int64:
        raise RuntimeError(f"edge_index must be int64, got {edge_index.dtype}")
    T, S, E = int(num_targets), int(num_sources), edge_index.size(1)
    if not (0 <= T < INT32_MAX and 0 <= S < INT32_MAX):
        raise RuntimeError(f"num_targets and num_sources must lie in [0, 2^31 - 1), got {T} and {S}")
    if E >= MAX_EDGES:
        raise RuntimeError(f"edge_index must have fewer than {MAX_EDGES} edges, got {E}")
    if E > 0 and edge_index.stride(1) != 1:
        edge_index = edge_index.contiguous()
    dev = edge_index.device
    src64, dst64 = edge_index[0].data_ptr(), edge_index[1].data_ptr()
    L = _lib.lib()
    with _lib.on_device(dev):
        _not_capturing("neighbor_index")
        stream = _lib.stream_of(dev)
        rows, row_start, src, cols, col_start, in_edge, in_dst = (
            torch.empty(n, dtype=torch.int32, device=dev) for n in (T, T + 1, E, S, S + 1, E, E))
        nbytes = ctypes.c_int64()
        _lib.check(L.dynb_neighbor_index_workspace_bytes(E, T, S, 0, ctypes.byref(nbytes)), "neighbor_index_workspace_bytes")
        ws = torch.empty(nbytes.value, dtype=torch.uint8, device=dev)   # this call's own: behind its wait another thread may use the stream before the fill
        words = take_host_words(2)
        try:
            _lib.check(L.dynb_neighbor_index_plan(src64, dst64, E, T, S, rows.data_ptr(), row_start.data_ptr(), src.data_ptr(), cols.data_ptr(),
                                                  col_start.data_ptr(), in_edge.data_ptr(), words.data_ptr(), ws.data_ptr(), ws.numel(), stream), "neighbor_index_plan")
            torch.cuda.current_stream(dev).synchronize()
        except BaseException:
            lose_host_words(words, dev)
            raise
        word = int(words[0])
        status, longest = word & 0xFFFFFFFF, (word >> 32) & 0xFFFFFFFF
        give_host_words(words)
        if status & 1:
            raise RuntimeError(f"neighbor_index: an edge has a target outside [0, {T}) or a source outside [0, {S})")
        if status & 2:
            raise RuntimeError("neighbor_index: the edges of a target must stand behind one another")
        if longest > LONGEST_LIST:
            planned = ws
            _lib.check(L.dynb_neighbor_index_workspace_bytes(E, T, S, longest, ctypes.byref(nbytes)), "neighbor_index_workspace_bytes")
            ws = torch.empty(nbytes.value, dtype=torch.uint8, device=dev)
            _lib.check(L.dynb_copy_async(ws.data_ptr(), planned.data_ptr(), planned.numel(), stream), "copy_async")
        _lib.check(L.dynb_neighbor_index_fill(dst64, E, T, S, src.data_ptr(), col_start.data_ptr(), longest, in_edge.data_ptr(), in_dst.data_ptr(),
                                              ws.data_ptr(), ws.numel(), stream), "neighbor_index_fill")
    return NeighborIndex(rows, row_start, src, cols, col_start, in_edge, in_dst)


def _heads_last(t: torch.Tensor) -> torch.Tensor:
    """``t`` as the kernels read it: any strides of rows (below 2^30 elements) and heads, the elements of a head consecutive."""
    if (t.stride(2) == 1 or t.size(2) == 1) and t.stride(0) < MAX_ROW:
        return t
    return t.clone(memory_format=torch.contiguous_format)   # contiguous() would keep the stride of a single row, whatever it is


def _pointer(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _attention_args(q, k, v, bias, index: NeighborIndex, scale: float) -> "_lib.Attention":
    a = _lib.Attention()
    a.q_dev, a.k_dev, a.v_dev = q.data_ptr(), k.data_ptr(), v.data_ptr()
    a.q_row, a.q_head = q.stride(0), q.stride(1)
    a.k_row, a.k_head = k.stride(0), k.stride(1)
    a.v_row, a.v_head = v.stride(0), v.stride(1)
    a.bias_dev = _pointer(bias)
    a.rows_dev, a.row_start_dev, a.src_dev = index.rows.data_ptr(), index.row_start.data_ptr(), index.src.data_ptr()
    a.n_targets, a.n_sources, a.n_edges = q.size(0), k.size(0), index.num_edges
    a.heads, a.kv_heads, a.dim, a.dtype = q.size(1), k.size(1), q.size(2), _DTYPES[q.dtype]
    a.scale = scale
    return a


class _NeighborAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, bias, index, scale, keep):
        dev = q.device
        q, k, v = _heads_last(q), _heads_last(k), _heads_last(v)
        with _lib.on_device(dev):
            out = torch.empty(q.shape, dtype=q.dtype, device=dev)
            out32 = stats = None
            if keep:
                out32 = out if q.dtype == torch.float32 else torch.empty(q.shape, dtype=torch.float32, device=dev)
                stats = torch.empty((q.size(0), 2, q.size(1)), dtype=torch.float32, device=dev)
            args = _attention_args(q, k, v, bias, index, scale)
            _lib.check(_lib.lib().dynb_neighbor_attention(ctypes.byref(args), out.data_ptr(), None if out32 is out else _pointer(out32),
                                                          _pointer(stats), _lib.stream_of(dev)), "neighbor_attention")
        if stats is not None:
            ctx.save_for_backward(q, k, v, bias, out32, stats)
            ctx.index, ctx.scale = index, scale
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, d_out):
        q, k, v, bias, out32, stats = ctx.saved_tensors
        want_q, want_k, want_v, want_bias = ctx.needs_input_grad[:4]
        index, dev = ctx.index, q.device
        d_out = _heads_last(d_out)
        with _lib.on_device(dev):
            dq = torch.empty(q.shape, dtype=q.dtype, device=dev) if want_q else None
            dk = torch.empty(k.shape, dtype=k.dtype, device=dev) if want_k else None
            dv = torch.empty(v.shape, dtype=v.dtype, device=dev) if want_v else None
            d_bias = torch.empty(bias.shape, dtype=torch.float32, device=dev) if want_bias else None
            delta = torch.empty((q.size(0), q.size(1), 4), dtype=torch.float32, device=dev)
            args = _attention_args(q, k, v, bias, index, ctx.scale)   # anew: hooks may have moved what was saved
            _lib.check(_lib.lib().dynb_neighbor_attention_backward(
                ctypes.byref(args), d_out.data_ptr(), d_out.stride(0), d_out.stride(1), out32.data_ptr(), stats.data_ptr(), index.cols.data_ptr(),
                index.col_start.data_ptr(), index.in_edge.data_ptr(), index.in_dst.data_ptr(), delta.data_ptr(), _pointer(dq), _pointer(dk),
                _pointer(dv), _pointer(d_bias), _lib.stream_of(dev)), "neighbor_attention_backward")
        return dq, dk, dv, d_bias, None, None, None


def neighbor_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, index: NeighborIndex, bias: Optional[torch.Tensor] = None,
                       scale: Optional[float] = None) -> torch.Tensor:
    """Attention of every target to its neighbours.  Per head and edge e from s to t: ``z_e = scale * q[t] . k[s] + bias[e]``, ``p`` = softmax of z
    over the edges of t, ``out[t] = sum_e p_e v[s]``.

    q [targets, heads, dim]; k, v [sources, kv_heads, dim], heads a multiple of kv_heads (query head h reads head
    ``h // (heads // kv_heads)``), dim at most 256; float32, float16 or bfloat16, all alike.  Rows and heads may have any strides (a slice of a joint
    projection is read in place).  bias [E, heads] float32; an edge whose bias is -inf takes no part for that head, whatever its rows
    hold.  scale: 1 / sqrt(dim) unless given.  A target without edges, or with none that takes part, gives zeros and gets zero gradients.

    Sums, maxima and probabilities are in 32 bits; the result and the gradients of q, k and v are rounded once to their type, the bias's
    gradient stays in 32 bits."""
    if not isinstance(index, NeighborIndex):
        raise RuntimeError("index must be a NeighborIndex (see neighbor_index)")
    for name, t in (("q", q), ("k", k), ("v", v)):
        if not isinstance(t, torch.Tensor) or not t.is_cuda:
            raise RuntimeError(f"{name} must be a CUDA tensor")
        if t.dim() != 3:
            raise RuntimeError(f"{name} must have shape [rows, heads, dim], got {list(t.shape)}")
    if q.dtype not in _DTYPES or k.dtype is not q.dtype or v.dtype is not q.dtype:
        raise RuntimeError(f"q, k and v must all be float32, float16 or bfloat16, got {q.dtype}, {k.dtype} and {v.dtype}")
    on = q.get_device()
    if k.get_device() != on or v.get_device() != on:
        raise RuntimeError("q, k and v must be on the same device")
    (targets, heads, dim), (sources, kv_heads, kv_dim) = q.shape, k.shape
    if k.shape != v.shape:
        raise RuntimeError(f"k and v must have the same shape, got {list(k.shape)} and {list(v.shape)}")
    if dim != kv_dim or not 1 <= dim <= MAX_DIM:
        raise RuntimeError(f"q, k and v must have the same dim in [1, {MAX_DIM}], got {dim} and {kv_dim}")
    if kv_heads < 1 or heads < 1 or heads % kv_heads != 0 or heads > 65535:
        raise RuntimeError(f"the heads of q must be a multiple of those of k and v, got {heads} and {kv_heads}")
    if targets != index.num_targets or sources != index.num_sources:
        raise RuntimeError(f"the index is of {index.num_targets} targets and {index.num_sources} sources, got {targets} and {sources} rows")
    if index.src.get_device() != on:
        raise RuntimeError("index and q must be on the same device")
    if bias is not None:
        if not isinstance(bias, torch.Tensor) or bias.get_device() != on or bias.dtype is not torch.float32:
            raise RuntimeError("bias must be a float32 tensor on the device of q")
        if bias.shape != (index.num_edges, heads):
            raise RuntimeError(f"bias must have shape [{index.num_edges}, {heads}], got {list(bias.shape)}")
        bias = bias.contiguous()
    scale = 1.0 / math.sqrt(dim) if scale is None else float(scale)
    if not -FLOAT_MAX <= scale <= FLOAT_MAX:
        raise RuntimeError(f"scale must be finite in single precision, got {scale}")
    # what the backward pass reads is kept where there can be one (needs_input_grad says yes under no_grad, too)
    keep = torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or (bias is not None and bias.requires_grad))
    return _NeighborAttention.apply(q, k, v, bias, index, scale, keep)


class _DistanceBias(torch.autograd.Function):
    @staticmethod
    def forward(ctx, dist, table, cutoff, smooth):
        dev, E, (buckets, heads) = dist.device, dist.size(0), table.shape
        with _lib.on_device(dev):
            bias = torch.empty((E, heads), dtype=torch.float32, device=dev)
            _lib.check(_lib.lib().dynb_distance_bias(dist.data_ptr(), E, table.data_ptr(), buckets, heads, cutoff, smooth, bias.data_ptr(),
                                                     _lib.stream_of(dev)), "distance_bias")
        ctx.save_for_backward(dist, table)
        ctx.cutoff, ctx.smooth = cutoff, smooth
        return bias

    @staticmethod
    @once_differentiable
    def backward(ctx, d_bias):
        dist, table = ctx.saved_tensors
        dev, E, (buckets, heads) = dist.device, dist.size(0), table.shape
        d_bias = d_bias.contiguous()
        L = _lib.lib()
        with _lib.on_device(dev):
            d_dist = torch.empty_like(dist) if ctx.needs_input_grad[0] else None
            d_table = ws = None
            if ctx.needs_input_grad[1]:
                d_table = torch.empty_like(table)
                nbytes = ctypes.c_int64()
                _lib.check(L.dynb_distance_bias_workspace_bytes(E, buckets, heads, ctypes.byref(nbytes)), "distance_bias_workspace_bytes")
                ws = torch.empty(nbytes.value, dtype=torch.uint8, device=dev)
            _lib.check(L.dynb_distance_bias_backward(dist.data_ptr(), E, table.data_ptr(), buckets, heads, ctx.cutoff, ctx.smooth, d_bias.data_ptr(),
                                                     _pointer(d_dist), _pointer(d_table), _pointer(ws), 0 if ws is None else ws.numel(),
                                                     _lib.stream_of(dev)), "distance_bias_backward")
        return d_dist, d_table, None, None


def distance_bias(dist: torch.Tensor, table: torch.Tensor, cutoff: float, smooth: bool = True) -> torch.Tensor:
    """A learned bias of attention logits, [E, heads] float32, from the distances ``dist`` [E] float32.

    ``table`` [buckets, heads] float32 holds ``buckets`` (4 to 1024) values a head over the distances [0, cutoff], joined by cubic B-splines: value and
    force are continuous in the distance.  With ``smooth`` the logarithm of the switch function ``(1 - u)^3 (1 + 3 u + 6 u^2)``,
    ``u = dist / cutoff``, is added, so that attention weights vanish smoothly at the cutoff.  Pairs at the cutoff and beyond (a list
    with a skin holds them) get -inf, that is, take no part, and zero gradients.  Distances are not negative.  The cutoff is
    rounded to single precision.  Gradients for ``dist`` and ``table``; sums over edges are joined in 64 bits."""
    if not isinstance(dist, torch.Tensor) or not dist.is_cuda:
        raise RuntimeError("dist must be a CUDA tensor")
    if dist.dim() != 1 or dist.dtype != torch.float32:
        raise RuntimeError(f"dist must be a 1-D float32 tensor, got {dist.dtype} {list(dist.shape)}")
    if not isinstance(table, torch.Tensor) or table.device != dist.device:
        raise RuntimeError("table must be on the device of dist")
    if table.dim() != 2 or table.dtype != torch.float32:
        raise RuntimeError(f"table must be a float32 tensor of shape [buckets, heads], got {table.dtype} {list(table.shape)}")
    if not 4 <= table.size(0) <= MAX_BUCKETS:
        raise RuntimeError(f"table must have 4 to {MAX_BUCKETS} buckets, got {table.size(0)}")
    if not 1 <= table.size(1) <= MAX_BIAS_HEADS:
        raise RuntimeError(f"table must have 1 to {MAX_BIAS_HEADS} heads, got {table.size(1)}")
    cutoff = float(cutoff)
    if not 0.0 < cutoff < 3.0e38 or ctypes.c_float(cutoff).value == 0.0:
        raise RuntimeError(f"cutoff must be positive and finite, got {cutoff}")
    return _DistanceBias.apply(dist.contiguous(), table.contiguous(), cutoff, int(bool(smooth)))


def type_index(types: torch.Tensor, num_types: int) -> TypeIndex:
    """Rows by type, for ``type_linear``: ``types`` [N] int64 in [0, num_types), num_types at most 4096.  Types change with a repartition, not
    from step to step: keep the index meanwhile.  Waits for the stream once; raises on a type out of range."""
    if not isinstance(types, torch.Tensor) or not types.is_cuda:
        raise RuntimeError("types must be a CUDA tensor")
    if types.dim() != 1 or types.dtype != torch.int64:
        raise RuntimeError(f"types must be a 1-D int64 tensor, got {types.dtype} {list(types.shape)}")
    T, N = int(num_types), types.size(0)
    if not 1 <= T <= MAX_TYPES:
        raise RuntimeError(f"num_types must lie in [1, {MAX_TYPES}], got {T}")
    if N >= INT32_MAX:
        raise RuntimeError(f"types must have fewer than 2^31 - 1 rows, got {N}")
    types = types.contiguous()
    dev = types.device
    L = _lib.lib()
    with _lib.on_device(dev):
        _not_capturing("type_index")
        order = torch.empty(N, dtype=torch.int32, device=dev)
        start = torch.empty(T + 1, dtype=torch.int32, device=dev)
        nbytes = ctypes.c_int64()
        _lib.check(L.dynb_type_index_workspace_bytes(N, ctypes.byref(nbytes)), "type_index_workspace_bytes")
        ws = torch.empty(nbytes.value, dtype=torch.uint8, device=dev)
        words = take_host_words(1)
        try:
            _lib.check(L.dynb_type_index(types.data_ptr(), N, T, order.data_ptr(), start.data_ptr(), words.data_ptr(), ws.data_ptr(), ws.numel(),
                                         _lib.stream_of(dev)), "type_index")
            torch.cuda.current_stream(dev).synchronize()
        except BaseException:
            lose_host_words(words, dev)
            raise
        bad = int(words[0])
        give_host_words(words)
        if bad:
            raise RuntimeError(f"type_index: a type lies outside [0, {T})")
    return TypeIndex(order, start)


_STATUS: dict = {}   # device -> (host word, device address): set by a kernel whose bounded wait ran out; kept as long as the process, graphs hold the address
_STATUS_LOCK = threading.Lock()


def _new_status_word():
    hp, dp = ctypes.c_void_p(), ctypes.c_void_p()
    _lib.check(_lib.lib().dynb_host_alloc_mapped(8, ctypes.byref(hp), ctypes.byref(dp)), "host_alloc_mapped")
    word = ctypes.c_uint32.from_address(hp.value)
    word.value = 0
    return word, dp.value


def _make_status_word(dev) -> None:
    """The device's status word, once, whichever thread comes first; none while the current stream is being captured, when memory cannot be had."""
    with _lib.on_device(dev):
        if torch.cuda.is_current_stream_capturing():
            return
        with _STATUS_LOCK:
            if dev.index not in _STATUS:
                _STATUS[dev.index] = _new_status_word()


def _status_word(dev) -> int:
    """Device address of the device's status word.  Raises when an earlier call's kernel gave up waiting."""
    found = _STATUS.get(dev.index)
    if found is None:
        _make_status_word(dev)
        found = _STATUS.get(dev.index)
        if found is None:
            raise RuntimeError("type_linear: the first index of a device must be made before a capture, so that a wait that runs out can be told")
    if found[0].value:
        found[0].value = 0
        raise RuntimeError("type_linear: a wait inside a kernel of an earlier call ran out; its results are not valid")
    return found[1]


def _linear_args(x, weight, index: TypeIndex) -> "_lib.TypeLinear":
    a = _lib.TypeLinear()
    a.status_dev = _status_word(x.device)
    a.weight_dev, a.order_dev, a.start_dev = weight.data_ptr(), index.order.data_ptr(), index.start.data_ptr()
    a.n_rows, a.types, a.inner, a.outer, a.dtype = x.size(0), weight.size(0), weight.size(1), weight.size(2), _DTYPES[x.dtype]
    return a


def _row_last(t: torch.Tensor) -> torch.Tensor:
    return t if t.stride(1) == 1 or t.size(1) == 1 else t.contiguous()


class _TypeLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, index):
        dev = x.device
        x, weight = _row_last(x), weight.contiguous()
        bias = None if bias is None else bias.contiguous()
        with _lib.on_device(dev):
            y = torch.empty((x.size(0), weight.size(2)), dtype=x.dtype, device=dev)
            args = _linear_args(x, weight, index)
            _lib.check(_lib.lib().dynb_type_linear(ctypes.byref(args), x.data_ptr(), x.stride(0), _pointer(bias), y.data_ptr(), _lib.stream_of(dev)),
                       "type_linear")
        ctx.save_for_backward(x, weight)
        ctx.index = index
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, d_y):
        x, weight = ctx.saved_tensors
        dev, d_y = x.device, _row_last(d_y)
        L = _lib.lib()
        with _lib.on_device(dev):
            args = _linear_args(x, weight, ctx.index)   # anew: hooks may have moved what was saved
            dx = torch.empty(x.shape, dtype=x.dtype, device=dev) if ctx.needs_input_grad[0] else None
            dw = torch.empty(weight.shape, dtype=x.dtype, device=dev) if ctx.needs_input_grad[1] else None
            db = torch.empty((weight.size(0), weight.size(2)), dtype=x.dtype, device=dev) if ctx.needs_input_grad[2] else None
            ws = None
            if dw is not None or db is not None:
                nbytes = ctypes.c_int64()
                _lib.check(L.dynb_type_linear_workspace_bytes(ctypes.byref(args), ctypes.byref(nbytes)), "type_linear_workspace_bytes")
                ws = torch.empty(nbytes.value, dtype=torch.uint8, device=dev)
            _lib.check(L.dynb_type_linear_backward(ctypes.byref(args), x.data_ptr(), x.stride(0), d_y.data_ptr(), d_y.stride(0), _pointer(dx), _pointer(dw),
                                                   _pointer(db), _pointer(ws), 0 if ws is None else ws.numel(), _lib.stream_of(dev)),
                       "type_linear_backward")
        return dx, dw, db, None


def type_linear(x: torch.Tensor, weight: torch.Tensor, index: TypeIndex, bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``y[i] = x[i] @ weight[type_i] (+ bias[type_i])``: x [N, inner], weight [types, inner, outer], bias [types, outer]; float32, float16 or bfloat16, all
    alike; widths at most 16384.  The rows of x may have any stride.  Products are summed in 32 bits and rounded once; gradients for x, weight and bias.

    y and its gradient for x run on the tensor cores while the summed dimension fits into shared memory: y up to 256 columns of x in float32 and 1344 in
    16 bits, the gradient up to 1088 and 5376 columns of y.  Wider ones take several times as long.
    float32 operands go to the tensor cores as three parts of 8 bits, which hold them whole (numbers below 2^-109 to within 2^-133); infinities and NaN give what IEEE arithmetic gives."""
    if not isinstance(index, TypeIndex):
        raise RuntimeError("index must be a TypeIndex (see type_index)")
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        raise RuntimeError("x must be a CUDA tensor")
    if x.dim() != 2 or x.dtype not in _DTYPES:
        raise RuntimeError(f"x must be a float32, float16 or bfloat16 tensor of shape [N, inner], got {x.dtype} {list(x.shape)}")
    if not isinstance(weight, torch.Tensor) or weight.device != x.device or weight.dtype != x.dtype:
        raise RuntimeError("weight must be on the device and of the type of x")
    if weight.dim() != 3 or weight.size(0) != index.num_types or weight.size(1) != x.size(1):
        raise RuntimeError(f"weight must have shape [{index.num_types}, {x.size(1)}, outer], got {list(weight.shape)}")
    if not (1 <= weight.size(1) <= MAX_WIDTH and 1 <= weight.size(2) <= MAX_WIDTH):
        raise RuntimeError(f"the widths of weight must lie in [1, {MAX_WIDTH}], got {weight.size(1)} and {weight.size(2)}")
    if index.order.numel() != x.size(0):
        raise RuntimeError(f"the index is of {index.order.numel()} rows, got {x.size(0)}")
    if index.order.device != x.device:
        raise RuntimeError("index and x must be on the same device")
    if bias is not None:
        if not isinstance(bias, torch.Tensor) or bias.device != x.device or bias.dtype != x.dtype:
            raise RuntimeError("bias must be on the device and of the type of x")
        if bias.shape != (weight.size(0), weight.size(2)):
            raise RuntimeError(f"bias must have shape [{weight.size(0)}, {weight.size(2)}], got {list(bias.shape)}")
    return _TypeLinear.apply(x, weight, bias, index)

"""Rows that choose their matrices: routing to experts, the experts' products and their weighted sums, with gradients.

``type_linear`` (message.py) gives a row the matrix of its atom type.  Here a row's logits choose:

* ``route_experts(logits, choices)``: experts and weights of every row, and the (row, choice) pairs by expert;
* ``expert_linear(x, weight, routing, bias, activation)``: the pairs' products with the matrices of their experts;
* ``expert_combine(z, routing, residual)``: every row's weighted sum.

A layer is ``expert_combine(expert_linear(expert_linear(x, w1, r, b1, "silu"), w2, r, b2), r, x)`` with ``r = route_experts(x @ gate, 2)``.

No counterpart in the reference: its model adapters leave this to their libraries (dynamis_model/src/dynamis_model/nnp/uma.py).

All work is enqueued on the current stream of the tensors' device; nothing waits for the host, and the calls can be captured into a graph.  Gradients are
formed without atomics on floating-point numbers: the same inputs give the same bits.  They can be taken once; a gradient of a gradient raises, and so does a tangent of forward mode.
"""

from __future__ import annotations

import ctypes
from dataclasses import dataclass
from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .message import _DTYPES, INT32_MAX, MAX_WIDTH, _STATUS, _differentiates, _each_once, _lists, _lists_refused, _make_status_word, _pointer, _row_last, _runs, _status_word

MAX_EXPERTS = 1024   # DYNB_ROUTING_MAX_EXPERTS
MAX_CHOICES = 32     # DYNB_ROUTING_MAX_CHOICES
_SCORES = {"softmax": 0, "sigmoid": 1}                  # DYNB_SCORE_*
_ACTIVATIONS = {None: 0, "silu": 1, "gelu": 2}          # DYNB_ACTIVATION_*


@dataclass(frozen=True)
class Routing:
    """Experts of rows.

    experts [rows, choices] int32   the experts of a row, -1 where a place has none
    weights [rows, choices] float32 their weights, 0 where a place has no expert; differentiable
    order [rows * choices] int32    the pairs ``row * choices + choice`` of expert 0, of expert 1, ..., ascending inside one, those without an expert behind
    start [experts + 1] int32       where every expert's pairs begin, and where those without an expert do

    ``route_experts`` makes it.  Lists made by hand have to be as described: entries out of range are passed over, but results of pairs that are left out or named
    twice are not defined (memory may show that was not written).  ``check_lists`` looks."""

    experts: torch.Tensor
    weights: torch.Tensor
    order: torch.Tensor
    start: torch.Tensor

    def __post_init__(self):
        e, w = self.experts, self.weights
        if not (isinstance(e, torch.Tensor) and e.is_cuda) or e.dtype is not torch.int32 or e.dim() != 2 or not e.is_contiguous():
            raise RuntimeError("Routing: experts must be a contiguous CUDA tensor of shape [rows, choices], int32")
        if not 1 <= e.size(1) <= MAX_CHOICES:
            raise RuntimeError(f"Routing: the choices must lie in [1, {MAX_CHOICES}], got {e.size(1)}")
        if not isinstance(w, torch.Tensor) or w.dtype is not torch.float32 or w.get_device() != e.get_device() or w.shape != e.shape:
            raise RuntimeError(f"Routing: weights must be a float32 tensor of shape {list(e.shape)} on the device of experts")
        _lists("Routing", ("order", "start"), (self.order, self.start))
        if self.order.get_device() != e.get_device():
            raise RuntimeError("Routing: all lists must be on the same device")
        if self.order.numel() != e.numel() or e.numel() >= INT32_MAX:
            raise RuntimeError(f"Routing: order must have one entry per pair (and fewer than 2^31 - 1), got {self.order.numel()} for {e.numel()}")
        if not 2 <= self.start.numel() <= MAX_EXPERTS + 1:
            raise RuntimeError(f"Routing: the number of experts must lie in [1, {MAX_EXPERTS}], got {self.start.numel() - 1}")
        if e.get_device() not in _STATUS:
            _make_status_word(e.device)

    def check_lists(self) -> None:
        """Waits and raises if the lists do not belong to one another: for a routing that ``route_experts`` did not make."""
        E, P = self.num_experts, self.order.numel()

        def by_expert():
            bounds = torch.cat([self.start.long(), self.start.new_tensor([P]).long()])
            want = torch.repeat_interleave(torch.arange(E + 1, device=bounds.device), bounds[1:] - bounds[:-1])
            of = self.experts.reshape(-1)[self.order.long()].long()
            return torch.equal(torch.where(of < 0, E, of), want)

        _lists_refused("Routing", (
            ("order must name every pair once", lambda: _each_once(self.order)),
            (f"start must rise from 0 to at most {P}", lambda: _runs(self.start, int(self.start[-1])) and int(self.start[-1]) <= P),
            (f"experts must lie in [-1, {E})", lambda: bool(((self.experts >= -1) & (self.experts < E)).all())),
            ("order must list the pairs by their experts", by_expert)))

    def check_status(self) -> None:
        """Synchronises and raises if a wait inside a kernel of an ``expert_linear`` (or ``type_linear``) on this device ran out, whose results are not valid
        then.  ``expert_linear`` looks, without waiting, before it launches; behind the last call, or where a graph replays the calls, look here."""
        dev = self.order.device
        torch.cuda.synchronize(dev)
        with _lib.on_device(dev):
            _status_word(dev)

    @property
    def num_rows(self) -> int:
        return self.experts.size(0)

    @property
    def choices(self) -> int:
        return self.experts.size(1)

    @property
    def num_experts(self) -> int:
        return self.start.numel() - 1


class _RouteExperts(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, bias, choices, score, groups, kept_groups, renormalize, scale):   # ctx None: without gradients nothing is kept for them
        dev, (rows, experts) = logits.device, logits.shape
        logits = _row_last(logits)
        L = _lib.lib()
        fixed = (bias, choices, score, groups, kept_groups, renormalize, scale)
        with _lib.on_device(dev):
            chosen = torch.empty((rows, choices), dtype=torch.int32, device=dev)
            weights = torch.empty((rows, choices), dtype=torch.float32, device=dev)
            order = torch.empty(rows * choices, dtype=torch.int32, device=dev)
            start = torch.empty(experts + 1, dtype=torch.int32, device=dev)
            args = _routing_args(logits, *fixed)
            nbytes = ctypes.c_int64()
            _lib.check(L.dynb_route_experts_workspace_bytes(ctypes.byref(args), ctypes.byref(nbytes)), "route_experts_workspace_bytes")
            ws = torch.empty(nbytes.value, dtype=torch.uint8, device=dev)
            _lib.check(L.dynb_route_experts(ctypes.byref(args), chosen.data_ptr(), weights.data_ptr(), order.data_ptr(), start.data_ptr(), ws.data_ptr(),
                                            ws.numel(), _lib.stream_of(dev)), "route_experts")
        if ctx is not None:
            ctx.mark_non_differentiable(chosen, order, start)
            ctx.set_materialize_grads(False)
            ctx.save_for_backward(logits, chosen, weights)
            ctx.fixed = fixed
        return chosen, weights, order, start

    @staticmethod
    @once_differentiable
    def backward(ctx, _, d_weights, *__):
        if d_weights is None:
            return (None,) * 8
        logits, chosen, weights = ctx.saved_tensors
        dev = logits.device
        d_weights = d_weights.contiguous()
        with _lib.on_device(dev):
            d_logits = torch.empty(logits.shape, dtype=logits.dtype, device=dev)
            args = _routing_args(logits, *ctx.fixed)
            _lib.check(_lib.lib().dynb_route_experts_backward(ctypes.byref(args), chosen.data_ptr(), weights.data_ptr(), d_weights.data_ptr(),
                                                              d_logits.data_ptr(), _lib.stream_of(dev)), "route_experts_backward")
        return d_logits, None, None, None, None, None, None, None


def _routing_args(logits, bias, choices, score, groups, kept_groups, renormalize, scale) -> "_lib.RoutingArgs":
    a = _lib.RoutingArgs()
    a.logits_dev, a.logits_row, a.bias_dev = logits.data_ptr(), logits.stride(0), _pointer(bias)
    a.n_rows, a.experts, a.choices, a.dtype = logits.size(0), logits.size(1), choices, _DTYPES[logits.dtype]
    a.score, a.groups, a.kept_groups, a.renormalize, a.scale = score, groups, kept_groups, renormalize, scale
    return a


def route_experts(logits: torch.Tensor, choices: int, score: str = "softmax", bias: Optional[torch.Tensor] = None, groups: int = 1, kept_groups: int = 1,
                  renormalize: bool = True, scale: float = 1.0) -> Routing:
    """Experts of rows from their logits [rows, experts] (float32, float16 or bfloat16; at most 1024 experts).

    Scores ``s`` are the softmax of a row's logits or their sigmoids (``score``).  Keys are ``s + bias`` (bias [experts] float32, for balance; it chooses, but does not
    weigh and has no gradient).  With ``groups`` the experts form that many groups of neighbours; the ``kept_groups`` groups whose two largest keys have the largest sums
    stay.  Of their experts the ``choices`` (at most 32) largest keys are chosen, in falling order, the lowest number first among equal ones.  Weights are ``scale * s``,
    with ``renormalize`` ``scale * s`` over the sum of the chosen ones.

    A logit or a bias of -inf closes an expert; places that no expert is left for have number -1 and weight 0.  A NaN comes before all numbers.  Keys are compared in
    64 bits; without bias and groups the logits are.  The gradient of the weights goes to the logits.  The choice has none: an energy whose logits depend on
    positions has a step where a row's choice changes."""
    if not isinstance(logits, torch.Tensor) or not logits.is_cuda:
        raise RuntimeError("logits must be a CUDA tensor")
    if logits.dim() != 2 or logits.dtype not in _DTYPES:
        raise RuntimeError(f"logits must be a float32, float16 or bfloat16 tensor of shape [rows, experts], got {logits.dtype} {list(logits.shape)}")
    rows, experts = logits.shape
    choices, groups, kept_groups, scale = int(choices), int(groups), int(kept_groups), float(scale)
    if not 1 <= experts <= MAX_EXPERTS:
        raise RuntimeError(f"the number of experts must lie in [1, {MAX_EXPERTS}], got {experts}")
    if not 1 <= choices <= min(MAX_CHOICES, experts):
        raise RuntimeError(f"choices must lie in [1, {min(MAX_CHOICES, experts)}], got {choices}")
    if rows * choices >= INT32_MAX:
        raise RuntimeError(f"rows times choices must be below 2^31 - 1, got {rows} times {choices}")
    if score not in _SCORES:
        raise RuntimeError(f"score must be 'softmax' or 'sigmoid', got {score!r}")
    if groups < 1 or experts % groups != 0 or not 1 <= kept_groups <= groups:
        raise RuntimeError(f"groups must divide the {experts} experts and kept_groups lie in [1, groups], got {groups} and {kept_groups}")
    if bias is not None:
        if not isinstance(bias, torch.Tensor) or bias.device != logits.device or bias.dtype is not torch.float32 or bias.shape != (experts,):
            raise RuntimeError(f"bias must be a float32 tensor of shape [{experts}] on the device of logits")
        if bias.requires_grad and torch.is_grad_enabled():
            raise RuntimeError("bias has no gradient: pass it detached")
        bias = bias.contiguous()
    if not 1e-30 <= scale <= 1e30:
        raise RuntimeError(f"scale must lie in [1e-30, 1e30], got {scale}")
    args = (logits, bias, choices, _SCORES[score], groups, kept_groups, int(bool(renormalize)), scale)
    if _differentiates(logits):
        return Routing(*_RouteExperts.apply(*args))
    return Routing(*_RouteExperts.forward(None, *args))     # a third of a small call's time is autograd's


def _linear_args(weight, routing: Routing, paired: bool, activation: int, dtype) -> "_lib.ExpertLinear":
    a = _lib.ExpertLinear()
    a.status_dev = _status_word(weight.device)
    a.weight_dev, a.order_dev, a.start_dev = weight.data_ptr(), routing.order.data_ptr(), routing.start.data_ptr()
    a.n_rows, a.choices, a.experts, a.inner, a.outer = routing.num_rows, routing.choices, weight.size(0), weight.size(1), weight.size(2)
    a.dtype, a.paired, a.activation = _DTYPES[dtype], int(paired), activation
    return a


def _unaligned(t: torch.Tensor) -> bool:
    """Whether rows of ``t`` start off 16-byte boundaries (they are copied then)."""
    return t.data_ptr() % 16 != 0 or t.stride(0) * t.element_size() % 16 != 0


def _linear_workspace(args, backward: int, want_x: int, want_weights: int, dev) -> torch.Tensor:
    nbytes = ctypes.c_int64()
    _lib.check(_lib.lib().dynb_expert_linear_workspace_bytes(ctypes.byref(args), backward, want_x, want_weights, ctypes.byref(nbytes)), "expert_linear_workspace_bytes")
    return torch.empty(nbytes.value, dtype=torch.uint8, device=dev)


def _pairs(t: torch.Tensor) -> torch.Tensor:
    """[rows, choices, width] as [pairs, width] with one stride from pair to pair and consecutive elements."""
    rows, choices, width = t.shape
    if t.stride(2) == 1 or width == 1:
        if choices == 1:
            return t[:, 0]
        if rows == 1:
            return t[0]
        if t.stride(0) == choices * t.stride(1):
            return t.as_strided((rows * choices, width), (t.stride(1), t.stride(2)))
    return t.reshape(-1, t.size(2)).contiguous()


class _ExpertLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, routing, activation):   # ctx None: without gradients nothing is kept for them
        dev, paired = x.device, x.dim() == 3
        flat, weight = _pairs(x) if paired else _row_last(x), weight.contiguous()
        bias = None if bias is None else bias.contiguous()
        with _lib.on_device(dev):
            z = torch.empty((routing.num_rows, routing.choices, weight.size(2)), dtype=x.dtype, device=dev)
            slope = None
            if ctx is not None and activation:
                slope = torch.empty((*z.shape[:2], -(-z.size(2) // 8) * 8), dtype=torch.float32 if x.dtype == torch.float32 else torch.int16, device=dev)
            args = _linear_args(weight, routing, paired, activation, x.dtype)
            args.unaligned = int(_unaligned(flat))
            ws = _linear_workspace(args, 0, 0, 0, dev)
            _lib.check(_lib.lib().dynb_expert_linear(ctypes.byref(args), flat.data_ptr(), flat.stride(0), _pointer(bias), z.data_ptr(), _pointer(slope),
                                                     ws.data_ptr(), ws.numel(), _lib.stream_of(dev)), "expert_linear")
        if ctx is not None:
            ctx.save_for_backward(flat, weight, slope)
            ctx.routing, ctx.activation, ctx.shape = routing, activation, x.shape
        return z

    @staticmethod
    @once_differentiable
    def backward(ctx, d_z):
        x, weight, slope = ctx.saved_tensors
        dev, d_z, routing, paired = x.device, _pairs(d_z), ctx.routing, len(ctx.shape) == 3
        want_x, want_w, want_b = ctx.needs_input_grad[:3]
        with _lib.on_device(dev):
            args = _linear_args(weight, routing, paired, ctx.activation, x.dtype)   # anew: hooks may have moved what was saved
            dx = torch.empty(ctx.shape, dtype=x.dtype, device=dev) if want_x else None
            dw = torch.empty(weight.shape, dtype=x.dtype, device=dev) if want_w else None
            db = torch.empty((weight.size(0), weight.size(2)), dtype=x.dtype, device=dev) if want_b else None
            args.unaligned = int(_unaligned(x)) + 2 * int(_unaligned(d_z) or (slope is not None and slope.data_ptr() % 16 != 0))
            ws = _linear_workspace(args, 1, int(want_x), int(want_w or want_b), dev)
            _lib.check(_lib.lib().dynb_expert_linear_backward(ctypes.byref(args), x.data_ptr(), x.stride(0), d_z.data_ptr(), d_z.stride(0), _pointer(slope),
                                                     routing.experts.data_ptr(), _pointer(dx), _pointer(dw), _pointer(db), ws.data_ptr(), ws.numel(),
                                                     _lib.stream_of(dev)), "expert_linear_backward")
        return dx, dw, db, None, None


def expert_linear(x: torch.Tensor, weight: torch.Tensor, routing: Routing, bias: Optional[torch.Tensor] = None, activation: Optional[str] = None) -> torch.Tensor:
    """``z[i, j] = act(x[i] @ weight[e] (+ bias[e]))`` with ``e = routing.experts[i, j]``: x [rows, inner], or [rows, choices, inner] (``x[i, j]`` then), weight
    [experts, inner, outer], bias [experts, outer]; float32, float16 or bfloat16, all alike; widths at most 16384.  z [rows, choices, outer]; places without an
    expert give zeros and get zero gradients.  activation: None, "silu" or "gelu" (with the normal distribution function).

    Products are summed in 32 bits and rounded once behind the activation; gradients for x, weight and bias.  For 16-bit types the backward pass takes the
    activation's slope in 16 bits (to within 2^-15, below 1/8 within 2^-11 of itself or 2^-25), and the gradient in front of the activation is rounded to the
    type before it is multiplied and summed.  float32 operands go to the tensor cores as three parts of 8 bits, which hold them whole.  Slopes (of the size of z) are
    kept for the backward pass, which holds the gradient in front of the activation beside them and, for x of rows, that of x by pairs in 32 bits."""
    if not isinstance(routing, Routing):
        raise RuntimeError("routing must be a Routing (see route_experts)")
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        raise RuntimeError("x must be a CUDA tensor")
    if x.dim() not in (2, 3) or x.dtype not in _DTYPES:
        raise RuntimeError(f"x must be a float32, float16 or bfloat16 tensor of shape [rows, inner] or [rows, choices, inner], got {x.dtype} {list(x.shape)}")
    if x.shape[:-1] != (routing.num_rows, routing.choices)[:x.dim() - 1]:
        raise RuntimeError(f"the routing is of {routing.num_rows} rows with {routing.choices} choices, got {list(x.shape)}")
    if not isinstance(weight, torch.Tensor) or weight.device != x.device or weight.dtype != x.dtype:
        raise RuntimeError("weight must be on the device and of the type of x")
    if weight.dim() != 3 or weight.size(0) != routing.num_experts or weight.size(1) != x.size(-1):
        raise RuntimeError(f"weight must have shape [{routing.num_experts}, {x.size(-1)}, outer], got {list(weight.shape)}")
    if not (1 <= weight.size(1) <= MAX_WIDTH and 1 <= weight.size(2) <= MAX_WIDTH):
        raise RuntimeError(f"the widths of weight must lie in [1, {MAX_WIDTH}], got {weight.size(1)} and {weight.size(2)}")
    if routing.order.device != x.device:
        raise RuntimeError("routing and x must be on the same device")
    if bias is not None:
        if not isinstance(bias, torch.Tensor) or bias.device != x.device or bias.dtype != x.dtype:
            raise RuntimeError("bias must be on the device and of the type of x")
        if bias.shape != (weight.size(0), weight.size(2)):
            raise RuntimeError(f"bias must have shape [{weight.size(0)}, {weight.size(2)}], got {list(bias.shape)}")
    if activation not in _ACTIVATIONS:
        raise RuntimeError(f"activation must be None, 'silu' or 'gelu', got {activation!r}")
    args = (x, weight, bias, routing, _ACTIVATIONS[activation])
    if _differentiates(x, weight, bias):
        return _ExpertLinear.apply(*args)
    return _ExpertLinear.forward(None, *args)


class _ExpertCombine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, z, weights, residual, experts):   # ctx None: without gradients nothing is kept for them
        dev, (rows, choices, width) = z.device, z.shape
        z, weights = z.contiguous(), weights.contiguous()
        if residual is not None:
            residual = _row_last(residual)
        with _lib.on_device(dev):
            y = torch.empty((rows, width), dtype=z.dtype, device=dev)
            _lib.check(_lib.lib().dynb_expert_combine(z.data_ptr(), weights.data_ptr(), experts.data_ptr(), _pointer(residual),
                                                      0 if residual is None else residual.stride(0), rows, choices, width, _DTYPES[z.dtype], y.data_ptr(),
                                                      _lib.stream_of(dev)), "expert_combine")
        if ctx is not None:
            ctx.save_for_backward(z, weights, experts)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, d_y):
        z, weights, experts = ctx.saved_tensors
        dev, (rows, choices, width) = z.device, z.shape
        want_z, want_w, want_r = ctx.needs_input_grad[:3]
        dz = dw = None
        if want_z or want_w:
            rows_of = _row_last(d_y)
            with _lib.on_device(dev):
                dz = torch.empty(z.shape, dtype=z.dtype, device=dev) if want_z else None
                dw = torch.empty(weights.shape, dtype=torch.float32, device=dev) if want_w else None
                _lib.check(_lib.lib().dynb_expert_combine_backward(z.data_ptr(), weights.data_ptr(), experts.data_ptr(), rows_of.data_ptr(), rows_of.stride(0),
                                                                   rows, choices, width, _DTYPES[z.dtype], _pointer(dz), _pointer(dw), _lib.stream_of(dev)),
                           "expert_combine_backward")
        return dz, dw, d_y if want_r else None, None


def expert_combine(z: torch.Tensor, routing: Routing, residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``y[i] = residual[i] + sum_j routing.weights[i, j] * z[i, j]`` over the places with an expert: z [rows, choices, width], residual [rows, width];
    float32, float16 or bfloat16, both alike; widths at most 16384.  What z holds where a place has no expert is not used.  Summed in 32 bits and rounded
    once; gradients for z, the routing's weights and the residual."""
    if not isinstance(routing, Routing):
        raise RuntimeError("routing must be a Routing (see route_experts)")
    if not isinstance(z, torch.Tensor) or not z.is_cuda:
        raise RuntimeError("z must be a CUDA tensor")
    if z.dim() != 3 or z.dtype not in _DTYPES:
        raise RuntimeError(f"z must be a float32, float16 or bfloat16 tensor of shape [rows, choices, width], got {z.dtype} {list(z.shape)}")
    if z.shape[:2] != routing.experts.shape:
        raise RuntimeError(f"the routing is of {routing.num_rows} rows with {routing.choices} choices, got {list(z.shape)}")
    if not 1 <= z.size(2) <= MAX_WIDTH:
        raise RuntimeError(f"the width must lie in [1, {MAX_WIDTH}], got {z.size(2)}")
    if routing.experts.device != z.device:
        raise RuntimeError("routing and z must be on the same device")
    if residual is not None:
        if not isinstance(residual, torch.Tensor) or residual.device != z.device or residual.dtype != z.dtype:
            raise RuntimeError("residual must be on the device and of the type of z")
        if residual.shape != (z.size(0), z.size(2)):
            raise RuntimeError(f"residual must have shape [{z.size(0)}, {z.size(2)}], got {list(residual.shape)}")
    args = (z, routing.weights, residual, routing.experts)
    if _differentiates(z, routing.weights, residual):
        return _ExpertCombine.apply(*args)
    return _ExpertCombine.forward(None, *args)

"""Expert layers and rotary heads on the GPU: calls and values at the limits of what they are for.  The bounds are derived beside the plain forms
(tests/_experts.py) and here."""

import ctypes
import math
import threading

import pytest
import torch
from torch.autograd import forward_ad

import dynamis_b200 as D
from dynamis_b200 import _lib
from tests import _experts as X
from tests import _message as M

pytestmark = pytest.mark.gpu
U = M.U


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(gen, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=gen, device="cuda").to(dtype)


def _routing(rows, experts, choices, absent=0.0, seed=1):
    return D.Routing(*X.routing_by_hand(rows, experts, choices, absent, seed, "cuda"))


# ------------------------------------------------------------------------------------------------ forward-mode derivatives
def test_forward_mode_derivatives_are_refused(cuda):
    """There is no formula for them: a tangent raises, also without gradients, and a level that is open changes nothing else."""
    gen = _gen(1)
    q, k, pos, wave = _normal(gen, 20, 2, 8), _normal(gen, 20, 2, 8), _normal(gen, 20, 3), _normal(gen, 4, 3)
    qw, kw = _normal(gen, 8), _normal(gen, 8)
    logits, balance = _normal(gen, 20, 5), _normal(gen, 5)
    routing = _routing(20, 5, 2)
    x, w, b = _normal(gen, 20, 8), _normal(gen, 5, 8, 8), _normal(gen, 5, 8)
    z, r = _normal(gen, 20, 2, 8), _normal(gen, 20, 8)
    by_weights = lambda z, weights, r: D.expert_combine(z, D.Routing(routing.experts, weights, routing.order, routing.start), r)  # noqa: E731
    calls = [(lambda *t: D.rotary_heads(*t)[0], (q, k, pos, wave, qw, kw)), (lambda t, c: D.route_experts(t, 2, bias=c).weights, (logits, balance)),
             (lambda x, w, b: D.expert_linear(x, w, routing, b, "silu"), (x, w, b)), (by_weights, (z, routing.weights, r))]
    for call, args in calls:
        want = call(*args)
        with forward_ad.dual_level():
            assert torch.equal(call(*args), want)
            for i, t in enumerate(args):
                for grad in (True, False):
                    with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="jvp"):
                        call(*args[:i], forward_ad.make_dual(t, torch.ones_like(t)), *args[i + 1:])
            assert torch.equal(call(*args), want)


# ------------------------------------------------------------------------------------------------ routing
def _sigmoid_gradient(logits, experts, g, renormalize, scale):
    """(value, bound) of the gradient of sigmoid weights.  1 - s = 1 / (1 + e^l) as a whole: exponential 4 u, addition and division 2 u, relative, whatever is
    left of it; products and the other factor (weights as in X.route) beside it.  1 - s below 2^-126 may be flushed before it meets g (e^l overflows from
    l = 88.7 on, where 1 - s is 2.9e-39): off by 2^-126 |g|, in p (g - sum p g) by twice the largest |g|; and the product by 2^-126."""
    l64, at = logits.detach().double(), experts.long()
    chosen, g = l64.gather(1, at), g.double() * scale
    s, rest = torch.sigmoid(chosen), torch.sigmoid(-chosen)
    if renormalize:
        logs = torch.nn.functional.logsigmoid(chosen)
        p = torch.softmax(logs, 1)
        r = (8 * logs.abs().max(1, keepdim=True).values + at.size(1) + 28) * U
        dot, off_dot = (p * g).sum(1, keepdim=True), (p * g.abs() * (r + (at.size(1) + 8) * U)).sum(1, keepdim=True)
        d = p * (g - dot) * rest
        off = p * (r * (g - dot).abs() + off_dot + 4 * U * (g.abs() + dot.abs())) * rest + 10 * U * d.abs() + 2.0 ** -125 * g.abs().max(1, keepdim=True).values
    else:
        d = g * s * rest
        off = 24 * U * d.abs() + 2.0 ** -126 * g.abs()
    put = lambda t: torch.zeros_like(l64).scatter_(1, at, t)  # noqa: E731
    return put(d), put(off) + 2.0 ** -126


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("experts,choices", [(16, 4), (200, 4), (64, 12)])
def test_route_gradients_of_open_gates(cuda, dtype, renormalize, experts, choices):
    """Sigmoids next to 1: what they leave of 1 keeps its digits, whichever kernel takes the rows."""
    gen = _gen(experts)
    logits = (10 + 20 * torch.rand(300, experts, generator=gen, device="cuda")).to(M.TYPES[dtype])
    logits[:20] += 60.0
    g = _normal(gen, 300, choices)
    leaf = logits.detach().requires_grad_()
    r = D.route_experts(leaf, choices, score="sigmoid", renormalize=renormalize, scale=1.5)
    got, = torch.autograd.grad(r.weights, [leaf], g)
    M.check(got, *_sigmoid_gradient(logits, r.experts, g, renormalize, 1.5), "d_logits")


@pytest.mark.parametrize("spread", [4.0, 8.0])
@pytest.mark.parametrize("experts,choices,groups,kept", [(64, 6, 8, 4), (128, 8, 1, 1), (32, 4, 4, 2)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route_of_peaked_logits(cuda, spread, experts, choices, groups, kept, score):
    """Scores far below the largest decide: many rows are looked at again in 64 bits, and all choices are those of 64 bits."""
    gen = _gen(experts + int(spread))
    logits = _normal(gen, 700, experts) * spread
    for bias in (None, 0.1 * _normal(gen, experts)):
        how = dict(score=score, groups=groups, kept_groups=kept, bias=bias)
        r, ref = D.route_experts(logits, choices, **how), X.route(logits, choices, **how)
        for name in ("experts", "order", "start"):
            assert torch.equal(getattr(r, name).cpu(), ref[name]), name
        M.check(r.weights.cpu(), *ref["weights"], "weights")


# ------------------------------------------------------------------------------------------------ products
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("activation", ["silu", "gelu"])
@pytest.mark.parametrize("wide", [16, 17])
def test_linear_small_slopes_keep_their_digits(cuda, dtype, activation, wide):
    """Far on the negative side slopes are small, and so are the gradients, but for their own digits: d_x = d_z act'(x) through a matrix of ones on the diagonal.
      slope in 32 bits: SiLU p (1 + u (1 - p)): exponential (2 + |u|) 2 u, addition and reciprocal 4 u, relative to p, twice in the product;
        GELU: 7.1.26 of Abramowitz and Stegun, 7.5e-8 in all and below -3 at most 2e-4 of the slope (evaluated down to -10)
      in memory: 2^-15 from 1/8 on, below 2^-11 of itself, or 2^-25 where that is more, on a scale of 31/32."""
    dtype = M.TYPES[dtype]
    x = torch.linspace(-16, 4, 40 * wide, device=cuda).to(dtype).view(40, wide)
    g = _normal(_gen(wide), 40, 1, wide, dtype=dtype)
    w = torch.eye(wide, device=cuda, dtype=dtype)[None]
    leaf = x.detach().requires_grad_()
    z = D.expert_linear(leaf, w, _routing(40, 1, 1), None, activation)
    got, = torch.autograd.grad(z, [leaf], g)
    u, gd = x.double(), g[:, 0].double()
    if activation == "silu":
        p = torch.sigmoid(u)
        slope, off = p * (1 + u * (1 - p)), p * (1 + u.abs()) * (20 + 4 * u.abs()) * U
    else:
        slope = 0.5 * torch.erfc(-u * math.sqrt(0.5)) + u * torch.exp(-0.5 * u * u) / math.sqrt(2 * math.pi)
        off = torch.where(u < -3, 3e-4 * slope.abs(), 1e-7 + 16 * U * (1 + u.abs()))
    off = off + torch.where(slope.abs() < 0.125, torch.maximum((2.0 ** -11 + 4 * U) * slope.abs(), torch.full_like(u, 1.04 * 2.0 ** -25)), 2.0 ** -15)
    M.check(got, slope * gd, gd.abs() * off + 2 * U * (slope * gd).abs(), "d_x")


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,experts,inner,outer,paired", [(50_000, 300, 64, 64, False), (17_000, 7, 1032, 520, True), (24_000, 90, 512, 128, False)])
def test_linear_walks_of_many_tiles(cuda, dtype, rows, experts, inner, outer, paired):
    """Blocks that take five tiles of rows and more, with changes of the expert among them, matrices that stay and that come with every stage."""
    gen, dtype = _gen(rows), M.TYPES[dtype]
    routing = _routing(rows, experts, 2, 0.02, inner)
    x, g = _normal(gen, *((rows, 2) if paired else (rows,)), inner, dtype=dtype), _normal(gen, rows, 2, outer, dtype=dtype)
    w, b = (_normal(gen, experts, inner, outer) * inner ** -0.5).to(dtype), _normal(gen, experts, outer, dtype=dtype)
    leaves = [t.detach().requires_grad_() for t in (x, w, b)]
    z = D.expert_linear(*leaves[:2], routing, leaves[2], "silu")
    grads = torch.autograd.grad(z, leaves, g)
    ref = X.linear(x, w, routing.experts, b, "silu", g)
    for name, got in zip(("z", "d_x", "d_weight", "d_bias"), (z, *grads)):
        M.check(got, *ref[name], name)
    routing.check_status()


@pytest.mark.parametrize("dtype,rows,steps", [("f32", 6000, 64), ("f16", 30_000, 470), ("bf16", 30_000, 470)])
def test_linear_cuts_a_sum_off_once_a_step(cuda, dtype, rows, steps):
    """Operands of one sign: the tensor cores cut a sum off towards zero at every step of 16 products, by half of its last place on average, at most 2^-23 of it.
    Partial sums grow evenly, so over n steps this costs at most (n + 1) / 4 * 2^-23 =: c of the whole on average.  n for the matrices' gradient: the pairs of
    a sum over 16, which are 1024 of 3000 in fp32 and a slice of 7500 in 16 bits (148 SMs, tiles of 128 x 128 and 128 x 256 of 1024 x 1024 elements); for rows
    64.  Parts of fp32 numbers have 8 bits, and their products end above the last place of sums as short as these.  Products of 16-bit numbers reach below it, and
    each of the 17 terms of a step may be cut off there: 17 c at most; and results in 16 bits are not to show it: an eighth of a step of the type.
    Beside it 2^-24.  The mean of the roundings to the type does not vanish where the values lie about a power of two (the step doubles there: exact sums of
    this kind, rounded to bfloat16, come out 2.8e-5 too small on average), so the exact sums are rounded, too.  Both roundings differ in a share c / eps of the
    elements, by a step: the mean over 2^20 of them or more is off by sqrt(c eps / 2^20), taken five times."""
    dtype = M.TYPES[dtype]
    gen, wide = _gen(rows), 1024
    experts = torch.zeros(rows, 1, dtype=torch.int32, device=cuda)
    routing = D.Routing(experts, torch.ones(rows, 1, device=cuda), torch.arange(rows, dtype=torch.int32, device=cuda), torch.tensor([0, rows], dtype=torch.int32, device=cuda))
    x, w, g = (torch.rand(*s, generator=gen, device="cuda").to(dtype) for s in ((rows, wide), (1, wide, wide), (rows, 1, wide)))
    leaves = [t.detach().requires_grad_() for t in (x, w)]
    z = D.expert_linear(*leaves, routing)
    dx, dw = torch.autograd.grad(z, leaves, g)
    xd, wd, gd = x.double(), w[0].double(), g[:, 0].double()
    for name, got, ref, n in (("z", z.detach()[:, 0], xd @ wd, 64), ("d_x", dx, gd @ wd.T, 64), ("d_weight", dw[0], xd.T @ gd, steps)):
        lost, most = float(((ref.to(dtype).double() - got.double()) / ref).mean()), (n + 1) / 4 * 2.0 ** -23
        if dtype != torch.float32:
            most = min(17 * most, torch.finfo(dtype).eps / 8)
        noise = 2.0 ** -24 + 5 * math.sqrt(most * torch.finfo(dtype).eps) / wide
        assert -noise <= lost <= most + noise, (name, lost)
        M.check(got, ref, (1 if dtype == torch.float32 else 17) * (n + 1) * 2.0 ** -23 * ref, name)


# ------------------------------------------------------------------------------------------------ threads
def _route_entry(experts):
    logits, (L, n) = _normal(_gen(experts), 40, experts), (_lib.lib(), ctypes.c_int64())
    a = _lib.RoutingArgs(logits_dev=logits.data_ptr(), logits_row=experts, n_rows=40, experts=experts, choices=4, groups=4, kept_groups=2, renormalize=1, scale=1.0)
    assert L.dynb_route_experts_workspace_bytes(ctypes.byref(a), ctypes.byref(n)) == 0
    out = [torch.empty(k, dtype=torch.int32, device="cuda") for k in (160, 160, 160, experts + 1)]
    ws = torch.empty(n.value, dtype=torch.uint8, device="cuda")
    return (logits, *out, ws), lambda s: L.dynb_route_experts(ctypes.byref(a), *(t.data_ptr() for t in (*out, ws)), n.value, s), out


def _route_backward_entry(experts):
    logits = _normal(_gen(experts), 40, experts)
    r = D.route_experts(logits, 4)
    a = _lib.RoutingArgs(logits_dev=logits.data_ptr(), logits_row=experts, n_rows=40, experts=experts, choices=4, groups=1, kept_groups=1, renormalize=1, scale=1.0)
    g, out = _normal(_gen(1), 40, 4), torch.empty_like(logits)
    return (logits, r, g, out), lambda s: _lib.lib().dynb_route_experts_backward(ctypes.byref(a), *(t.data_ptr() for t in (r.experts, r.weights, g, out)), s), [out]


def _type_linear_entry(inner):
    x, w = _normal(_gen(inner), 300, inner), _normal(_gen(1), 2, inner, 64)
    index, out = D.type_index(torch.arange(300, device="cuda") % 2, 2), torch.empty(300, 64, device="cuda")
    a = _lib.TypeLinear(weight_dev=w.data_ptr(), order_dev=index.order.data_ptr(), start_dev=index.start.data_ptr(), n_rows=300, types=2, inner=inner, outer=64)
    return (x, w, index, out), lambda s: _lib.lib().dynb_type_linear(ctypes.byref(a), x.data_ptr(), inner, None, out.data_ptr(), s), [out]


def _type_linear_backward_entry(outer):
    x, w, g = _normal(_gen(outer), 300, 64), _normal(_gen(1), 2, 64, outer), _normal(_gen(2), 300, outer)
    index, out, n = D.type_index(torch.arange(300, device="cuda") % 2, 2), torch.empty_like(w), ctypes.c_int64()
    a = _lib.TypeLinear(weight_dev=w.data_ptr(), order_dev=index.order.data_ptr(), start_dev=index.start.data_ptr(), n_rows=300, types=2, inner=64, outer=outer)
    assert _lib.lib().dynb_type_linear_workspace_bytes(ctypes.byref(a), ctypes.byref(n)) == 0
    ws = torch.empty(n.value, dtype=torch.uint8, device="cuda")
    return (x, w, g, index, out, ws), lambda s: _lib.lib().dynb_type_linear_backward(ctypes.byref(a), x.data_ptr(), 64, g.data_ptr(), outer, None, out.data_ptr(), None, ws.data_ptr(),
                                                                                  n.value, s), [out]


def _distance_bias_entry(buckets):
    dist, table, g = torch.rand(500, device="cuda") * 5, _normal(_gen(buckets), buckets, 8), _normal(_gen(1), 500, 8)
    out, n = [torch.empty_like(dist), torch.empty_like(table)], ctypes.c_int64()
    assert _lib.lib().dynb_distance_bias_workspace_bytes(500, buckets, 8, ctypes.byref(n)) == 0
    ws = torch.empty(n.value, dtype=torch.uint8, device="cuda")
    return (dist, table, g, *out, ws), lambda s: _lib.lib().dynb_distance_bias_backward(dist.data_ptr(), 500, table.data_ptr(), buckets, 8, 5.0, 1, g.data_ptr(), out[0].data_ptr(),
                                                                                     out[1].data_ptr(), ws.data_ptr(), n.value, s), out


@pytest.mark.parametrize("entry,sizes", [(_route_entry, (128, 96)), (_route_entry, (1024, 800)), (_route_backward_entry, (128, 100)), (_type_linear_entry, (256, 64)),
                                         (_type_linear_backward_entry, (128, 16)), (_distance_bias_entry, (64, 300)), (_distance_bias_entry, (1024, 300))])
def test_entries_in_two_threads(cuda, entry, sizes):
    """Calls of one kernel that need unlike amounts of shared memory: no thread takes from the other what its launch needs."""
    cases = [entry(n) for n in sizes]
    codes, together = [set() for _ in cases], threading.Barrier(len(cases))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]

    def work(call, stream, seen):
        together.wait()
        for _ in range(3000):
            seen.add(call(stream.cuda_stream))

    threads = [threading.Thread(target=work, args=(c[1], s, seen)) for c, s, seen in zip(cases, streams, codes)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert codes == [{0}, {0}]
    for (_, call, out), stream in zip(cases, streams):
        beside = [t.clone() for t in out]
        assert call(torch.cuda.current_stream().cuda_stream) == 0
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, beside))

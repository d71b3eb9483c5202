"""Rotary heads, routing and the experts' products on the GPU against plain forms in 64 bits, at sizes, masks, strides and types where they can go
wrong.  The bounds are derived beside the plain forms (tests/_experts.py) and here."""

import math

import pytest
import torch

import dynamis_b200 as D
from tests import _experts as X
from tests import _message as M

pytestmark = pytest.mark.gpu
U = M.U


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(gen, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=gen, device="cuda").to(dtype)


# ------------------------------------------------------------------------------------------------ rotary heads
def _rotary_case(n_q, n_k, heads, kv_heads, dim, dtype, axes=3, seed=1, pos_dtype=torch.float32, far=1.0, weights=True):
    gen = _gen(seed)
    q, k = _normal(gen, n_q, heads, dim, dtype=dtype), _normal(gen, n_k, kv_heads, dim, dtype=dtype)
    pos = (torch.randn(max(n_q, n_k), axes, generator=gen, device="cuda", dtype=torch.float64) * far).to(pos_dtype)
    wave = _normal(gen, dim // 2, axes)
    w = [1 + 0.3 * _normal(gen, dim) for _ in range(2)] if weights else [None, None]
    return q, k, pos, wave, *w, _normal(gen, n_q, heads, dim, dtype=dtype), _normal(gen, n_k, kv_heads, dim, dtype=dtype)


def _compare_rotary(case, eps=1e-6, interleaved=False):
    q, k, pos, wave, qw, kw, d_q, d_k = case
    leaves = {n: t.detach().requires_grad_() for n, t in (("q", q), ("k", k), ("pos", pos), ("q_weight", qw), ("k_weight", kw)) if t is not None}
    got_q, got_k = D.rotary_heads(leaves["q"], leaves["k"], leaves["pos"], wave, leaves.get("q_weight"), leaves.get("k_weight"), eps, interleaved)
    grads = torch.autograd.grad([got_q, got_k], list(leaves.values()), [d_q, d_k])
    ref = X.rotary(q, k, pos, wave, qw, kw, eps, interleaved, d_q, d_k)
    M.check(got_q, *ref["q"], "q")
    M.check(got_k, *ref["k"], "k")
    for name, grad in zip(leaves, grads):
        value, off = ref["d_" + name]
        if grad.dtype == torch.float64:      # formed in 32 bits all the same
            off = off + U * value.abs()
        M.check(grad, value, off, "d_" + name)
    with torch.no_grad():
        again = D.rotary_heads(q, k, pos, wave, qw, kw, eps, interleaved)
    assert torch.equal(again[0], got_q) and torch.equal(again[1], got_k)
    return got_q, got_k, grads


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 8, 16), (1, 1, 2), (3, 1, 6), (6, 2, 20), (4, 4, 64), (5, 5, 34), (2, 1, 256), (7, 7, 50), (3, 3, 130), (40, 8, 8), (1, 2, 254),
                                                (12, 12, 4), (9, 3, 48)])
def test_rotary_and_gradients(cuda, dtype, interleaved, heads, kv_heads, dim):
    _compare_rotary(_rotary_case(97, 131, heads, kv_heads, dim, M.TYPES[dtype], seed=heads * 1000 + dim), interleaved=interleaved)


@pytest.mark.parametrize("n_q,n_k", [(1, 1), (0, 3), (3, 0), (0, 0), (5, 2), (1, 70), (4099, 5003), (33, 33)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_rotary_rows(cuda, n_q, n_k, dtype):
    _compare_rotary(_rotary_case(n_q, n_k, 4, 2, 16, M.TYPES[dtype], seed=n_q + n_k))


@pytest.mark.parametrize("axes", [1, 2, 3])
@pytest.mark.parametrize("pos_dtype", [torch.float32, torch.float64])
def test_rotary_axes_and_far_positions(cuda, axes, pos_dtype):
    """Positions of up to a million turns: 32-bit angles would be off by several per cent of a turn."""
    _compare_rotary(_rotary_case(60, 80, 4, 4, 32, torch.float32, axes, 5, pos_dtype, far=1e6))
    _compare_rotary(_rotary_case(60, 80, 4, 4, 32, torch.float32, axes, 6, pos_dtype, weights=False), eps=None)
    _compare_rotary(_rotary_case(60, 80, 4, 4, 32, torch.float16, axes, 7, pos_dtype, weights=False), eps=0.25)


def test_rotary_images_of_a_periodic_box(cuda):
    """Whole waves on fractional coordinates: rows in other images turn alike, to the bit, and zero waves leave a head as it is."""
    q, k, pos, wave, qw, kw, _, _ = _rotary_case(50, 50, 4, 4, 16, torch.float32)
    pos = torch.round(pos * 256) / 256
    wave = torch.randint(-3, 4, wave.shape, device=cuda).float()
    one = D.rotary_heads(q, k, pos, wave, qw, kw)
    two = D.rotary_heads(q, k, pos + torch.randint(-9, 10, pos.shape, device=cuda), wave, qw, kw)
    assert torch.equal(one[0], two[0]) and torch.equal(one[1], two[1])
    still = D.rotary_heads(q, k, pos, torch.zeros_like(wave), eps=None)
    assert torch.equal(still[0], q) and torch.equal(still[1], k)


def test_rotary_strides(cuda):
    """Slices of one projection, heads before rows, elements apart, one row of any stride, gradients as slices and as an expanded number."""
    q, k, pos, wave, qw, kw, d_q, d_k = _rotary_case(70, 90, 4, 4, 16, torch.float32, seed=9)
    gen = _gen(10)
    joint = _normal(gen, 90, 3, 4, 16)
    wide = _normal(gen, 90, 4, 40)
    for qq, kk in ((joint[:70, 0], joint[:, 1]), (_normal(gen, 4, 70, 16).transpose(0, 1), wide[..., 8:24]), (wide[:70, :, 1:17], wide[..., 24:]),
                   (_normal(gen, 70, 16, 4).transpose(1, 2), wide[..., ::2][..., :16]), (wide[:70, :, 2:18], wide[..., 4:20])):
        for mixed in (False, True):
            _compare_rotary((qq, kk, pos, wave, qw, kw, wide[:70, :, 3:19], joint[:, 2]), interleaved=mixed)
    one = torch.randn(1, 4, 16, device=cuda).as_strided((1, 4, 16), (2 ** 33, 16, 1))
    _compare_rotary((one, one, pos[:1], wave, qw, kw, d_q[:1], d_k[:1]))
    leaves = [t.detach().requires_grad_() for t in (q, k, pos)]
    ones = torch.autograd.grad(sum(t.sum() for t in D.rotary_heads(*leaves, wave, qw, kw)), leaves)
    want = torch.autograd.grad(D.rotary_heads(*leaves, wave, qw, kw), leaves, [torch.ones_like(q), torch.ones_like(k)])
    assert all(torch.equal(a, b) for a, b in zip(ones, want))


def test_rotary_zero_rows_and_numbers_that_are_none(cuda):
    q, k, pos, wave, qw, kw, d_q, d_k = _rotary_case(40, 40, 4, 2, 16, torch.float32, seed=2)
    q[3] = 0.0
    _compare_rotary((q, k, pos, wave, qw, kw, d_q, d_k), eps=1e-3)
    q[5, 1, 2], pos[7, 0], k[9, 0] = math.nan, math.inf, 1e30       # squares overflow: the head becomes zeros
    a, b = D.rotary_heads(q, k, pos, wave, qw, kw)
    assert torch.isnan(a[5, 1]).all() and torch.isfinite(a[5, [0, 2, 3]]).all() and torch.isnan(a[7]).all() and torch.isnan(b[7]).all()
    rest = [i for i in range(40) if i not in (5, 7)]
    assert torch.isfinite(a[rest]).all() and torch.isfinite(b[rest]).all() and not b[9, 0].any()


def test_rotary_wants_some_gradients_only(cuda):
    q, k, pos, wave, qw, kw, d_q, d_k = _rotary_case(300, 400, 4, 2, 16, torch.bfloat16, seed=3)
    leaves = [t.detach().requires_grad_() for t in (q, k, pos, qw, kw)]
    call = lambda t: D.rotary_heads(t[0], t[1], t[2], wave, t[3], t[4])  # noqa: E731
    every = torch.autograd.grad(call(leaves), leaves, [d_q, d_k])
    for i in range(5):
        one, = torch.autograd.grad(call([t if j == i else t.detach() for j, t in enumerate(leaves)]), [leaves[i]], [d_q, d_k], allow_unused=True)
        assert torch.equal(one, every[i])
    half, = torch.autograd.grad(call(leaves)[0], [leaves[2]], d_q)       # nothing asked of the keys
    want, = torch.autograd.grad(call(leaves), [leaves[2]], [d_q, torch.zeros_like(d_k)])
    assert torch.equal(half, want)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        grad, = torch.autograd.grad(call(leaves)[0], [leaves[0]], d_q.requires_grad_(), create_graph=True)
        grad.sum().backward()


def test_rotary_refusals(cuda):
    q, k, pos, wave, qw, kw, _, _ = _rotary_case(4, 5, 4, 2, 8, torch.float32)

    def refused(match, *args, **more):
        with pytest.raises(RuntimeError, match=match):
            D.rotary_heads(*args, **more)

    refused("CUDA", q.cpu(), k, pos, wave)
    refused("shape", q[0], k, pos, wave)
    refused("float32, float16", q.double(), k.double(), pos, wave)
    refused("float32, float16", q, k.half(), pos, wave)
    refused("even dim", q[..., :7], k[..., :7], pos, wave)
    refused("even dim", q, k[..., :6], pos, wave)
    refused("even dim", torch.zeros(4, 4, 258, device=cuda), torch.zeros(5, 2, 258, device=cuda), pos, wave)
    refused("pos must have shape", q, k, pos[:4], wave)
    refused("pos must have shape", q, k, torch.zeros(5, 4, device=cuda), wave)
    refused("pos must be", q, k, pos.half(), wave)
    refused("wave must have shape", q, k, pos, wave[:, :2])
    refused("wave must be", q, k, pos, wave.double())
    refused("no gradient", q, k, pos, wave.clone().requires_grad_())
    refused("belongs to the norm", q, k, pos, wave, qw, None, None)
    refused("q_weight must be", q, k, pos, wave, qw[:4])
    refused("k_weight must be", q, k, pos, wave, qw, kw.double())
    for eps in (-1.0, math.nan, math.inf):
        refused("eps", q, k, pos, wave, eps=eps)


# ------------------------------------------------------------------------------------------------ routing
def _compare_route(logits, choices, **how):
    g = _normal(_gen(77), logits.size(0), choices)
    leaf = logits.detach().requires_grad_()
    r = D.route_experts(leaf, choices, **how)
    grad, = torch.autograd.grad(r.weights, [leaf], g)
    ref = X.route(logits, choices, d_weights=g, **how)
    for name in ("experts", "order", "start"):
        got = getattr(r, name)
        assert got.dtype == torch.int32 and torch.equal(got.cpu(), ref[name]), name
    M.check(r.weights.cpu(), *ref["weights"], "weights")
    assert grad.dtype == logits.dtype
    M.check(grad.cpu(), *ref["d_logits"], "d_logits")
    r.check_lists()
    return r


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("score,renormalize", [("softmax", True), ("softmax", False), ("sigmoid", True), ("sigmoid", False)])
@pytest.mark.parametrize("rows,experts,choices,groups,kept,bias", [(300, 8, 2, 1, 1, False), (1, 1, 1, 1, 1, False), (77, 5, 5, 1, 1, True), (500, 64, 6, 8, 4, True),
                                                                   (203, 33, 3, 11, 2, False), (64, 128, 8, 4, 1, True), (31, 1024, 32, 32, 5, True), (40, 300, 4, 1, 1, False),
                                                                   (900, 12, 2, 12, 3, True)])
def test_route_and_gradients(cuda, dtype, score, renormalize, rows, experts, choices, groups, kept, bias):
    gen = _gen(rows + experts)
    logits = (_normal(gen, rows, experts) * 1.5).to(M.TYPES[dtype])       # 16 bits: many equal ones
    _compare_route(logits, choices, score=score, renormalize=renormalize, groups=groups, kept_groups=kept, bias=_normal(gen, experts) * 0.1 if bias else None, scale=2.5)


@pytest.mark.parametrize("score,renormalize", [("softmax", True), ("softmax", False), ("sigmoid", True), ("sigmoid", False)])
@pytest.mark.parametrize("closed", [0.3, 0.9, 1.0])
@pytest.mark.parametrize("groups", [1, 4])
def test_route_closed_experts(cuda, score, renormalize, closed, groups):
    gen = _gen(5)
    logits = _normal(gen, 400, 16)
    logits[torch.rand(400, 16, generator=gen, device="cuda") < closed] = -math.inf
    bias = torch.zeros(16, device=cuda)
    bias[3] = -math.inf
    for b in (None, bias):
        r = _compare_route(logits, 4, score=score, renormalize=renormalize, groups=groups, kept_groups=min(2, groups), bias=b)
        assert b is None or not (r.experts == 3).any()
    assert closed < 1.0 or (not r.weights.any() and (r.experts == -1).all() and not r.start.any())


@pytest.mark.parametrize("rows", [0, 1, 7, 8, 9, 31, 4735, 4736, 4737, 150_001])
def test_route_lists_of_any_length(cuda, rows):
    logits = _normal(_gen(rows), rows, 8)
    r = D.route_experts(logits, 3)
    top = torch.sort(logits, dim=1, descending=True, stable=True).indices[:, :3]
    assert torch.equal(r.experts.long(), top)
    flat = top.reshape(-1)
    assert torch.equal(r.order.long(), torch.sort(flat, stable=True).indices)
    assert torch.equal(r.start.long(), torch.cat([flat.new_zeros(1), torch.bincount(flat, minlength=8).cumsum(0)]))


def test_route_extremes(cuda):
    """Logits of hundreds: sigmoids that are zero in 32 bits still give weights that add up, large ones do not overflow."""
    logits = torch.tensor([[-300.0, -301.0, -302.0, -400.0], [300.0, 299.0, 100.0, -100.0], [88.0, 89.0, 90.0, 91.0], [0.0, 0.0, 0.0, 0.0]], device=cuda)
    for score in ("softmax", "sigmoid"):
        r = _compare_route(logits, 2, score=score)
        assert torch.allclose(r.weights.sum(1), torch.ones(4, device=cuda), atol=1e-6)
        _compare_route(logits, 3, score=score, renormalize=False)
    wide = _normal(_gen(3), 50, 96)[:, ::3]
    assert torch.equal(D.route_experts(wide, 3).experts, D.route_experts(wide.contiguous(), 3).experts)
    row = _normal(_gen(3), 50, 96)[:, 10:42]
    assert torch.equal(D.route_experts(row, 3).experts, D.route_experts(row.contiguous(), 3).experts)


@pytest.mark.parametrize("experts", [8, 64, 200])
@pytest.mark.parametrize("groups", [1, 4])
def test_route_close_and_equal_keys(cuda, experts, groups):
    """Keys that 32 bits cannot tell apart, equal ones, and zeros of both signs: chosen as 64 bits choose, the lowest number first among equal ones."""
    gen = _gen(experts)
    logits = torch.randint(-2, 3, (600, experts), generator=gen, device="cuda").float() * 2.0 ** -20      # sigmoids 2^-22 apart, many of them equal
    logits[::3] = 0.0
    logits[::3][torch.rand(200, experts, generator=gen, device="cuda") < 0.5] *= -1.0
    bias = torch.randint(-3, 4, (experts,), generator=gen, device="cuda").float() * 2.0 ** -23
    for score in ("softmax", "sigmoid"):
        for b in (None, bias, 1000 * bias + 0.5):
            _compare_route(logits, 5, score=score, groups=groups, kept_groups=(groups + 1) // 2, bias=b)


def test_route_numbers_that_are_none(cuda):
    """A NaN comes first, its row's weights are NaN (sigmoids without sums: its own alone), other rows are as they were; every number stays in range."""
    logits = _normal(_gen(8), 9, 8)
    clean = D.route_experts(logits, 2)
    bad = logits.clone()
    bad[4, 5], bad[6, 1] = math.nan, math.inf
    rest = [i for i in range(9) if i not in (4, 6)]
    for bias in (None, torch.zeros(8, device=cuda)):
        r = D.route_experts(bad, 2, bias=bias)
        assert ((r.experts >= 0) & (r.experts < 8)).all() and torch.isnan(r.weights[4]).all() and torch.isnan(r.weights[6]).all()
        assert torch.equal(r.experts[rest], clean.experts[rest]) and torch.equal(r.weights[rest], clean.weights[rest])
        r.check_lists()
    s = D.route_experts(bad, 2, score="sigmoid", renormalize=False)
    assert s.experts[4, 0] == 5 and torch.isnan(s.weights[4, 0]) and torch.isfinite(s.weights[4, 1]) and s.weights[6, 0] == 1.0


def test_route_refusals(cuda):
    logits = torch.zeros(4, 8, device=cuda)

    def refused(match, *args, **more):
        with pytest.raises(RuntimeError, match=match):
            D.route_experts(*args, **more)

    refused("CUDA", logits.cpu(), 2)
    refused("shape", logits[0], 2)
    refused("float32, float16", logits.double(), 2)
    refused("choices", logits, 0)
    refused("choices", logits, 9)
    refused("choices", torch.zeros(4, 64, device=cuda), 33)
    refused("number of experts", torch.zeros(4, 1025, device=cuda), 2)
    refused("score", logits, 2, score="tanh")
    refused("groups", logits, 2, groups=3)
    refused("groups", logits, 2, groups=4, kept_groups=5)
    refused("bias", logits, 2, bias=torch.zeros(7, device=cuda))
    refused("bias", logits, 2, bias=torch.zeros(8, device=cuda, dtype=torch.float16))
    refused("no gradient", logits, 2, bias=torch.zeros(8, device=cuda, requires_grad=True))
    for scale in (0.0, -1.0, math.nan, math.inf):
        refused("scale", logits, 2, scale=scale)
    r = D.route_experts(logits, 2)
    for change, match in (({"experts": r.experts.long()}, "int32"), ({"weights": r.weights[:, :1]}, "weights"), ({"order": r.order[:-1]}, "one entry per pair"),
                          ({"start": r.start[:1]}, "number of experts"), ({"order": r.order.long()}, "int32")):
        with pytest.raises(RuntimeError, match=match):
            D.Routing(**{**{n: getattr(r, n) for n in ("experts", "weights", "order", "start")}, **change})
    twisted = D.Routing(r.experts, r.weights, r.order.flip(0), r.start)
    with pytest.raises(RuntimeError, match="by their experts"):
        twisted.check_lists()


# ------------------------------------------------------------------------------------------------ products
def _linear_case(rows, experts, choices, inner, outer, dtype, paired, offset, absent=0.1, seed=1):
    gen = _gen(seed + rows)
    routing = D.Routing(*X.routing_by_hand(rows, experts, choices, absent, seed, "cuda"))
    x = _normal(gen, *((rows, choices) if paired else (rows,)), inner, dtype=dtype)
    w = (_normal(gen, experts, inner, outer) * inner ** -0.5).to(dtype)
    return routing, x, w, _normal(gen, experts, outer, dtype=dtype) if offset else None, _normal(gen, rows, choices, outer, dtype=dtype)


def _compare_linear(routing, x, w, b, g, activation):
    leaves = [t.detach().requires_grad_() for t in (x, w, b) if t is not None]
    z = D.expert_linear(leaves[0], leaves[1], routing, leaves[2] if b is not None else None, activation)
    grads = torch.autograd.grad(z, leaves, g)
    ref = X.linear(x, w, routing.experts, b, activation, g)
    M.check(z, *ref["z"], "z")
    for name, grad in zip(("d_x", "d_weight", "d_bias"), grads):
        assert grad.dtype == x.dtype
        M.check(grad, *ref[name], name)
    with torch.no_grad():
        assert torch.equal(D.expert_linear(x, w, routing, b, activation), z)
    return z, grads


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("activation,paired", [(None, False), ("silu", False), ("gelu", True)])
@pytest.mark.parametrize("rows,experts,choices,inner,outer,offset", [(1, 1, 1, 1, 1, True), (1, 3, 2, 16, 8, True), (63, 2, 1, 7, 5, True), (64, 4, 2, 64, 64, False),
                                                                     (500, 8, 2, 128, 256, True), (333, 37, 3, 256, 128, True), (129, 89, 4, 64, 256, True), (2500, 3, 2, 130, 70, True),
                                                                     (4501, 2, 2, 33, 129, False), (2049, 1, 1, 256, 16, True), (300, 7, 2, 1, 300, True), (300, 7, 2, 300, 1, True),
                                                                     (3001, 16, 3, 96, 192, True), (777, 4, 2, 512, 384, True), (256, 2, 1, 8, 1024, True), (70, 2, 1, 1200, 40, True)])
def test_linear_and_gradients(cuda, dtype, activation, paired, rows, experts, choices, inner, outer, offset):
    _compare_linear(*_linear_case(rows, experts, choices, inner, outer, M.TYPES[dtype], paired, offset, seed=inner), activation)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("paired", [False, True])
def test_linear_places_without_an_expert(cuda, dtype, paired):
    """Zeros and zero gradients there, whatever the rows of x hold; also where no place has one, and where experts have no rows."""
    routing, x, w, b, g = _linear_case(200, 9, 3, 40, 24, M.TYPES[dtype], paired, True, absent=0.5)
    none = routing.experts < 0
    gone = none if paired else none.all(1)
    x[gone], g[none] = math.nan, math.nan
    leaves = [t.detach().requires_grad_() for t in (x, w, b)]
    z = D.expert_linear(*leaves[:2], routing, leaves[2], "silu")
    dx, dw, db = torch.autograd.grad(z, leaves, g)
    assert not z[none].any() and torch.isfinite(z).all() and not dx[gone].any() and all(torch.isfinite(t).all() for t in (dx, dw, db))
    x[gone], g[none] = 0.0, 0.0
    _compare_linear(routing, x, w, b, g, "silu")
    for absent in (1.0, 0.0):
        routing, x, w, b, g = _linear_case(150, 9, 2, 40, 24, M.TYPES[dtype], paired, True, absent=absent)
        w = torch.cat([w, w])
        start = torch.cat([routing.start, routing.start[-1:].expand(9)])
        _compare_linear(D.Routing(routing.experts, routing.weights, routing.order, start.contiguous()), x, w, torch.cat([b, b]), g, None)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_linear_strides(cuda, dtype):
    dtype = M.TYPES[dtype]
    routing, x, w, b, g = _linear_case(300, 5, 2, 64, 48, dtype, False, True)
    gen = _gen(4)
    wide, pairs = _normal(gen, 300, 200, dtype=dtype), _normal(gen, 300, 2, 200, dtype=dtype)
    slice_of_g = _normal(gen, 300, 2, 96, dtype=dtype)[..., 48:]
    for t in (wide[:, 8:72], wide[:, 4:68], wide[:, 3:67], wide[:, ::3][:, :64], _normal(gen, 64, 300, dtype=dtype).t(), pairs[..., 8:72], pairs[..., 1:65], pairs.transpose(0, 1).contiguous().transpose(0, 1)[..., :64]):
        _compare_linear(routing, t, w, b, slice_of_g, "silu")
    _compare_linear(routing, x, _normal(gen, 5, 48, 64, dtype=dtype).transpose(1, 2), b, g, "gelu")
    leaves = [t.detach().requires_grad_() for t in (x, w, b)]
    call = lambda t: D.expert_linear(t[0], t[1], routing, t[2], "silu")  # noqa: E731
    ones = torch.autograd.grad(call(leaves).sum(), leaves)
    assert all(torch.equal(a, c) for a, c in zip(ones, torch.autograd.grad(call(leaves), leaves, torch.ones_like(g))))
    every = torch.autograd.grad(call(leaves), leaves, g)
    for i in range(3):
        one, = torch.autograd.grad(call([t if j == i else t.detach() for j, t in enumerate(leaves)]), [leaves[i]], g)
        assert torch.equal(one, every[i])
    with pytest.raises(RuntimeError, match="once_differentiable"):
        grad, = torch.autograd.grad(call(leaves), [leaves[0]], g.requires_grad_(), create_graph=True)
        grad.sum().backward()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_linear_rows_off_16_bytes_give_the_same_bits(cuda, dtype):
    dtype = M.TYPES[dtype]
    routing, x, w, b, g = _linear_case(700, 4, 3, 72, 136, dtype, False, True)

    def off(t):
        moved = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)[1:].view(t.shape)
        return moved.copy_(t)

    def run(x, g, want, activation):
        leaves = [t.detach().requires_grad_(i in want) for i, t in enumerate((x, w, b))]
        z = D.expert_linear(*leaves[:2], routing, leaves[2], activation)
        return [z.detach(), *torch.autograd.grad(z, [leaves[i] for i in want], g)]

    odd = torch.cat([x, x], 1)[:, :73]
    odd = odd.contiguous()[:, :72]
    for activation in (None, "silu"):
        for want in ((0,), (1, 2), (0, 1, 2)):
            one = run(x, g, want, activation)
            for xx, gg in ((off(x), g), (odd, g), (x, off(g)), (off(x), off(g))):
                assert all(torch.equal(a, c) for a, c in zip(one, run(xx, gg, want, activation)))
            with torch.autograd.graph.saved_tensors_hooks(off, lambda t: t):   # slopes among them
                assert all(torch.equal(a, c) for a, c in zip(one, run(x, g, want, activation)))


def test_linear_of_no_rows(cuda):
    routing = D.Routing(*X.routing_by_hand(0, 3, 2, 0.0, 1, "cuda"))
    x, w, b = (torch.randn(*s, device=cuda, requires_grad=True) for s in ((0, 8), (3, 8, 4), (3, 4)))
    z = D.expert_linear(x, w, routing, b, "silu")
    assert z.shape == (0, 2, 4)
    dx, dw, db = torch.autograd.grad(z.sum(), (x, w, b))
    assert dx.shape == (0, 8) and not dw.any() and not db.any()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,experts,choices,inner,outer,paired", [(600, 3, 2, 1032, 520, False), (50, 1000, 2, 24, 40, False), (9000, 1, 1, 64, 64, True), (700, 5, 32, 16, 24, False),
                                                                     (40, 2, 2, 2050, 1030, True)])
def test_linear_wide_matrices_and_many_experts(cuda, dtype, rows, experts, choices, inner, outer, paired):
    """Matrices that come in pieces, more experts than rows, one expert for all, and the same experts several times in a row."""
    gen = _gen(rows)
    of = torch.randint(0, experts, (rows, choices), generator=torch.Generator().manual_seed(inner)).to(torch.int32)
    flat = of.reshape(-1).long()
    start = torch.cat([flat.new_zeros(1), torch.bincount(flat, minlength=experts).cumsum(0)]).to(torch.int32)
    routing = D.Routing(of.to(cuda), torch.rand(rows, choices, device=cuda), torch.sort(flat, stable=True).indices.to(torch.int32).to(cuda), start.to(cuda))
    routing.check_lists()
    dtype = M.TYPES[dtype]
    x = _normal(gen, *((rows, choices) if paired else (rows,)), inner, dtype=dtype)
    w = (_normal(gen, experts, inner, outer) * inner ** -0.5).to(dtype)
    _compare_linear(routing, x, w, _normal(gen, experts, outer, dtype=dtype), _normal(gen, rows, choices, outer, dtype=dtype), "silu")


def test_offsets_beyond_32_bits(cuda):
    """More than 2^31 elements of pairs: the last rows have the bits that they have in a small call, and so have their gradients."""
    rows, tail, wide = 2_200_000, 300, 512
    gen = _gen(1)
    x_tail, g_tail, z_tail = (_normal(gen, tail, *s, dtype=torch.bfloat16) for s in ((16,), (2, wide), (2, wide)))
    w = _normal(gen, 3, 16, wide, dtype=torch.bfloat16)
    logits = _normal(gen, rows, 3)
    big, small = (D.route_experts(t, 2) for t in (logits, logits[-tail:]))
    assert torch.equal(big.experts[-tail:], small.experts) and torch.equal(big.weights[-tail:], small.weights)
    assert rows * 2 * wide > 2 ** 31
    x = torch.zeros(rows, 16, device=cuda, dtype=torch.bfloat16)
    x[-tail:] = x_tail
    g = torch.zeros(rows, 2, wide, device=cuda, dtype=torch.bfloat16)
    g[-tail:] = g_tail

    def products(t, routing, grad):
        t = t.detach().requires_grad_()
        z = D.expert_linear(t, w, routing, None, "silu")
        return z.detach()[-tail:], torch.autograd.grad(z, [t], grad)[0][-tail:]

    for a, b in zip(products(x, big, g), products(x_tail, small, g_tail)):
        assert torch.equal(a, b)
    del x
    g[-tail:] = z_tail

    def sums(z, routing, grad):
        z, weights = z.detach().requires_grad_(), routing.weights.detach().requires_grad_()
        y = D.expert_combine(z, D.Routing(routing.experts, weights, routing.order, routing.start))
        return [t[-tail:] for t in (y.detach(), *torch.autograd.grad(y, [z, weights], grad))]

    d_y = torch.zeros(rows, wide, device=cuda, dtype=torch.bfloat16)
    d_y[-tail:] = g_tail[:, 0]
    for a, b in zip(sums(g, big, d_y), sums(z_tail, small, g_tail[:, 0])):
        assert torch.equal(a, b)


@pytest.mark.parametrize("activation", ["silu", "gelu"])
def test_linear_of_large_arguments(cuda, activation):
    """Far from zero the activations are 0 or their argument and the slopes 0 or 1, without overflow on the way."""
    routing = D.Routing(*X.routing_by_hand(4, 1, 1, 0.0, 1, "cuda"))
    w = torch.eye(16, device=cuda)[None].clone().requires_grad_()
    for dtype, far in ((torch.float32, 1e30), (torch.float32, 200.0), (torch.bfloat16, 300.0), (torch.float16, 60000.0)):
        x = torch.full((4, 16), far, device=cuda, dtype=dtype)
        x[:, ::2] *= -1
        leaf, ww = x.requires_grad_(), w.detach().to(dtype)
        z = D.expert_linear(leaf, ww, routing, None, activation)[:, 0]
        assert torch.equal(z[:, 1::2], x[:, 1::2]) and not z[:, ::2].any()
        dx, = torch.autograd.grad(z, [leaf], torch.ones_like(z))
        assert (dx[:, 1::2] == 1).all() and not dx[:, ::2].any()


def test_linear_numbers_that_are_none(cuda):
    """A NaN or an infinity of a row reaches that row's pairs alone, and the gradients of its experts."""
    routing, x, w, b, g = _linear_case(120, 4, 2, 32, 16, torch.float32, False, True, absent=0.0)
    x[7, 3], x[9, 0] = math.nan, math.inf
    for dtype in (torch.float32, torch.bfloat16):
        z = D.expert_linear(x.to(dtype), w.to(dtype), routing, b.to(dtype))
        assert torch.isnan(z[7]).all() and not torch.isfinite(z[9]).any()
        rest = [i for i in range(120) if i not in (7, 9)]
        assert torch.isfinite(z[rest]).all()


def test_linear_refusals(cuda):
    routing, x, w, b, _ = _linear_case(6, 3, 2, 8, 4, torch.float32, False, True)

    def refused(match, *args):
        with pytest.raises(RuntimeError, match=match):
            D.expert_linear(*args)

    refused("CUDA", x.cpu(), w, routing)
    refused("rows", x[:5], w, routing)
    refused("rows", x[:, None].expand(6, 3, 8), w, routing)
    refused("shape", x[0], w, routing)
    refused("float32, float16", x.double(), w.double(), routing)
    refused("type of x", x, w.half(), routing)
    refused("weight must have shape", x, w[:2], routing)
    refused("weight must have shape", x, w[:, :7], routing)
    refused("bias must have shape", x, w, routing, b[:, :3])
    refused("bias must be", x, w, routing, b.half())
    refused("activation", x, w, routing, b, "relu")


# ------------------------------------------------------------------------------------------------ sums
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("residual", [True, False])
@pytest.mark.parametrize("rows,choices,width", [(1, 1, 1), (7, 3, 5), (100, 2, 128), (65, 32, 33), (3, 4, 2049), (1001, 8, 64), (0, 2, 8), (301, 5, 40), (50, 1, 16384)])
def test_combine_and_gradients(cuda, dtype, residual, rows, choices, width):
    gen, dtype = _gen(rows + width), M.TYPES[dtype]
    experts, weights, order, start = X.routing_by_hand(rows, 40, choices, 0.2, width, "cuda")
    z, g = _normal(gen, rows, choices, width, dtype=dtype), _normal(gen, rows, width, dtype=dtype)
    z[experts < 0] = math.nan            # not used
    r = _normal(gen, rows, width, dtype=dtype) if residual else None
    leaves = [t.detach().requires_grad_() for t in (z, weights, r) if t is not None]
    y = D.expert_combine(leaves[0], D.Routing(experts, leaves[1], order, start), leaves[2] if residual else None)
    grads = torch.autograd.grad(y, leaves, g)
    ref = X.combine(z, weights, experts, r, g)
    M.check(y, *ref["y"], "y")
    for name, grad in zip(("d_z", "d_weights"), grads):
        M.check(grad, *ref[name], name)
    assert not residual or torch.equal(grads[2], g)


def test_combine_strides_and_refusals(cuda):
    gen = _gen(2)
    routing = D.Routing(*X.routing_by_hand(30, 5, 2, 0.1, 3, "cuda"))
    z, r = _normal(gen, 30, 2, 24), _normal(gen, 30, 24)
    want = D.expert_combine(z, routing, r)
    wide = torch.cat([r, r], 1)
    for zz in (z, torch.cat([z, z], 2)[..., :24], z.transpose(1, 2).contiguous().transpose(1, 2)):
        for rr in (r, wide[:, 24:], r.t().contiguous().t(), torch.cat([r[:, :1], r], 1)[:, 1:]):
            assert torch.equal(D.expert_combine(zz, routing, rr), want)
    leaves = [z.requires_grad_(), routing.weights.requires_grad_()]
    ones = torch.autograd.grad(D.expert_combine(z, routing).sum(), leaves)
    assert all(torch.equal(a, b) for a, b in zip(ones, torch.autograd.grad(D.expert_combine(z, routing), leaves, torch.ones_like(r))))

    def refused(match, *args):
        with pytest.raises(RuntimeError, match=match):
            D.expert_combine(*args)

    refused("CUDA", z.cpu(), routing)
    refused("shape", z[0], routing)
    refused("choices", z[:, :1], routing)
    refused("float32, float16", z.double(), routing)
    refused("residual must have shape", z, routing, r[:, :3])
    refused("residual must be", z, routing, r.half())


# ------------------------------------------------------------------------------------------------ together
def _layer(x, pos, wave, index, p):
    """A layer as a model has it: attention of turned heads to the neighbours, then two products by the experts that the rows choose."""
    n, heads = index.num_targets, 4
    q, k, v = (t.view(t.size(0), heads, -1) for t in (x[:n] @ p["wq"], x @ p["wk"], x @ p["wv"]))
    q, k = D.rotary_heads(q, k, pos, wave, p["gq"], p["gk"])
    h = x[:n] + D.neighbor_attention(q, k, v, index).reshape(n, -1)
    routing = D.route_experts(h @ p["gate"], 2, score="sigmoid", bias=p["balance"], scale=1.5)
    z = D.expert_linear(D.expert_linear(h, p["w1"], routing, p["b1"], "silu"), p["w2"], routing, p["b2"])
    return D.expert_combine(z, routing, h)


def _layer_64(x, pos, wave, src, dst, p, experts):
    n, heads = int(dst.max()) + 1, 4
    q, k, v = (t.view(t.size(0), heads, -1) for t in (x[:n] @ p["wq"], x @ p["wk"], x @ p["wv"]))

    def turn(t, w):
        a, b = (t * torch.rsqrt((t * t).mean(-1, keepdim=True) + 1e-6) * w).chunk(2, -1)
        angle = (2 * math.pi * (pos[:t.size(0)] @ wave.T))[:, None]
        return torch.cat([a * angle.cos() - b * angle.sin(), a * angle.sin() + b * angle.cos()], -1)

    q, k = turn(q, p["gq"]), turn(k, p["gk"])
    e = torch.exp((q[dst] * k[src]).sum(-1) * q.size(2) ** -0.5)
    a = e / torch.zeros(n, heads, dtype=x.dtype, device=x.device).index_add(0, dst, e)[dst]
    h = x[:n] + torch.zeros_like(q).index_add(0, dst, a[..., None] * v[src]).reshape(n, -1)
    s = torch.sigmoid(h @ p["gate"]).gather(1, experts)
    w = 1.5 * s / s.sum(1, keepdim=True)
    u = torch.nn.functional.silu(torch.einsum("ni,ncio->nco", h, p["w1"][experts]) + p["b1"][experts])
    z = torch.einsum("nci,ncio->nco", u, p["w2"][experts]) + p["b2"][experts]
    return h + (w[..., None] * z).sum(1)


def _layer_case(seed=3, n=400, wide=32, experts=6):
    gen = _gen(seed)
    ei, src, dst = M.ragged_graph([9] * n, n + 60, seed, "cuda")
    shapes = {"wq": (wide, wide), "wk": (wide, wide), "wv": (wide, wide), "gate": (wide, experts), "w1": (experts, wide, 48), "b1": (experts, 48),
              "w2": (experts, 48, wide), "b2": (experts, wide)}
    p = {name: _normal(gen, *s) * (s[-2] ** -0.5 if len(name) > 1 and name[0] in "wg" else 0.1) for name, s in shapes.items()}
    p["gq"], p["gk"] = (1 + 0.1 * _normal(gen, wide // 4) for _ in range(2))
    p["balance"] = _normal(gen, experts) * 0.05
    return ei, src, dst, _normal(gen, n + 60, wide), torch.rand(n + 60, 3, generator=gen, device="cuda"), torch.randint(-2, 3, (wide // 8, 3), device="cuda").float(), p, _normal(gen, n, wide)


def test_a_layer_and_its_gradients(cuda):
    """Rotation, attention, routing, products and sums as they are used together, against the same layer in 64 bits with the same experts."""
    ei, src, dst, x, pos, wave, p, g = _layer_case()
    index = D.neighbor_index(ei, 400, 460)
    leaves = {"x": x, "pos": pos, **{n: t for n, t in p.items() if n != "balance"}}
    leaves = {n: t.detach().requires_grad_() for n, t in leaves.items()}
    out = _layer(leaves["x"], leaves["pos"], wave, index, {**leaves, "balance": p["balance"]})
    grads = torch.autograd.grad(out, list(leaves.values()), g)
    # the experts that the layer chose: from its own h, made once more
    with torch.no_grad():
        q, k, v = (t.view(t.size(0), 4, -1) for t in (x[:400] @ p["wq"], x @ p["wk"], x @ p["wv"]))
        q, k = D.rotary_heads(q, k, pos, wave, p["gq"], p["gk"])
        h = x[:400] + D.neighbor_attention(q, k, v, index).reshape(400, -1)
        experts = D.route_experts(h @ p["gate"], 2, score="sigmoid", bias=p["balance"], scale=1.5).experts.long()
    wide = {n: t.detach().double().requires_grad_() for n, t in leaves.items()}
    ref = _layer_64(wide["x"], wide["pos"], wave.double(), src, dst, wide, experts)
    want = torch.autograd.grad(ref, list(wide.values()), g.double())
    # Chains of six sums of at most 60 terms, each off by some hundred u of its magnitudes: 1e4 u of the largest value is about 30 times above what they add up to
    out, ref = out.detach(), ref.detach()
    assert float((out.double() - ref).abs().max()) <= 1e4 * U * float(ref.abs().max())
    for name, a, b in zip(leaves, grads, want):
        assert float((a.double() - b).abs().max()) <= 1e4 * U * float(b.abs().max()), name


def test_a_captured_layer_replays_on_new_inputs(cuda):
    """Forward and gradients in one graph, routing included, replayed on other values on which other experts are chosen; two graphs side by side."""
    ei, _, _, x, pos, wave, p, g = _layer_case(5)
    index = D.neighbor_index(ei, 400, 460)
    x, pos = x.requires_grad_(), pos.requires_grad_()
    params = [p[n].requires_grad_() for n in ("gate", "w1", "b1", "w2", "b2", "gq")]

    def work():
        out = _layer(x, pos, wave, index, p)
        return (out, *torch.autograd.grad(out, [x, pos, *params], g))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = work()
    torch.cuda.current_stream().wait_stream(side)
    first = [t.detach().clone() for t in first]
    graphs, results = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            results.append(work())
        graphs.append(graph)
    with torch.no_grad():
        x.copy_(torch.randn_like(x))
        pos.copy_(torch.rand_like(pos))
    want = work()
    assert not torch.equal(want[0], first[0])
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for graph, s in zip(graphs, streams):
        with torch.cuda.stream(s):
            graph.replay()
    torch.cuda.synchronize()
    for result in results:
        assert all(torch.equal(a, b) for a, b in zip(result, want))


def test_layers_on_other_streams_repeat_their_bits(cuda):
    ei, _, _, x, pos, wave, p, g = _layer_case(7)
    index = D.neighbor_index(ei, 400, 460)
    x, w = x.requires_grad_(), p["w1"].requires_grad_()

    def work():
        out = _layer(x, pos, wave, index, p)
        return (out, *torch.autograd.grad(out, [x, w], g))

    want = work()
    torch.cuda.synchronize()
    got = []
    for _ in range(3):
        with torch.cuda.stream(torch.cuda.Stream()):
            got.append(work())
    torch.cuda.synchronize()
    for values in got:
        assert all(torch.equal(a, b) for a, b in zip(values, want))


def test_gradients_of_tensors_that_hooks_moved(cuda):
    """Saved tensors that went to the host and came back elsewhere, dense."""
    ei, _, _, x, pos, wave, p, g = _layer_case(9)
    index = D.neighbor_index(ei, 400, 460)
    x = torch.cat([x, x], 1)[:, 32:].requires_grad_()
    w = p["w2"].requires_grad_()

    def grads(moved):
        if moved:
            with torch.autograd.graph.save_on_cpu():
                out = _layer(x, pos, wave, index, p)
            junk = [torch.full((1 << 16,), float("nan"), device=cuda) for _ in range(20)]   # where the tensors were
            del junk
        else:
            out = _layer(x, pos, wave, index, p)
        return torch.autograd.grad(out, [x, w], g)

    assert all(torch.equal(a, c) for a, c in zip(grads(False), grads(True)))


def test_a_wait_that_ran_out_is_told_at_the_next_call(cuda):
    """The word that a kernel sets when one of its bounded waits runs out (set from the host here)."""
    from dynamis_b200 import message

    routing, x, w, b, _ = _linear_case(6, 3, 2, 8, 4, torch.float32, False, True)
    z = D.expert_linear(x, w, routing, b)
    torch.cuda.synchronize()
    for look in (lambda: D.expert_linear(x, w, routing, b), routing.check_status):
        message._STATUS[x.device.index][0].value = 1
        with pytest.raises(RuntimeError, match="ran out"):
            look()
    assert torch.equal(D.expert_linear(x, w, routing, b), z)

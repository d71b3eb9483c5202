"""Message-passing operators on the GPU against plain forms in 64 bits, at sizes, masks, strides and types where they can go wrong.  The
bounds are derived beside the plain forms (tests/_message.py) and here."""

import math

import numpy as np
import pytest
import torch

import dynamis_b200 as D
from tests import _message as M

pytestmark = pytest.mark.gpu
U = M.U
RAGGED = [0, 1, 2, 3, 31, 32, 33, 0, 64, 129, 5, 700, 0, 7]


def _normal(gen, *shape, dtype=torch.float32, dev="cuda"):
    return torch.randn(*shape, generator=gen, device=dev).to(dtype)


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


# ------------------------------------------------------------------------------------------------ lists
@pytest.mark.parametrize("degrees,sources", [([], 0), ([], 5), ([0], 1), ([1], 1), ([0, 0, 0], 2), (RAGGED, 40), (RAGGED, 3000), ([3000, 1, 0, 2500], 2),
                                             ([53] * 700, 900), ([1] * 5000, 5000), ([300] * 40, 12000)])
def test_neighbor_index_lists(cuda, degrees, sources):
    if sources == 0 and sum(degrees):
        pytest.skip("no sources")
    ei, src, dst = M.ragged_graph(degrees, sources, 3, cuda)
    index = D.neighbor_index(ei, len(degrees), sources)
    for name, want in M.index_lists(src, dst, len(degrees), sources).items():
        got = getattr(index, name)
        assert got.dtype == torch.int32 and got.tolist() == want, name


def test_neighbor_index_of_a_graph_and_of_a_strided_edge_list(cuda):
    rng = np.random.default_rng(1)
    pos = torch.as_tensor((rng.random((3000, 3)) * 31.0).astype(np.float32), device=cuda)
    ei, _, _ = D.owned_graph(pos, torch.eye(3) * 31.0, torch.tensor([True] * 3), 5.0, 2000)
    index = D.neighbor_index(ei, 2000, 3000)
    want = M.index_lists(ei[0], ei[1], 2000, 3000)
    both = ei.t().contiguous().t()      # [2, E] with the endpoints of an edge beside one another
    again = D.neighbor_index(both, 2000, 3000)
    for name in want:
        assert getattr(index, name).tolist() == want[name], name
        assert torch.equal(getattr(index, name), getattr(again, name))


def test_neighbor_index_hub(cuda):
    """One source in every list, one target with most edges."""
    T, S = 20000, 20001
    dst = torch.cat([torch.zeros(30000, dtype=torch.int64), torch.arange(1, T)])
    src = torch.cat([torch.arange(30000) % S, torch.full((T - 1,), 7)])
    index = D.neighbor_index(torch.stack([src, dst]).to(cuda), T, S)
    want = M.index_lists(src, dst, T, S)
    for name in want:
        assert getattr(index, name).tolist() == want[name], name


def test_neighbor_index_refusals(cuda):
    ei, _, _ = M.ragged_graph([2, 3, 4], 5, 1, cuda)
    for T, S in ((2, 5), (3, 4 if int(ei[0].max()) == 4 else int(ei[0].max()))):
        with pytest.raises(RuntimeError, match="outside"):
            D.neighbor_index(ei, T, S)
    low = ei.clone()
    low[0, 3] = -1
    with pytest.raises(RuntimeError, match="outside"):
        D.neighbor_index(low, 3, 5)
    apart = torch.tensor([[0, 1, 2], [0, 1, 0]], device=cuda)
    with pytest.raises(RuntimeError, match="behind one another"):
        D.neighbor_index(apart, 2, 3)
    with pytest.raises(RuntimeError, match="int64"):
        D.neighbor_index(ei.int(), 3, 5)
    with pytest.raises(RuntimeError, match="shape"):
        D.neighbor_index(ei.t(), 3, 5)
    with pytest.raises(RuntimeError, match="num_targets"):
        D.neighbor_index(ei, -1, 5)
    # and after the refusals the next call answers
    assert D.neighbor_index(ei, 3, 5).num_edges == 9


# ------------------------------------------------------------------------------------------------ attention
def _attention_case(degrees, sources, heads, kv_heads, dim, dtype, bias, seed, masked=0.1):
    gen = _gen(seed)
    ei, src, dst = M.ragged_graph(degrees, sources, seed, "cuda")
    T, E = len(degrees), src.numel()
    q, k, v = _normal(gen, T, heads, dim, dtype=dtype), _normal(gen, sources, kv_heads, dim, dtype=dtype), _normal(gen, sources, kv_heads, dim, dtype=dtype)
    b = None
    if bias:
        b = _normal(gen, E, heads) * 2
        b[torch.rand(E, heads, generator=gen, device="cuda") < masked] = -math.inf
        if T > 4:
            b[dst == 4] = -math.inf     # a target whose edges are all masked
    g = _normal(gen, T, heads, dim, dtype=dtype)
    return ei, src, dst, q, k, v, b, g


def _compare_attention(case, scale=None, index=None):
    ei, src, dst, q, k, v, b, g = case
    index = index or D.neighbor_index(ei, q.size(0), k.size(0))
    leaves = [t.detach().requires_grad_() for t in (q, k, v)] + ([b.detach().requires_grad_()] if b is not None else [])
    out = D.neighbor_attention(*leaves[:3], index, leaves[3] if b is not None else None, scale)
    grads = torch.autograd.grad(out, leaves, g)
    ref = M.attention(q, k, v, src, dst, b, scale if scale is not None else q.size(2) ** -0.5, g)
    M.check(out, *ref["out"], "out")
    for name, got in zip(("dq", "dk", "dv", "d_bias"), grads):
        M.check(got, *ref[name], name)
    with torch.no_grad():
        assert torch.equal(D.neighbor_attention(q, k, v, index, b, scale), out)
    return out, grads


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,dim,bias", [(8, 8, 16, True), (8, 8, 16, False), (1, 1, 1, True), (6, 3, 20, True), (4, 1, 64, True), (3, 3, 33, False),
                                                     (16, 16, 8, True), (40, 10, 4, True), (2, 2, 128, True), (2, 1, 256, True), (5, 5, 130, True),
                                                     (12, 4, 24, False), (64, 64, 2, True), (9, 3, 48, True)])
def test_attention_and_gradients(cuda, dtype, heads, kv_heads, dim, bias):
    _compare_attention(_attention_case(RAGGED, 60, heads, kv_heads, dim, M.TYPES[dtype], bias, heads * 1000 + dim))


@pytest.mark.parametrize("degrees,sources", [([0], 1), ([0, 0], 3), ([1], 1), ([5000], 100), ([20000, 0, 3], 7), ([52] * 3000, 3100), ([2] * 9000, 9000)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attention_lengths(cuda, degrees, sources, dtype):
    _compare_attention(_attention_case(degrees, sources, 8, 4, 16, M.TYPES[dtype], True, len(degrees)))


def test_attention_without_rows(cuda):
    for T, S in ((0, 0), (0, 5), (4, 0), (3, 3)):
        index = D.neighbor_index(torch.empty((2, 0), dtype=torch.int64, device=cuda), T, S)
        q, k, v = (torch.randn(n, 2, 8, device=cuda, requires_grad=True) for n in (T, S, S))
        out = D.neighbor_attention(q, k, v, index, torch.empty(0, 2, device=cuda))
        assert out.shape == (T, 2, 8) and not out.any()
        for t, grad in zip((q, k, v), torch.autograd.grad(out.sum(), (q, k, v))):
            assert grad.shape == t.shape and not grad.any()


def test_attention_strides(cuda):
    """Queries, keys and values as slices of one projection, rows of a wider table, heads before rows; gradients of the result as a slice and
    as an expanded number."""
    gen = _gen(3)
    degrees, S, H, dim = RAGGED, 50, 4, 16
    ei, src, dst = M.ragged_graph(degrees, S, 5, "cuda")
    T = len(degrees)
    joint = _normal(gen, S, 3, H, dim)
    index = D.neighbor_index(ei, T, S)
    k, v = joint[:, 1], joint[:, 2]
    q = _normal(gen, H, T, dim).transpose(0, 1)
    g = _normal(gen, T, H, 2 * dim)[..., :dim]
    _compare_attention((ei, src, dst, q, k, v, None, g), index=index)
    odd = _normal(gen, S, H, dim + 1)[..., 1:]                # heads off the 16-byte boundaries
    half = _normal(gen, S, H, dim + 4)[..., 4:]               # on 16 bytes, not on 32
    _compare_attention((ei, src, dst, q, half, v, None, g), index=index)
    last = _normal(gen, S, dim, H).transpose(1, 2)            # the elements of a head apart
    _compare_attention((ei, src, dst, q, odd, last, None, g), index=index)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    ones = torch.autograd.grad(D.neighbor_attention(*leaves, index).sum(), leaves)
    want = torch.autograd.grad(D.neighbor_attention(*leaves, index), leaves, torch.ones(T, H, dim, device=cuda))
    assert all(torch.equal(a, b) for a, b in zip(ones, want))


def test_attention_masks_of_any_kind(cuda):
    case = list(_attention_case(RAGGED, 60, 4, 4, 16, torch.float32, True, 77, masked=0.5))
    ei, src, dst, q, k, v, b, g = case
    # edges of source 9 are all masked, and its rows hold NaN and infinities
    b[src == 9] = -math.inf
    k[9], v[9] = math.nan, math.inf
    out, grads = _compare_attention(tuple(case))
    assert all(torch.isfinite(t).all() for t in (out, *grads))
    assert not grads[1][9].any() and not grads[2][9].any()
    # masks of the type's lowest value: a target with nothing else weighs its edges alike
    low = b.clone()
    low[:] = torch.finfo(torch.float32).min
    index = D.neighbor_index(ei, q.size(0), k.size(0))
    k[9], v[9] = 0.5, 0.5
    # q . k vanishes beside 3e38: every edge weighs 1 / n exactly
    n = torch.bincount(dst, minlength=q.size(0))
    leaves = [t.detach().requires_grad_() for t in (q, k, v, low)]
    out = D.neighbor_attention(*leaves[:3], index, leaves[3])
    mean = torch.zeros(q.shape, dtype=torch.float64, device=cuda).index_add_(0, dst, v[src].double()) / n.clamp(min=1)[:, None, None]
    size = torch.zeros(q.shape, dtype=torch.float64, device=cuda).index_add_(0, dst, v[src].double().abs()) / n.clamp(min=1)[:, None, None]
    M.check(out, mean, size * (n[:, None, None] + 8) * U, "mean")
    dv = torch.autograd.grad(out, leaves, g)[2]
    w = 1.0 / n.clamp(min=1).double()
    ref = torch.zeros(v.shape, dtype=torch.float64, device=cuda).index_add_(0, src, w[dst][:, None, None] * g.double()[dst])
    mag = torch.zeros(v.shape, dtype=torch.float64, device=cuda).index_add_(0, src, w[dst][:, None, None] * g.double()[dst].abs())
    M.check(dv, ref, mag * (n.max() + torch.bincount(src).max() + 8) * U, "dv of the mean")


def test_attention_large_logits_and_nan(cuda):
    """Logits of hundreds on both sides neither overflow nor underflow to zero sums; a NaN that takes part reaches its target alone."""
    case = list(_attention_case(RAGGED, 60, 2, 2, 16, torch.float32, True, 5, masked=0.0))
    case[3], case[4] = case[3] * 20, case[4] * 20
    _compare_attention(tuple(case))
    ei, src, dst, q, k, v, b, g = _attention_case([3, 2, 4], 9, 2, 2, 16, torch.float32, False, 6)
    e = 1
    src[e] = ei[0, e] = 8
    ei[0][torch.arange(9, device=cuda) != e] %= 8
    k[8, 0] = math.nan
    out = D.neighbor_attention(q, k, v, D.neighbor_index(ei, 3, 9))
    t = int(ei[1, e])
    assert torch.isnan(out[t, 0]).all() and torch.isfinite(out[t, 1]).all()
    assert torch.isfinite(out[[i for i in range(3) if i != t]]).all()


def test_attention_wants_some_gradients_only(cuda):
    ei, src, dst, q, k, v, b, g = _attention_case(RAGGED, 60, 4, 2, 16, torch.float32, True, 8)
    index = D.neighbor_index(ei, q.size(0), k.size(0))
    leaves = [t.detach().requires_grad_() for t in (q, k, v, b)]
    every = torch.autograd.grad(D.neighbor_attention(*leaves[:3], index, leaves[3]), leaves, g)
    for i in range(4):
        some = [t if j == i else t.detach() for j, t in enumerate(leaves)]
        one, = torch.autograd.grad(D.neighbor_attention(*some[:3], index, some[3]), [leaves[i]], g)
        assert torch.equal(one, every[i])
    with pytest.raises(RuntimeError, match="once_differentiable"):
        out = D.neighbor_attention(*leaves[:3], index, leaves[3])
        grad, = torch.autograd.grad(out, [leaves[0]], g.requires_grad_(), create_graph=True)
        grad.sum().backward()


def test_attention_refusals(cuda):
    ei, _, _ = M.ragged_graph([2, 3], 4, 1, cuda)
    index = D.neighbor_index(ei, 2, 4)
    q, k = torch.randn(2, 4, 8, device=cuda), torch.randn(4, 2, 8, device=cuda)
    assert D.neighbor_attention(q, k, k, index).shape == q.shape

    def refused(match, *args):
        with pytest.raises(RuntimeError, match=match):
            D.neighbor_attention(*args)

    refused("same shape", q, k, k[:, :1], index)
    refused("multiple", q[:, :3], k, k, index)
    refused("targets", q[:1], k, k, index)
    refused("sources", q, k[:3], k[:3], index)
    refused("dim", q[..., :4], k, k, index)
    refused("float32, float16 or bfloat16", q.double(), k.double(), k.double(), index)
    refused("float32, float16 or bfloat16", q, k.half(), k.half(), index)
    refused("shape", q[0], k, k, index)
    refused("bias must have shape", q, k, k, index, torch.zeros(5, 1, device=cuda))
    refused("bias must be", q, k, k, index, torch.zeros(5, 4, device=cuda, dtype=torch.bfloat16))
    refused("scale", q, k, k, index, None, math.nan)
    refused("CUDA", q.cpu(), k, k, index)
    wide = torch.zeros(4, 2, 257, device=cuda)
    refused("dim", torch.zeros(2, 4, 257, device=cuda), wide, wide, index)
    with pytest.raises(RuntimeError, match="one entry more"):
        D.NeighborIndex(index.rows, index.rows, index.src, index.cols, index.col_start, index.in_edge, index.in_dst)
    with pytest.raises(RuntimeError, match="int32"):
        D.NeighborIndex(index.rows.long(), index.row_start, index.src, index.cols, index.col_start, index.in_edge, index.in_dst)


def test_attention_of_lists_with_bad_entries(cuda):
    """Lists that a caller made: entries out of range are passed over, not followed."""
    ei, src, dst, q, k, v, b, g = _attention_case([3, 4, 2], 6, 2, 2, 16, torch.float32, True, 3, masked=0.0)
    index = D.neighbor_index(ei, 3, 6)
    src_bad, in_dst_bad = index.src.clone(), index.in_dst.clone()
    e = 4
    src_bad[e] = 1 << 30
    in_dst_bad[index.in_edge == e] = -5
    bad = D.NeighborIndex(index.rows, index.row_start, src_bad, index.cols, index.col_start, index.in_edge, in_dst_bad)
    leaves = [t.detach().requires_grad_() for t in (q, k, v, b)]
    grads = torch.autograd.grad(D.neighbor_attention(*leaves[:3], bad, leaves[3]), leaves, g)
    masked = b.clone()
    masked[e] = -math.inf
    ref = M.attention(q, k, v, src, dst, masked, 0.25, g)
    for name, got in zip(("dq", "dk", "dv", "d_bias"), grads):
        M.check(got, *ref[name], name)


# ------------------------------------------------------------------------------------------------ distance bias
def _bias_bounds(r, table, cutoff, smooth):
    """Value and bounds: the place x = u (K - 3) is off by 3 u x (three roundings), the spline moves by at most its slope times that, its four
    products and weights are off by 12 u of their magnitudes; the logarithms' arguments are off by 3 u relative (1 - u is one exact difference and a
    division; the polynomial's terms are positive), so 3 log(.) by 9 u, and their values by 4 u relative, all sums by 4 u."""
    K = table.size(0)
    rd = r.double().requires_grad_()
    td = table.double().requires_grad_()
    value = M.spline(rd, td, cutoff, smooth)
    plain = M.spline(rd.detach(), td.detach().abs(), cutoff, smooth=False)
    x = rd.detach() / cutoff * (K - 3)
    reach = torch.stack([td.detach().abs()[(x.long().clamp(0, K - 4) + j)] for j in range(4)]).amax(0)     # largest value nearby
    slack = 12 * U * plain + 2 * reach * (3 * U * x)[:, None]
    if smooth:
        u = rd.detach() / cutoff
        logs = (3 * torch.log1p(-u.clamp(max=1 - 1e-16)).abs() + torch.log1p(3 * u + 6 * u * u))[:, None]
        slack = slack + 8 * U * logs + 14 * U
    return value, slack + 4 * U * torch.where(torch.isinf(value), 0.0, value.abs()).detach(), rd, td, x, reach


@pytest.mark.parametrize("edges,buckets,heads,smooth", [(0, 8, 2, True), (1, 4, 1, True), (777, 4, 3, False), (5000, 64, 8, True), (30011, 64, 8, True),
                                                        (4099, 1024, 5, True), (2500, 17, 33, True), (3001, 100, 64, False), (20000, 9, 16, True), (1000, 300, 130, True)])
def test_distance_bias_and_gradients(cuda, edges, buckets, heads, smooth):
    gen, cutoff = _gen(edges + heads), 5.0
    r = 5.5 * torch.rand(edges, generator=gen, device="cuda")
    if edges > 500:
        c = torch.tensor(cutoff)
        r[:6] = torch.stack([c, torch.nextafter(c, c * 0), torch.nextafter(c, c * 2), c * 0, c / (buckets - 3), c * 2])
    table = _normal(gen, buckets, heads)
    g = _normal(gen, edges, heads)
    leaves = [r.requires_grad_(), table.requires_grad_()]
    bias = D.distance_bias(*leaves, cutoff, smooth)
    d_dist, d_table = torch.autograd.grad(bias, leaves, g)
    value, slack, rd, td, x, reach = _bias_bounds(r.detach(), table.detach(), cutoff, smooth)
    M.check(bias, value.detach(), slack, "bias")
    gd = torch.where(torch.isinf(value), 0.0, g.double())
    want_r, want_t = torch.autograd.grad(torch.where(torch.isinf(value), 0.0, value), [rd, td], gd) if edges else (torch.zeros(0), torch.zeros(buckets, heads))
    want_r, want_t = want_r.cuda().double(), want_t.cuda().double()
    # slopes: second derivatives are at most 4 reach a bucket, weights' derivatives off by 8 u; the switch's term by 10 u; sums of heads
    G = gd.abs()
    pull = (30 * x * x / (buckets - 3) ** 2)[:, None] if smooth else torch.zeros_like(x)[:, None]
    u = rd.detach() / cutoff
    pull = pull / ((1 - u).clamp(min=1e-30) * (1 + 3 * u + 6 * u * u))[:, None]
    pull = torch.where(torch.isinf(value), 0.0, pull.expand_as(value))
    slope_off = (buckets - 3) * reach * (12 * U * x + 16 * U)[:, None] + 12 * U * pull
    size = (buckets - 3) * 2 * reach + pull
    M.check(d_dist, want_r, (G * (slope_off + (heads + 4) * U * size)).sum(1).detach() / cutoff, "d_dist")
    # the table: weights off by 3 u x of their slopes (at most 0.75) and 8 u; sums of a stretch in 32 bits
    w_off = torch.zeros_like(td.detach())
    at = x.long().clamp(0, buckets - 4)
    per = (edges + 147) // 148 + 40
    for j in range(4):
        w_off.index_add_(0, at + j, G * (0.75 * 3 * U * x + 8 * U + per * U)[:, None])
    M.check(d_table, want_t, w_off, "d_table")
    again = torch.autograd.grad(D.distance_bias(*leaves, cutoff, smooth), leaves, g)
    assert torch.equal(again[0], d_dist) and torch.equal(again[1], d_table)


def test_distance_bias_against_differences(cuda):
    """Slopes against differences of the values: forces are the energy's own."""
    gen = _gen(9)
    r = (torch.rand(2000, generator=gen, device="cuda") * 4.8 + 0.05).requires_grad_()
    table = _normal(gen, 12, 4)
    bias = D.distance_bias(r, table, 5.0)
    slope, = torch.autograd.grad(bias.sum(), [r])
    h = 0.01
    r64 = r.detach().double()
    up, down = (M.spline(r64 + s * h, table.double(), 5.0) for s in (1, -1))
    diff = ((up - down) / (2 * h)).sum(1)
    # third derivatives: of the spline at most 8 largest value (9 / 5)^3 a head, of the switch 2 * 3 / (5 - r)^3; times h^2 / 6
    third = 4 * (8 * table.abs().max().double() * 1.8 ** 3 + 6 / (5 - r64 - h) ** 3)
    assert ((slope.double() - diff).abs() <= third * h * h / 6 * 1.1 + 1e-4).all()


def test_distance_bias_refusals_and_odd_values(cuda):
    r, t = torch.rand(10, device=cuda) * 5, torch.randn(8, 2, device=cuda)
    for args, match in (((r.double(), t, 5.0), "float32"), ((r[None], t, 5.0), "1-D"), ((r, t.half(), 5.0), "float32"), ((r, t[:3], 5.0), "buckets"),
                        ((r, t[:, :0], 5.0), "heads"), ((r, t, 0.0), "cutoff"), ((r, t, -1.0), "cutoff"), ((r, t, math.inf), "cutoff"), ((r, t, math.nan), "cutoff"),
                        ((r, t.cpu(), 5.0), "device"), ((r, t, 1e-60), "cutoff"), ((r, torch.zeros(1025, 2, device=cuda), 5.0), "buckets")):
        with pytest.raises(RuntimeError, match=match):
            D.distance_bias(*args)
    odd = torch.tensor([math.nan, math.inf, 5.0, 1.0], device=cuda)
    b = D.distance_bias(odd, t, 5.0)
    assert torch.isnan(b[0]).all() and (b[1:3] == -math.inf).all() and torch.isfinite(b[3]).all()
    # masked pairs take nothing from gradients of any kind
    odd = torch.tensor([5.0, 6.0, 1.0], device=cuda, requires_grad=True)
    tt = t.clone().requires_grad_()
    g = torch.tensor([[math.nan, 1.0], [math.inf, math.nan], [0.0, 0.0]], device=cuda)
    d, dt = torch.autograd.grad(D.distance_bias(odd, tt, 5.0), [odd, tt], g)
    assert not d.any() and not dt.any()
    strided = torch.rand(20, 3, device=cuda)[:, 1] * 5
    assert torch.equal(D.distance_bias(strided, t, 5.0), D.distance_bias(strided.contiguous(), t, 5.0))


# ------------------------------------------------------------------------------------------------ products by type
def _kinds(rows, types, seed, skew=True):
    gen = torch.Generator().manual_seed(seed)
    share = 1.0 / torch.arange(1, types + 1) if skew else torch.ones(types)
    return torch.multinomial(share, rows, replacement=True, generator=gen) if rows else torch.empty(0, dtype=torch.int64)


@pytest.mark.parametrize("rows,types", [(0, 1), (0, 7), (1, 1), (1, 9), (257, 1), (1000, 5), (5003, 300), (20011, 89), (70000, 3), (100, 4096)])
def test_type_index(cuda, rows, types):
    kinds = _kinds(rows, types, rows)
    index = D.type_index(kinds.to(cuda), types)
    assert index.order.tolist() == torch.argsort(kinds, stable=True).tolist()
    assert index.start.tolist() == [0] + torch.cumsum(torch.bincount(kinds, minlength=types), 0).tolist()


def _compare_linear(x, weight, offset, kinds, g):
    dtype = x.dtype
    index = D.type_index(kinds, weight.size(0))
    leaves = [x.detach().requires_grad_(), weight.detach().requires_grad_()] + ([offset.detach().requires_grad_()] if offset is not None else [])
    y = D.type_linear(leaves[0], leaves[1], index, leaves[2] if offset is not None else None)
    grads = torch.autograd.grad(y, leaves, g)
    n, (T, a, b) = x.size(0), weight.shape
    xd, wd, gd = x.double(), weight.double(), g.double()
    ref = {"y": [], "dx": []}
    want_y, off_y = torch.zeros(n, b, dtype=torch.float64, device="cuda"), torch.zeros(n, b, dtype=torch.float64, device="cuda")
    want_x, off_x = torch.zeros(n, a, dtype=torch.float64, device="cuda"), torch.zeros(n, a, dtype=torch.float64, device="cuda")
    want_w, off_w, want_b, off_b = (torch.zeros(s, dtype=torch.float64, device="cuda") for s in (weight.shape, weight.shape, (T, b), (T, b)))
    # products of fp32 operands may leave 2^-20 out (16 u); sums of `inner`, `outer` or `rows` products
    for t in range(T):
        m = torch.nonzero(kinds == t)[:, 0]
        want_y[m], off_y[m] = xd[m] @ wd[t], (a + 17) * U * (xd[m].abs() @ wd[t].abs())
        if offset is not None:
            want_y[m] += offset[t].double()
            off_y[m] += 2 * U * (offset[t].double().abs() + xd[m].abs() @ wd[t].abs())
        want_x[m], off_x[m] = gd[m] @ wd[t].T, (b + 17) * U * (gd[m].abs() @ wd[t].abs().T)
        want_w[t], off_w[t] = xd[m].T @ gd[m], (m.numel() + 17) * U * (xd[m].abs().T @ gd[m].abs())
        want_b[t], off_b[t] = gd[m].sum(0), (m.numel() + 2) * U * gd[m].abs().sum(0)
    M.check(y, want_y, off_y, "y")
    for name, got, want, off in zip(("dx", "dw", "db"), grads, (want_x, want_w, want_b), (off_x, off_w, off_b)):
        assert got.dtype == dtype
        M.check(got, want, off, name)
    return y, grads


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,types,inner,outer,offset", [(1, 1, 1, 1, True), (1, 3, 16, 8, True), (63, 2, 7, 5, True), (64, 1, 64, 64, False), (65, 1, 64, 64, True),
                                                           (1000, 5, 128, 128, True), (1003, 5, 128, 64, True), (129, 89, 64, 256, True), (5000, 3, 130, 70, True),
                                                           (9001, 2, 33, 129, False), (4097, 1, 256, 16, True), (300, 7, 1, 300, True), (300, 7, 300, 1, True),
                                                           (20000, 12, 96, 192, True), (777, 4, 512, 384, True), (256, 2, 8, 1024, True), (70, 2, 1200, 40, True), (70, 3, 24, 1300, True)])
def test_type_linear_and_gradients(cuda, dtype, rows, types, inner, outer, offset):
    gen, dtype = _gen(rows + inner), M.TYPES[dtype]
    kinds = _kinds(rows, types, rows + outer).to(cuda)
    _compare_linear(_normal(gen, rows, inner, dtype=dtype), _normal(gen, types, inner, outer, dtype=dtype),
                    _normal(gen, types, outer, dtype=dtype) if offset else None, kinds, _normal(gen, rows, outer, dtype=dtype))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_type_linear_strides_and_missing_types(cuda, dtype):
    gen, dtype = _gen(1), M.TYPES[dtype]
    kinds = (_kinds(900, 3, 1) * 2 + 1).to(cuda)      # types 0, 2, 4 and 6 have no rows
    wide = _normal(gen, 900, 200, dtype=dtype)
    for x in (wide[:, 8:72], wide[:, 3:67], wide[:, ::3][:, :64], _normal(gen, 64, 900, dtype=dtype).t()):
        g = _normal(gen, 900, 2 * 48, dtype=dtype)[:, 48:]
        y, (dx, dw, db) = _compare_linear(x, _normal(gen, 7, 64, 48, dtype=dtype), _normal(gen, 7, 48, dtype=dtype), kinds, g)
        assert not dw[0::2].any() and not db[0::2].any()


@pytest.mark.parametrize("inner,outer", [(128, 128), (384, 250)])
def test_type_linear_long_sums_of_one_sign(cuda, inner, outer):
    """Operands of one sign, where sums that are cut off towards zero lose the most.  A step of 16 products cuts at most 2^-23 of the sum so far off, and a
    leading sum has at most 1024 / 16 = 64 of them (y, dx: one for every 16 columns); parts of 24 bits and the rest of the rounding stay within 2^-21."""
    gen = _gen(31)
    n = 150_001
    kinds = _kinds(n, 2, 3).to(cuda)
    x, w, g = (torch.rand(*s, generator=gen, device="cuda") for s in ((n, inner), (2, inner, outer), (n, outer)))
    leaves = [t.requires_grad_() for t in (x, w)]
    y = D.type_linear(x, w, D.type_index(kinds, 2))
    dx, dw = torch.autograd.grad(y, leaves, g)
    for t in range(2):
        m = torch.nonzero(kinds == t)[:, 0]
        for got, ref, steps in ((y[m], x[m].double() @ w[t].double(), inner // 16), (dx[m], g[m].double() @ w[t].double().T, -(-outer // 16)),
                                (dw[t], x[m].double().T @ g[m].double(), 64)):
            assert float(((got.double() - ref) / ref).abs().max()) <= steps * 2.0 ** -23 + 2.0 ** -21


def test_type_linear_of_no_rows(cuda):
    index = D.type_index(torch.empty(0, dtype=torch.int64, device=cuda), 3)
    x, w, b = (torch.randn(*s, device=cuda, requires_grad=True) for s in ((0, 8), (3, 8, 4), (3, 4)))
    y = D.type_linear(x, w, index, b)
    assert y.shape == (0, 4)
    dx, dw, db = torch.autograd.grad(y.sum(), (x, w, b))
    assert dx.shape == (0, 8) and not dw.any() and not db.any()


def test_type_linear_repeats_its_bits_and_wants_some_gradients_only(cuda):
    gen = _gen(2)
    kinds = _kinds(9000, 4, 2).to(cuda)
    index = D.type_index(kinds, 4)
    leaves = [_normal(gen, 9000, 64).requires_grad_(), _normal(gen, 4, 64, 32).requires_grad_(), _normal(gen, 4, 32).requires_grad_()]
    g = _normal(gen, 9000, 32)
    every = torch.autograd.grad(D.type_linear(leaves[0], leaves[1], index, leaves[2]), leaves, g)
    for i in range(3):
        some = [t if j == i else t.detach() for j, t in enumerate(leaves)]
        one, = torch.autograd.grad(D.type_linear(some[0], some[1], index, some[2]), [leaves[i]], g)
        assert torch.equal(one, every[i])


def test_type_linear_refusals(cuda):
    kinds = torch.tensor([0, 1, 1], device=cuda)
    index = D.type_index(kinds, 2)
    x, w = torch.randn(3, 4, device=cuda), torch.randn(2, 4, 5, device=cuda)

    def refused(match, *args):
        with pytest.raises(RuntimeError, match=match):
            D.type_linear(*args)

    refused("shape", x, w[:1], index)
    refused("shape", x, w[:, :3], index)
    refused("rows", x[:2], w, index)
    refused("type of x", x, w.half(), index)
    refused("float32, float16", x.double(), w.double(), index)
    refused("bias must have shape", x, w, index, torch.zeros(2, 4, device=cuda))
    refused("bias must be", x, w, index, torch.zeros(2, 5, device=cuda, dtype=torch.float16))
    for bad in (torch.tensor([0, 2], device=cuda), torch.tensor([-1, 0], device=cuda)):
        with pytest.raises(RuntimeError, match="outside"):
            D.type_index(bad, 2)
    with pytest.raises(RuntimeError, match="int64"):
        D.type_index(kinds.int(), 2)
    for n in (0, 4097):
        with pytest.raises(RuntimeError, match="num_types"):
            D.type_index(kinds, n)


# ------------------------------------------------------------------------------------------------ together
def _layer(x, types, dist, table, index, wq, wk, wv, heads):
    """One layer as a model has it: projections by type of all rows, attention of the owned rows with the learned bias."""
    n = index.num_targets
    tall, town = types
    q = D.type_linear(x[:n], wq, town).view(n, heads, -1)
    k, v = (D.type_linear(x, w, tall).view(x.size(0), heads, -1) for w in (wk, wv))
    return D.neighbor_attention(q, k, v, index, D.distance_bias(dist, table, 5.0)).reshape(n, -1)


def test_layers_over_ranks_give_the_forces_of_the_whole(cuda):
    """Two layers of a model over three ranks driven from one process (partition, halo maps, owned graphs, exchange of the embeddings and of
    their gradients) against the same model over one graph, and that one against 64 bits."""
    rng = np.random.default_rng(4)
    N, L, W, F, H = 1500, 24.0, 3, 32, 4
    pos = torch.as_tensor((rng.random((N, 3)) * L).astype(np.float32), device=cuda)
    cell, pbc = torch.eye(3) * L, torch.tensor([True] * 3)
    kinds = torch.as_tensor(rng.integers(0, 3, N), device=cuda)
    gen = _gen(11)
    emb = _normal(gen, N, F)
    layers = [[_normal(gen, 3, F, F) * F ** -0.5 for _ in range(3)] + [_normal(gen, 16, H)] for _ in range(2)]
    head = _normal(gen, F)

    def vectors(p, ei, shifts):
        return torch.linalg.norm(p[ei[0]] + shifts - p[ei[1]], dim=1)

    # the whole system at once
    def whole(p):
        ei, _, shifts = D.owned_graph(p.detach(), cell, pbc, 5.0, N, negate_shifts=False)
        index, tt = D.neighbor_index(ei, N, N), D.type_index(kinds, 3)
        d, x = vectors(p, ei, shifts), emb
        for wq, wk, wv, table in layers:
            x = x + _layer(x, (tt, tt), d, table, index, wq, wk, wv, H)
        return (x @ head).sum(), (ei, shifts)

    p1 = pos.clone().requires_grad_()
    energy, (ei, shifts) = whole(p1)
    force, = torch.autograd.grad(energy, [p1])

    # in 64 bits with elementary operations
    p2 = pos.double().requires_grad_()
    src, dst = ei[0], ei[1]
    d = torch.linalg.norm(p2[src] + shifts.double() - p2[dst], dim=1)
    x = emb.double()
    for wq, wk, wv, table in layers:
        q, k, v = (torch.einsum("ni,nio->no", x, w.double()[kinds]).view(N, H, -1) for w in (wq, wk, wv))
        z = (q[dst] * k[src]).sum(-1) * (F // H) ** -0.5 + M.spline(d, table.double(), 5.0)
        e = torch.exp(z - z.max())
        p = e / torch.zeros(N, H, dtype=torch.float64, device=cuda).index_add(0, dst, e)[dst]
        x = x + torch.zeros(N, H, F // H, dtype=torch.float64, device=cuda).index_add(0, dst, p[..., None] * v[src]).reshape(N, -1)
    e64 = (x @ head.double()).sum()
    f64, = torch.autograd.grad(e64, [p2])
    # Two layers of sums of at most 200 terms: values are off by some hundred u relative to the magnitudes, which the projections and the
    # softmax (its logits enter with factors of up to 10) carry on twice: 1e5 u of the largest force is 100 times above that estimate's typical value
    energy, e64 = energy.detach(), e64.detach()
    assert abs(float(energy) - float(e64)) <= 1e5 * U * float((x.detach().abs() @ head.double().abs()).sum())
    assert float((force.double() - f64).abs().max()) <= 1e5 * U * float(f64.abs().max())

    # the same over three ranks
    st = D.MolecularInfo()
    st.num_atoms, st.atom_positions = N, pos
    st.atom_vertex_numbers = torch.arange(N, dtype=torch.int64, device=cuda)
    cfg = D.SimulationConfig()
    cfg.cutoff, cfg.ghost_cutoff_buffer, cfg.cell, cfg.pbc = 5.0, 0.5, cell, pbc
    infos, meta, exs = [], [], []
    for r in range(W):
        env = D.DistEnvironment()
        env.global_rank, env.world_size = r, W
        info = D.SFCPartitioner().partition(st, env)
        D.SFCPartitioner().build_halo_maps(info, st, env, cfg)
        ex = D.FeatureExchanger(wait_ns=5_000_000_000)
        meta.append(ex.local_setup(info.send_offsets, info.send_local_indices, info.recv_offsets, info.partition_indices.numel(), F, r, W, cuda))
        infos.append(info)
        exs.append(ex)
    for ex in exs:
        ex.connect(meta)
    ranks = []
    for info in infos:
        n = info.partition_indices.numel()
        atoms = torch.cat([info.partition_indices, info.recv_atom_global])
        p = pos[atoms].requires_grad_()
        ei, _, shifts = D.owned_graph(p.detach(), cell, pbc, 5.0, n, negate_shifts=False)
        index = D.neighbor_index(ei, n, atoms.numel())
        ranks.append({"n": n, "atoms": atoms, "p": p, "d": vectors(p, ei, shifts), "index": index,
                      "types": (D.type_index(kinds[atoms], 3), D.type_index(kinds[atoms[:n]], 3))})
    # layer 1 on every rank (its inputs are known everywhere), exchange, layer 2
    for rank in ranks:
        wq, wk, wv, table = layers[0]
        rank["x0"] = emb[rank["atoms"]]
        rank["x1"] = rank["x0"][:rank["n"]] + _layer(rank["x0"], rank["types"], rank["d"], table, rank["index"], wq, wk, wv, H)
    pend = [ex.forward_begin(r["x1"].detach()) for ex, r in zip(exs, ranks)]
    total = 0.0
    for ex, r, (o, gen_) in zip(exs, ranks, pend):
        r["all1"] = ex.forward_end(o, gen_).requires_grad_()
        wq, wk, wv, table = layers[1]
        x2 = r["all1"][:r["n"]] + _layer(r["all1"], r["types"], r["d"], table, r["index"], wq, wk, wv, H)
        r["energy"] = (x2 @ head).sum()
        total += float(r["energy"].detach())
    for r in ranks:
        r["g1"], r["gp"] = torch.autograd.grad(r["energy"], [r["all1"], r["p"]], retain_graph=True)
    pend = [ex.backward_begin(r["g1"].contiguous()) for ex, r in zip(exs, ranks)]
    forces = torch.zeros(N, 3, dtype=torch.float64, device=cuda)
    for ex, r, (g, gen_) in zip(exs, ranks, pend):
        own = ex.backward_end(g, gen_)
        more, = torch.autograd.grad(r["x1"], [r["p"]], own)
        forces.index_add_(0, r["atoms"], (r["gp"] + more).double())
    assert abs(total - float(e64)) <= 1e5 * U * float((x.detach().abs() @ head.double().abs()).sum())
    assert float((forces - f64).abs().max()) <= 1e5 * U * float(f64.abs().max())
    for ex in exs:
        ex.check_status()
        ex.teardown()


def test_streams_devices_and_repeats(cuda):
    """On another stream than the default one, with other work of the same kind beside it, the bits are the same."""
    case = _attention_case([40] * 500, 600, 8, 8, 16, torch.float32, True, 1)
    ei, src, dst, q, k, v, b, g = case
    index = D.neighbor_index(ei, 500, 600)
    leaves = [t.detach().requires_grad_() for t in (q, k, v, b)]
    r, table = torch.rand(5000, device=cuda).mul_(5).requires_grad_(), torch.randn(32, 8, device=cuda, requires_grad=True)
    gr = torch.randn(5000, 8, device=cuda)

    def work():
        out = D.neighbor_attention(*leaves[:3], index, leaves[3])
        bias = D.distance_bias(r, table, 5.0)
        return (out, *torch.autograd.grad(out, leaves, g), bias, *torch.autograd.grad(bias, [r, table], gr))

    want = work()
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got.append((work(), D.neighbor_index(ei, 500, 600)))
    torch.cuda.synchronize()
    for values, lists in got:
        assert all(torch.equal(x, y) for x, y in zip(values, want))
        assert torch.equal(lists.in_edge, index.in_edge) and torch.equal(lists.cols, index.cols)


def test_captured_layer_replays_on_new_inputs(cuda):
    """Forward and gradients in one graph, replayed on other values; two graphs replayed side by side, and a capture that is refused."""
    ei, src, dst, q, k, v, b, g = _attention_case([30] * 300, 350, 4, 4, 16, torch.float32, False, 2)
    index = D.neighbor_index(ei, 300, 350)
    kinds = _kinds(350, 3, 1).to(cuda)
    tall = D.type_index(kinds, 3)
    dist = torch.rand(9000, device=cuda) * 5.2
    params = [torch.randn(20, 4, device=cuda, requires_grad=True), torch.randn(3, 64, 64, device=cuda, requires_grad=True)]
    x, qq, r = torch.randn(350, 64, device=cuda, requires_grad=True), q.detach().requires_grad_(), dist.requires_grad_()

    def work():
        kv = D.type_linear(x, params[1], tall).view(350, 4, 16)
        out = D.neighbor_attention(qq, kv, kv, index, D.distance_bias(r, params[0], 5.0))
        return (out, *torch.autograd.grad(out, [x, qq, r, *params], g))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    graphs, results = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            results.append(work())
        graphs.append(graph)
    with torch.no_grad():
        x.copy_(torch.randn(350, 64, device=cuda))
        qq.mul_(0.5)
        r.copy_(torch.rand(9000, device=cuda) * 5.2)
    want = work()
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for graph, s in zip(graphs, streams):
        with torch.cuda.stream(s):
            graph.replay()
    torch.cuda.synchronize()
    for result in results:
        assert all(torch.equal(a, b) for a, b in zip(result, want))
    with pytest.raises(RuntimeError, match="captured"):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            D.neighbor_index(ei, 300, 350)
    assert D.neighbor_index(ei, 300, 350).num_edges == 9000


def test_gradients_of_tensors_that_hooks_moved(cuda):
    """Saved tensors that went to the host and came back elsewhere, dense: the backward passes read them where they are then."""
    ei, src, dst, q, k, v, b, g = _attention_case(RAGGED, 60, 4, 2, 16, torch.float32, True, 12)
    index = D.neighbor_index(ei, q.size(0), k.size(0))
    wide = torch.cat([k, v], dim=2)
    k, v = wide[..., :16], wide[..., 16:]
    kinds = _kinds(60, 3, 1).to(cuda)
    tall, w = D.type_index(kinds, 3), torch.randn(3, 32, 16, device=cuda, requires_grad=True)
    r, table = torch.rand(ei.size(1), device=cuda).mul_(5).requires_grad_(), torch.randn(12, 4, device=cuda, requires_grad=True)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    x = torch.randn(60, 64, device=cuda)[:, ::2].requires_grad_()

    def grads(moved):
        if moved:
            with torch.autograd.graph.save_on_cpu():
                out, y = D.neighbor_attention(*leaves, index, D.distance_bias(r, table, 5.0)), D.type_linear(x, w, tall)
            junk = [torch.full((1 << 16,), float("nan"), device=cuda) for _ in range(20)]   # where the tensors were
            del junk
        else:
            out, y = D.neighbor_attention(*leaves, index, D.distance_bias(r, table, 5.0)), D.type_linear(x, w, tall)
        return torch.autograd.grad([out, y], [*leaves, r, table, x, w], [g, torch.ones_like(y)])

    assert all(torch.equal(a, c) for a, c in zip(grads(False), grads(True)))


def test_a_wait_that_ran_out_is_told_at_the_next_call(cuda):
    """The word that a kernel sets when one of its bounded waits runs out (set from the host here): the next call raises, the one behind it works."""
    from dynamis_b200 import message

    index = D.type_index(torch.tensor([0, 1, 1], device=cuda), 2)
    x, w = torch.randn(3, 8, device=cuda), torch.randn(2, 8, 4, device=cuda)
    y = D.type_linear(x, w, index)
    torch.cuda.synchronize()
    message._STATUS[x.device.index][0].value = 1
    with pytest.raises(RuntimeError, match="ran out"):
        D.type_linear(x, w, index)
    assert torch.equal(D.type_linear(x, w, index), y)

"""Message-passing operators at the borders of what they promise: bytes behind a result, large and small values, calls without gradients, captures.
The bounds are derived beside the tests."""

import ctypes
import math
import threading

import pytest
import torch

import dynamis_b200 as D
from dynamis_b200 import _lib
from tests import _message as M

pytestmark = pytest.mark.gpu
U = M.U


# ------------------------------------------------------------------------------------------------ lists
@pytest.mark.parametrize("sources", [3000, 17_000_000])
def test_plan_writes_sixteen_bytes_to_the_host(cuda, sources):
    """The words of the plan are four of 32 bits: what stands behind them in the caller's pinned memory stays.  (Both ways to the host: from the
    scan's last block, and by a kernel of its own where the scan has many tiles.)"""
    L, n = _lib.lib(), ctypes.c_int64()
    degrees = [3, 0, 5, 1]
    ei, src, dst = M.ragged_graph(degrees, 3000, 1, cuda)
    E, T = ei.size(1), len(degrees)
    words = torch.full((64,), -7, dtype=torch.int64).pin_memory()
    rows, row_start, src32, cols, col_start, in_edge = (torch.empty(m, dtype=torch.int32, device=cuda) for m in (T, T + 1, E, sources, sources + 1, E))
    _lib.check(L.dynb_neighbor_index_workspace_bytes(E, T, sources, 0, ctypes.byref(n)), "workspace_bytes")
    ws = torch.empty(n.value, dtype=torch.uint8, device=cuda)
    _lib.check(L.dynb_neighbor_index_plan(ei[0].data_ptr(), ei[1].data_ptr(), E, T, sources, rows.data_ptr(), row_start.data_ptr(), src32.data_ptr(),
                                          cols.data_ptr(), col_start.data_ptr(), in_edge.data_ptr(), words.data_ptr(), ws.data_ptr(), ws.numel(),
                                          _lib.stream_of(cuda)), "plan")
    torch.cuda.synchronize()
    assert int(words[0]) & 0xFFFFFFFF == 0 and int(words[0]) >> 32 == int(torch.bincount(src).max())
    assert (words[2:] == -7).all()
    assert src32.tolist() == src.tolist() and row_start.tolist() == [0] + torch.cumsum(torch.bincount(dst, minlength=T)[rows.long()], 0).tolist()


def test_weights_gradient_with_a_workspace_off_sixteen_bytes(cuda):
    """The sums of stretches go to a workspace on any 4-byte boundary, by whole pieces where it allows."""
    L, n = _lib.lib(), ctypes.c_int64()
    x, w, g = (torch.randn(*s, device=cuda) for s in ((300, 64), (2, 64, 32), (300, 32)))
    index = D.type_index((torch.arange(300, device=cuda) % 2), 2)
    a = _lib.TypeLinear()
    a.weight_dev, a.order_dev, a.start_dev = w.data_ptr(), index.order.data_ptr(), index.start.data_ptr()
    a.n_rows, a.types, a.inner, a.outer, a.dtype = 300, 2, 64, 32, _lib.DYNB_F32
    _lib.check(L.dynb_type_linear_workspace_bytes(ctypes.byref(a), ctypes.byref(n)), "workspace_bytes")
    got = []
    for off in (0, 4):
        ws, dw, db = torch.empty(n.value + 16, dtype=torch.uint8, device=cuda), torch.empty_like(w), torch.empty(2, 32, device=cuda)
        _lib.check(L.dynb_type_linear_backward(ctypes.byref(a), x.data_ptr(), 64, g.data_ptr(), 32, None, dw.data_ptr(), db.data_ptr(),
                                               ws.data_ptr() + off, n.value, _lib.stream_of(cuda)), "backward")
        torch.cuda.synchronize()
        got.append((dw, db))
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])


# ------------------------------------------------------------------------------------------------ distance bias
@pytest.mark.parametrize("buckets,heads,smooth", [(64, 8, False), (300, 8, False), (300, 8, True), (1024, 8, False), (1024, 3, True), (1000, 40, False)])
def test_distance_bias_keeps_its_place_among_many_buckets(cuda, buckets, heads, smooth):
    """The place between two buckets is off by 2 u (the sum of its exact leading part and a small one, and that small one's own roundings) however many
    buckets stand below it: no bound here grows with the place.  Bias: the spline's slope is at most 2 of the largest value nearby (reach), its products and
    weights are off by 12 u of their magnitudes, the logarithms as in test_message_gpu.py.  d_dist: the second derivative is at most 4 reach a bucket,
    the weights' derivatives are off by 8 u twice over, sums of heads.  d_table: the weights' slopes are at most 0.75."""
    gen, cutoff, edges = torch.Generator(device="cuda").manual_seed(buckets + heads), 5.0, 20011
    r = 5.0 * torch.rand(edges, generator=gen, device="cuda")
    r[:3] = torch.stack([torch.nextafter(torch.tensor(cutoff), torch.tensor(0.0)), torch.tensor(0.0), torch.tensor(cutoff / (buckets - 3))])
    table = torch.randn(buckets, heads, generator=gen, device="cuda")
    g = torch.randn(edges, heads, generator=gen, device="cuda")
    leaves = [r.requires_grad_(), table.requires_grad_()]
    bias = D.distance_bias(*leaves, cutoff, smooth)
    d_dist, d_table = torch.autograd.grad(bias, leaves, g)
    rd, td = r.detach().double(), table.detach().double()
    x = rd / cutoff * (buckets - 3)
    at = x.long().clamp(0, buckets - 4)
    t = x - at
    near = torch.stack([td[at + j] for j in range(4)])
    w = torch.stack([(1 - t) ** 3, 3 * t ** 3 - 6 * t ** 2 + 4, -3 * t ** 3 + 3 * t ** 2 + 3 * t + 1, t ** 3]) / 6
    dw = torch.stack([-(1 - t) ** 2, 3 * t ** 2 - 4 * t, -3 * t ** 2 + 2 * t + 1, t ** 2]) / 2
    reach = near.abs().amax(0)
    value = (w[..., None] * near).sum(0)
    slack = 12 * U * (w[..., None] * near.abs()).sum(0) + 2 * reach * 2 * U
    slope = (dw[..., None] * near).sum(0) * (buckets - 3)
    pull = torch.zeros_like(rd)[:, None]
    if smooth:
        u = rd / cutoff
        logs = (3 * torch.log1p(-u).abs() + torch.log1p(3 * u + 6 * u * u))[:, None]
        value = value + (3 * torch.log1p(-u) + torch.log1p(3 * u + 6 * u * u))[:, None]
        slack = slack + 8 * U * logs + 14 * U
        pull = (30 * u * u / ((1 - u) * (1 + 3 * u + 6 * u * u)))[:, None]
    M.check(bias.detach(), value, slack + 4 * U * value.abs(), "bias")
    G, gd = g.double().abs(), g.double()
    size = (buckets - 3) * 2 * reach + pull
    off = (buckets - 3) * reach * (4 * 2 + 16) * U + 12 * U * pull
    M.check(d_dist, (gd * (slope - pull)).sum(1) / cutoff, (G * (off + (heads + 4) * U * size)).sum(1) / cutoff, "d_dist")
    want, w_off = torch.zeros_like(td), torch.zeros_like(td)
    per = (edges + 147) // 148 + 40
    for j in range(4):
        want.index_add_(0, at + j, w[j][:, None] * gd)
        w_off.index_add_(0, at + j, G * (0.75 * 2 + 8 + per) * U)
    M.check(d_table, want, w_off, "d_table")


@pytest.mark.parametrize("edges,buckets,heads", [(1000, 64, 8), (5000, 64, 1), (777, 17, 33), (30, 1024, 3), (4000, 700, 8)])
def test_distance_bias_wants_some_gradients_only(cuda, edges, buckets, heads):
    gen = torch.Generator(device="cuda").manual_seed(edges)
    r, table = 5.2 * torch.rand(edges, generator=gen, device="cuda"), torch.randn(buckets, heads, generator=gen, device="cuda")
    g = torch.randn(edges, heads, generator=gen, device="cuda")
    both = [t.detach().requires_grad_() for t in (r, table)]
    every = torch.autograd.grad(D.distance_bias(*both, 5.0), both, g)
    for i in range(2):
        some = [t if j == i else t.detach() for j, t in enumerate(both)]
        assert torch.equal(torch.autograd.grad(D.distance_bias(*some, 5.0), [both[i]], g)[0], every[i])


# ------------------------------------------------------------------------------------------------ products by type
def test_a_wait_that_ran_out_in_a_replay_is_told(cuda, monkeypatch):
    """Making the index makes the word, so that the first product may be a captured one; behind a replay the index tells (the word is set from the host here)."""
    from dynamis_b200 import message

    monkeypatch.setattr(message, "_STATUS", {})
    index = D.type_index(torch.tensor([0, 1, 1], device=cuda), 2)
    x, w = torch.randn(3, 8, device=cuda), torch.randn(2, 8, 4, device=cuda)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = D.type_linear(x, w, index)
    graph.replay()
    index.check_status()
    M.check(y, torch.stack([x[0].double() @ w[0].double(), *(x[1:].double() @ w[1].double())]), 25 * U * torch.full((3, 4), 8.0, device=cuda) * x.abs().max() * w.abs().max(), "y")
    message._STATUS[x.device.index][0].value = 1
    with pytest.raises(RuntimeError, match="ran out"):
        index.check_status()
    index.check_status()
    # lists made by hand under a capture, on a device without a word: refused, and the next call answers
    monkeypatch.setattr(message, "_STATUS", {})
    with pytest.raises(RuntimeError, match="before a capture"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            D.type_linear(x, w, D.TypeIndex(index.order, index.start))
    assert torch.equal(D.type_linear(x, w, D.TypeIndex(index.order, index.start)), y)


# ------------------------------------------------------------------------------------------------ lists made by hand
def test_lists_made_by_hand_are_looked_at(cuda):
    ei, src, dst = M.ragged_graph([3, 0, 4, 2], 6, 3, cuda)
    good = D.neighbor_index(ei, 4, 6)
    good.check_lists()
    names = ("rows", "row_start", "src", "cols", "col_start", "in_edge", "in_dst")

    def changed(match, name, at, to):
        lists = {n: getattr(good, n).clone() for n in names}
        lists[name][at] = to
        with pytest.raises(RuntimeError, match=match):
            D.NeighborIndex(**lists).check_lists()

    changed("rows must name", "rows", 0, int(good.rows[1]))
    changed("rows must name", "rows", 0, 4)
    changed("cols must name", "cols", 2, -1)
    changed("in_edge must name", "in_edge", 3, int(good.in_edge[4]))
    changed("row_start must rise", "row_start", 0, 1)
    changed("row_start must rise", "row_start", 4, 8)
    changed("row_start must rise", "row_start", 1, 1 + int(good.row_start[2]))
    changed("col_start must rise", "col_start", 6, 10)
    changed("src must lie", "src", 5, 6)
    other = (int(good.src[0]) + 1) % 6
    changed("in_edge must list", "src", 0, other)
    changed("in_dst must hold", "in_dst", 0, (int(good.in_dst[0]) + 1) % 4)
    for T, S in ((0, 0), (0, 5), (4, 0)):
        D.neighbor_index(torch.empty((2, 0), dtype=torch.int64, device=cuda), T, S).check_lists()

    types = D.type_index(torch.tensor([2, 0, 2, 0], device=cuda), 4)
    types.check_lists()
    D.type_index(torch.empty(0, dtype=torch.int64, device=cuda), 3).check_lists()
    for order, start, match in (([1, 3, 0, 0], [0, 2, 2, 4, 4], "order must name"), ([1, 3, 0, 4], [0, 2, 2, 4, 4], "order must name"),
                                ([1, 3, 0, 2], [0, 2, 2, 3, 3], "start must rise"), ([1, 3, 0, 2], [1, 2, 2, 4, 4], "start must rise"),
                                ([1, 3, 0, 2], [0, 3, 2, 4, 4], "start must rise")):
        with pytest.raises(RuntimeError, match=match):
            D.TypeIndex(*(torch.tensor(t, dtype=torch.int32, device=cuda) for t in (order, start))).check_lists()


# ------------------------------------------------------------------------------------------------ attention
def test_attention_of_a_single_row_with_any_stride(cuda):
    """A dimension of one element may carry any stride: a row stride beyond what the kernels take is of no meaning here."""
    index = D.neighbor_index(torch.zeros((2, 1), dtype=torch.int64, device=cuda), 1, 1)
    base = torch.randn(3, 2, 8, device=cuda)
    q, k, v = (torch.as_strided(base, (1, 2, 8), (1 << 30, 8, 1), 16 * i) for i in range(3))
    assert q.stride(0) == 1 << 30
    assert torch.equal(D.neighbor_attention(q, k, v, index), base[2:])   # one edge: its values
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    g = torch.as_strided(torch.randn(16, device=cuda), (1, 2, 8), (1 << 30, 8, 1))
    grads = torch.autograd.grad(D.neighbor_attention(*leaves, index), leaves, g)
    # bounds beside the plain form: by source the logit is rounded in another order than the largest logit was, so that p is not exactly 1 there
    zero = torch.zeros(1, dtype=torch.int64, device=cuda)
    ref = M.attention(q, k, v, zero, zero, None, 8 ** -0.5, g)
    for name, got in zip(("dq", "dk", "dv"), grads):
        M.check(got, *ref[name], name)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attention_of_broadcast_operands(cuda, dtype):
    """One row of keys for all sources, one head of values for all heads, one row of the result's gradient for all targets, read where they are: the bits of the
    dense tensors."""
    gen, T, S = torch.Generator(device="cuda").manual_seed(2), 14, 60
    ei, _, _ = M.ragged_graph([0, 1, 2, 3, 31, 32, 33, 0, 64, 129, 5, 70, 0, 7], S, 4, cuda)
    index = D.neighbor_index(ei, T, S)
    q, k, v, g = (torch.randn(*s, generator=gen, device="cuda").to(M.TYPES[dtype]) for s in ((T, 4, 16), (1, 2, 16), (S, 1, 16), (1, 4, 16)))
    wide = [q, k.expand(S, 2, 16), v.expand(S, 2, 16), g.expand(T, 4, 16)]
    results = []
    for q, k, v, g in (wide, [t.contiguous() for t in wide]):
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        out = D.neighbor_attention(*leaves, index)
        results.append((out, *torch.autograd.grad(out, leaves, g)))
    assert all(torch.equal(a, b) for a, b in zip(*results))


def test_attention_refuses_a_scale_beyond_single_precision(cuda):
    index = D.neighbor_index(torch.zeros((2, 1), dtype=torch.int64, device=cuda), 1, 1)
    q = torch.ones(1, 1, 4, device=cuda)
    for scale in (1e39, -1e300, math.inf, math.nan):
        with pytest.raises(RuntimeError, match="scale must be finite"):
            D.neighbor_attention(q, q, q, index, None, scale)
    assert torch.equal(D.neighbor_attention(q, q, q, index, None, 1e30), q)


def test_attention_without_gradients_keeps_nothing_for_them(cuda):
    """Under no_grad the operands of a trained model still ask for gradients: no unrounded result and no statistics are written then (three times the
    memory of a result in 16 bits)."""
    ei, _, _ = M.ragged_graph([2] * 4000, 4000, 1, cuda)
    index = D.neighbor_index(ei, 4000, 4000)
    leaves = [torch.randn(4000, 8, 32, device=cuda).bfloat16().requires_grad_() for _ in range(3)]
    want = D.neighbor_attention(*leaves, index).detach()
    for mode in (torch.no_grad, torch.inference_mode):
        with mode():
            torch.cuda.synchronize()
            torch.cuda.reset_peak_memory_stats()
            before = torch.cuda.memory_allocated()
            out = D.neighbor_attention(*leaves, index)
            assert torch.cuda.max_memory_allocated() - before <= want.numel() * 2 + (1 << 16)
        assert torch.equal(out, want) and not out.requires_grad
    grads = torch.autograd.grad(D.neighbor_attention(*leaves, index), leaves, torch.ones_like(want))
    with torch.no_grad():
        again = [t.detach() for t in leaves]
    again[1].requires_grad_()     # only one of them asks
    assert torch.equal(torch.autograd.grad(D.neighbor_attention(*again, index), [again[1]], torch.ones_like(want))[0], grads[1])


def test_type_linear_cuts_a_sum_off_once_a_step(cuda):
    """Operands of one sign in float32: the tensor cores cut a sum off towards zero at every addition, by half of its last place on average, which is at most
    2^-23 of it.  Partial sums grow evenly, so over n steps of 16 products one addition a step costs at most (n + 1) / 4 * 2^-23 of the whole on average.  The
    products that are left out and the other roundings have either sign and are below 2^-24.  n: 16 for 256 summed columns, 64 for a stretch of 1024 rows.
    Bounds 5.7e-7 and 2.0e-6; measured 3.1e-7 and 1.7e-6, and with all six part-products of a step in one sum 1.4e-6 and 4.1e-6, which must not pass."""
    gen = torch.Generator(device="cuda").manual_seed(41)
    rows, wide = 152_000, 256
    kinds = (torch.arange(rows, device="cuda") * 7 % 3 == 0).long()
    x, w, g = (torch.rand(*s, generator=gen, device="cuda") for s in ((rows, wide), (2, wide, wide), (rows, wide)))
    leaves = [t.requires_grad_() for t in (x, w)]
    y = D.type_linear(x, w, D.type_index(kinds, 2)).detach()
    dx, dw = torch.autograd.grad(D.type_linear(x, w, D.type_index(kinds, 2)), leaves, g)
    xd, wd, gd = x.detach().double(), w.detach().double(), g.double()
    lost = {"y": [], "dx": [], "dw": []}
    for t in range(2):
        m = torch.nonzero(kinds == t)[:, 0]
        for name, got, ref in (("y", y[m], xd[m] @ wd[t]), ("dx", dx[m], gd[m] @ wd[t].T), ("dw", dw[t], xd[m].T @ gd[m])):
            lost[name].append(float(((ref - got.double()) / ref).mean()))
    for name, values in lost.items():
        n = 64 if name == "dw" else 16
        assert all(-2.0 ** -24 <= v <= (n + 1) / 4 * 2.0 ** -23 + 2.0 ** -24 for v in values), (name, values)


def _same_kinds(got, want, off, what):
    """NaN where the 64-bit form has NaN, infinities of its sign where it has them, and the rest within the bounds."""
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    inf = torch.isinf(want)
    assert torch.equal(torch.isinf(got), inf) and torch.equal(got[inf].double(), want[inf]), what
    ok = torch.isfinite(want)
    M.check(torch.where(ok, got, 0.0), torch.where(ok, want, 0.0), torch.where(ok, off, 0.0), what)


@pytest.mark.parametrize("inner,outer", [(64, 48), (33, 130), (300, 40), (40, 1200)])
def test_type_linear_infinities_and_the_largest_numbers(cuda, inner, outer):
    """float32 operands with infinities, NaN and numbers that round to an infinity in 8 bits, in rows, matrices and gradients: what 64 bits give, whatever the width (the
    last two are beyond the tensor cores forward and back).  Bounds as in test_message_gpu.py: the parts of the largest numbers leave out 2^-25."""
    gen, top = torch.Generator(device="cuda").manual_seed(inner), torch.finfo(torch.float32).max
    kinds = torch.arange(500, device="cuda") % 3

    def away(*shape):      # no zeros: infinity times zero would be a NaN on both sides, and is tested by hand below
        t = torch.rand(*shape, generator=gen, device="cuda") * 0.1 + 0.05
        return torch.where(torch.rand(*shape, generator=gen, device="cuda") < 0.5, -t, t)

    for what in ("x", "w", "g"):
        x, w, g = away(500, inner), away(3, inner, outer), away(500, outer)
        odd = {"x": x, "w": w.view(-1, outer), "g": g}[what]
        odd[4, 3], odd[7, 5], odd[9, 2], odd[9, 6], odd[13, 1], odd[16, 0] = math.inf, -math.inf, math.inf, -math.inf, top, -top
        odd[19, 4], odd[22, 7], odd[25, 9] = math.nan, 3.395e38, 3.3895e38
        odd[28, 2:10] = torch.tensor([1.0, -1.0, 2.0, -2.0, 0.5, -0.5, 0.25, -0.25], device="cuda") * 2.0 ** 127 * 0.1
        leaves = [x.requires_grad_(), w.requires_grad_()]
        y = D.type_linear(x, w, D.type_index(kinds, 3))
        dx, dw = torch.autograd.grad(y, leaves, g)
        xd, wd, gd = x.detach().double(), w.detach().double(), g.double()
        for t in range(3):
            m = torch.nonzero(kinds == t)[:, 0]
            for got, a, b, name in ((y.detach()[m], xd[m], wd[t], "y"), (dx[m], gd[m], wd[t].T, "dx"), (dw[t], xd[m].T, gd[m], "dw")):
                ref = (a[:, :, None] * b[None]).sum(1) if a.size(0) * a.size(1) * b.size(1) < 40_000_000 else a @ b
                _same_kinds(got, ref, (a.size(1) + 17) * U * (a.abs() @ b.abs()), f"{name} with odd {what}")
    # an infinity times zero is a NaN, two infinities meet in one
    x, w = torch.zeros(2, 32, device="cuda"), torch.ones(1, 32, 16, device="cuda")
    x[0, 3], w[0, 3, 1], w[0, 3, 2] = math.inf, 0.0, -math.inf
    y = D.type_linear(x, w, D.type_index(torch.zeros(2, dtype=torch.int64, device="cuda"), 1))
    assert y[0, 0] == math.inf and torch.isnan(y[0, 1]) and y[0, 2] == -math.inf and torch.isnan(y[1, 2]) and y[1, 0] == 0


@pytest.mark.parametrize("inner,outer", [(64, 48), (256, 64)])
def test_type_linear_of_the_smallest_numbers(cuda, inner, outer):
    """float32 operands below 2^-109 have parts below the smallest steps of bfloat16, 2^-133, and are taken to within that; above, whole.  Beside bounds as in
    test_message_gpu.py every product may be off by 2^-133 of its other operand."""
    gen = torch.Generator(device="cuda").manual_seed(outer)
    kinds = torch.arange(300, device="cuda") % 2
    for power in (-100, -108, -116, -124, -130):
        x = (torch.randn(300, inner, generator=gen, device="cuda").double() * 2.0 ** power).float()
        w = torch.randn(2, inner, outer, generator=gen, device="cuda") * 2.0 ** 100
        y = D.type_linear(x, w, D.type_index(kinds, 2))
        for t in range(2):
            m = torch.nonzero(kinds == t)[:, 0]
            M.check(y[m], x[m].double() @ w[t].double(), (inner + 17) * U * (x[m].double().abs() @ w[t].double().abs()) + 2.0 ** -133 * w[t].double().abs().sum(0), f"y at 2^{power}")


# ------------------------------------------------------------------------------------------------ threads
class _Wait:
    """A stream behind whose first wait another thread makes a call on the same stream, before the waiting one goes on."""

    def __init__(self, stream, pending):
        self.stream, self.pending = stream, pending

    def __getattr__(self, name):
        return getattr(self.stream, name)

    def synchronize(self):
        self.stream.synchronize()
        if self.pending:
            t = threading.Thread(target=self.pending.pop())
            t.start()
            t.join()


@pytest.mark.parametrize("hub", [False, True])
def test_neighbor_index_beside_another_thread(cuda, monkeypatch, hub):
    """Between the two phases of the lists another thread makes lists of another graph on the same stream: each gets its own."""
    mine = M.ragged_graph([5, 0, 700 if hub else 40, 3] * 3, 1 if hub else 90, 1, cuda)
    other = M.ragged_graph([9] * 50, 30, 2, cuda)
    got, pending, me, real = [], [], threading.get_ident(), torch.cuda.current_stream
    pending.append(lambda: got.append(D.neighbor_index(other[0], 50, 30)))
    monkeypatch.setattr(torch.cuda, "current_stream", lambda dev=None: _Wait(real(dev), pending) if threading.get_ident() == me else real(dev))
    index = D.neighbor_index(mine[0], 12, 1 if hub else 90)
    assert not pending
    for lists, (_, src, dst), T, S in ((index, mine, 12, 1 if hub else 90), (got[0], other, 50, 30)):
        for name, want in M.index_lists(src, dst, T, S).items():
            assert getattr(lists, name).tolist() == want, name

"""CPU tests of rotary heads, routing and the experts' products: refusals that need no GPU, and the plain forms that the GPU tests compare with."""

import ctypes
import math

import pytest
import torch

import dynamis_b200 as D
from dynamis_b200 import _lib
from tests import _experts as X


def test_python_refuses_host_tensors():
    f, i = torch.zeros(4, 2, 8), torch.zeros(4, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="q must be a CUDA tensor"):
        D.rotary_heads(f, f, torch.zeros(4, 3), torch.zeros(4, 3))
    with pytest.raises(RuntimeError, match="logits must be a CUDA tensor"):
        D.route_experts(torch.zeros(4, 8), 2)
    with pytest.raises(RuntimeError, match="experts must be a contiguous CUDA tensor"):
        D.Routing(i.view(2, 2), torch.zeros(2, 2), i, i)
    with pytest.raises(RuntimeError, match="routing must be a Routing"):
        D.expert_linear(torch.zeros(3, 4), torch.zeros(2, 4, 4), None)
    with pytest.raises(RuntimeError, match="routing must be a Routing"):
        D.expert_combine(f, None)


def _set(a, values, change):
    for name, value in {**values, **change}.items():
        setattr(a, name, value)
    return a


def _rotary(**change):
    return _set(_lib.Rotary(), dict(n_q=3, n_k=4, heads=4, kv_heads=2, dim=16, axes=3, dtype=_lib.DYNB_F32, pos_dtype=_lib.DYNB_F32, norm=1, eps=1e-6), change)


@pytest.mark.parametrize("change", [{"dtype": _lib.DYNB_F64}, {"pos_dtype": _lib.DYNB_F16}, {"n_q": -1}, {"n_k": 2 ** 31}, {"heads": 0}, {"kv_heads": 65536}, {"dim": 15},
                                    {"dim": 0}, {"dim": 258}, {"axes": 0}, {"axes": 4}, {"eps": -1.0}, {"eps": math.nan}, {"eps": math.inf}, {}])
def test_rotary_entry_refuses(change):
    """The last case: null pointers."""
    L, a, n = _lib.lib(), _rotary(**change), ctypes.c_int64()
    assert L.dynb_rotary_heads(ctypes.byref(a), None, None, None) == -1
    assert L.dynb_rotary_heads_backward(ctypes.byref(a), None, 0, 0, None, 0, 0, None, None, None, None, None, None, 0, None) == -1
    assert L.dynb_rotary_heads(None, None, None, None) == -1
    assert L.dynb_rotary_heads_workspace_bytes(None, ctypes.byref(n)) == -1


def test_rotary_entry_checks_its_workspace():
    L, at, n = _lib.lib(), 4096, ctypes.c_int64()
    a = _rotary(q_dev=at, k_dev=at, pos_dev=at, wave_dev=at)
    assert L.dynb_rotary_heads_workspace_bytes(ctypes.byref(a), ctypes.byref(n)) == 0 and n.value >= 2 * 16 * 4
    assert L.dynb_rotary_heads_backward(ctypes.byref(a), at, 64, 16, at, 32, 16, None, None, None, at, None, None, 0, None) == -1
    assert L.dynb_rotary_heads_backward(ctypes.byref(a), at, 64, 16, at, 32, 16, None, None, None, at, None, at, n.value - 1, None) == -1
    assert b"workspace" in L.dynb_last_error()


def _routing(**change):
    return _set(_lib.RoutingArgs(), dict(n_rows=5, experts=8, choices=2, dtype=_lib.DYNB_F32, score=0, groups=1, kept_groups=1, renormalize=1, scale=1.0), change)


@pytest.mark.parametrize("change", [{"dtype": _lib.DYNB_F64}, {"experts": 0}, {"experts": 1025}, {"choices": 0}, {"choices": 9}, {"experts": 64, "choices": 33}, {"n_rows": -1},
                                    {"n_rows": 2 ** 30}, {"groups": 3}, {"groups": 0}, {"groups": 4, "kept_groups": 5}, {"kept_groups": 0}, {"score": 2}, {"scale": 0.0},
                                    {"scale": math.nan}, {}])
def test_routing_entry_refuses(change):
    """The last case: null pointers."""
    L, a = _lib.lib(), _routing(**change)
    assert L.dynb_route_experts(ctypes.byref(a), None, None, None, None, None, 0, None) == -1
    assert L.dynb_route_experts_backward(ctypes.byref(a), None, None, None, None, None) == -1
    assert L.dynb_route_experts(None, None, None, None, None, None, 0, None) == -1


def test_routing_entry_checks_its_workspace():
    L, at, n = _lib.lib(), 4096, ctypes.c_int64()
    a = _routing(logits_dev=at, logits_row=8)
    assert L.dynb_route_experts_workspace_bytes(ctypes.byref(a), ctypes.byref(n)) == 0 and n.value >= 4 * 9
    assert L.dynb_route_experts(ctypes.byref(a), at, at, at, at, at, n.value - 1, None) == -1 and b"workspace" in L.dynb_last_error()
    assert L.dynb_route_experts(ctypes.byref(a), at, at, at, at, at + 2, n.value, None) == -1 and b"4-byte" in L.dynb_last_error()


def _linear(**change):
    return _set(_lib.ExpertLinear(), dict(n_rows=5, choices=2, experts=3, inner=8, outer=4, dtype=_lib.DYNB_F32), change)


@pytest.mark.parametrize("change", [{"dtype": _lib.DYNB_F64}, {"choices": 0}, {"choices": 33}, {"n_rows": -1}, {"n_rows": 2 ** 30}, {"experts": 0}, {"experts": 1025},
                                    {"inner": 0}, {"outer": 16385}, {"activation": 3}, {"activation": -1}, {}])
def test_linear_entry_refuses(change):
    """The last case: null pointers."""
    L, a, n = _lib.lib(), _linear(**change), ctypes.c_int64()
    assert L.dynb_expert_linear(ctypes.byref(a), None, 8, None, None, None, None, 0, None) == -1
    assert L.dynb_expert_linear_backward(ctypes.byref(a), None, 8, None, 4, None, None, None, None, None, None, 0, None) == -1
    assert L.dynb_expert_linear_workspace_bytes(ctypes.byref(a), 1, 1, 1, ctypes.byref(n)) == -1
    assert L.dynb_expert_linear(None, None, 8, None, None, None, None, 0, None) == -1


def test_linear_entry_checks_its_workspace():
    L, at, n = _lib.lib(), 4096, ctypes.c_int64()
    a = _linear(weight_dev=at, order_dev=at, start_dev=at, activation=1)
    assert L.dynb_expert_linear_workspace_bytes(ctypes.byref(a), 0, 0, 0, ctypes.byref(n)) == 0 and n.value > 0
    for ws, size in ((None, 0), (at, n.value - 1), (at + 8, n.value)):
        assert L.dynb_expert_linear(ctypes.byref(a), at, 8, None, at, None, ws, size, None) == -1 and b"workspace" in L.dynb_last_error()
    assert L.dynb_expert_linear_workspace_bytes(ctypes.byref(a), 1, 1, 1, ctypes.byref(n)) == 0 and n.value > 0
    args = (ctypes.byref(a), at, 8, at, 4, at, at, at, at, at)
    assert L.dynb_expert_linear_backward(*args, None, 0, None) == -1
    assert L.dynb_expert_linear_backward(*args, at, n.value - 1, None) == -1 and b"workspace" in L.dynb_last_error()
    assert L.dynb_expert_linear_backward(*args, at + 8, n.value, None) == -1
    assert L.dynb_expert_linear_backward(ctypes.byref(a), at, 8, at, 4, None, at, at, at, at, at, n.value, None) == -1   # an activation without its slopes


def test_linear_entry_checks_the_workspace_of_rows_off_16_bytes():
    L, at, n = _lib.lib(), 4096, ctypes.c_int64()
    a = _linear(weight_dev=at, order_dev=at, start_dev=at, outer=16, activation=1)
    sizes = {}
    for back in (0, 1):
        for flags in range(4):
            a.unaligned = flags
            assert L.dynb_expert_linear_workspace_bytes(ctypes.byref(a), back, 1, 1, ctypes.byref(n)) == 0
            sizes[back, flags] = n.value
    assert sizes[0, 0] == sizes[0, 2] < sizes[0, 1] and sizes[1, 0] < sizes[1, 1]
    for x, row in ((at + 4, 8), (at, 9)):
        assert L.dynb_expert_linear(ctypes.byref(a), x, row, None, at, None, at, sizes[0, 0], None) == -1 and b"workspace" in L.dynb_last_error()
        assert L.dynb_expert_linear_backward(ctypes.byref(a), x, row, at, 16, at, at, at, at, at, at, sizes[1, 0], None) == -1 and b"workspace" in L.dynb_last_error()
    a.activation = 0                                   # without slopes no rows of d_z are kept, unless they are copied
    a.unaligned = 0
    assert L.dynb_expert_linear_workspace_bytes(ctypes.byref(a), 1, 1, 1, ctypes.byref(n)) == 0
    assert L.dynb_expert_linear_backward(ctypes.byref(a), at, 8, at, 17, None, at, at, at, at, at, n.value, None) == -1 and b"workspace" in L.dynb_last_error()


@pytest.mark.parametrize("n,choices,width,dtype", [(-1, 2, 8, 0), (3, 0, 8, 0), (3, 33, 8, 0), (2 ** 30, 2, 8, 0), (3, 2, 0, 0), (3, 2, 16385, 0), (3, 2, 8, 1), (3, 2, 8, 0)])
def test_combine_entry_refuses(n, choices, width, dtype):
    """The last case: null pointers."""
    L = _lib.lib()
    assert L.dynb_expert_combine(None, None, None, None, 0, n, choices, width, dtype, None, None) == -1
    assert L.dynb_expert_combine_backward(None, None, None, None, 0, n, choices, width, dtype, 4096, None, None) == -1


def test_empty_calls_launch_nothing():
    L = _lib.lib()
    a = _rotary(n_q=0, n_k=0)
    assert L.dynb_rotary_heads(ctypes.byref(a), None, None, None) == 0
    assert L.dynb_rotary_heads_backward(ctypes.byref(a), None, 0, 0, None, 0, 0, None, None, None, None, None, None, 0, None) == 0
    assert L.dynb_route_experts_backward(ctypes.byref(_routing(n_rows=0)), None, None, None, None, None) == 0
    b = _linear(n_rows=0, weight_dev=4096, start_dev=4096)
    assert L.dynb_expert_linear(ctypes.byref(b), None, 8, None, None, None, None, 0, None) == 0
    assert L.dynb_expert_linear_backward(ctypes.byref(b), None, 8, None, 4, None, None, 4096, None, None, None, 0, None) == 0
    assert L.dynb_expert_combine(None, None, None, None, 0, 0, 2, 8, 0, None, None) == 0


# ------------------------------------------------------------------------------------------------ the plain forms themselves
def _differences(value, leaves, grads, step=1e-5, limit=1e-7):
    """Central differences: third derivatives times step^2 and 2^-53 / step, both below 1e-8 for the functions here."""
    for name, t in leaves.items():
        flat = t.view(-1)
        for at in range(0, flat.numel(), max(flat.numel() // 9, 1)):
            keep = float(flat[at])
            flat[at] = keep + step
            up = value()
            flat[at] = keep - step
            down = value()
            flat[at] = keep
            assert abs((up - down) / (2 * step) - float(grads[name].reshape(-1)[at])) < limit, name


@pytest.mark.parametrize("eps,interleaved", [(1e-3, False), (1e-3, True), (None, False)])
def test_plain_rotary_gradients_against_differences(eps, interleaved):
    gen = torch.Generator().manual_seed(3)
    q, k, d_q, d_k = (torch.randn(n, h, 6, generator=gen, dtype=torch.float64) for n, h in ((4, 3), (5, 2), (4, 3), (5, 2)))
    pos, wave = torch.rand(5, 2, generator=gen, dtype=torch.float64), torch.randn(3, 2, generator=gen, dtype=torch.float64) * 0.3
    w = [torch.rand(6, generator=gen, dtype=torch.float64) + 0.5 for _ in range(2)] if eps is not None else [None, None]
    run = lambda: X.rotary(q, k, pos, wave, *w, eps, interleaved, d_q, d_k)  # noqa: E731
    value = lambda: float((run()["q"][0] * d_q).sum() + (run()["k"][0] * d_k).sum())  # noqa: E731
    r = run()
    leaves = {"d_q": q, "d_k": k, "d_pos": pos}
    if eps is not None:
        leaves.update(d_q_weight=w[0], d_k_weight=w[1])
    _differences(value, leaves, {n: r[n][0] for n in leaves})


def test_plain_rotary_products_depend_on_displacements_alone():
    gen = torch.Generator().manual_seed(4)
    q, k = (torch.randn(6, 2, 8, generator=gen, dtype=torch.float64) for _ in range(2))
    pos, wave = torch.rand(6, 3, generator=gen, dtype=torch.float64), torch.randint(-3, 4, (4, 3), generator=gen).double()
    dots = lambda p: (lambda r: torch.einsum("nhd,mhd->hnm", r["q"][0], r["k"][0]))(X.rotary(q, k, p, wave, None, None, 1e-6, False, q, k))  # noqa: E731
    moved = pos + torch.tensor([0.2, -0.7, 5.1], dtype=torch.float64)
    moved[3] += torch.tensor([1.0, -2.0, 0.0], dtype=torch.float64)       # another image of the box
    assert float((dots(pos) - dots(moved)).abs().max()) < 1e-12


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [True, False])
def test_plain_routing_gradients_against_differences(score, renormalize):
    gen = torch.Generator().manual_seed(6)
    logits, g = torch.randn(6, 8, generator=gen, dtype=torch.float64), torch.randn(6, 3, generator=gen, dtype=torch.float64)
    bias = torch.randn(8, generator=gen) * 0.1
    run = lambda: X.route(logits, 3, score, bias, 4, 2, renormalize, 1.7, g)  # noqa: E731
    _differences(lambda: float((run()["weights"][0] * g).sum()), {"d_logits": logits}, {"d_logits": run()["d_logits"][0]})


def test_plain_routing_closes_and_breaks_ties():
    inf = math.inf
    logits = torch.tensor([[1.0, 2.0, 2.0, 0.0], [-inf, -inf, 3.0, -inf], [-inf] * 4, [5.0, 5.0, 5.0, 5.0]])
    r = X.route(logits, 2)
    assert r["experts"].tolist() == [[1, 2], [2, -1], [-1, -1], [0, 1]]
    assert r["order"].tolist() == [6, 0, 7, 1, 2, 3, 4, 5] and r["start"].tolist() == [0, 1, 3, 5, 5]
    assert r["weights"][0][1].tolist() == [1.0, 0.0] and not r["weights"][0][2].any()


@pytest.mark.parametrize("activation", [None, "silu", "gelu"])
@pytest.mark.parametrize("paired", [False, True])
def test_plain_linear_gradients_against_differences(activation, paired):
    gen = torch.Generator().manual_seed(7)
    experts = X.routing_by_hand(7, 3, 2, 0.2, 5, "cpu")[0]
    x = torch.randn(*((7, 2) if paired else (7,)), 5, generator=gen, dtype=torch.float64)
    w, b, g = (torch.randn(*s, generator=gen, dtype=torch.float64) for s in ((3, 5, 4), (3, 4), (7, 2, 4)))
    run = lambda: X.linear(x, w, experts, b, activation, g)  # noqa: E731
    _differences(lambda: float((run()["z"][0] * g).sum()), {"d_x": x, "d_weight": w, "d_bias": b}, {n: run()[n][0] for n in ("d_x", "d_weight", "d_bias")})


def test_plain_combine_gradients_against_differences():
    gen = torch.Generator().manual_seed(8)
    experts, weights, _, _ = X.routing_by_hand(5, 4, 3, 0.3, 5, "cpu")
    weights = weights.double()
    z, r, g = (torch.randn(*s, generator=gen, dtype=torch.float64) for s in ((5, 3, 4), (5, 4), (5, 4)))
    run = lambda: X.combine(z, weights, experts, r, g)  # noqa: E731
    _differences(lambda: float((run()["y"][0] * g).sum()), {"d_z": z, "d_weights": weights}, {n: run()[n][0] for n in ("d_z", "d_weights")})

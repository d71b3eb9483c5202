"""CPU tests of the message-passing operators: refusals that need no GPU, and the plain forms that the GPU tests compare with."""

import ctypes
import math

import pytest
import torch

import dynamis_b200 as D
from dynamis_b200 import _lib
from tests import _message as M


def test_python_refuses_host_tensors():
    f, i = torch.zeros(4, 2, 8), torch.zeros(4, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="edge_index must be a CUDA tensor"):
        D.neighbor_index(torch.zeros(2, 3, dtype=torch.int64), 2, 2)
    with pytest.raises(RuntimeError, match="rows must be a CUDA tensor"):
        D.NeighborIndex(i, i, i, i, i, i, i)
    with pytest.raises(RuntimeError, match="index must be a NeighborIndex"):
        D.neighbor_attention(f, f, f, None)
    with pytest.raises(RuntimeError, match="dist must be a CUDA tensor"):
        D.distance_bias(torch.zeros(3), torch.zeros(8, 2), 5.0)
    with pytest.raises(RuntimeError, match="types must be a CUDA tensor"):
        D.type_index(torch.zeros(3, dtype=torch.int64), 2)
    with pytest.raises(RuntimeError, match="order must be a CUDA tensor"):
        D.TypeIndex(i, i)
    with pytest.raises(RuntimeError, match="index must be a TypeIndex"):
        D.type_linear(torch.zeros(3, 4), torch.zeros(2, 4, 4), None)


def _attention_args(**change):
    a = _lib.Attention()
    a.n_targets, a.n_sources, a.n_edges, a.heads, a.kv_heads, a.dim, a.dtype, a.scale = 4, 4, 4, 4, 2, 16, _lib.DYNB_F32, 0.25
    for name, value in change.items():
        setattr(a, name, value)
    return a


@pytest.mark.parametrize("change", [{"dtype": _lib.DYNB_F64}, {"n_targets": -1}, {"n_edges": 2 ** 31}, {"heads": 3}, {"kv_heads": 0}, {"dim": 0},
                                    {"dim": 257}, {"heads": 65538}, {}])
def test_attention_entry_refuses(change):
    """The last case: null pointers."""
    L = _lib.lib()
    a = _attention_args(**change)
    assert L.dynb_neighbor_attention(ctypes.byref(a), None, None, None, None) == -1
    assert L.dynb_neighbor_attention_backward(ctypes.byref(a), None, 0, 0, *[None] * 12) == -1
    assert L.dynb_neighbor_attention(None, None, None, None, None) == -1


def test_empty_calls_launch_nothing():
    L = _lib.lib()
    a = _attention_args(n_targets=0, n_sources=0, n_edges=0)
    assert L.dynb_neighbor_attention(ctypes.byref(a), None, None, None, None) == 0
    assert L.dynb_neighbor_attention_backward(ctypes.byref(a), None, 0, 0, *[None] * 12) == 0
    assert L.dynb_distance_bias(None, 0, None, 8, 2, 5.0, 1, None, None) == 0


def test_other_entries_refuse():
    L, n = _lib.lib(), ctypes.c_int64()
    assert L.dynb_neighbor_index_workspace_bytes(-1, 2, 2, 0, ctypes.byref(n)) == -1
    assert L.dynb_neighbor_index_workspace_bytes(2 ** 31, 2, 2, 0, ctypes.byref(n)) == -1
    assert L.dynb_neighbor_index_workspace_bytes(1000, 20, 20, 0, ctypes.byref(n)) == 0 and n.value >= 8000
    assert L.dynb_neighbor_index_plan(None, None, 5, 2, 2, None, None, None, None, None, None, None, None, 0, None) == -1
    assert L.dynb_neighbor_index_fill(None, 5, 2, 2, None, None, 3, None, None, None, 0, None) == -1
    for buckets, heads, cutoff in ((3, 4, 5.0), (1025, 4, 5.0), (8, 0, 5.0), (8, 1025, 5.0), (8, 4, 0.0), (8, 4, math.nan), (8, 4, math.inf)):
        assert L.dynb_distance_bias(None, 3, None, buckets, heads, cutoff, 1, None, None) == -1
        assert L.dynb_distance_bias_backward(None, 3, None, buckets, heads, cutoff, 1, None, None, None, None, 0, None) == -1
    assert L.dynb_distance_bias(None, 3, None, 8, 4, 5.0, 1, None, None) == -1   # null pointers
    assert L.dynb_type_index(None, 3, 0, None, None, None, None, 0, None) == -1
    assert L.dynb_type_index(None, 3, 4097, None, None, None, None, 0, None) == -1
    for change in ({"types": 0}, {"types": 4097}, {"inner": 0}, {"outer": 16385}, {"dtype": 1}, {"n_rows": -1}, {}):
        a = _lib.TypeLinear()
        a.n_rows, a.types, a.inner, a.outer, a.dtype = 3, 2, 4, 4, _lib.DYNB_F32
        for name, value in change.items():
            setattr(a, name, value)
        assert L.dynb_type_linear(ctypes.byref(a), None, 4, None, None, None) == -1
        assert L.dynb_type_linear_backward(ctypes.byref(a), None, 4, None, 4, None, None, None, None, 0, None) == -1


def test_plain_attention_gradients_against_differences():
    """The formulas of the gradients, in 64 bits, against central differences."""
    gen = torch.Generator().manual_seed(5)
    ei, src, dst = M.ragged_graph([3, 0, 1, 5], 6, 2, "cpu")
    q, k, v = (torch.randn(n, h, 5, generator=gen, dtype=torch.float64) for n, h in ((4, 4), (6, 2), (6, 2)))
    bias, g = torch.randn(9, 4, generator=gen, dtype=torch.float64), torch.randn(4, 4, 5, generator=gen, dtype=torch.float64)
    bias[2, 1] = -math.inf
    r = M.attention(q, k, v, src, dst, bias, 0.4, g)
    value = lambda: float((M.attention(q, k, v, src, dst, bias, 0.4)["out"][0] * g).sum())  # noqa: E731
    h = 1e-5
    for name, t in (("dq", q), ("dk", k), ("dv", v), ("d_bias", bias)):
        for at in range(0, t.numel(), 7):
            flat = t.view(-1)
            if math.isinf(float(flat[at])):
                continue
            keep = float(flat[at])
            flat[at] = keep + h
            up = value()
            flat[at] = keep - h
            down = value()
            flat[at] = keep
            # differences: third derivatives times h^2 and 2^-53 / h, both below 1e-9 here
            assert abs((up - down) / (2 * h) - float(r[name][0].reshape(-1)[at])) < 1e-8, name


def test_plain_spline_sums_to_one_and_is_smooth():
    table = torch.ones(9, 1, dtype=torch.float64)
    x = torch.linspace(0, 4.999, 400, dtype=torch.float64)
    assert torch.allclose(M.spline(x, table, 5.0, smooth=False), torch.ones(400, 1, dtype=torch.float64), atol=1e-12)
    w = torch.exp(M.spline(torch.tensor([4.999999], dtype=torch.float64), table, 5.0))
    assert float(w) < 1e-15


def test_walk_of_the_lists():
    src, dst = torch.tensor([2, 0, 2, 2]), torch.tensor([3, 3, 1, 0])
    lists = M.index_lists(src, dst, 5, 4)
    assert lists == {"rows": [3, 1, 0, 2, 4], "row_start": [0, 2, 3, 4, 4, 4], "src": [2, 0, 2, 2], "cols": [2, 0, 1, 3], "col_start": [0, 3, 4, 4, 4],
                     "in_edge": [0, 2, 3, 1], "in_dst": [3, 1, 0, 3]}


def test_workspace_of_the_weights_gradient_follows_the_rows():
    """Sums of stretches for the types that can have rows, and no more than about twice the room of wide rows (no memory is touched here)."""
    L, n = _lib.lib(), ctypes.c_int64()

    def room(rows, types, inner, outer):
        a = _lib.TypeLinear()
        a.weight_dev = a.order_dev = a.start_dev = 4096
        a.n_rows, a.types, a.inner, a.outer, a.dtype = rows, types, inner, outer, _lib.DYNB_F32
        assert L.dynb_type_linear_workspace_bytes(ctypes.byref(a), ctypes.byref(n)) == 0
        return n.value

    assert room(100, 4096, 128, 128) <= 102 * 4 * (128 * 128 + 128)
    assert room(0, 4096, 128, 128) <= 2 * 4 * (128 * 128 + 128)
    rows, wide = 1_000_000, 16384
    assert room(rows, 1, wide, wide) <= 2.1 * rows * 2 * wide * 4

"""Message-passing operators at the borders of what they promise: bytes behind a result, large and small values, calls without gradients, captures.
The bounds are derived beside the tests."""

import ctypes
import math

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

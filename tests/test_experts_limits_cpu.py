"""CPU tests of the entries of the expert layers at the limits of what they take; nothing is launched."""

import ctypes

import pytest
import torch

from dynamis_b200 import _lib, message

AT = 4096       # an address that no refused call touches


@pytest.mark.parametrize("n_rows", [2 ** 31 - 1, 2 ** 58, 2 ** 59, 2 ** 59 + 1, 2 ** 62, 2 ** 63 - 1])
def test_numbers_of_rows_whose_pairs_wrap_are_refused(n_rows):
    """2^59 rows of 32 choices are 2^64 pairs, none in 64 bits."""
    L, n = _lib.lib(), ctypes.c_int64()
    r = _lib.RoutingArgs(logits_dev=AT, logits_row=64, n_rows=n_rows, experts=64, choices=32, dtype=0, score=0, groups=1, kept_groups=1, renormalize=1, scale=1.0)
    e = _lib.ExpertLinear(weight_dev=AT, order_dev=AT, start_dev=AT, n_rows=n_rows, choices=32, experts=3, inner=8, outer=8, dtype=0)
    for call in (lambda: L.dynb_route_experts_workspace_bytes(ctypes.byref(r), ctypes.byref(n)),
                 lambda: L.dynb_route_experts(ctypes.byref(r), AT, AT, AT, AT, AT, 0, None),
                 lambda: L.dynb_route_experts_backward(ctypes.byref(r), None, AT, AT, AT, None),
                 lambda: L.dynb_expert_linear_workspace_bytes(ctypes.byref(e), 1, 1, 1, ctypes.byref(n)),
                 lambda: L.dynb_expert_linear(ctypes.byref(e), AT, 8, None, AT, None, AT, 0, None),
                 lambda: L.dynb_expert_linear_backward(ctypes.byref(e), AT, 8, AT, 8, None, None, AT, None, None, AT, 0, None),
                 lambda: L.dynb_expert_combine(None, AT, AT, None, 0, n_rows, 32, 8, 0, AT, None),
                 lambda: L.dynb_expert_combine_backward(None, AT, AT, AT, 8, n_rows, 32, 8, 0, AT, None, None)):
        assert call() == -1 and b"rows times choices" in L.dynb_last_error()


@pytest.mark.parametrize("scale", [0.0, 1e-38, 0.99e-30, 1.01e30, 3e38])
def test_scales_that_the_weights_do_not_survive_are_refused(scale):
    """The gradient divides the weights by the scale: as from Python, it lies in [1e-30, 1e30]."""
    L, n = _lib.lib(), ctypes.c_int64()
    for value, rc in ((scale, -1), (1e-30, 0), (1e30, 0)):
        r = _lib.RoutingArgs(logits_dev=AT, logits_row=64, n_rows=5, experts=64, choices=2, dtype=0, score=0, groups=1, kept_groups=1, renormalize=1, scale=value)
        assert L.dynb_route_experts_workspace_bytes(ctypes.byref(r), ctypes.byref(n)) == rc
        assert rc == 0 or b"scale" in L.dynb_last_error()


def test_waits_that_ran_out_are_told_of_both_products(monkeypatch):
    """The word of a device is set by ``type_linear`` and ``expert_linear`` alike, and either call may be the one that finds it."""
    dev, word = torch.device("cuda:0"), ctypes.c_uint32(1)
    monkeypatch.setattr(message, "_STATUS", {0: (word, AT)})
    with pytest.raises(RuntimeError, match="^type_linear or expert_linear: a wait inside a kernel of an earlier call ran out"):
        message._status_word(dev)
    assert message._status_word(dev) == AT
    monkeypatch.setattr(message, "_STATUS", {})
    monkeypatch.setattr(message, "_make_status_word", lambda dev: None)          # as under a capture
    with pytest.raises(RuntimeError, match="^the first TypeIndex or Routing of a device must be made before a capture"):
        message._status_word(dev)

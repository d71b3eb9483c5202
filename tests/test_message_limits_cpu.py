"""Message-passing entries at the borders of what they promise, as far as no GPU is needed."""

import contextlib
import ctypes
import threading
import time

import pytest
import torch

from dynamis_b200 import _lib, message


def _last():
    return _lib.lib().dynb_last_error().decode()


@pytest.mark.parametrize("off", [4, 8])
def test_entries_refuse_addresses_that_kernels_cannot_read_whole(off):
    """Workspaces off 16 bytes, statistics off 16 and the unrounded result off 8: refused before anything is launched.  (No memory is touched here.)"""
    L, at, n = _lib.lib(), 4096, ctypes.c_int64()
    assert L.dynb_neighbor_index_workspace_bytes(5, 2, 2, 0, ctypes.byref(n)) == 0
    assert L.dynb_neighbor_index_plan(at, at, 5, 2, 2, at, at, at, at, at, at, at, at + off, n.value, None) == -1 and "16-byte" in _last()
    assert L.dynb_neighbor_index_fill(at, 5, 2, 2, at, at, 3, at, at, at + off, n.value, None) == -1 and "16-byte" in _last()
    assert L.dynb_type_index_workspace_bytes(5, ctypes.byref(n)) == 0
    assert L.dynb_type_index(at, 5, 2, at, at, at, at + off, n.value, None) == -1 and "16-byte" in _last()
    a = _lib.Attention()
    a.n_targets, a.n_sources, a.n_edges, a.heads, a.kv_heads, a.dim, a.dtype, a.scale = 4, 4, 4, 4, 2, 16, _lib.DYNB_BF16, 0.25
    for name in ("q_dev", "k_dev", "v_dev", "rows_dev", "row_start_dev", "src_dev"):
        setattr(a, name, at)
    if off == 4:
        assert L.dynb_neighbor_attention(ctypes.byref(a), at, at + off, at, None) == -1 and "8-byte" in _last()
    assert L.dynb_neighbor_attention_backward(ctypes.byref(a), at, 64, 16, at, at, at, at, at, at, at + off, at, at, at, None, None) == -1
    assert "16-byte" in _last()


def test_threads_share_one_status_word(monkeypatch):
    """The word of a device is made once, however many threads ask for it first (the allocation is a fake that takes its time)."""
    made = []

    def slow():
        time.sleep(0.05)
        made.append(object())
        return ctypes.c_uint32(0), 4096 * len(made)

    monkeypatch.setattr(message, "_STATUS", {})
    monkeypatch.setattr(message, "_new_status_word", slow)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(_lib, "on_device", lambda dev: contextlib.nullcontext())
    start, got = threading.Barrier(6), []

    def ask():
        start.wait()
        got.append(message._status_word(torch.device("cuda", 0)))

    threads = [threading.Thread(target=ask) for _ in range(6)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(made) == 1 and got == [4096] * 6
    # set by a kernel: told once
    message._STATUS[0][0].value = 1
    with pytest.raises(RuntimeError, match="ran out"):
        message._status_word(torch.device("cuda", 0))
    assert message._status_word(torch.device("cuda", 0)) == 4096


def test_a_capture_without_a_status_word_is_refused(monkeypatch):
    monkeypatch.setattr(message, "_STATUS", {})
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    monkeypatch.setattr(_lib, "on_device", lambda dev: contextlib.nullcontext())
    with pytest.raises(RuntimeError, match="before a capture"):
        message._status_word(torch.device("cuda", 0))

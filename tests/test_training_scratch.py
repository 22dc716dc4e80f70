"""Scratch memory of training calls: each host thread has its own, for as long as it lives (no GPU)."""
import threading

import pytest
import torch

from kfold_b200 import functional as F

CPU = torch.device("cpu")


@pytest.fixture(autouse=True)
def _streams(monkeypatch):
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(F.L, "raw_stream", lambda at=None: 7)
    F.release_workspaces()
    yield
    F.release_workspaces()


def _in_threads(n, work):
    """Run `work` in n threads that are all alive until each has done it; what it raised or returned."""
    results, gate = [], threading.Barrier(n)

    def run():
        try:
            results.append(work())
        finally:
            gate.wait(timeout=60)

    threads = [threading.Thread(target=run) for _ in range(n)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    return results


def test_threads_have_memory_of_their_own_and_leave_none():
    mine = F._call_workspace(CPU, 4096)

    def work():
        ws = F._call_workspace(CPU, 8192)
        assert F._call_workspace(CPU, 100) is ws
        return ws.data_ptr(), set(F._workspaces)

    for _ in range(3):
        seen = _in_threads(4, work)
        assert len(seen) == 4 and len({at for at, _ in seen} | {mine.data_ptr()}) == 5
        assert len(F._workspaces) == 1 and F._call_workspace(CPU, 4096) is mine


def test_a_thread_that_ends_takes_no_other_memory_with_it():
    shared, mine = F._workspace(CPU, 1000), F._call_workspace(CPU, 1000)
    assert shared is not mine
    _in_threads(2, lambda: (F._workspace(CPU, 500), F._call_workspace(CPU, 500)))
    assert F._workspace(CPU, 1000) is shared and F._call_workspace(CPU, 1000) is mine and len(F._workspaces) == 2


def test_released_scratch_is_taken_anew():
    first = F._call_workspace(CPU, 4096)
    F.release_workspaces()
    assert not F._workspaces and F._call_workspace(CPU, 4096) is not first
    F.withdraw_workspaces([F._call_workspace(CPU, 4096)])
    assert not F._workspaces


def test_sizes_of_a_call_and_of_any_call():
    """Of widths whose launches keep their hidden channels."""
    from kfold_b200 import _lib, build
    build.build()
    lib = _lib.lib()
    for rows, c, hidden, dtype in ((1, 136, 512, 0), (5000, 72, 1024, 0), (1 << 20, 384, 1536, 0), (300, 72, 64, 2), (1 << 20, 8, 8192, 2)):
        need = [lib.kfb_feed_forward_call_bytes(rows, c, hidden, dtype, wanted) for wanted in range(8)]
        assert 0 < need[0] <= lib.kfb_feed_forward_workspace_bytes(rows, c, hidden, dtype, 0)
        assert 0 < min(need[1:]) and max(need) == max(need[0], need[7]) and need[7] == lib.kfb_feed_forward_workspace_bytes(rows, c, hidden, dtype, 1)
        for wanted in range(1, 8):
            assert all(need[wanted] >= need[part] for part in range(1, 8) if part & wanted == part)
    for bad in ((0, 128, 512, 0, 1), (1 << 31, 128, 512, 0, 1), (5, 0, 512, 0, 1), (5, 12, 512, 0, 0), (5, 128, 512, 0, 8), (5, 128, 512, 0, -1)):
        assert lib.kfb_feed_forward_call_bytes(*bad) == 0

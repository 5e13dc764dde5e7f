"""Workspaces of the Python entry points (siliconfer_amd/_lib.py), without a GPU: an entry's launches
are issued without the interpreter's lock, so two host threads on one stream must not share one."""

import threading

import pytest
import torch

from siliconfer_amd import _lib
from siliconfer_amd.kernels import attention

CPU = torch.device("cpu")


@pytest.mark.parametrize("get", [_lib.scratch, attention.workspace], ids=["scratch", "attention"])
def test_a_thread_has_its_own(monkeypatch, get):
    monkeypatch.setattr(torch._C, "_cuda_isCurrentStreamCapturing", lambda: False)
    mine, other, both = get(CPU, 7, 1000), [], threading.Barrier(3)

    def work():
        other.append(get(CPU, 7, 1000))
        both.wait()  # (both threads live at once)
        other.append(get(CPU, 7, 1000))

    threads = [threading.Thread(target=work) for _ in range(2)]
    for t in threads:
        t.start()
    both.wait()
    for t in threads:
        t.join()
    at = sorted(t.data_ptr() for t in other)
    assert at[0] == at[1] and at[2] == at[3] and len({*at, mine.data_ptr()}) == 3
    # a thread's calls share one a stream, grown on demand
    assert get(CPU, 7, 500).data_ptr() == mine.data_ptr() != get(CPU, 8, 500).data_ptr()
    big = get(CPU, 7, 1 << 20)
    assert big.numel() >= 1 << 20 and get(CPU, 7, 1000).data_ptr() == big.data_ptr()


@pytest.mark.parametrize("get", [_lib.scratch, attention.workspace], ids=["scratch", "attention"])
def test_a_recorded_call_has_its_own(monkeypatch, get):
    monkeypatch.setattr(torch._C, "_cuda_isCurrentStreamCapturing", lambda: False)
    eager = get(CPU, 9, 1000)
    monkeypatch.setattr(torch._C, "_cuda_isCurrentStreamCapturing", lambda: True)
    a, b = get(CPU, 9, 1000), get(CPU, 9, 1000)
    assert len({t.data_ptr() for t in (eager, a, b)}) == 3

"""Workspaces of calls that several host threads make on one stream (no GPU
needed: the stream and the device are stand-ins)."""

import threading
import types

import pytest
import torch

from qgemv_roofline_b200 import _tensors, gemv


def multi_type(nbytes):
    return _tensors.workspace(torch.device("cpu"), nbytes, None)[1]


def gemv_batch(nbytes):
    return gemv._workspace(torch.device("cpu"), nbytes, None).data_ptr()


@pytest.mark.parametrize("get", [multi_type, gemv_batch])
def test_threads_on_one_stream_have_buffers_of_their_own(get, monkeypatch):
    monkeypatch.setattr(_tensors, "_raw_stream", lambda index: 7)
    monkeypatch.setattr(torch.cuda, "current_stream",
                        lambda device=None: types.SimpleNamespace(stream_id=3, cuda_stream=7))
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    got, meet = {}, threading.Barrier(3)

    def work(name):
        first = get(4096)
        meet.wait(20)  # both hold a buffer
        got[name] = (first, get(1024), get(1 << 20))
        meet.wait(20)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    mine = get(4096)
    meet.wait(20)
    meet.wait(20)
    for t in threads:
        t.join(20)
    assert len({mine, got[0][0], got[1][0]}) == 3
    for first, smaller, larger in got.values():
        assert smaller == first and larger != first  # a thread's calls share theirs
    assert len({got[0][2], got[1][2], mine}) == 3
    assert get(4096) == mine

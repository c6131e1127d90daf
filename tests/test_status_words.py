"""The status words that the dense, softmax and update kernels write to."""
import threading
import time

import pytest
import torch

from parameter_server_b200.ops import dense


def test_threads_that_ask_at_once_get_the_same_words(monkeypatch):
    """The address goes to kernels: words that another thread's replaced would be freed under them."""
    monkeypatch.setattr(dense, "_status", {})
    zeros, start, got = torch.zeros, threading.Barrier(4), []

    def slow(*a, **k):
        t = zeros(*a, **k)
        time.sleep(0.05)
        return t

    monkeypatch.setattr(torch, "zeros", slow)

    def ask():
        start.wait()
        got.append(dense._status_for(torch.device("cpu")))

    threads = [threading.Thread(target=ask) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(got) == 4 and len({t.data_ptr() for t in got}) == 1 and got[0] is dense._status_for(torch.device("cpu"))


def test_a_gpu_without_an_index_is_the_current_one(monkeypatch):
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 3)
    assert dense._key(torch.device("cuda")) == dense._key(torch.device("cuda", 3)) == ("cuda", 3)
    assert dense._key(torch.device("cuda", 1)) == ("cuda", 1) and dense._key(torch.device("cpu")) == ("cpu", None)


@pytest.mark.gpu
def test_a_report_is_found_by_either_name_of_the_gpu():
    from parameter_server_b200.ops import softmax

    x, w = torch.zeros(2, 4, device="cuda"), torch.zeros(3, 4, device="cuda")
    for dev in (torch.device("cuda"), torch.device("cuda", torch.cuda.current_device())):
        dense.check_status(dev)
        softmax.softmax_loss(x, w, torch.tensor([0, 3], device="cuda"))
        with pytest.raises(RuntimeError):
            dense.check_status(dev)

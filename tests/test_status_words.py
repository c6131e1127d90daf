"""The status words that the dense, softmax and update kernels write to."""
import threading
import time

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

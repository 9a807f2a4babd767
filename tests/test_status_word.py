"""The status word of a device is made once, whichever threads ask for it first."""

import threading
import time

import torch

from flaggems_vllm_b200 import _lib


def test_threads_that_ask_at_once_get_one_word(monkeypatch):
    given = []

    class Host:
        @staticmethod
        def set_status(device, pointer):
            given.append((device, pointer))

    zeros = torch.zeros

    def slow(*size, dtype=None, device=None):  # making it lets other threads run
        time.sleep(0.05)
        return zeros(*size, dtype=dtype)

    monkeypatch.setattr(_lib, "_status", {})
    monkeypatch.setattr(_lib, "host", lambda: Host)
    monkeypatch.setattr(torch, "zeros", slow)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    barrier, words = threading.Barrier(8), []

    def body():
        barrier.wait()
        words.append(_lib.status_word(torch.device("cuda", 5)))

    threads = [threading.Thread(target=body) for _ in range(8)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(words) == 8 and len({w.data_ptr() for w in words}) == 1
    assert given == [(5, words[0].data_ptr())]  # what the kernels write is what is read

"""The operators' error word: made once."""
import threading
import time

import pytest
import torch


def test_error_word_is_made_once(built_lib, monkeypatch):
    """Threads that make a device's first call together share one word (a second one would be given back in use)."""
    from hackthenorth_b200 import ops

    def slow_zeros(*size, dtype=None, device=None):
        time.sleep(0.05)
        return torch.empty(*size, dtype=dtype)

    monkeypatch.setattr(ops, "_scratch", {})
    monkeypatch.setattr(ops.torch, "zeros", slow_zeros)
    monkeypatch.setattr(ops.torch.cuda, "is_current_stream_capturing", lambda: False)
    words = []
    threads = [threading.Thread(target=lambda: words.append(ops._status(0))) for _ in range(8)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(set(words)) == 1 and words[0] == ops._scratch[0].data_ptr()

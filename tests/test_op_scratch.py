"""The operators' error word: made once, and zero before any call can report to it."""
import threading
import time

import pytest
import torch

DEV = "cuda:0"


@pytest.mark.gpu
def test_error_word_is_zero_for_every_stream(built_lib, monkeypatch):
    """Its first use lies behind long work of one stream; another stream's call and check do not wait for that."""
    from hackthenorth_b200 import ops

    x, u = torch.zeros(1, 100, device=DEV), torch.zeros(1, device=DEV)
    ops.sample_token(x, u)
    size = int(built_lib.qb_op_scratch_bytes())
    one, other = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(one):
        torch.full((size,), 255, dtype=torch.uint8, device=DEV)  # the memory that the allocator hands out next
    torch.cuda.synchronize()
    monkeypatch.setattr(ops, "_scratch", {})
    with torch.cuda.stream(one):
        torch.cuda._sleep(2 * 10 ** 9)  # about a second
        ops.sample_token(x, u)
    with torch.cuda.stream(other):
        assert int(ops.sample_token(x, u)) == 0
        ops.check_device_errors(DEV)
    torch.cuda.synchronize()


def test_error_word_is_made_once(built_lib, monkeypatch):
    """Threads that make a device's first call together share one word (a second one would be given back in use)."""
    from hackthenorth_b200 import ops

    def slow_zeros(*size, dtype=None, device=None):
        time.sleep(0.05)
        return torch.empty(*size, dtype=dtype)

    class Stream:
        def synchronize(self):
            pass

    monkeypatch.setattr(ops, "_scratch", {})
    monkeypatch.setattr(ops.torch, "zeros", slow_zeros)
    monkeypatch.setattr(ops.torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(ops.torch.cuda, "current_stream", lambda device=None: Stream())
    words = []
    threads = [threading.Thread(target=lambda: words.append(ops._status(0))) for _ in range(8)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(set(words)) == 1 and words[0] == ops._scratch[0].data_ptr()

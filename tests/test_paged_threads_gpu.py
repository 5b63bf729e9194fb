"""Paged attention from several host threads that share one stream."""
import threading

import pytest
import torch

from paged_reference import make_batch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"

CASES = [  # of every kernel and number of launches
    dict(lens=[(40, 5000), (1, 300)], prefix=0),
    dict(lens=[(700, 700)], prefix=0),
    dict(lens=[(1, 9000), (1, 4), (1, 700)], prefix=0),
    dict(lens=[(1, 30)] * 50, prefix=4000),
    dict(lens=[(30, 60), (2, 900)], prefix=1500),
]


def _attend(bt):
    from hackthenorth_b200 import ops

    tail = (bt["table"], bt["q_start"], bt["kv_lens"])
    n = max(n for n, _ in bt["lens"])
    if bt["prefix"]:
        return ops.shared_prefix_attention(bt["q"], bt["k"], bt["v"], bt["prefix_table"], bt["prefix"], *tail, max_queries=n)
    return ops.paged_attention(bt["q"], bt["k"], bt["v"], *tail, max_queries=n)


@pytest.mark.parametrize("own_stream", [False, True])
def test_threads_that_share_a_stream(built_lib, own_stream):
    """Every thread's results are those of the same calls made alone."""
    from hackthenorth_b200 import ops

    batches = [make_batch(c["lens"], 16, 4, 32, 40 + i, DEV, prefix=c["prefix"]) for i, c in enumerate(CASES)]
    want = [_attend(bt) for bt in batches]
    torch.cuda.synchronize()
    stream = torch.cuda.Stream() if own_stream else torch.cuda.default_stream()
    got, start = [[] for _ in batches], threading.Barrier(len(batches))

    def work(i):
        with torch.cuda.stream(stream), torch.no_grad():
            start.wait(30)
            for _ in range(40):
                got[i].append(_attend(batches[i]))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(batches))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    ops.check_device_errors(DEV)
    for outs, w in zip(got, want):
        assert len(outs) == 40 and all(torch.equal(o, w) for o in outs)

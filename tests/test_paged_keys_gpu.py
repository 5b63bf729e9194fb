"""Paged attention over long caches where every key counts.

A flat softmax over many random keys averages their values down to where a
missing key tile hides below the bound of P's rounding. Here the scores are all
equal, so that every weight is exactly 1 and the sums are exact, or one key
carries the whole weight.
"""
import pytest
import torch

from paged_reference import BF16, D, attention64, make_batch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module", autouse=True)
def _ready(built_lib):
    yield
    from hackthenorth_b200 import ops

    ops.check_device_errors(DEV)


def _attend(bt, window=0, sinks=0):
    from hackthenorth_b200 import ops

    tail = (bt["table"], bt["q_start"], bt["kv_lens"])
    n = max(n for n, _ in bt["lens"])
    if bt["prefix"]:
        return ops.shared_prefix_attention(bt["q"], bt["k"], bt["v"], bt["prefix_table"], bt["prefix"], *tail, max_queries=n)
    return ops.paged_attention(bt["q"], bt["k"], bt["v"], *tail, window=window, sinks=sinks, max_queries=n)


def _fill(bt, values):
    """V of the first sequence's keys: ``values`` [keys, D], for every KV head (prefix keys first)."""
    page, at = bt["page"], 0
    for ids, count in ((bt["prefix_table"], bt["prefix"]), (bt["pages"][0], bt["lens"][0][1])):
        for c in range(0, count, page):
            m = min(page, count - c)
            bt["v"][int(ids[c // page]), :, :m] = values[at:at + m].to(BF16)
            at += m


@pytest.mark.parametrize("n,prefix", [(1, 0), (20, 0), (40, 0), (2, 30000), (40, 30000)])
def test_the_weights_of_equal_scores_sum_exactly(n, prefix):
    """Values 1 and 1 + 2^-7 whose mean lies 2^-19 to 2^-17 below the middle between the two.

    Weights are 1, sums of values multiples of 2^-7 below 2^16, both exact in
    fp32; the quotient's two roundings leave 2^-23 at most, so the result is
    the nearest bf16, and an error of the row sum of 2^-16 is not hidden."""
    kv = 2 ** 15 - prefix
    bt = make_batch([(n, kv)], 8, 2, 64, 31, DEV, prefix=prefix)
    bt["q"].zero_()
    total = 2 ** 15
    high = (total - n + 1) // 2 - 8
    order = torch.randperm(total - n + 1, generator=torch.Generator().manual_seed(1))[:high]
    values = torch.ones(total, D, device=DEV)
    values[order.to(DEV)] += 2.0 ** -7
    values[:, 1::2] *= -1
    _fill(bt, values)
    assert torch.equal(_attend(bt), attention64(bt)[0].to(BF16))

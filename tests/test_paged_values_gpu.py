"""Paged attention where single values are extreme: keys that are not finite,
and masked values at the type's lowest. Bound: ``paged_reference.attention_bound``."""
import pytest
import torch

from paged_reference import attention64, attention_bound, make_batch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module", autouse=True)
def _ready(built_lib):
    yield
    from hackthenorth_b200 import ops

    ops.check_device_errors(DEV)


def _attend(bt, **kw):
    from hackthenorth_b200 import ops

    tail = (bt["table"], bt["q_start"], bt["kv_lens"])
    if bt["prefix"]:
        return ops.shared_prefix_attention(bt["q"], bt["k"], bt["v"], bt["prefix_table"], bt["prefix"], *tail, **kw)
    return ops.paged_attention(bt["q"], bt["k"], bt["v"], *tail, **kw)


@pytest.mark.parametrize("lens,prefix", [([(1, 9), (1, 70)], 200), ([(20, 30), (1, 70)], 200), ([(1, 9)] * 70, 3000),
                                         ([(1, 500), (1, 3)], 0), ([(30, 500), (1, 3)], 0)])
@pytest.mark.parametrize("key", [0, 1, 4, 5, 63, 64, 130])
def test_a_key_that_is_nan_makes_its_rows_nan(lens, prefix, key):
    """All rows that see the key, of its KV head; never a finite result without it."""
    hq, hkv, page = 8, 4, 16
    bt = make_batch(lens, hq, hkv, page, 21, DEV, prefix=prefix)
    ref, mag = attention64(bt)
    ids = bt["prefix_table"] if prefix else bt["pages"][0]
    bt["k"][int(ids[key // page]), 2, key % page, 5] = float("nan")
    out = _attend(bt, max_queries=max(n for n, _ in lens))
    rows = bt["rows"] if prefix else lens[0][0]
    assert bool(out[:rows, 4:6].isnan().all())
    other = torch.ones(bt["rows"], hq, dtype=torch.bool, device=DEV)
    other[:rows, 4:6] = False
    assert bool(((out.double() - ref).abs() <= attention_bound(ref, mag))[other].all())


@pytest.mark.parametrize("hq,hkv,page", [(16, 4, 16), (8, 8, 64), (10, 2, 128)])
def test_values_that_a_row_does_not_see_do_not_reach_it(hq, hkv, page):
    """Later keys of a chunk hold the lowest value of the type: rows before them are as without."""
    n, kv, late = 200, 700, 90
    bt = make_batch([(n, kv), (1, 40)], hq, hkv, page, 22, DEV)
    low = torch.finfo(torch.bfloat16).min
    for c in range(kv - late, kv):
        bt["v"][int(bt["pages"][0, c // page]), :, c % page] = low
    ref, mag = attention64(bt)
    out = _attend(bt, max_queries=n)
    rows = n - late
    assert bool(((out[:rows].double() - ref[:rows]).abs() <= attention_bound(ref[:rows], mag[:rows])).all())


@pytest.mark.parametrize("n", [1, 200])
def test_values_before_the_window_do_not_reach_a_row(n):
    """Keys that only the first rows' windows reach hold the lowest value."""
    kv, window, page = 900, 128, 32
    bt = make_batch([(n, kv)], 16, 4, page, 23, DEV)
    early = kv - n - window + n // 2  # the rows from n / 2 on do not see the keys up to here
    for c in range(early + 1):
        bt["v"][int(bt["pages"][0, c // page]), :, c % page] = torch.finfo(torch.bfloat16).min
    ref, mag = attention64(bt, window)
    out = _attend(bt, max_queries=n, window=window)
    rows = slice(n // 2 + 1 if n > 1 else 0, n)
    assert bool(((out[rows].double() - ref[rows]).abs() <= attention_bound(ref[rows], mag[rows])).all())

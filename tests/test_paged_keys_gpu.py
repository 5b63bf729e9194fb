"""Paged attention over long caches where every key counts.

A flat softmax over many random keys averages their values down to where a
missing key tile hides below the bound of P's rounding. Here the scores are all
equal, so that every weight is exactly 1 and the sums are exact, or one key
carries the whole weight.
"""
import pytest
import torch

from paged_reference import BF16, D, attention64, attention_bound, make_batch

DEV = "cuda:0"


@pytest.fixture(scope="module", autouse=True)
def _ready(built_lib):
    yield
    if torch.cuda.is_available():
        from hackthenorth_b200 import ops

        ops.check_device_errors(DEV)


def _attend(bt, window=0, sinks=0):
    from hackthenorth_b200 import ops

    tail = (bt["table"], bt["q_start"], bt["kv_lens"])
    n = max(n for n, _ in bt["lens"])
    if bt["prefix"]:
        return ops.shared_prefix_attention(bt["q"], bt["k"], bt["v"], bt["prefix_table"], bt["prefix"], *tail, max_queries=n)
    return ops.paged_attention(bt["q"], bt["k"], bt["v"], *tail, window=window, sinks=sinks, max_queries=n)


def _fill(bt, values, seq=0):
    """V of a sequence's keys: ``values`` [keys, D], for every KV head (the prefix's keys first)."""
    page, at = bt["page"], 0
    for ids, count in ((bt["prefix_table"], bt["prefix"]), (bt["pages"][seq], bt["lens"][seq][1])):
        whole = count // page
        bt["v"][ids[:whole].long()] = values[at:at + whole * page].view(whole, 1, page, D).to(BF16)
        at += whole * page
        if count % page:
            bt["v"][int(ids[whole]), :, :count % page] = values[at:at + count % page].to(BF16)
            at += count % page


@pytest.mark.gpu
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


GROUP = 16  # keys whose values are 1 in one dim: a quarter of a key tile, the smallest page


def _coded(keys, shift=0):
    """Values [keys, D] that are 0 but for a 1 in the dim of the key's group (neighbours far apart)."""
    dims = ((torch.arange(keys) // GROUP + shift) * 37) % D
    return torch.nn.functional.one_hot(dims, D).float()


def test_a_missing_or_repeated_tile_would_show():
    """With equal scores a row's result is the share of its keys in each dim, off by half a bf16 step (2^-8) at
    most. Leaving out or repeating any whole 64-key tile of up to 131072 keys moves some dim by more than twice
    that. (A shorter last tile is the next test's.)"""
    for keys in (700, 20000, 40001, 131072):
        values = _coded(keys).double()
        count = values.sum(0)
        tiles = torch.stack([values[c:c + 64].sum(0) for c in range(0, keys - 63, 64)])
        share = count / keys
        for sign in (-1, 1):
            moved = (count + sign * tiles) / (keys + sign * tiles.sum(1, keepdim=True))
            assert bool(((moved - share).abs() > 2 * 2.0 ** -8 * share.maximum(moved)).any(1).all())


EQUAL = [
    ([(1, 20000)], 4, 1, 128, 0, 0, 0),
    ([(2, 40000)], 16, 2, 64, 0, 0, 0),
    ([(1, 131072)], 32, 8, 64, 0, 0, 0),
    ([(1, 33000), (1, 900), (0, 70), (1, 64 * 37 + 1), (1, 64)], 8, 4, 16, 0, 0, 0),
    ([(1, 30000), (4, 5000)], 8, 4, 32, 4096, 4, 0),
    ([(40, 40001)], 8, 2, 64, 0, 0, 0),
    ([(300, 20000)], 4, 1, 128, 0, 0, 0),
    ([(65, 300), (1, 9000), (33, 20049), (5, 5)], 32, 8, 32, 0, 0, 0),
    ([(260, 30000), (1, 700)], 5, 1, 16, 3000, 130, 0),
    ([(1, 70), (1, 900), (1, 5)], 8, 2, 64, 0, 0, 30000),
    ([(1, 1 + 7 * i) for i in range(70)], 16, 4, 16, 0, 0, 9001),
    ([(40, 700), (3, 3)], 8, 2, 32, 0, 0, 20000),
]


@pytest.mark.gpu
@pytest.mark.parametrize("lens,hq,hkv,page,window,sinks,prefix", EQUAL)
def test_every_key_counts_once(lens, hq, hkv, page, window, sinks, prefix):
    """Equal scores: exact sums, and a quotient within half a bf16 step and 2^-22 for its two fp32 roundings."""
    bt = make_batch(lens, hq, hkv, page, 32, DEV, prefix=prefix)
    bt["q"].zero_()
    for b, (_, kv) in enumerate(lens):
        _fill(bt, torch.cat((_coded(prefix), _coded(kv, b))).to(DEV), b)
    ref, _ = attention64(bt, window, sinks)
    out = _attend(bt, window, sinks).double()
    assert bool(((out - ref).abs() <= (2.0 ** -8 + 2.0 ** -21) * ref).all()), ((out - ref).abs() / ref.clamp(min=1e-9)).max().item()


NEEDLES = [
    ([(1, 40000)], 8, 2, 64, 0, 0, 0),
    ([(3, 20001), (1, 300)], 8, 2, 16, 0, 0, 0),
    ([(1, 20000)], 8, 2, 128, 5000, 100, 0),
    ([(20, 30000)], 8, 2, 64, 0, 0, 0),
    ([(200, 12000)], 8, 2, 32, 0, 0, 0),
    ([(20, 20000), (1, 90)], 8, 2, 64, 5000, 100, 0),
    ([(1, 50), (1, 3)], 8, 2, 64, 0, 0, 20000),
    ([(30, 300)], 8, 2, 16, 0, 0, 12000),
]


@pytest.mark.gpu
@pytest.mark.parametrize("lens,hq,hkv,page,window,sinks,prefix", NEEDLES)
def test_one_key_that_outweighs_the_others(lens, hq, hkv, page, window, sinks, prefix):
    """One key of each tile in turn, at another place of it each time, and at the borders: its score is 33.9, the
    others' are below 7 (normal, of 4e4 keys), so they weigh less than 4e4 e^-26.9 = 2^-23 together, and the result
    is the key's value within half a bf16 step and 2^-20 (values below 6). Rows that do not see the key keep their
    result, within the bound of the exact one: not bit for bit, since the tcgen05 kernel moves the reference maxima
    of a warp's rows together, and another reference rounds P elsewhere."""
    n, kv = lens[0]
    bt = make_batch(lens, hq, hkv, page, 33, DEV, prefix=prefix)
    direction = (torch.randint(0, 2, (D,), generator=torch.Generator().manual_seed(3)) * 2.0 - 1.0).to(DEV)
    bt["q"][:n] = direction.to(BF16)
    ref, mag = (x[:n].view(n, hkv, hq // hkv, D) for x in attention64(bt, window, sinks))
    ids = torch.cat((bt["prefix_table"], bt["pages"][0][:-(-kv // page)])).tolist()
    slots = [(ids[c // page], c % page) for c in range(prefix)]
    first = -(-prefix // page)
    slots += [(ids[first + c // page], c % page) for c in range(kv)]
    total = prefix + kv
    places = sorted({min(c + 37 * (c // 64) % 64, total - 1) for c in range(0, total, 64)}
                    | {c for b in (prefix, total, total - n, total - window if window else 0, sinks) for c in (b - 1, b, b + 1)
                       if 0 <= c < total} | {0, 1, 63, 64, 65, page - 1, page})
    got = []
    for c in places:
        pg, sl = slots[c]
        kept = bt["k"][pg, :, sl].clone()
        bt["k"][pg, :, sl] = (3 * direction).to(BF16)
        got.append(_attend(bt, window, sinks)[:n])
        bt["k"][pg, :, sl] = kept
    got = torch.stack(got).view(len(places), n, hkv, hq // hkv, D).double()
    value = torch.stack([bt["v"][pg, :, sl] for pg, sl in (slots[c] for c in places)]).double()[:, None, :, None]
    c = torch.tensor(places, device=DEV)[:, None]
    p = torch.arange(total - n, total, device=DEV)[None]
    seen = c <= p
    if window:
        seen = seen & ((c > p - window) | (c < sinks))
    right = ((got - value).abs() <= 2.0 ** -8 * value.abs() + 2.0 ** -20).flatten(2).all(2)
    same = ((got - ref).abs() <= attention_bound(ref, mag)).flatten(2).all(2)
    assert bool(right[seen].all()), (c.expand_as(seen)[seen & ~right].unique().tolist(), n)
    assert bool(same[~seen].all())

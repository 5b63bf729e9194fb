"""The paged-cache operators on the GPU against 64-bit plain forms.

Attention tolerance: ``paged_reference.attention_bound``. Append: fp32
arithmetic and one rounding, so half a bf16 step (2^-8 of the value) and the
fp32 error of the two products of the rotation (below 2^-20 of their sum of
magnitudes); V and untouched slots are bit-exact.
"""
import pytest
import torch

from paged_reference import BF16, D, attention64, attention_bound, make_batch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module", autouse=True)
def _ready(built_lib):
    yield
    from hackthenorth_b200 import ops

    ops.check_device_errors(DEV)


def _tables(positions):
    from hackthenorth_b200.config import QWEN3_0P6B
    from hackthenorth_b200.weights import rotary_table

    cos, sin = rotary_table(QWEN3_0P6B, positions)
    return cos.to(DEV), sin.to(DEV)


def _append64(bt, qkv, qn, kn, cos, sin, eps, first):
    """(q, K pool, V pool, summed magnitudes of q) in 64 bits."""
    hq, hkv, page = bt["hq"], bt["hkv"], bt["page"]
    q = torch.full((bt["rows"], hq, D), float("nan"), dtype=torch.float64, device=DEV)
    k, v = bt["k"].double(), bt["v"].double()
    magq, magk = q.clone(), torch.zeros_like(k)
    for b, (n, kv) in enumerate(bt["lens"]):
        for i in range(n):
            t, p = bt["starts"][b] + i, kv - n + i
            x = qkv[t].double().view(hq + 2 * hkv, D)
            c, s = cos[first + p].double(), sin[first + p].double()

            def turn(y, gain):
                if gain is not None:
                    y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps) * gain.double()
                half = torch.cat((-y[..., 64:], y[..., :64]), -1)
                return y * c + half * s, (y * c).abs() + (half * s).abs()

            q[t], magq[t] = turn(x[:hq], qn)
            pg, sl = int(bt["table"][b, p // page]), p % page
            k[pg, :, sl], magk[pg, :, sl] = turn(x[hq:hq + hkv], kn)
            v[pg, :, sl] = x[hq + hkv:]
    return q, k, v, magq, magk


@pytest.mark.parametrize("lens,hq,hkv,page,pad,norm,first", [
    ([(1, 1)], 16, 8, 16, 0, True, 0),
    ([(1, 4097)], 32, 8, 64, 0, True, 0),
    ([(3, 3), (0, 7), (1, 130), (20, 33)], 32, 8, 16, 5, True, 0),
    ([(1, 9), (2, 2), (0, 0)], 4, 1, 32, 1, False, 100),
    ([(1, 1 + i % 70) for i in range(300)], 8, 4, 16, 0, True, 3),
    ([(40, 300)], 5, 5, 256, 0, True, 0),
])
def test_append_matches_formula(lens, hq, hkv, page, pad, norm, first):
    from hackthenorth_b200 import ops

    bt = make_batch(lens, hq, hkv, page, 7, DEV, pad=pad)
    g = torch.Generator(device=DEV).manual_seed(8)
    qkv = (1.5 * torch.randn(bt["rows"], (hq + 2 * hkv) * D, generator=g, device=DEV)).to(BF16)
    qn = (1 + 0.3 * torch.randn(D, generator=g, device=DEV)).to(BF16) if norm else None
    kn = (1 + 0.3 * torch.randn(D, generator=g, device=DEV)).to(BF16) if norm else None
    cos, sin = _tables(first + max(kv for _, kv in lens))
    ref_q, ref_k, ref_v, magq, magk = _append64(bt, qkv, qn, kn, cos, sin, 1e-6, first)
    out = torch.full((bt["rows"], hq, D), 7.0, dtype=BF16, device=DEV)
    k, v = bt["k"].clone(), bt["v"].clone()
    got = ops.rope_paged_append(qkv, qn, kn, cos, sin, k, v, bt["table"], bt["q_start"], bt["kv_lens"],
                                first_position=first, out=out)
    ops.check_device_errors(DEV)
    used = bt["starts"][-1]
    assert got is out and bool((out[used:] == 7.0).all())
    assert torch.equal(v.double(), ref_v)
    for got, ref, mag in ((out[:used].double(), ref_q[:used], magq[:used]), (k.double(), ref_k, magk)):
        assert bool(((got - ref).abs() <= 2.0 ** -8 * ref.abs() + 2.0 ** -20 * mag).all())


def _attend(bt, **kw):
    from hackthenorth_b200 import ops

    out = torch.full_like(bt["q"], 7.0)
    got = ops.paged_attention(bt["q"], bt["k"], bt["v"], bt["table"], bt["q_start"], bt["kv_lens"], out=out, **kw)
    ops.check_device_errors(DEV)
    assert got is out
    return out


def _check(bt, out, window=0, sinks=0):
    ref, mag = attention64(bt, window, sinks)
    used = bt["starts"][-1]
    assert bool((out[used:] == 7.0).all())  # rows of no sequence stay
    diff = (out[:used].double() - ref[:used]).abs()
    assert bool((diff <= attention_bound(ref[:used], mag[:used])).all()), diff.max().item()


def _poison(bt, window=0, sinks=0):
    """NaN into every slot that no query sees, and an impossible id for the pages with nothing but such slots."""
    page = bt["page"]
    seen = torch.zeros(bt["k"].shape[0], page, dtype=torch.bool)
    table = bt["table"].cpu().clone()
    for b, (n, kv) in enumerate(bt["lens"]):
        lo = max(0, kv - n - window + 1) if window else 0
        for c in range(kv if n else 0):
            if c >= lo or c < sinks:
                seen[int(table[b, c // page]), c % page] = True
    for b in range(table.shape[0]):
        for j in range(table.shape[1]):
            if table[b, j] >= 0 and not bool(seen[table[b, j]].any()):
                table[b, j] = 1 << 30
    dead = ~seen.to(DEV)[:, None, :, None]
    bt["k"].masked_fill_(dead, float("nan"))
    bt["v"].masked_fill_(dead, float("nan"))
    bt["table"] = table.to(DEV)


DECODE = [
    ([(1, 1)], 16, 8, 16),
    ([(1, 512)], 16, 8, 16),
    ([(1, 64)], 32, 8, 64),
    ([(1, 65), (1, 1), (0, 40), (1, 129), (1, 63)], 32, 8, 32),
    ([(1, 20000)], 4, 1, 128),
    ([(1, 7000), (1, 3), (1, 2500)], 32, 8, 256),
    ([(4, 4), (3, 100), (0, 0), (1, 1)], 8, 4, 16),
    ([(1, 77)], 16, 1, 16),
    ([(3, 50), (2, 333)], 5, 1, 64),
    ([(1, 1 + 37 * i % 400) for i in range(700)], 8, 8, 16),
    ([(int(i % 3 > 0), 5 + 13 * i % 150) for i in range(1024)], 4, 2, 16),
    ([(2, 40000)], 16, 2, 64),
]


@pytest.mark.parametrize("lens,hq,hkv,page", DECODE)
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (50, 4), (64, 64), (1000, 130)])
def test_few_rows_match_formula(lens, hq, hkv, page, window, sinks):
    bt = make_batch(lens, hq, hkv, page, 3, DEV, pad=2, scale=1.5)
    _poison(bt, window, sinks)
    kw = dict(window=window, sinks=sinks, max_queries=max(n for n, _ in lens))
    out = _attend(bt, **kw)
    _check(bt, out, window, sinks)
    assert torch.equal(out, _attend(bt, **kw))  # joins in a fixed order, tickets back at zero


MANY = [
    ([(17, 17)], 16, 8, 16),
    ([(5, 9000)], 32, 8, 64),
    ([(64, 64)], 32, 8, 64),
    ([(65, 300), (1, 1), (0, 40), (129, 129), (1, 700), (33, 2049)], 32, 8, 32),
    ([(17, 6000)], 4, 1, 128),
    ([(700, 700)], 8, 4, 16),
    ([(300, 1000), (7, 100)], 5, 1, 256),
    ([(100, 100), (3, 200)], 16, 1, 16),
    ([(260, 400)], 4, 4, 64),
    ([(1 + i % 9, 20 + 37 * i % 400) for i in range(300)], 8, 8, 16),
]


@pytest.mark.parametrize("lens,hq,hkv,page", MANY)
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (50, 4), (128, 128), (1000, 130)])
def test_many_rows_match_formula(lens, hq, hkv, page, window, sinks):
    bt = make_batch(lens, hq, hkv, page, 5, DEV, pad=3, scale=1.5)
    _poison(bt, window, sinks)
    kw = dict(window=window, sinks=sinks, max_queries=max(max(n for n, _ in lens), 17))
    out = _attend(bt, **kw)
    _check(bt, out, window, sinks)
    assert torch.equal(out, _attend(bt, **kw))


def test_rows_before_the_first_key_give_zero():
    # more queries than cached keys: the first rows sit at negative positions and see nothing
    for n, kv, hq in ((3, 1, 8), (2, 0, 8), (40, 9, 32)):
        bt = make_batch([(n, kv), (1, 70)], hq, 8, 16, 11, DEV)
        out = _attend(bt, max_queries=n)
        assert bool((out[:n - kv] == 0).all())
        _check(bt, out)


def test_growing_scores_move_the_reference_maximum():
    """Keys whose scores grow along the sequence: every tile lifts the running
    maximum, the largest by far the last."""
    for lens in ([(1, 700)], [(40, 700)]):
        bt = make_batch(lens, 8, 8, 64, 13, DEV)
        direction = torch.randn(D, generator=torch.Generator().manual_seed(1)).to(DEV)
        bt["q"] = (direction.to(BF16).expand_as(bt["q"])).contiguous()
        for c in range(700):
            bt["k"][int(bt["pages"][0, c // 64]), :, c % 64] = (direction * (c / 700.0) ** 2 * 3).to(BF16)
        ref, mag = attention64(bt)
        out = _attend(bt, max_queries=lens[0][0])
        # scores reach 40: a score's fp32 error is below 128 * 2^-24 * 40 = 2^-11.6, and so is its weight's
        assert bool(((out.double() - ref).abs() <= attention_bound(ref, mag) + 2.0 ** -11 * mag).all())


PREFIX = [
    ([(1, 1)], 16, 8, 16, 1),
    ([(1, 5), (1, 90), (1, 1)], 4, 1, 16, 1000),
    ([(1, 1 + 7 * i) for i in range(40)], 32, 8, 64, 3001),
    ([(4, 4), (1, 40), (0, 3), (2, 130)], 8, 4, 32, 129),
    ([(9, 30), (40, 300), (1, 2)], 32, 8, 16, 777),
    ([(30, 30)] * 9, 5, 1, 128, 256),
    ([(1, 9), (2, 20)], 16, 8, 16, 0),
    ([(2, 0), (1, 5), (3, 1)], 16, 8, 16, 40),
    ([(20, 0), (1, 5)], 16, 8, 16, 300),
]


@pytest.mark.parametrize("lens,hq,hkv,page,prefix", PREFIX)
def test_shared_prefix_matches_formula(lens, hq, hkv, page, prefix):
    from hackthenorth_b200 import ops

    bt = make_batch(lens, hq, hkv, page, 17, DEV, pad=2, scale=1.5, prefix=prefix)
    own = torch.zeros(bt["k"].shape[0], page, dtype=torch.bool)
    for ids, kv in [(bt["pages"][b].tolist(), kv if n else 0) for b, (n, kv) in enumerate(lens)] + [
            (bt["prefix_table"].tolist(), prefix)]:
        for c in range(kv):
            own[ids[c // page], c % page] = True
    for pool in (bt["k"], bt["v"]):
        pool.masked_fill_(~own.to(DEV)[:, None, :, None], float("nan"))
    outs = []
    for _ in range(2):
        out = torch.full_like(bt["q"], 7.0)
        ops.shared_prefix_attention(bt["q"], bt["k"], bt["v"], bt["prefix_table"], prefix, bt["table"], bt["q_start"],
                                    bt["kv_lens"], max_queries=max(n for n, _ in lens), out=out)
        ops.check_device_errors(DEV)
        _check(bt, out)
        outs.append(out)
    assert torch.equal(*outs)


def _fresh(bt):
    """The result of a call on the current stream, checked later."""
    from hackthenorth_b200 import ops

    return ops.paged_attention(bt["q"], bt["k"], bt["v"], bt["table"], bt["q_start"], bt["kv_lens"],
                               max_queries=max(n for n, _ in bt["lens"]))


def test_calls_on_several_streams_overlap():
    """Long calls of both kernels on three streams at once, each with data made on its own stream."""
    streams = [torch.cuda.Stream() for _ in range(3)]
    cases = [[(1, 9000)] * 3, [(40, 3000), (1, 5000)], [(1, 12000), (1, 4)]]
    batches = [make_batch(c, 32, 8, 64, 60 + i, DEV) for i, c in enumerate(cases)]
    torch.cuda.synchronize()
    outs = [[] for _ in streams]
    for _ in range(4):
        for s, bt, o in zip(streams, batches, outs):
            with torch.cuda.stream(s):
                o.append(_fresh(bt))
    torch.cuda.synchronize()
    for bt, o in zip(batches, outs):
        ref, mag = attention64(bt)
        for x in o:
            assert torch.equal(x, o[0])
        assert bool(((o[0].double() - ref).abs() <= attention_bound(ref, mag)).all())


def test_graphs_follow_the_lengths_and_share_no_workspace():
    """Two captured graphs replayed on two streams at once, then again with longer sequences."""
    from hackthenorth_b200 import ops

    batches = [make_batch([(1, 6000), (1, 900)], 32, 8, 32, 70, DEV), make_batch([(30, 4000)], 32, 8, 64, 71, DEV)]
    for bt in batches:
        _fresh(bt)
    graphs, outs = [], []
    side = torch.cuda.Stream()
    for bt in batches:
        g, out = torch.cuda.CUDAGraph(), torch.zeros_like(bt["q"])
        with torch.cuda.graph(g, stream=side):
            ops.paged_attention(bt["q"], bt["k"], bt["v"], bt["table"], bt["q_start"], bt["kv_lens"],
                                max_queries=max(n for n, _ in bt["lens"]), out=out)
        graphs.append(g)
        outs.append(out)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for shorter in (0, 700):
        for bt in batches:
            bt["lens"] = [(n, kv - shorter) for n, kv in bt["lens"]]
            bt["kv_lens"].copy_(torch.tensor([kv for _, kv in bt["lens"]], dtype=torch.int32))
        torch.cuda.synchronize()
        for _ in range(3):
            for g, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        for bt, out in zip(batches, outs):
            ref, mag = attention64(bt)
            assert bool(((out.double() - ref).abs() <= attention_bound(ref, mag)).all())
    ops.check_device_errors(DEV)


@pytest.mark.parametrize("what,message", [("page", "page id"), ("negative page", "page id"), ("length", "lie outside"),
                                          ("rows", "lie outside"), ("queries", "lie outside")])
@pytest.mark.parametrize("n", [1, 40])
def test_numbers_out_of_range_are_reported_and_spoil_no_other_sequence(what, message, n):
    """The kernels check every page id, length and row range before they use it."""
    from hackthenorth_b200 import ops

    bt = make_batch([(n, 200), (1, 150), (1, 90)], 16, 8, 16, 80, DEV)
    ref, mag = attention64(bt)
    kw = dict(max_queries=n)
    if what == "page":
        bt["table"][1, 4] = bt["k"].shape[0]
    elif what == "negative page":
        bt["table"][1, 4] = -5
    elif what == "length":
        bt["kv_lens"][1] = bt["table"].shape[1] * 16 + 1
    elif what == "rows":
        bt["q_start"][3] = bt["rows"] + 7
    else:
        kw = dict(max_queries=n)
        bt["q_start"][1:] = torch.tensor([0, n + 1, n + 2], dtype=torch.int32)  # the second sequence has n + 1 rows
    out = torch.zeros_like(bt["q"])
    ops.paged_attention(bt["q"], bt["k"], bt["v"], bt["table"], bt["q_start"], bt["kv_lens"], out=out, **kw)
    with pytest.raises(ValueError, match=message):
        ops.check_device_errors(DEV)
    ops.check_device_errors(DEV)
    if what != "queries":
        good = out[:n].double()
        assert bool(((good - ref[:n]).abs() <= attention_bound(ref[:n], mag[:n])).all())
    again = make_batch([(n, 200), (1, 150), (1, 90)], 16, 8, 16, 80, DEV)  # and the next call is whole
    _check(again, _attend(again, max_queries=n))


def test_append_reports_pages_and_positions_out_of_range():
    from hackthenorth_b200 import ops

    bt = make_batch([(2, 20), (1, 40)], 16, 8, 16, 81, DEV)
    qkv = torch.randn(3, 32 * D, device=DEV).to(BF16)
    cos, sin = _tables(64)
    for spoil, message in ((lambda: bt["table"].index_put_((torch.tensor([0], device=DEV), torch.tensor([1], device=DEV)),
                                                           torch.tensor(99, dtype=torch.int32, device=DEV)), "page id"),
                           (lambda: bt["kv_lens"].fill_(1), "KV capacity"), (lambda: bt["kv_lens"].fill_(1 << 20), "lie outside")):
        table, lens = bt["table"].clone(), bt["kv_lens"].clone()
        spoil()
        k, v = bt["k"].clone(), bt["v"].clone()
        ops.rope_paged_append(qkv, None, None, cos, sin, k, v, bt["table"], bt["q_start"], bt["kv_lens"])
        with pytest.raises(ValueError, match=message):
            ops.check_device_errors(DEV)
        bt["table"], bt["kv_lens"] = table, lens
    with_table = ops.rope_paged_append(qkv, None, None, cos[:30].contiguous(), sin[:30].contiguous(), bt["k"].clone(),
                                       bt["v"].clone(), bt["table"], bt["q_start"], bt["kv_lens"])  # position 39 of 30 rows
    assert with_table.shape == (3, 16, D)
    with pytest.raises(ValueError, match="KV capacity"):
        ops.check_device_errors(DEV)


def test_pools_beyond_32_bits():
    """Page ids whose elements lie past 2^32 in the pool."""
    from hackthenorth_b200 import ops

    pages, hkv, page = 70000, 8, 64  # 4.6e9 elements a pool
    k = torch.empty(pages, hkv, page, D, dtype=BF16, device=DEV)
    v = torch.empty_like(k)
    ids = torch.tensor([69999, 3, 65536, 69998], dtype=torch.int32, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(1)
    for i in ids.tolist():
        k[i] = torch.randn(hkv, page, D, generator=g, device=DEV).to(BF16)
        v[i] = torch.randn(hkv, page, D, generator=g, device=DEV).to(BF16)
    lens = [(1, 250)]
    for n in (1, 20):
        bt = dict(lens=[(n, 250)], hq=32, hkv=hkv, page=page, starts=[0, n], rows=n, prefix=0, prefix_table=ids[:0],
                  q=torch.randn(n, 32, D, generator=g, device=DEV).to(BF16), k=k, v=v, table=ids[None].contiguous(),
                  pages=ids[None], q_start=torch.tensor([0, n], dtype=torch.int32, device=DEV),
                  kv_lens=torch.tensor([250], dtype=torch.int32, device=DEV))
        _check(bt, _attend(bt, max_queries=n))
    qkv = torch.randn(1, 48 * D, generator=g, device=DEV).to(BF16)
    cos, sin = _tables(256)
    ops.rope_paged_append(qkv, None, None, cos, sin, k, v, ids[None].contiguous(), bt["q_start"] // 20, bt["kv_lens"])
    ops.check_device_errors(DEV)
    assert torch.equal(v[69998, :, 249 - 192], qkv.view(48, D)[40:])


def test_serving_steps_match_the_contiguous_operators():
    """Prompt appended and attended in one chunk, then single tokens, on pages:
    as ``rope_attention`` and ``grouped_attention`` on a contiguous cache, and a
    second sequence that shares the prompt as a prefix; the last row's token drawn."""
    from hackthenorth_b200 import ops

    hq, hkv, page, prompt, steps = 32, 8, 32, 75, 4
    g = torch.Generator(device=DEV).manual_seed(90)
    rnd = lambda *s: torch.randn(*s, generator=g, device=DEV).to(BF16)
    rows = rnd(prompt + steps, (hq + 2 * hkv) * D)
    qn, kn = (1 + 0.1 * torch.randn(2, D, generator=g, device=DEV)).to(BF16)
    cos, sin = _tables(128)
    kc, vc = (torch.zeros(hkv, 128, D, dtype=BF16, device=DEV) for _ in range(2))
    want = [ops.rope_attention(rows[p], qn, kn, cos, sin, kc, vc, torch.tensor([p], device=DEV), n_heads=hq)
            for p in range(prompt + steps)]
    k, v = (torch.full((12, hkv, page, D), float("nan"), dtype=BF16, device=DEV) for _ in range(2))
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)
    table = i32(7, 2, 9, 4)[None].contiguous()
    q = ops.rope_paged_append(rows[:prompt].contiguous(), qn, kn, cos, sin, k, v, table, i32(0, prompt), i32(prompt))
    got = list(ops.paged_attention(q, k, v, table, i32(0, prompt), i32(prompt)))
    own = i32(0, 11)[None].contiguous()
    for p in range(prompt, prompt + steps):
        row = rows[p][None].contiguous()
        q = ops.rope_paged_append(row, qn, kn, cos, sin, k, v, table, i32(0, 1), i32(p + 1))
        got.append(ops.paged_attention(q, k, v, table, i32(0, 1), i32(p + 1))[0])
        # the same token behind the prompt as a shared prefix, its own keys on other pages
        q = ops.rope_paged_append(row, qn, kn, cos, sin, k, v, own, i32(0, 1), i32(p + 1 - prompt), first_position=prompt)
        shared = ops.shared_prefix_attention(q, k, v, table[0], prompt, own, i32(0, 1), i32(p + 1 - prompt))[0]
        # two results of the same rows: each within the bound of the exact one
        assert ((shared.float() - got[-1].float()).abs().max() / got[-1].float().abs().max()).item() <= 2e-2
    ops.check_device_errors(DEV)
    for a, b in zip(got, want):  # the cache rows differ by bf16 ulps (products rounded or not), so the outputs do
        assert ((a.float() - b.float()).abs().max() / b.float().abs().max()).item() <= 2e-2
    token = ops.sample_token(got[-1].reshape(1, -1), torch.full((1,), 0.5, device=DEV), top_k=1)
    assert int(token) == int(got[-1].float().argmax())

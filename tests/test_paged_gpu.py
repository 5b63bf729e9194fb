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

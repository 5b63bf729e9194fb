"""Token sampling at the ends of the temperature's range.

At temperature infinity every token that can be drawn weighs exactly 1 (beside
an infinite logit nothing else weighs anything), so the definition is in whole
numbers and the drawn token has to be equal. The products of a uniform number
or ``top_p`` (24 bits) with a count (18 bits) are exact in 64 bits.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16 = torch.bfloat16
INF = float("inf")


@pytest.fixture(scope="module", autouse=True)
def _ready(built_lib):
    yield
    from hackthenorth_b200 import ops

    ops.check_device_errors(DEV)


def flat_token(x, u, top_k=0, top_p=1.0, min_p=0.0):
    """The token of one row whose drawable tokens all weigh 1."""
    x = x.double()
    x = torch.where(x.isnan(), -INF, x)
    top = x.max()
    order = torch.argsort(-x, stable=True)
    order = order[x[order] > -INF]
    weight = torch.ones_like(x) if top < INF else (x == INF).double()
    if top_k > 0:
        order = order[:top_k]
    if top_p < 1:
        ahead = weight[order].cumsum(0) - weight[order]
        keep = ahead < float(torch.tensor(top_p, dtype=torch.float32)) * weight[order].sum()
        keep[0] = True
        order = order[keep]
    order = order[weight[order] >= min_p]
    order = order[weight[order] > 0]
    return int(order.sort().values[math.floor(float(u) * len(order))])


FLAT = [dict(), dict(top_k=1), dict(top_k=5), dict(top_k=100), dict(top_k=3000), dict(top_k=5000), dict(top_p=0.003),
        dict(top_p=0.3), dict(top_p=0.999), dict(min_p=0.5), dict(top_k=40, top_p=0.5), dict(top_k=6000, top_p=0.9, min_p=1.0)]


@pytest.mark.parametrize("vocab", [1, 7, 200, 6001, 151936])
@pytest.mark.parametrize("dtype", [BF16, torch.float32])
def test_infinite_temperature_draws_evenly_of_what_is_kept(vocab, dtype):
    from hackthenorth_b200 import ops

    g = torch.Generator().manual_seed(vocab)
    rows = 4
    for kw in FLAT:
        x = (3 * torch.randn(rows, vocab, generator=g)).to(dtype)
        u = torch.rand(rows, generator=g)
        want = [flat_token(x[r], u[r], **kw) for r in range(rows)]
        for t in (INF, torch.full((rows,), INF, device=DEV)):
            out = torch.full((rows,), -7, dtype=torch.int64, device=DEV)
            ops.sample_token(x.to(DEV), u.to(DEV), t, out=out, **kw)
            assert out.tolist() == want, kw


def test_infinite_temperature_beside_finite_ones():
    from hackthenorth_b200 import ops

    g = torch.Generator().manual_seed(2)
    x = torch.randn(6, 5003, generator=g)
    u = torch.rand(6, generator=g)
    t = torch.tensor([INF, 0.7, INF, 0.0, 1.0, INF])
    for kw in (dict(), dict(top_k=50), dict(top_p=0.6)):
        out = torch.full((6,), -7, dtype=torch.int64, device=DEV)
        ops.sample_token(x.to(DEV), u.to(DEV), t.to(DEV), out=out, **kw)
        for r in range(6):
            if t[r] == INF:
                assert int(out[r]) == flat_token(x[r], u[r], **kw)
            else:
                assert int(out[r]) == int(ops.sample_token(x[r].to(DEV), u[r:r + 1].to(DEV), float(t[r]), **kw))


@pytest.mark.parametrize("vocab", [100, 6001])
def test_infinite_temperature_and_values_at_the_ends(vocab):
    """Masked places, the type's ends (their difference is past fp32) and infinite logits."""
    from hackthenorth_b200 import ops

    g = torch.Generator().manual_seed(3)
    x = torch.randn(4, vocab, generator=g)
    x[0, ::3] = -INF
    x[0, 1::3] = float("nan")
    x[1, ::2] = torch.finfo(torch.float32).min
    x[1, 5] = torch.finfo(torch.float32).max
    x[2, [4, 50, vocab - 1]] = INF
    x[3] = torch.finfo(torch.float32).min
    u = torch.tensor([0.8, 0.3, 0.7, 0.999])
    for kw in FLAT[1:]:
        out = torch.full((4,), -7, dtype=torch.int64, device=DEV)
        ops.sample_token(x.to(DEV), u.to(DEV), INF, out=out, **kw)
        assert out.tolist() == [flat_token(x[r], u[r], **kw) for r in range(4)], kw


def test_infinite_logits_take_all_the_mass_at_any_temperature():
    from hackthenorth_b200 import ops

    x = torch.zeros(64, 5000, device=DEV)
    x[:, [7, 4000]] = INF
    u = (torch.arange(64, device=DEV) / 64).float()
    for t in (1e-45, 1.0, 1e37, 3e38, INF):
        for kw in (dict(), dict(top_k=3), dict(top_p=0.999), dict(top_k=4500, top_p=0.9999)):
            got = ops.sample_token(x, u, t, **kw).tolist()
            assert got == [7] * 32 + [4000] * 32, (t, kw)


def test_temperatures_below_the_normal_numbers_count_as_the_least_of_them():
    from hackthenorth_b200 import ops

    least = 2.0 ** -126
    u = torch.rand(50, generator=torch.Generator().manual_seed(4)).to(DEV)
    near = (-torch.arange(300, device=DEV).float() * least).repeat(50, 1)  # weights e^-i at the least temperature
    far = (-torch.arange(300, device=DEV).float() * 1e-20).repeat(50, 1)
    for kw in (dict(), dict(top_k=20), dict(top_p=0.9), dict(top_k=280, top_p=0.95)):
        want = ops.sample_token(near / least, u, 1.0, **kw)
        for t in (least, 1e-40, 1e-45):
            assert torch.equal(ops.sample_token(near, u, t, **kw), want), (t, kw)
            assert bool((ops.sample_token(far, u, t, **kw) == 0).all())

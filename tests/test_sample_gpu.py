"""Token sampling on the GPU against the definition in 64 bits.

The drawn token is a whole number and has to be equal. The kernel's weights
carry a relative error of a few 2^-24 and its sums none, so a uniform number
chosen without regard to the logits falls on the other side of a token's edge
about once in 10^6 rows; the inputs here are fixed, and the ones that sit on an
edge on purpose have weights that are exact on both sides (equal logits).
"""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16 = torch.bfloat16


@pytest.fixture(scope="module", autouse=True)
def _ready(built_lib):
    yield
    from hackthenorth_b200 import ops

    ops.check_device_errors(DEV)


def draw64(x, u, temperature, top_k, top_p, min_p):
    """One row's token by the definition (numpy, 64 bits)."""
    x = x.astype(np.float64)
    x = np.where(np.isnan(x), -np.inf, x)
    top = x.max()
    if top == -np.inf:
        return -1
    if not temperature > 0:
        return int(x.argmax())
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.where(x == top, 1.0, np.exp(-np.minimum(np.where(x == top, 0.0, top - x) / np.float64(temperature), 1e300)))
    order = np.argsort(-x, kind="stable")
    order = order[x[order] > -np.inf]
    if top_k > 0:
        order = order[:top_k]
    if top_p < 1:
        ahead = np.concatenate(([0.0], np.cumsum(w[order])[:-1]))
        order = order[:max(1, int((ahead < np.float64(top_p) * w[order].sum()).sum()))]
    order = order[w[order] >= min(np.float64(min_p), 1.0)]
    idx = np.sort(order)
    mass = np.cumsum(w[idx])
    target = np.float64(u) * mass[-1]
    return int(idx[min(np.searchsorted(mass, target, side="right"), len(idx) - 1)])


def check(logits, uniforms, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    from hackthenorth_b200 import ops

    rows = logits.shape[0]

    def spread(v, dtype):
        return torch.as_tensor(v, dtype=dtype).expand(rows).contiguous()

    settings = [spread(temperature, torch.float32), spread(top_k, torch.int32), spread(top_p, torch.float32),
                spread(min_p, torch.float32)]
    got = ops.sample_token(logits.to(DEV), uniforms.to(DEV), *[s.to(DEV) for s in settings]).cpu()
    want = [draw64(logits[r].float().numpy(), float(uniforms[r]), *[s[r].item() for s in settings]) for r in range(rows)]
    assert got.tolist() == want
    scalars = [temperature, top_k, top_p, min_p]
    if not any(torch.is_tensor(s) for s in scalars):  # one number for all rows: the same
        assert torch.equal(ops.sample_token(logits.to(DEV), uniforms.to(DEV), *scalars).cpu(), got)


SETTINGS = [dict(), dict(top_k=1), dict(top_k=20), dict(top_k=3000), dict(top_p=0.9), dict(top_p=0.05), dict(min_p=0.05),
            dict(temperature=0.6, top_k=20, top_p=0.95), dict(temperature=1.7, top_k=500, top_p=0.5, min_p=0.01),
            dict(temperature=0.0), dict(temperature=0.01), dict(temperature=50.0, top_p=0.7), dict(top_k=2 ** 31 - 1),
            dict(top_p=1e-6), dict(min_p=1.0), dict(top_k=64), dict(top_k=65, top_p=0.7), dict(top_k=2500, top_p=0.99),
            dict(top_k=4097), dict(top_k=200, top_p=0.97, min_p=0.02), dict(temperature=1.2, top_p=0.999), dict(temperature=3.0, top_p=0.4)]


@pytest.mark.parametrize("vocab", [1, 7, 100, 4096, 50257, 151936, 262144])
@pytest.mark.parametrize("dtype", [BF16, torch.float32])
def test_draws_match_the_definition(vocab, dtype):
    g = torch.Generator().manual_seed(vocab)
    for i, kw in enumerate(SETTINGS):
        rows = 3
        x = 2.5 * torch.randn(rows, vocab, generator=g)
        x[:, torch.randint(0, vocab, (5,), generator=g)] += 7 * torch.rand(5, generator=g)
        check(x.to(dtype), torch.rand(rows, generator=g), **kw)


def test_rows_with_their_own_settings():
    g = torch.Generator().manual_seed(5)
    rows = 40
    x = (3 * torch.randn(rows, 5003, generator=g)).to(BF16)  # an odd width: rows without 16-byte alignment
    check(x, torch.rand(rows, generator=g), temperature=torch.rand(rows, generator=g) * 1.5 * (torch.rand(rows, generator=g) > 0.2),
          top_k=torch.randint(0, 300, (rows,), generator=g), top_p=0.2 + 0.9 * torch.rand(rows, generator=g),
          min_p=0.2 * torch.rand(rows, generator=g))


@pytest.mark.parametrize("dtype", [BF16, torch.float32])
def test_equal_logits_are_cut_by_index(dtype):
    # weights are exactly 1, so every edge is exact: a uniform number on an edge belongs to the next token
    rows = 64
    for value in (0.0, -7.5, torch.finfo(dtype).min):
        x = torch.full((rows, 6000), value, dtype=dtype)
        x[:, 1::2] = float("-inf")  # 3000 tokens, the even ones
        u = torch.arange(rows) / rows
        check(x, u, top_k=1024)
        check(x, u, top_p=0.5)
        check(x, u, top_k=1500, top_p=0.25)
        check(x, u)


def test_values_far_apart_and_within_one_sub_bin():
    g = torch.Generator().manual_seed(9)
    rows = 12
    u = torch.rand(rows, generator=g)
    near = 1.0 + torch.randint(0, 64, (rows, 3001), generator=g) * 2.0 ** -20  # fp32 values a few 2^-20 apart
    for kw in (dict(top_k=700), dict(top_p=0.3), dict(top_k=2000, top_p=0.6)):
        check(near, u, **kw)
    far = torch.randn(rows, 3001, generator=g) * 1e4
    far[:, ::7] = 3e38
    far[:, 3::7] = -3e38
    for kw in (dict(top_k=700), dict(top_p=0.3), dict(temperature=1e5, top_k=2900, top_p=0.999), dict(temperature=1e-30)):
        check(far, u, **kw)


def test_masked_infinite_and_nan_logits():
    g = torch.Generator().manual_seed(11)
    x = 2 * torch.randn(6, 1000, generator=g)
    x[0, :999] = float("-inf")
    x[1, 5:] = float("nan")
    x[2, [3, 700]] = float("inf")
    x[3] = torch.finfo(torch.float32).min
    x[3, 17] = 0.0
    x[4, ::2] = 0.0
    x[4, 1::2] = -0.0
    for kw in (dict(), dict(top_k=600), dict(top_p=0.9), dict(temperature=0.0), dict(top_k=100, top_p=0.5, min_p=0.1)):
        check(x, torch.rand(6, generator=g), **kw)


def test_a_row_without_a_token_is_reported():
    from hackthenorth_b200 import ops

    x = torch.full((2, 300), float("-inf"), device=DEV)
    x[1, 5] = 1.0
    assert ops.sample_token(x, torch.full((2,), 0.5, device=DEV)).tolist() == [-1, 5]
    with pytest.raises(ValueError, match="no token"):
        ops.check_device_errors(DEV)
    ops.check_device_errors(DEV)


def test_uniform_numbers_at_and_beyond_the_ends():
    from hackthenorth_b200 import ops

    x = torch.zeros(5, 10, device=DEV)
    u = torch.tensor([0.0, 1.0 - 2.0 ** -24, 1.0, -1.0, float("nan")], device=DEV)
    assert ops.sample_token(x, u).tolist() == [0, 9, 9, 0, 0]


def test_evenly_spread_numbers_give_the_probabilities():
    n = 4000
    x = torch.tensor([0.3, -1.0, 2.0, 0.3, float("-inf"), 1.1]).repeat(n, 1)
    from hackthenorth_b200 import ops

    got = ops.sample_token(x.to(DEV), ((torch.arange(n) + 0.5) / n).to(DEV)).cpu()
    want = torch.softmax(x[0].double(), 0) * n
    counts = torch.bincount(got, minlength=6).double()
    assert bool(((counts - want).abs() <= 1.0).all())  # each token owns one interval of the numbers
    assert bool((got.diff() >= 0).all())


def test_settings_greedy_and_captured_replay_agree():
    from hackthenorth_b200 import ops

    g = torch.Generator(device=DEV).manual_seed(3)
    x = torch.randn(4, 151936, generator=g, device=DEV).to(BF16)
    u = torch.rand(4, generator=g, device=DEV)
    out = torch.empty(4, dtype=torch.int64, device=DEV)
    eager = ops.sample_token(x, u, top_k=50, top_p=0.9)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.sample_token(x, u, top_k=50, top_p=0.9, out=out)
    graph.replay()
    assert torch.equal(out, eager)
    u.copy_(torch.rand(4, generator=g, device=DEV))
    graph.replay()
    assert torch.equal(out, ops.sample_token(x, u, top_k=50, top_p=0.9))
    assert torch.equal(ops.sample_token(x, u, temperature=0.0), x.float().argmax(1))

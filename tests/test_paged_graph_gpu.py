"""A serving step captured as one graph: append, attention (with and without a
shared prefix) and sampling, replayed while lengths, tables and rows change."""
import pytest
import torch

from paged_reference import BF16, D, attention64, attention_bound, make_batch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
HQ, HKV, PAGE, VOCAB = 16, 4, 32, 1000


@pytest.fixture(scope="module", autouse=True)
def _ready(built_lib):
    yield
    from hackthenorth_b200 import ops

    ops.check_device_errors(DEV)


@pytest.mark.parametrize("n,prefix", [(1, 0), (1, 700), (30, 0), (30, 700)])
def test_a_captured_step_follows_its_inputs(n, prefix):
    from hackthenorth_b200 import ops
    from hackthenorth_b200.config import QWEN3_0P6B
    from hackthenorth_b200.weights import rotary_table

    bt = make_batch([(n, 900), (1, 333), (0, 40)], HQ, HKV, PAGE, 51, DEV, pad=2, prefix=prefix)
    cos, sin = (t.to(DEV) for t in rotary_table(QWEN3_0P6B, 2000))
    g = torch.Generator(device=DEV).manual_seed(52)
    rows = torch.empty(bt["rows"], (HQ + 2 * HKV) * D, dtype=BF16, device=DEV)
    head = torch.randn(VOCAB, HQ * D, generator=g, device=DEV).to(BF16)
    u = torch.empty(bt["rows"], device=DEV)
    q, out = torch.full_like(bt["q"], 7.0), torch.full_like(bt["q"], 7.0)
    token = torch.empty(bt["rows"], dtype=torch.int64, device=DEV)
    tail = (bt["table"], bt["q_start"], bt["kv_lens"])

    def step():
        ops.rope_paged_append(rows, None, None, cos, sin, bt["k"], bt["v"], *tail, first_position=prefix, out=q)
        if prefix:
            ops.shared_prefix_attention(q, bt["k"], bt["v"], bt["prefix_table"], prefix, *tail, max_queries=n, out=out)
        else:
            ops.paged_attention(q, bt["k"], bt["v"], *tail, max_queries=n, out=out)
        ops.sample_token(out.view(bt["rows"], -1) @ head.T, u, 0.8, top_k=50, top_p=0.9, out=token)

    rows.normal_(generator=g)
    u.uniform_(generator=g)
    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for shorter in (0, 100, 301):
        bt["lens"] = [(m, max(kv - shorter, m)) for m, kv in [(n, 900), (1, 333), (0, 40)]]
        bt["kv_lens"].copy_(torch.tensor([kv for _, kv in bt["lens"]], dtype=torch.int32))
        order = torch.randperm(bt["pages"].shape[1], generator=torch.Generator().manual_seed(shorter)).to(DEV)
        if shorter:  # the first sequence's pages in another order
            bt["table"][0, :29] = bt["pages"][0, :29][order[order < 29]]
            bt["pages"] = bt["table"].clone()
        rows.normal_(generator=g)
        u.uniform_(generator=g)
        graph.replay()
        replayed = (q.clone(), out.clone(), token.clone())
        ops.check_device_errors(DEV)
        step()
        for a, b in zip(replayed, (q, out, token)):
            assert torch.equal(a, b)
        bt["q"] = q
        ref, mag = attention64(bt)
        used = bt["starts"][-1]
        assert bool(((out[:used].double() - ref[:used]).abs() <= attention_bound(ref[:used], mag[:used])).all())
        assert bool((out[used:] == 7.0).all())

"""Sampled generation through the Engine: settings are checked on the CPU; on
the GPU the drawn tokens are those of ``ops.sample_token`` on the step's logits."""
import pytest
import torch

DEV = "cuda:0"
PROMPT = [645, 610, 926, 2984, 3233, 1274, 986, 2860]


@pytest.mark.parametrize("kw", [dict(temperature=-0.1), dict(temperature=float("inf")), dict(temperature=float("nan")),
                                dict(top_k=-1), dict(top_k=1.5), dict(top_p=0.0), dict(top_p=1.1), dict(min_p=-0.1),
                                dict(min_p=2.0)])
def test_settings_are_checked(kw):
    from hackthenorth_b200 import Sampling

    with pytest.raises(ValueError):
        Sampling(**kw)


@pytest.fixture(scope="module")
def engine(built_lib):
    from hackthenorth_b200 import Engine
    from hackthenorth_b200.config import QWEN3_SMALL

    return Engine.from_random(QWEN3_SMALL, seed=0)


@pytest.mark.gpu
def test_greedy_settings_give_the_greedy_tokens(engine):
    from hackthenorth_b200 import Sampling

    greedy = [s[0] for s in engine.generate([PROMPT], 12, draft_tokens=0)]
    for sampling in (Sampling(temperature=0.0), Sampling(top_k=1, seed=3), Sampling(top_p=1e-9)):
        assert [s[0] for s in engine.generate([PROMPT], 12, sampling=sampling)] == greedy
    assert [s[0] for s in engine.generate([PROMPT], 12)] == greedy  # and plain calls are as before
    engine.state.check()


@pytest.mark.gpu
@pytest.mark.parametrize("batch", [1, 3])
def test_steps_draw_from_their_logits(engine, batch):
    from hackthenorth_b200 import Sampling, ops

    s = Sampling(temperature=1.3, top_k=200, top_p=0.95, min_p=0.001, seed=5)
    state = engine.new_state(len(PROMPT), 6, batch=batch, sampling=s)
    numbers = torch.Generator(device=DEV)
    numbers.manual_seed(5)
    ids = torch.tensor([PROMPT] * batch if batch > 1 else PROMPT, device=DEV)
    tokens = []
    for step in range(6):
        if step == 0:
            state.prefill(ids)
        else:
            state.step()
        u = torch.empty(batch, device=DEV).uniform_(generator=numbers)
        want = ops.sample_token(state.logits, u, s.temperature, s.top_k, s.top_p, s.min_p)
        assert torch.equal(state.token, want)
        tokens.append(state.read_token())
    assert state.position.tolist() == [len(PROMPT) + 5] * batch
    state.check()
    if batch > 1:  # the sequences draw numbers of their own
        assert len({tuple(t[b] for t in tokens) for b in range(batch)}) == batch


@pytest.mark.gpu
def test_a_seed_repeats_and_another_differs(engine):
    from hackthenorth_b200 import Sampling

    run = lambda seed, prompts: [tuple(s) for s in engine.generate(prompts, 10, sampling=Sampling(temperature=1.5, seed=seed))]
    first = run(1, [PROMPT])
    assert run(1, [PROMPT]) == first and run(2, [PROMPT]) != first
    many = run(1, [PROMPT] * 11)  # two chunks
    assert run(1, [PROMPT] * 11) == many and len({t[i] for t in many for i in range(11)}) > 11
    assert len(set(zip(*many))) == 11


@pytest.mark.gpu
def test_sampling_is_refused_beside_speculation(engine):
    from hackthenorth_b200 import Sampling

    with pytest.raises(ValueError, match="speculation"):
        next(engine.generate([PROMPT], 4, draft_tokens=2, sampling=Sampling()))
    state = engine.new_state(len(PROMPT), 4, draft_tokens=2, sampling=Sampling())
    state.prefill(torch.tensor(PROMPT, device=DEV))
    with pytest.raises(ValueError, match="greedy"):
        state.verify(1, [2])
    plain = engine.new_state(len(PROMPT), 4)
    with pytest.raises(ValueError, match="without sampling"):
        plain.set_sampling(Sampling())

"""Sampled decode states: reuse by greedy calls, their own checks, and steps
taken outside of ``generate``."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
PROMPT = [645, 610, 926, 2984, 3233, 1274, 986, 2860]


@pytest.fixture(scope="module")
def engine(built_lib):
    from hackthenorth_b200 import Engine
    from hackthenorth_b200.config import QWEN3_SMALL

    return Engine.from_random(QWEN3_SMALL, seed=0)


def test_speculation_does_not_reuse_a_sampled_state(engine):
    from hackthenorth_b200 import Sampling

    greedy = [s[0] for s in engine.generate([PROMPT], 10, draft_tokens=0)]
    for seed in range(3):
        engine.new_state(len(PROMPT), 10, draft_tokens=3, sampling=Sampling(temperature=1e4, seed=seed))
        assert [s[0] for s in engine.generate([PROMPT], 10, draft_tokens=3)] == greedy


@pytest.mark.parametrize("batch", [1, 2])
def test_check_reports_logits_without_a_token(engine, batch):
    from hackthenorth_b200 import Sampling, ops

    state = engine.new_state(len(PROMPT), 4, batch=batch, sampling=Sampling())
    state.prefill(torch.tensor([PROMPT] * batch if batch > 1 else PROMPT, device=DEV))
    state.check()
    state.logits.fill_(float("nan"))
    state._draw()
    assert state.read_token() == [-1] * batch
    with pytest.raises(ValueError, match="no token"):
        state.check()
    state.check()  # reported once
    ops.check_device_errors(DEV)  # and not to the operators' callers


def test_steps_outside_of_generate(engine):
    """A state that ``generate`` made (in inference mode) takes further steps outside of it."""
    from hackthenorth_b200 import Sampling

    tokens = list(engine.generate([PROMPT], 3, sampling=Sampling(seed=1)))
    assert len(tokens) == 3
    state = engine.new_state(len(PROMPT), 6, sampling=Sampling(seed=1))
    state.prefill(torch.tensor(PROMPT, device=DEV))
    with torch.inference_mode():
        state.set_sampling(Sampling(seed=1))
    state.step()
    state.check()

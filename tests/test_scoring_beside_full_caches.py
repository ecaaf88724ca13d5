"""Scores where running requests hold every state slot, and forks whose scores are switched on and off."""
import pytest
import torch

import helpers
from kungfu_b200 import api
from kungfu_b200.cache import CacheError
from kungfu_b200.engine.engine import Engine
from kungfu_b200.sampling import Sampling

CFG = helpers.TINY_A


@pytest.fixture(scope="module")
def folder(tmp_path_factory):
    return helpers.write_model(str(tmp_path_factory.mktemp("full") / "m"), CFG, seed=4, dtype=torch.float32, draw="loud")


@pytest.fixture
def engine(folder, cpu_ops):
    cfg, model = api.load_model(folder, dtype="float32", device="cpu")
    return Engine(runner=api.make_runner(cfg, model, dtype="float32", device="cpu", page_size=4, max_tokens=256, max_requests=3, max_context=64),
                  batch=16, parallel=3)


def test_a_score_without_a_state_slot_says_so(engine):
    ids = [engine.add_request([i, 2, 3], Sampling(temperature=0.0), max_tokens=5, ignore_eos=True) for i in range(3)]
    while not all(engine.requests[i].output for i in ids):
        engine.step()
    with pytest.raises(CacheError, match="state slot"):
        engine.score([[1, 2, 3]])
    while not engine.idle:
        engine.step()
    assert len(engine.score([[1, 2, 3]])[0]) == 2 and all(len(engine.requests[i].output) == 5 for i in ids)


def test_a_fork_without_its_parents_scores(engine):
    a = engine.add_request([5, 2, 3], Sampling(temperature=0.0), max_tokens=7, ignore_eos=True, logprobs=2)
    while len(engine.requests[a].output) < 3:
        engine.step()
    b, c = engine.fork(a, logprobs=None), engine.fork(a)
    with pytest.raises(ValueError):
        engine.fork(a, logprobs=65)
    while not engine.idle:
        engine.step()
    assert engine.requests[b].scores == [] and engine.requests[b].logprobs is None
    assert [len(engine.requests[i].scores) for i in (a, c)] == [7, 7] and engine.requests[a].output == engine.requests[b].output

"""Scores with alternatives beside captured decode graphs: the logits they look at are none of the steps' buffers."""
import pytest
import torch

import helpers
from kungfu_b200 import api
from kungfu_b200.engine.engine import Engine
from kungfu_b200.sampling import Sampling

CFG = helpers.TINY_A


@pytest.fixture(scope="module")
def folder(tmp_path_factory):
    return helpers.write_model(str(tmp_path_factory.mktemp("buffers") / "m"), CFG, seed=4, dtype=torch.float32, draw="loud")


def test_scores_leave_the_steps_buffers_alone(folder, cpu_ops):
    cfg, model = api.load_model(folder, dtype="float32", device="cpu")
    runner = api.make_runner(cfg, model, dtype="float32", device="cpu", page_size=4, max_tokens=256, max_requests=4,
                             max_context=CFG["max_position_embeddings"])
    eng = Engine(runner=runner, batch=16, parallel=4)
    eng.score([helpers.random_tokens(17, 512, 1)])            # every buffer of a step of 16 rows has its size now
    generation, held = runner.buffers.generation, runner.buffers.nbytes()
    for n in (3, 9, 17):
        eng.score([helpers.random_tokens(n, 512, n)], top=3)
    assert (runner.buffers.generation, runner.buffers.nbytes()) == (generation, held)


@pytest.mark.gpu
def test_scores_leave_captured_graphs_alone(folder):
    eng = Engine(folder, dtype="bfloat16", device="cuda:0", ctx=512, batch=64, parallel=2, page_size=16, cuda_graphs=True)
    eng.warm_up()
    prompt = helpers.random_tokens(57, 512, 1)
    eng.score([prompt])
    first = eng.generate([prompt[:9]], Sampling(temperature=0.0), max_tokens=8, ignore_eos=True)
    captured = {k: g["graph"] for k, g in eng.runner._graphs.items() if g["graph"] is not None}
    assert captured
    for n in (5, 33, 57):
        eng.score([prompt[:n]], top=5)
    assert eng.generate([prompt[:9]], Sampling(temperature=0.0), max_tokens=8, ignore_eos=True) == first
    assert all(eng.runner._graphs[k]["graph"] is g for k, g in captured.items())

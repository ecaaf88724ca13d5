"""A beam search whose next best tokens are mostly ids that end an answer still keeps as many open ones as it was asked for."""
import pytest
import torch

import helpers
import plain_gemma2
import scoring_cases as sc
from kungfu_b200 import api
from kungfu_b200.engine.engine import Engine

CFG = helpers.TINY_A


@pytest.fixture(scope="module")
def model(tmp_path_factory):
    folder = helpers.write_model(str(tmp_path_factory.mktemp("ends") / "m"), CFG, seed=4, dtype=torch.float32, draw="loud")
    return folder, helpers.read_tensors(folder)


@pytest.mark.parametrize("beams,ends", [(1, 2), (1, 7), (2, 4), (3, 6), (3, 20), (4, 9)])
def test_the_best_first_tokens_all_end_an_answer(model, cpu_ops, beams, ends):
    folder, tensors = model
    cfg, m = api.load_model(folder, dtype="float32", device="cpu")
    eng = Engine(runner=api.make_runner(cfg, m, dtype="float32", device="cpu", page_size=4, max_tokens=256, max_requests=8, max_context=64),
                 batch=16, parallel=8)
    prompt = helpers.random_tokens(9, 512, 4)                 # the prompt of `check_beams`
    first = plain_gemma2.forward(CFG, tensors, prompt)[-1]
    eos = tuple(torch.argsort(first, descending=True)[:ends].tolist())
    sc.check_beams(eng, CFG, tensors, 1.6e-3, beams=beams, max_tokens=6, eos=eos, length_penalty=2.5)

"""The commands that report log probabilities, in this process: on the CPU stand-in, and what a device has recorded on the GPU."""
import json
from types import SimpleNamespace

import pytest
import torch

import helpers
from kungfu_b200 import api, cli, ops
from kungfu_b200.engine.engine import Engine
from kungfu_b200.sampling import TokenScore

CFG = helpers.TINY_A
IDS = helpers.random_tokens(9, 512, 2)


@pytest.fixture(scope="module")
def folder(tmp_path_factory):
    return helpers.write_model(str(tmp_path_factory.mktemp("cli_scoring") / "m"), CFG, seed=4, dtype=torch.float32, draw="loud")


@pytest.fixture
def program(folder, cpu_ops, monkeypatch, capsys):
    """A function that runs a command on the CPU stand-in and gives what it prints; `.engines`: the engines it made, `.eos`: the ids
    that end a text."""
    engines = []

    def engine(args, parallel=1):
        cfg, model = api.load_model(folder, dtype="float32", device="cpu")
        runner = api.make_runner(cfg, model, dtype="float32", device="cpu", page_size=4, max_tokens=256, max_requests=max(parallel, 2), max_context=64)
        engines.append(Engine(runner=runner, batch=16, parallel=max(parallel, 2)))
        engines[-1].cfg = SimpleNamespace(eos_token_id=run.eos)
        return engines[-1]

    def run(*args):
        assert cli.main([*args, "--model", folder, "--ids", json.dumps(IDS)]) == 0
        return json.loads(capsys.readouterr().out)

    monkeypatch.setattr(cli, "_engine", engine)
    run.engines, run.eos = engines, ()
    return run


@pytest.mark.gpu
def test_a_scored_generation_raises_what_the_device_recorded(folder, capsys):
    with pytest.raises(ops.KernelError, match="gave up waiting"):
        ops._dev_scratch(torch.device("cuda", 0))["error"].fill_(1)          # as a product that gave up would leave it
        try:
            cli.main(["generate", "--model", folder, "--ids", json.dumps(IDS), "--max-tokens", "3", "--ignore-eos", "--ctx", "64", "--logprobs", "1"])
        finally:
            ops.clear_device_error(torch.device("cuda", 0))
    assert cli.main(["generate", "--model", folder, "--ids", json.dumps(IDS), "--max-tokens", "3", "--ignore-eos", "--ctx", "64", "--logprobs", "1"]) == 0
    assert len(json.loads(capsys.readouterr().out)["scores"]) == 3


def test_a_scored_generation_runs_as_the_plain_one(program, monkeypatch):
    ends = []
    monkeypatch.setattr(Engine, "run_to_end", lambda self, ids, run=Engine.run_to_end: (ends.append(list(ids)), run(self, ids))[1])
    plain = program("generate", "--max-tokens", "6", "--ignore-eos")
    scored = program("generate", "--max-tokens", "6", "--ignore-eos", "--logprobs", "2")
    assert scored["generated"] == plain["generated"] and [s["token"] for s in scored["scores"]] == plain["generated"]
    assert len(ends) == 2


def test_the_id_that_ends_a_text_is_taken_off_its_scores_too(program):
    ids = program("generate", "--max-tokens", "8", "--ignore-eos")["generated"]
    program.eos = (ids[4],)
    n = ids.index(ids[4])
    plain = program("generate", "--max-tokens", "8")
    scored = program("generate", "--max-tokens", "8", "--logprobs", "0")
    assert plain["generated"] == scored["generated"] == ids[:n] and [s["token"] for s in scored["scores"]] == ids[:n]
    whole = program("generate", "--max-tokens", "8", "--logprobs", "0", "--emit-ids")
    assert whole["generated"] == ids[:n + 1] and [s["token"] for s in whole["scores"]] == ids[:n + 1]


def test_the_id_that_ends_a_text_is_taken_off_beams(program):
    program.eos = tuple(range(0, 512, 5))
    bare = program("generate", "--max-tokens", "6", "--beams", "4")["beams"]
    whole = program("generate", "--max-tokens", "6", "--beams", "4", "--emit-ids")["beams"]
    assert any(b["finish"] == "eos" for b in whole)
    for a, b in zip(bare, whole):
        ended = b["finish"] == "eos"
        assert (b["generated"][-1] in program.eos) == ended and a["logprob"] == b["logprob"]
        assert a["generated"] == (b["generated"][:-1] if ended else b["generated"])


@pytest.mark.parametrize("args", [("generate", "--beams", "0"), ("generate", "--beams", "-3")] + [("generate", "--beams", "2", *more) for more in (
    ("--temperature", "0.7"), ("--repeat-penalty", "1.2"), ("--min-p", "0.1"), ("--logprobs", "0"))] + [
        ("score", "--logprobs", "--prefix", "3"), ("score", "--logprobs", "--ignore-eos")])
def test_options_that_would_have_no_effect_are_refused(program, args):
    with pytest.raises(SystemExit, match="error: .*--"):
        program(*args)
    assert not program.engines


@pytest.mark.parametrize("logprob,perplexity", [(-2.0, 7.38905609893065), (-700.0, 1.0142320547350045e304), (-5000.0, float("inf")),
                                                (float("-inf"), float("inf")), (float("nan"), float("nan"))])
def test_the_perplexity_of_any_text(program, monkeypatch, logprob, perplexity):
    monkeypatch.setattr(Engine, "score", lambda self, prompts, top=0: [[TokenScore(t, logprob, 1.0) for t in p[1:]] for p in prompts])
    doc = program("score", "--logprobs")
    assert doc["perplexity"] == pytest.approx(perplexity, nan_ok=True)

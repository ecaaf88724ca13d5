"""The commands that report log probabilities, in this process: on the CPU stand-in, and what a device has recorded on the GPU."""
import json

import pytest
import torch

import helpers
from kungfu_b200 import api, cli, ops
from kungfu_b200.engine.engine import Engine

CFG = helpers.TINY_A
IDS = helpers.random_tokens(9, 512, 2)


@pytest.fixture(scope="module")
def folder(tmp_path_factory):
    return helpers.write_model(str(tmp_path_factory.mktemp("cli_scoring") / "m"), CFG, seed=4, dtype=torch.float32, draw="loud")


@pytest.fixture
def program(folder, cpu_ops, monkeypatch, capsys):
    """A function that runs a command on the CPU stand-in and gives what it prints; `.engines`: the engines it made."""
    engines = []

    def engine(args, parallel=1):
        cfg, model = api.load_model(folder, dtype="float32", device="cpu")
        runner = api.make_runner(cfg, model, dtype="float32", device="cpu", page_size=4, max_tokens=256, max_requests=max(parallel, 2), max_context=64)
        engines.append(Engine(runner=runner, batch=16, parallel=max(parallel, 2)))
        engines[-1].cfg = cfg
        return engines[-1]

    def run(*args):
        assert cli.main([*args, "--model", folder, "--ids", json.dumps(IDS)]) == 0
        return json.loads(capsys.readouterr().out)

    monkeypatch.setattr(cli, "_engine", engine)
    run.engines = engines
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

"""What the log probabilities and the copies of pages refuse, before anything reaches a device."""
import pytest
import torch

from kungfu_b200 import ops
from kungfu_b200.ops import KernelError

I32 = torch.int32


def _t(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype)


@pytest.mark.parametrize("change", [
    dict(logits=_t(4, 10, dtype=torch.float16)), dict(logits=_t(40)), dict(logits=_t(4, 0)), dict(logits=_t(10, 4).T),
    dict(tokens=_t(4, dtype=torch.int64)), dict(tokens=_t(3, dtype=I32)), dict(tokens=_t(8, dtype=I32)[::2]), dict(tokens=None),
    dict(out_logprob=_t(5)), dict(out_logprob=_t(4, dtype=torch.bfloat16)), dict(out_logprob=_t(8)[::2]),
    dict(out_entropy=_t(4, 1)), dict(out_rank=_t(4)), dict(out_top_ids=_t(4, 0, dtype=I32)), dict(out_top_ids=_t(4, 11, dtype=I32)),
    dict(out_top_ids=_t(4, 3)), dict(out_top_ids=_t(4, 3, dtype=I32), out_top_logprobs=_t(4, 2)), dict(out_top_logprobs=_t(3, 2)),
    dict(out_top_logprobs=_t(4)), dict(logits=_t(4, 100), out_top_ids=_t(4, 65, dtype=I32)),
    dict(out_logprob=None),
])
def test_token_logprobs_refuses(change):
    args = dict(logits=_t(4, 10), tokens=_t(4, dtype=I32), out_logprob=_t(4))
    args.update(change)
    with pytest.raises(KernelError, match="token_logprobs"):
        ops.token_logprobs(args.pop("logits"), args.pop("tokens"), args.pop("out_logprob"), **args)


@pytest.mark.parametrize("change", [
    dict(x=_t(4, 6)), dict(x=_t(4, 16)[:, ::2]), dict(x=_t(4, 8, dtype=torch.float16)), dict(weight=_t(8)), dict(weight=_t(0, 8)),
    dict(tokens=_t(3, dtype=I32)), dict(tokens=_t(4)), dict(tokens=None), dict(out_logprob=None), dict(out_logprob=_t(2)), dict(out_entropy=_t(5)),
    dict(softcap=-1.0), dict(softcap=float("nan")), dict(softcap=float("inf")), dict(weight=_t(20, 8, dtype=torch.int32)),
])
def test_head_logprobs_refuses(change):
    args = dict(x=_t(4, 8), weight=_t(20, 8), tokens=_t(4, dtype=I32), out_logprob=_t(4))
    args.update(change)
    with pytest.raises(KernelError, match="head_logprobs"):
        ops.head_logprobs(args.pop("x"), args.pop("weight"), args.pop("tokens"), args.pop("out_logprob"), **args)


@pytest.mark.parametrize("stores,src,dst", [
    ([_t(5, 3)], [0, 1], [2]), ([_t(5, 3)], [0], [2, 3]), ([_t(5, 3)], [0, 1], [2, 2]), ([_t(5, 3)], [0, 2], [2, 3]), ([_t(5, 3)], [1], [1]),
    ([_t(5, 3)], [-1], [2]), ([_t(5, 3)], [0], [-2]), ([_t(5, 3)], [0], [5]), ([_t(5, 3)], [7], [0]), ([_t(5, 3), _t(4, 3)], [0], [4]),
    ([_t(5, 6)[:, ::2]], [0], [1]), ([torch.tensor(1.0)], [0], [1]),
])
def test_copy_pages_refuses(stores, src, dst):
    with pytest.raises(KernelError, match="copy_pages"):
        ops.copy_pages(stores, src, dst)


def test_there_is_no_cpu_path():
    for call in (lambda: ops.token_logprobs(_t(2, 5), _t(2, dtype=I32), _t(2)),
                 lambda: ops.head_logprobs(_t(2, 8), _t(5, 8), _t(2, dtype=I32), _t(2)),
                 lambda: ops.copy_pages([_t(4, 2)], [0], [1])):
        with pytest.raises(KernelError, match="CUDA"):
            call()


def test_tensors_of_another_device_than_the_current_one_are_refused(monkeypatch):
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 1)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 1)
    with pytest.raises(KernelError, match="current device is cuda:1"):
        ops._current("token_logprobs", 0)
    with pytest.raises(KernelError, match="another device"):
        ops._checked("token_logprobs", 0, (("tokens", _t(4, dtype=I32), (4,), I32),))

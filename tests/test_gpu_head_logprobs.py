"""Log probabilities straight from the rows that enter the output head, against the product, cap and softmax in 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
UNIT = 2.0 ** -24


def make(R, K, V, dtype, seed=0, spread=2.5):
    g = torch.Generator(device=DEV).manual_seed(seed + R + K + V)
    w = (torch.randn(V, K, generator=g, device=DEV) * spread / math.sqrt(K)).to(dtype)
    t = torch.randint(0, V, (R,), generator=g, device=DEV)
    x = torch.randn(R, K, generator=g, device=DEV)
    x += w[t].float() * 2.0 * torch.rand(R, 1, generator=g, device=DEV)
    return x.to(dtype), w, t.to(torch.int32)


def plain(x, w, tokens, cap):
    """(logprob, entropy, how far a logit may be off) in 64 bits.  A logit is a sum of K products accumulated in 32-bit numbers:
    on the tensor cores sixteen exact products at a time (each addition within one step, 2^-23, of the running magnitude), on the FMA
    units one at a time (half a step); the cap's slope is at most 1, its tanh within 4 steps of 2^-23."""
    K = x.shape[1]
    lp, ent, off = [], [], 0.0
    for a in range(0, x.shape[0], 64):
        xs = x[a:a + 64].double()
        v = xs @ w.double().T
        sizes = xs.abs() @ w.double().abs().T
        off = max(off, float(sizes.max()) * ((K / 16 + 18) * 2.0 ** -23 if x.dtype == torch.bfloat16 else (K + 2) * UNIT))
        if cap > 0:
            v = cap * torch.tanh(v / cap)
        lse = torch.logsumexp(v, 1)
        p = torch.exp(v - lse[:, None])
        lp.append(v.gather(1, tokens[a:a + 64].long()[:, None])[:, 0] - lse)
        ent.append(lse - (p * v).sum(1))
    return torch.cat(lp), torch.cat(ent), off + (4 * 2.0 ** -23 * cap if cap > 0 else 0.0)


def run(x, w, tokens, cap):
    from kungfu_b200 import ops
    lp, ent = (torch.full((x.shape[0],), 7.0, device=DEV) for _ in range(2))
    ops.head_logprobs(x, w, tokens, lp, out_entropy=ent, softcap=cap)
    return lp, ent


def check(x, w, tokens, cap):
    from kungfu_b200 import ops
    V = w.shape[0]
    lp, ent = run(x, w, tokens, cap)
    want_lp, want_ent, off = plain(x, w, tokens, cap)
    # log s: as far off as the farthest logit, plus the sums (chains under V / 1024 additions, trees under 96, arguments 26);
    # the entropy moves with the logits by at most their error times (1 + the spread of x - lse under p, itself below 1 + log V)
    sums = (V / 1024 + 122) * UNIT
    assert bool(((lp.double() - want_lp).abs() <= 2 * off + sums * (1 + want_lp.abs())).all()), float((lp.double() - want_lp).abs().max())
    assert bool(((ent.double() - want_ent).abs() <= 2 * off * (2 + math.log(V)) + sums * (1 + want_ent.abs())).all()), \
        float((ent.double() - want_ent).abs().max())
    ops.raise_on_device_error()
    return lp, ent


# rows below, at and above the tiles (16, 32, 64, 128, 256); widths below a stage, ending inside one, of many; vocabularies likewise
@pytest.mark.parametrize("cap", [0.0, 30.0])
@pytest.mark.parametrize("R,K,V", [(1, 8, 1), (1, 64, 2), (2, 72, 255), (16, 128, 256), (17, 136, 257), (33, 192, 511), (64, 64, 1000), (65, 256, 3000),
                                   (127, 200, 777), (128, 512, 32003), (129, 520, 5000), (255, 64, 513), (256, 640, 4096), (257, 1000, 20001),
                                   (513, 328, 999), (1000, 96, 300)])
def test_bfloat16_rows_of_any_size(R, K, V, cap):
    check(*make(R, K, V, torch.bfloat16), cap)


@pytest.mark.parametrize("cap", [0.0, 30.0])
@pytest.mark.parametrize("R,K,V", [(1, 1, 1), (1, 5, 3), (3, 33, 100), (40, 512, 3000), (130, 100, 1001)])
def test_32_bit_rows(R, K, V, cap):
    check(*make(R, K, V, torch.float32), cap)


@pytest.mark.parametrize("K", [4, 7, 33, 100])
def test_bfloat16_rows_that_no_tile_load_takes(K):
    check(*make(21, K, 400, torch.bfloat16), 0.0)


def test_mixed_types():
    x, w, t = make(9, 64, 500, torch.bfloat16)
    lp, _ = run(x.float(), w, t, 0.0)
    want, _, off = plain(x.float(), w.float(), t, 0.0)
    assert bool(((lp.double() - want).abs() <= 2 * off + 200 * UNIT * (1 + want.abs())).all())


def test_whole_vocabulary():
    check(*make(70, 2304, 256000, torch.bfloat16), 30.0)


def test_more_rows_than_one_launch_takes(monkeypatch):
    from kungfu_b200 import ops
    x, w, t = make(700, 64, 3000, torch.bfloat16)
    for rows in (256, 100):                                   # (which worker sums which tile depends on the rows of a launch: not the same bits)
        monkeypatch.setattr(ops, "HEAD_ROWS", rows)
        check(x, w, t, 30.0)
    xf, wf = x.float(), w.float()
    whole = run(xf, wf, t, 30.0)
    monkeypatch.setattr(ops, "LOGITS_PIECE_BYTES", 100 * 4 * 3000)
    assert all(torch.equal(a, b) for a, b in zip(run(xf, wf, t, 30.0), whole))


def test_padding_rows_and_strange_tokens():
    x, w, t = make(150, 128, 3001, torch.bfloat16)
    whole, ent = run(x, w, t, 0.0)
    for r, v in ((0, -1), (3, 3001), (149, -7), (64, 2 ** 31 - 1)):
        t[r] = v
    lp, en = run(x, w, t, 0.0)
    for r in (0, 149):
        assert float(lp[r]) == float(en[r]) == 7.0
    for r in (3, 64):
        assert math.isnan(float(lp[r])) and float(en[r]) == float(ent[r])
    others = [r for r in range(150) if r not in (0, 3, 64, 149)]
    assert torch.equal(lp[others], whole[others]) and torch.equal(en[others], ent[others])


def test_logits_that_are_no_numbers():
    x, w, t = make(5, 64, 700, torch.bfloat16)
    x[2, 3] = float("nan")
    lp, ent = run(x, w, t, 0.0)
    keep = [0, 1, 3, 4]
    want, want_ent = run(x[keep].contiguous(), w, t[keep].contiguous(), 0.0)
    assert math.isnan(float(lp[2])) and math.isnan(float(ent[2]))
    assert torch.equal(lp[keep], want) and torch.equal(ent[keep], want_ent)


def test_huge_logits():
    x, w, t = make(20, 256, 2000, torch.bfloat16, spread=900.0)
    check(x, w, t, 0.0)
    check(x, w, t, 30.0)


def test_no_entropy_and_no_rows():
    from kungfu_b200 import ops
    x, w, t = make(6, 64, 300, torch.bfloat16)
    lp = torch.empty(6, device=DEV)
    ops.head_logprobs(x, w, t, lp)
    assert torch.equal(lp, run(x, w, t, 0.0)[0])
    ops.head_logprobs(x[:0], w, t[:0], lp[:0])


def test_streams_and_graphs():
    """Calls on two streams at a time, and two graphs captured from the same operands and replayed at a time, do not share sums."""
    from kungfu_b200 import ops
    cases = [make(300, 256, 9000, torch.bfloat16), make(40, 512, 30000, torch.bfloat16, seed=9)]
    want = [run(x, w, t, 30.0) for x, w, t in cases]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [None, None]
    for _ in range(4):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i] = run(*cases[i], 30.0)
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(p, q) for p, q in zip(a, b))
    outs, graphs = [torch.empty_like(w[0]) for w in want], []
    for (x, w, t), lp in zip(cases, outs):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ops.head_logprobs(x, w, t, lp, softcap=30.0)
        graphs.append(graph)
    for _ in range(3):
        for lp in outs:
            lp.fill_(0.0)
        torch.cuda.synchronize()
        for graph, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(lp, w[0]) for lp, w in zip(outs, want))
    ops.raise_on_device_error()


# pairs and single blocks; the loads stop before the first stage, inside the first run of K and beyond the ring (a pair's only tile has
# 1,024 / 128 = 8 stages)
@pytest.mark.parametrize("R", [20, 300])
@pytest.mark.parametrize("drop", [0, 3, 6])
def test_a_product_whose_operands_never_arrive(R, drop):
    """A test hook makes the producers leave out their loads from a stage on, with a limit of 2 ms: the kernel comes back by itself with its
    code and NaN, and is right again after."""
    import ctypes
    from kungfu_b200 import ops
    lib = ops.library()
    x, w, t = make(R, 1024, 3000, torch.bfloat16)
    right = run(x, w, t, 0.0)
    torch.cuda.synchronize()
    assert ops.device_error() == 0
    assert lib.kf_test_head_give_up(ctypes.c_ulonglong(2_000_000), drop) == 0
    try:
        lp, _ = run(x, w, t, 0.0)
        torch.cuda.synchronize()
        assert ops.device_error() == 65
        with pytest.raises(ops.KernelError, match="the head's log probabilities, operands never arrived"):
            ops.raise_on_device_error()
        assert bool(torch.isnan(lp).all())
    finally:
        assert lib.kf_test_head_give_up(ctypes.c_ulonglong(0), -1) == 0
        ops.clear_device_error()
    again = run(x, w, t, 0.0)
    ops.raise_on_device_error()
    assert all(torch.equal(a, b) for a, b in zip(again, right))

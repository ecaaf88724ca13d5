"""How exact the fused head's sums and its cap are, where one logit can be read off: weights of two rows, the first of them zeros, so that the log
probability of the less likely token is minus the other logit."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
STEP = 2.0 ** -23                                             # of a 32-bit number, relative to it


def less_likely(x, w, cap):
    """(log probability of the less likely of the two tokens, the same in 64 bits)."""
    from kungfu_b200 import ops
    v = x.double() @ w[1].double()
    if cap > 0:
        v = cap * torch.tanh(v / cap)
    tokens = torch.where(v > 0, 0, 1).to(torch.int32)
    lp = torch.empty(x.shape[0], device=DEV)
    ops.head_logprobs(x, w, tokens, lp, softcap=cap)
    ops.raise_on_device_error()
    return lp.double(), -torch.nn.functional.softplus(v.abs(), threshold=1e9)


@pytest.mark.parametrize("R", [40, 256, 600])
@pytest.mark.parametrize("K", [512, 1000, 2304, 4608])
def test_sums_of_positive_products(R, K):
    """Sums that only grow, where a rounding towards zero at every step of 16 products loses most.  A run of at most 768 products has 48 steps; a step loses
    half of STEP of the running sum on average (all of it at most), and the running sum is half of the whole on average: 48 / 2 * STEP / 2 = 12 STEP at
    most on average.  The additions of runs' sums, at most ten of 512 or six of 768, lose STEP / 2 of the sum at most and nothing on average: 2.5.  The
    difference to the maximum, the logarithm and their difference lose half a step each: 1.5.  One sum of K = 2304 has 144 steps and loses
    144 / 2 * STEP / 4 = 18 STEP at least on average, since a step of a number is no less than STEP / 2 of it."""
    g = torch.Generator(device=DEV).manual_seed(R + K)
    x = (0.5 + torch.rand(R, K, generator=g, device=DEV)).to(torch.bfloat16)
    w = torch.zeros(2, K, dtype=torch.bfloat16, device=DEV)
    w[1] = ((0.5 + torch.rand(K, generator=g, device=DEV)) * 30.0 / K).to(torch.bfloat16)
    got, want = less_likely(x, w, 0.0)
    off = float((got - want).norm() / want.norm())
    assert off <= 16 * STEP, off / STEP


@pytest.mark.parametrize("R", [40, 300])
@pytest.mark.parametrize("cap", [30.0, 64.0, 65.0, 100.0, 1000.0, 1e4, 1e30])
def test_caps_of_any_size(R, cap):
    """Logits that are exact (one product of a row is not zero).  The capped logit is within 4 steps of a logit's size, or of 64 where the
    cap is below that (a quotient's error counts with the cap); the log probability adds at most two."""
    g = torch.Generator(device=DEV).manual_seed(R)
    x = torch.zeros(R, 64, device=DEV)
    x[:, 3] = 120.0 * torch.rand(R, generator=g, device=DEV) - 60.0
    x[0, 3], x[1, 3], x[2, 3], x[3, 3] = 250.0, -250.0, 0.25, 0.0
    x = x.to(torch.bfloat16)
    w = torch.zeros(2, 64, dtype=torch.bfloat16, device=DEV)
    w[1, 3] = 1.0
    got, want = less_likely(x, w, cap)
    size = want.abs().clamp(min=64.0 if cap <= 64.0 else 0.6)
    assert bool(((got - want).abs() <= 6 * STEP * size).all()), float(((got - want).abs() / size).max() / STEP)

"""The sums behind token_logprobs, held to the error that their order of addition allows."""
import math

import pytest
import torch

DEV = "cuda"
THREADS, PER, SPLITS = 512, 16, 32                       # csrc/logprobs.hip: kThreads, kPer, kMaxSplits


def bound(T, V):
    """Relative error of S, in units of 2^-24: a thread adds 16 terms of each of its split's blocks one after the other; its sum is
    rescaled once a block at most (an exponential and a product, 3); six joins across a wave, seven across the waves, six across the
    splits (two products, an addition, an exponential's two: 5 each); every term's exponential is off by two units and by 4 |d| from
    its argument's roundings, and |d| weighted by e^d / S is log V at most."""
    blocks = -(-(V + 15) // (THREADS * PER))
    per = -(-blocks // min(max(512 // T, 1), SPLITS, blocks))
    return PER * per + 3 * per + 5 * 19 + 2 + 4 * math.log(V)


@pytest.mark.gpu
@pytest.mark.parametrize("T,V", [(1, 128256), (1, 600), (3, 50001), (64, 128256), (600, 128256), (600, 9000)])
@pytest.mark.parametrize("kind", ["flat", "spread", "rising"])
def test_log_s(T, V, kind):
    from mi355_attn import ops
    g = torch.Generator().manual_seed(T + V)
    x = torch.randn((T, V), generator=g) * (0.01 if kind == "flat" else 6.0)
    if kind == "rising":
        x = x.sort(dim=1).values                                           # every block moves the maximum
    top = x.argmax(1)
    got = ops.token_logprobs(x.to(DEV), top.to(DEV)).logprobs.double().cpu()
    want = -torch.logsumexp(x.double() - x.double().amax(1, keepdim=True), 1)
    # (the logarithm's own rounding and the subtraction's: three units of the result)
    tol = 2.0 ** -24 * (bound(T, V) + 3 * want.abs())
    assert bool(((got - want).abs() <= tol).all())


def test_this_bound_is_the_tighter_one():
    from oracle.scored_ref import logprobs_bound
    for T, V in ((1, 128256), (64, 128256), (600, 128256)):
        assert 2.0 ** -24 * bound(T, V) < logprobs_bound(torch.empty(0, V), 1.0)

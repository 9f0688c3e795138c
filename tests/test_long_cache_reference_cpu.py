"""The check of attention on long caches fails for what it is there to find: parts of a cache that are lost, counted twice, or taken for others."""
import pytest
import torch

from long_cache_reference import attend_long, roundings, stretches
from paged_reference import HALF_STEP, check


def _weighted(q, k, v, scale, times):
    """The result with every key counted times[j] times."""
    w = torch.exp(scale * k[:, 0].double() @ q.double().T)
    w = w * times[:, None] / (w * times[:, None]).sum(0)
    return w.T @ v[:, 0].double()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,D,weight", [(50000, 256, 2.0 ** -11), (20000, 256, 2.0 ** -11), (131071, 256, 2.0 ** -11), (30000, 128, 2.0 ** -11),
                                        (12000, 64, 2.0 ** -11), (2052, 128, None), (5130, 64, None)])
def test_losses_fail(n, D, weight, dtype):
    g = torch.Generator().manual_seed(n)
    q, k, v = torch.randn(2, D, generator=g).to(dtype), torch.randn(n, 1, D, generator=g).to(dtype), stretches(n, D, dtype, g, "cpu")
    scale, seen = D ** -0.5, torch.ones(n, dtype=torch.bool)
    want, allow = attend_long(q, k, v, scale, seen, weight or HALF_STEP[dtype], roundings(n, 1184))
    once = torch.ones(n, dtype=torch.float64)
    check(_weighted(q, k, v, scale, once).to(dtype), want, allow)                # what is right passes, rounded to the type
    wrong = [torch.zeros_like(want), want * (1 + 2.0 ** -5), want.roll(1, 1)]
    for first in (0, n // 2 // 64 * 64, (n - 1) // 16 * 16 - 16):
        for keys in (16, 64):
            for times in (0.0, 2.0):
                some = once.clone()
                some[first:first + keys] = times
                wrong.append(_weighted(q, k, v, scale, some))
    for got in wrong:
        with pytest.raises(AssertionError):
            check(got.to(dtype), want, allow)

"""ops.paged_attention_nvfp4 where a scale times the size of a head's queries leaves fp32, while the scores do not."""
import pytest
import torch

from nvfp4_cache_reference import held, pack, quantise

pytestmark = pytest.mark.gpu


def _problem(device, n, D, keys):
    """One sequence whose keys are `keys` [n, D], 8 on 1 heads; (run, the values held)."""
    from turbopi_b200 import ops
    g = torch.Generator(device=device).manual_seed(D)
    P = -(-n // 16)
    k = torch.zeros(P * 16, D, dtype=torch.bfloat16, device=device)
    k[:n] = keys
    v = torch.randn((P * 16, D), generator=g, device=device, dtype=torch.bfloat16)
    pages = [pack(*quantise(x.view(P, 16, 1, D).transpose(1, 2))) for x in (k, v)]
    table = torch.arange(P, dtype=torch.int32, device=device)[None]
    lengths = torch.tensor([n], dtype=torch.int32, device=device)
    assert torch.equal(held(pages[0], D).flatten(0, 1)[:n, 0], k[:n].double())         # these keys are held exactly

    def run(q, scale, **kw):
        return ops.paged_attention_nvfp4(q, *pages, table, lengths, scale, **kw)
    return run, held(pages[1], D).flatten(0, 1)[:n, 0]


def _mean(out, v, factor=1.0):
    """Equal weights are 1, exactly: of the mean the sum in 32 bits is rounded, and the output."""
    want = factor * v.mean(0)
    allow = want.abs() * 2.0 ** -8 + 2 * v.shape[0] * 2.0 ** -23 * v.abs().mean(0) * factor
    assert bool(((out.double() - want).abs() <= allow).all())


QUERIES = [(2.0 ** 126, 8.0, 1.0), (2.0 ** 100, 2.0 ** 20, 2.0 ** 10), (2.0 ** 64, 1.0, 2.0 ** 64), (2.0 ** 127, -2.0 ** 60, 2.0 ** 3)]


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("size,scale,k_scale", QUERIES)
def test_keys_of_zero(cuda_device, D, size, scale, k_scale):
    """Every score is 0, whatever the queries: the mean of the values."""
    run, v = _problem(cuda_device, 100, D, 0.0)
    q = torch.full((1, 8, D), size, dtype=torch.bfloat16, device=cuda_device)
    q[0, 1] = 1.0
    _mean(run(q, scale, k_scale=k_scale)[0], v)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("size,scale", [(2.0 ** 126, 8.0), (2.0 ** 126, -8.0), (2.0 ** 100, 2.0 ** 30)])
def test_scores_that_fp32_holds(cuda_device, D, size, scale):
    """The keys are 6 * 2^-9, 0 and -6 * 2^-9 in one column: scores of up to 2^124 and their opposites, so that the keys with the
    largest one share the weight, one each."""
    n = 100
    keys = torch.zeros(n, D, device=cuda_device)
    sign = torch.tensor([1.0, 0.0, -1.0], device=cuda_device)[torch.arange(n, device=cuda_device) % 3]
    keys[:, 5] = sign * 6 * 2.0 ** -9
    run, v = _problem(cuda_device, n, D, keys)
    q = torch.zeros(1, 8, D, dtype=torch.bfloat16, device=cuda_device)
    q[0, :, 5] = size
    q[0, 4:, 5] = -size
    out = run(q, scale)[0]
    for h in range(8):
        best = sign == (1.0 if (h < 4) == (scale > 0) else -1.0)
        _mean(out[h], v[best])


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("scale,size", [(0.0, 2.0 ** 126), (0.0, 2.0 ** 110), (2.0 ** -149, 2.0 ** 10)])
def test_a_scale_of_nothing(cuda_device, D, scale, size):
    """scale q k is 0, or below 2^-120: the mean of the values."""
    g = torch.Generator(device=cuda_device).manual_seed(1)
    keys = torch.randint(-1, 2, (100, D), generator=g, device=cuda_device).float() * 6       # of 16 values the scale is 1 (all zeros: 0)
    run, v = _problem(cuda_device, 100, D, keys)
    q = torch.randn((1, 8, D), generator=g, device=cuda_device).sign().to(torch.bfloat16) * size
    _mean(run(q, scale)[0], v)

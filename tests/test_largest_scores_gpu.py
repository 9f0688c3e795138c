"""Attention whose scores lie past 2^24, where fp32 no longer holds them to a unit: the keys with the largest score share the weight."""
import pytest
import torch

from nvfp4_cache_reference import held, pack, quantise

pytestmark = pytest.mark.gpu

STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
N = 200


def _keys(D, dtype, device):
    """One column decides: 6 for every seventh key, 4, 3 and -6 for the others.  With queries of one number in that column scores are exact products, and
    2 times the query apart at least."""
    level = torch.tensor([6.0, 4.0, 3.0, -6.0, 4.0, 3.0, -6.0], device=device)[torch.arange(N, device=device) % 7]
    k = torch.zeros(N, 1, D, dtype=dtype, device=device)
    k[:, 0, 5] = level.to(dtype)
    return k, level


def _check(out, v, best, dtype):
    """Weights of 1 and 0, exactly, but for the reference's factor, a power of two times one that rounds once: the mean over `best` with a rounding of the
    weight (fp32 2^-23 for the sums, half a step of 16 bits for the product) and one of the output."""
    v = v[best]
    want = v.mean(0)
    allow = want.abs() * STEP[dtype] + v.abs().mean(0) * (2 * STEP[dtype] + 2 * N * 2.0 ** -23) + 2.0 ** -25
    assert bool(out.isfinite().all()), "not finite"
    assert bool(((out.double() - want).abs() <= allow).all())


SIZES = {torch.float16: [(2.0 ** a, s) for a in (9, 12, 15) for s in (1.0, 16.0, 300.0, -777.0, 2.0 ** 20)],
         torch.bfloat16: [(2.0 ** a, s) for a in (10, 20, 22, 25, 31, 40, 60, 100) for s in (1.0, 1.7, -1.3, 11.0)]}


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 72, 128, 256])
@pytest.mark.parametrize("bits", [4, 16])
def test_single_tokens(cuda_device, bits, D, dtype):
    from turbopi_b200 import ops
    k, level = _keys(D, dtype, cuda_device)
    g = torch.Generator(device=cuda_device).manual_seed(D)
    v = torch.randn((N, 1, D), generator=g, device=cuda_device, dtype=dtype)
    P = -(-N // 16)
    pages = []
    for x in (k, v):
        x = torch.nn.functional.pad(x, (0, 0, 0, 0, 0, P * 16 - N)).view(P, 16, 1, D)
        pages.append(pack(*quantise(x.transpose(1, 2))) if bits == 4 else x.contiguous())
    values = held(pages[1], D).flatten(0, 1)[:N, 0] if bits == 4 else v[:, 0].double()
    table, lengths = torch.arange(P, dtype=torch.int32, device=cuda_device)[None], torch.tensor([N], dtype=torch.int32, device=cuda_device)
    call = ops.paged_attention_nvfp4 if bits == 4 else ops.paged_attention
    for hq in (8, 16):
        for size, scale in SIZES[dtype]:
            q = torch.zeros(1, hq, D, dtype=dtype, device=cuda_device)
            q[0, ::2, 5], q[0, 1::2, 5] = size, -size
            for window in (None, 50):
                out = call(q, *pages, table, lengths, scale, window=window)[0]
                shown = torch.arange(N, device=cuda_device) >= N - (window or N)
                for h in range(hq):
                    up = (h % 2 == 0) == (scale > 0)
                    _check(out[h], values, shown & (level == (6.0 if up else -6.0)), dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 72, 128, 256])
@pytest.mark.parametrize("window", [None, 50])
def test_prompts(cuda_device, window, D, dtype):
    from turbopi_b200 import ops
    k, level = _keys(D, dtype, cuda_device)
    g = torch.Generator(device=cuda_device).manual_seed(D)
    v = torch.randn((N, 1, D), generator=g, device=cuda_device, dtype=dtype)
    cu = torch.tensor([0, N], dtype=torch.int32, device=cuda_device)
    for size, scale in SIZES[dtype]:
        q = torch.zeros(N, 2, D, dtype=dtype, device=cuda_device)
        q[:, 0, 5], q[:, 1, 5] = size, -size
        out = ops.packed_attention(q, k, v, cu, scale, window=window)
        for i in (13, 60, 127, 128, N - 1):
            at = torch.arange(N, device=cuda_device)
            shown = (at <= i) & (at > i - (window or N))
            for h in range(2):
                up = (h == 0) == (scale > 0)
                _check(out[i, h], v[:, 0].double(), shown & (level == (6.0 if up else -6.0)), dtype)

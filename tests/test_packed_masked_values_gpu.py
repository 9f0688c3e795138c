"""Infinities and NaN among the values of tiles with masked pairs, in every form of the kernel and both types; infinities in visible keys."""
import pytest
import torch

pytestmark = pytest.mark.gpu

# (query heads, key heads, head size, empty sequences behind): the mean length decides between one and two row tiles
FORMS = [(4, 2, 64, 0), (4, 2, 64, 30), (3, 1, 40, 0), (8, 2, 128, 0), (8, 2, 128, 60), (2, 1, 72, 0), (8, 1, 256, 0), (2, 2, 136, 0)]


def _offsets(lens, device):
    return torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device=device)


def _problem(hq, hk, D, empty, dtype, device):
    lens, klens = [300, 200] + [0] * empty, [300, 3000] + [0] * empty
    g = torch.Generator(device=device).manual_seed(D)
    q = torch.randn((500, hq, D), generator=g, device=device, dtype=dtype)
    k, v = torch.randn((2, 3300, hk, D), generator=g, device=device, dtype=dtype)
    return q, k, v, _offsets(lens, device), _offsets(klens, device)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,hk,D,empty", FORMS)
def test_values(cuda_device, hq, hk, D, empty, dtype):
    """A bad value reaches the queries that see it and no other, in its columns alone."""
    from turbopi_b200 import _lib, ops
    q, k, v, cu, cuk = _problem(hq, hk, D, empty, dtype, cuda_device)
    clean = ops.packed_attention(q, k, v, cu, D ** -0.5, cu_keys=cuk)
    g, half = hq // hk, D // 2
    for value in (float("nan"), float("inf"), float("-inf")):
        for at in (2802, 2850, 2943, 2944, 2999):                # the first query sees 2801
            v2 = v.clone()
            v2[300 + at, 0, half:] = value
            out = ops.packed_attention(q, k, v2, cu, D ** -0.5, cu_keys=cuk)
            sees = torch.arange(200, device=cuda_device) + 2800 >= at
            assert torch.equal(out[:300], clean[:300]) and torch.equal(out[300:][~sees], clean[300:][~sees])
            bad = out[300:][sees][:, :g, half:]
            assert bool((bad.isnan() if value != value else (bad == value)).all())
            assert torch.equal(out[300:, :, :half], clean[300:, :, :half]) and torch.equal(out[300:, g:], clean[300:, g:])
        v2 = v.clone()                                           # a whole key behind the first sequence's end: the second's first
        v2[300] = value
        out = ops.packed_attention(q, k, v2, cu, D ** -0.5, cu_keys=cuk)
        assert torch.equal(out[:300], clean[:300])
        assert bool((out[300:].isnan() if value != value else out[300:] == value).all())
    assert _lib.load().tpb200_device_error(0) == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,hk,D,empty", FORMS)
def test_keys(cuda_device, hq, hk, D, empty, dtype):
    """A masked key's score is selected away whatever it is; a visible one of minus infinity has no weight, the last query's too."""
    from turbopi_b200 import _lib, ops
    q, k, v, cu, cuk = _problem(hq, hk, D, empty, dtype, cuda_device)
    q[300:] = q[300:].abs().clamp_(min=0.25)
    for value in (float("nan"), float("inf"), float("-inf")):
        for at in (2850, 2999):
            clean = ops.packed_attention(q, k, v, cu, D ** -0.5, cu_keys=cuk)
            k2 = k.clone()
            k2[300 + at] = value
            out = ops.packed_attention(q, k2, v, cu, D ** -0.5, cu_keys=cuk)
            sees = torch.arange(200, device=cuda_device) + 2800 >= at
            assert torch.equal(out[:300], clean[:300]) and torch.equal(out[300:][~sees], clean[300:][~sees])
            seen = out[300:][sees]
            assert bool((seen.isfinite() if value == float("-inf") else seen.isnan()).all())
    assert _lib.load().tpb200_device_error(0) == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D,page", [(64, 16), (128, 24), (256, 16)])
def test_single_tokens_with_infinities_in_sight(cuda_device, D, page, dtype):
    """Keys of minus infinity have no weight, of plus infinity or NaN make the row NaN; an infinite value with weight is the output."""
    from turbopi_b200 import ops
    n, hq, hk = 900, 4, 2
    pages = -(-n // page)
    g = torch.Generator(device=cuda_device).manual_seed(D)
    pool = torch.randn((2, pages, page, hk, D), generator=g, device=cuda_device, dtype=dtype)
    q = torch.randn((1, hq, D), generator=g, device=cuda_device, dtype=dtype).abs().clamp_(min=0.25)
    table = torch.arange(pages, dtype=torch.int32, device=cuda_device)[None]
    lengths = torch.tensor([n], dtype=torch.int32, device=cuda_device)

    def run(p):
        return ops.paged_attention(q, p[0], p[1], table, lengths, D ** -0.5)
    clean = run(pool)
    for at in (0, 450, 899):
        for value in (float("nan"), float("inf"), float("-inf")):
            p = pool.clone()
            p[0, at // page, at % page, 1] = value
            out = run(p)
            assert torch.equal(out[:, :2], clean[:, :2])
            assert bool((out[:, 2:].isfinite() if value == float("-inf") else out[:, 2:].isnan()).all())
            p = pool.clone()
            p[1, at // page, at % page, 1, D // 2:] = value
            out = run(p)
            assert torch.equal(out[:, :2], clean[:, :2]) and torch.equal(out[..., :D // 2], clean[..., :D // 2])
            bad = out[:, 2:, D // 2:]
            assert bool((bad.isnan() if value != value else bad == value).all())

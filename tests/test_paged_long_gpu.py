"""Single tokens on long caches, on 4 bits and on 16 under a window: no part of a cache is lost or counted twice where it is split over warps and joined."""
import pytest
import torch

from long_cache_reference import attend_long, roundings, stretches
from nvfp4_cache_reference import held, pack, quantise, seen
from paged_reference import HALF_STEP, check, deal_pages

pytestmark = pytest.mark.gpu

CASES = [(8, 1, 256, [50000]), (8, 1, 256, [20000, 1, 1, 1]), (8, 1, 256, [131071, 60000]), (32, 8, 128, [8192, 3, 5000, 0, 1]), (16, 16, 64, [12000, 700]),
         (16, 1, 128, [30000]), (40, 1, 64, [30000, 20]), (12, 1, 200, [20000, 20000, 20000]), (6, 2, 72, [20000]), (4, 4, 256, [343, 11600])]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("bits,page", [(4, 16), (4, 64), (16, 32), (16, 24)])
@pytest.mark.parametrize("hq,hk,D,lens", CASES)
def test_every_stretch_counts(cuda_device, hq, hk, D, lens, bits, page, dtype):
    from turbopi_b200 import _lib, ops
    g = torch.Generator(device=cuda_device).manual_seed(D + len(lens))
    rows, pool = deal_pages(lens, page, D)
    q = torch.randn((len(lens), hq, D), generator=g, device=cuda_device, dtype=dtype)
    windows = [(None, 0), (2048, 4), (5000, 130)] if bits == 4 else [(2048, 4), (5000, 130), (19000, 0)]
    for window, sinks in windows:
        x = torch.randn((2, pool * page, hk, D), generator=g, device=cuda_device, dtype=dtype)
        x[1] = 0
        masks = []
        for row, n in zip(rows, lens):           # the keys that are seen, cut into stretches
            mask = seen(1, n, window, sinks, cuda_device)[0]
            at = torch.arange(n, device=cuda_device)
            place = torch.tensor(row, dtype=torch.long, device=cuda_device)[at // page] * page + at % page
            x[1][place[mask]] = stretches(int(mask.sum()), D, dtype, g, cuda_device).expand(-1, hk, -1)
            masks.append((mask, place))
        x = x.view(2, pool, page, hk, D)
        pages = [pack(*quantise(s.transpose(1, 2))) for s in x] if bits == 4 else list(x)
        full = [(held(p, D) if bits == 4 else p).flatten(0, 1) for p in pages]
        call = ops.paged_attention_nvfp4 if bits == 4 else ops.paged_attention
        table, lengths = (torch.tensor(t, dtype=torch.int32, device=cuda_device) for t in (rows, lens))
        out = call(q, *pages, table, lengths, D ** -0.5, window=window, sinks=sinks)
        tiles = hk * -(-hq // hk // 8)
        workers = 8 * torch.cuda.get_device_properties(cuda_device).multi_processor_count
        steps = roundings(tiles * sum(int(m.sum()) for m, _ in masks), workers)
        for i, (mask, place) in enumerate(masks):
            k, v = (f[place] for f in full)
            want, allow = attend_long(q[i], k, v, D ** -0.5, mask, 2.0 ** -11 if bits == 4 else HALF_STEP[dtype], steps)
            check(out[i], want, allow)
    assert _lib.load().tpb200_device_error(0) == 0

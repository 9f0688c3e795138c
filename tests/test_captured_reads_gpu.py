"""What the documents offer for a captured prompt behind a growing cache: reads with room for what is to come, attention on their rows by key offsets."""
import pytest
import torch

from nvfp4_cache_reference import attend, held, seen
from paged_reference import check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["nvfp4", torch.bfloat16])
def test_a_captured_prompt_follows_its_batch(cuda_device, dtype):
    from turbopi_b200 import _lib, ops
    from turbopi_b200.paged_cache import PagedCache
    cache = PagedCache(1, 60, 16, 1, 128, 30, dtype=dtype, device=cuda_device)
    g = torch.Generator(device=cuda_device).manual_seed(0)
    seqs, room = [cache.add(), cache.add()], 300

    def rows(n, h):
        return torch.randn((n, h, 128), generator=g, device=cuda_device, dtype=torch.bfloat16)
    cache.append(0, cache.extend(seqs, [60, 33]), rows(93, 1), rows(93, 1))
    batch = cache.extend(seqs, [5, 4])
    q, k, v = rows(9, 4), rows(9, 1), rows(9, 1)

    def step():
        cache.append(0, batch, k, v)
        if dtype == "nvfp4":
            kk, vv = ops.paged_read_nvfp4(*cache.layer(0), batch.table, batch.cu_keys, batch.lengths, 128, room)
        else:
            kk, vv = ops.paged_read(*cache.layer(0), batch.table, batch.cu_keys, batch.lengths, room)
        return ops.packed_attention(q, kk, vv, batch.cu, 0.1, cu_keys=batch.cu_keys)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for turn in range(12):
        if turn:
            cache.extend(seqs, [5, 4], out=batch)
            for t in (q, k, v):
                t.normal_(generator=g)
        graph.replay()
        at = 0
        for s, n in zip(seqs, (5, 4)):
            m = cache.length(s)
            ids = torch.tensor(cache.page_ids(s), device=cuda_device)
            kk, vv = ((held(p[ids], 128) if dtype == "nvfp4" else p[ids]).flatten(0, 1)[:m] for p in cache.layer(0))
            want, allow = attend(q[at:at + n], kk, vv, 0.1, seen(n, m, None, 0, cuda_device))
            check(out[at:at + n], want, allow)
            at += n
        assert _lib.load().tpb200_device_error(0) == 0

"""ops.paged_read, ops.paged_read_nvfp4 and PagedCache.prompt_attention captured: what a replay does after the batch has grown or shrunk."""
import pytest
import torch

from nvfp4_cache_reference import attend, held, seen
from paged_reference import check

pytestmark = pytest.mark.gpu


def _ints(x, device):
    return torch.tensor(x, dtype=torch.int32, device=device)


def _captured(call):
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        result = call()
    return graph, result


@pytest.mark.parametrize("bits", [4, 16])
@pytest.mark.parametrize("seqs", [1, 3, 40])
def test_offsets_beyond_the_rows_are_reported(cuda_device, bits, seqs):
    """The rows that there are get their tokens, whether the offsets end with them or go past them."""
    from turbopi_b200 import _lib, ops
    lib, page, n = _lib.load(), 16, 9
    P = 2 * seqs
    table = torch.arange(P, dtype=torch.int32, device=cuda_device).view(seqs, 2)
    lengths, rows = _ints([n + 3] * seqs, cuda_device), n * seqs
    cu = _ints([n * i for i in range(seqs + 1)], cuda_device)
    if bits == 4:
        pages = torch.randint(0, 120, (2, P, 2, 1, 576), device=cuda_device, dtype=torch.uint8)
        out = torch.zeros(2, rows, 2, 64, dtype=torch.bfloat16, device=cuda_device)
        graph, _ = _captured(lambda: ops.paged_read_nvfp4(pages[0], pages[1], table, cu, lengths, 64, rows, out=(out[0], out[1])))
    else:
        pages = torch.randn(2, P, page, 2, 64, dtype=torch.bfloat16, device=cuda_device)
        out = torch.zeros(2, rows, 2, 64, dtype=torch.bfloat16, device=cuda_device)
        graph, _ = _captured(lambda: ops.paged_read(pages[0], pages[1], table, cu, lengths, rows, out=(out[0], out[1])))
    full = torch.stack([held(p, 64) for p in pages]) if bits == 4 else pages.double()

    def want(offsets):
        x = torch.full((2, rows, 2, 64), 7.0, dtype=torch.float64, device=cuda_device)
        for s, (lo, hi) in enumerate(zip(offsets, offsets[1:])):
            for t in range(lo, min(hi, rows)):
                pos = n + 3 - (hi - t)
                x[:, t] = full[:, 2 * s + pos // page, pos % page]
        return x
    assert lib.tpb200_device_error(1) == 0
    for more, code in ((0, 0), (1, 501), (3, 501), (-2, 0)):
        offsets = [n * i for i in range(seqs)] + [rows + more]
        cu.copy_(_ints(offsets, cuda_device))
        out.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert lib.tpb200_device_error(1) == code, more
        assert torch.equal(out.double(), want(offsets)), more


@pytest.mark.parametrize("dtype", ["nvfp4", torch.bfloat16])
def test_a_replayed_prompt_attention_says_that_its_batch_has_grown(cuda_device, dtype):
    from turbopi_b200 import _lib
    from turbopi_b200.paged_cache import PagedCache
    lib = _lib.load()
    cache = PagedCache(1, 40, 16, 1, 128, 20, dtype=dtype, device=cuda_device)
    g = torch.Generator(device=cuda_device).manual_seed(0)
    seqs = [cache.add(), cache.add()]

    def rows(n, h):
        return torch.randn((n, h, 128), generator=g, device=cuda_device, dtype=torch.bfloat16)
    cache.append(0, cache.extend(seqs, [60, 33]), rows(93, 1), rows(93, 1))
    batch = cache.extend(seqs, [5, 4])
    q, k, v = rows(9, 4), rows(9, 1), rows(9, 1)

    def step():
        cache.append(0, batch, k, v)
        return cache.prompt_attention(0, batch, q, 0.1)
    graph, out = _captured(step)
    assert lib.tpb200_device_error(1) == 0
    # the same batch, and one of as many keys and tokens: right, and nothing is reported
    for turn in range(3):
        if turn:
            for s, n in zip(seqs, (5, 4)):
                cache.truncate(s, cache.length(s) - n)
            cache.extend(seqs, [5, 4], out=batch)
            for t in (q, k, v):
                t.normal_(generator=g)
        graph.replay()
        torch.cuda.synchronize()
        at = 0
        for s, n in zip(seqs, (5, 4)):
            m = cache.length(s)
            ids = torch.tensor(cache.page_ids(s), device=cuda_device)
            kk, vv = ((held(p[ids], 128) if dtype == "nvfp4" else p[ids]).flatten(0, 1)[:m] for p in cache.layer(0))
            want, allow = attend(q[at:at + n], kk, vv, 0.1, seen(n, m, None, 0, cuda_device))
            check(out[at:at + n], want, allow)
            at += n
        assert lib.tpb200_device_error(1) == 0
    # nine keys more than the captured rows: reported, not left out in silence
    cache.extend(seqs, [5, 4], out=batch)
    graph.replay()
    torch.cuda.synchronize()
    assert lib.tpb200_device_error(1) == 501
    eager = cache.prompt_attention(0, batch, q, 0.1)
    torch.cuda.synchronize()
    assert lib.tpb200_device_error(1) == 0 and bool(eager.isfinite().all())

"""ops.packed_attention with a window and sinks against attention in 64 bits: windows around the tiles' edges, queries behind cached keys and
with fewer keys than queries, what stands in hidden places."""
import pytest
import torch

from nvfp4_cache_reference import attend, seen
from paged_reference import check

pytestmark = pytest.mark.gpu

WINDOWS = [(1, 0), (1, 1), (7, 130), (64, 4), (127, 0), (128, 128), (129, 127), (200, 16), (300, 300), (513, 1), (1000, 129), (10 ** 9, 3), (3, 10 ** 9)]


def _offsets(lens, device):
    return torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device=device)


def _no_error():
    from turbopi_b200 import _lib
    assert _lib.load().tpb200_device_error(0) == 0


def _run(device, lens, klens, hq, hk, D, dtype, windows, seed=0, scale=None):
    from turbopi_b200 import ops
    scale = D ** -0.5 if scale is None else scale
    g = torch.Generator(device=device).manual_seed(seed)
    q = torch.randn((sum(lens) + 3, hq, D), generator=g, device=device, dtype=dtype)
    k, v = torch.randn((2, sum(klens) + 3, hk, D), generator=g, device=device, dtype=dtype)
    for t, n in ((q, sum(lens)), (k, sum(klens)), (v, sum(klens))):
        t[n:] = float("nan")
    for window, sinks in windows:
        out = torch.full_like(q, 9.0)
        got = ops.packed_attention(q, k, v, _offsets(lens, device), scale, out=out, cu_keys=None if lens == klens else _offsets(klens, device),
                                   window=window, sinks=sinks)
        assert got is out and bool((out[sum(lens):] == 9).all())
        q0 = k0 = 0
        for n, m in zip(lens, klens):
            want, allow = attend(q[q0:q0 + n], k[k0:k0 + m], v[k0:k0 + m], scale, seen(n, m, window, sinks, device))
            check(out[q0:q0 + n], want, allow)
            q0, k0 = q0 + n, k0 + m
        _no_error()


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("n", [1, 128, 700])
def test_one_sequence(cuda_device, n, D):
    _run(cuda_device, [n], [n], 1, 1, D, torch.bfloat16, WINDOWS)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,hk,D,empty", [(4, 2, 64, 0), (4, 2, 64, 30), (3, 1, 40, 0), (8, 2, 128, 0), (8, 2, 128, 60), (2, 1, 72, 0), (8, 1, 256, 0),
                                           (2, 2, 136, 0), (16, 1, 64, 0)])
def test_batches(cuda_device, hq, hk, D, empty, dtype):
    """Every form of the kernel: lengths around a tile, keys from before, fewer keys than queries, none at all."""
    lens = [1, 0, 127, 130, 600, 40, 257, 5] + [0] * empty
    klens = [1, 0, 127, 130, 600, 900, 300, 2] + [0] * empty
    _run(cuda_device, lens, klens, hq, hk, D, dtype, WINDOWS, seed=D)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_long_sequences(cuda_device, D):
    """Many tiles left out between the sinks and the window, two row tiles to a CTA."""
    _run(cuda_device, [5000, 300], [5000, 4300], 2, 1, D, torch.bfloat16, [(100, 0), (256, 4), (1000, 200), (128, 640)], seed=D)


def test_a_negative_scale(cuda_device):
    _run(cuda_device, [300, 77], [300, 77], 4, 4, 64, torch.float16, [(50, 3)], scale=-0.2)


def test_the_window_of_everything_gives_the_same_bits(cuda_device):
    from turbopi_b200 import ops
    q = torch.randn((700, 8, 128), device=cuda_device, dtype=torch.bfloat16)
    k, v = torch.randn((2, 700, 2, 128), device=cuda_device, dtype=torch.bfloat16)
    cu = _offsets([300, 400], cuda_device)
    assert torch.equal(ops.packed_attention(q, k, v, cu, 0.1, window=700), ops.packed_attention(q, k, v, cu, 0.1))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,hk,D,empty", [(4, 2, 64, 0), (4, 2, 64, 30), (8, 2, 128, 0), (8, 2, 128, 60), (2, 1, 72, 0), (8, 1, 256, 0)])
def test_infinities_and_nan(cuda_device, hq, hk, D, empty, dtype):
    """A bad key or value reaches the queries that see it and no other."""
    from turbopi_b200 import ops
    lens, klens = [300, 200] + [0] * empty, [300, 3000] + [0] * empty
    g = torch.Generator(device=cuda_device).manual_seed(D)
    q = torch.randn((500, hq, D), generator=g, device=cuda_device, dtype=dtype)
    k, v = torch.randn((2, 3300, hk, D), generator=g, device=cuda_device, dtype=dtype)
    cu, cuk, group, half = _offsets(lens, cuda_device), _offsets(klens, cuda_device), hq // hk, D // 2
    for window, sinks in ((150, 70), (700, 4), (1, 129)):
        def run(k, v):
            return ops.packed_attention(q, k, v, cu, D ** -0.5, cu_keys=cuk, window=window, sinks=sinks)
        clean = run(k, v)
        mask = seen(200, 3000, window, sinks, cuda_device)
        for value in (float("nan"), float("inf"), float("-inf")):
            for at in (0, 3, 69, 70, 128, 500, 2100, 2175, 2660, 2700, 2801, 2850, 2943, 2999):
                v2 = v.clone()
                v2[300 + at, 0, half:] = value
                out = run(k, v2)
                sees = mask[:, at]
                assert torch.equal(out[:300], clean[:300]) and torch.equal(out[300:][~sees], clean[300:][~sees])
                bad = out[300:][sees][:, :group, half:]
                assert bool((bad.isnan() if value != value else (bad == value)).all())
                assert torch.equal(out[300:, :, :half], clean[300:, :, :half]) and torch.equal(out[300:, group:], clean[300:, group:])
            for at in (3, 69, 70, 2175, 2850, 2999):
                k2 = k.clone()
                k2[300 + at] = float("nan")
                out = run(k2, v)
                sees = mask[:, at]
                assert torch.equal(out[:300], clean[:300]) and torch.equal(out[300:][~sees], clean[300:][~sees]) and bool(out[300:][sees].isnan().all())
    _no_error()


def test_a_graph_follows_the_offsets(cuda_device):
    from turbopi_b200 import ops
    q = torch.randn((600, 8, 64), device=cuda_device, dtype=torch.bfloat16)
    k, v = torch.randn((2, 600, 2, 64), device=cuda_device, dtype=torch.bfloat16)
    cu, out = _offsets([300, 300], cuda_device), torch.empty_like(q)
    ops.packed_attention(q, k, v, cu, 0.1, window=100, sinks=4)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.packed_attention(q, k, v, cu, 0.1, out=out, window=100, sinks=4)
    for lens in ([1, 599], [600, 0]):
        cu.copy_(_offsets(lens, cuda_device))
        graph.replay()
        assert torch.equal(out, ops.packed_attention(q, k, v, cu, 0.1, window=100, sinks=4))
        q0 = 0
        for n in lens:
            want, allow = attend(q[q0:q0 + n], k[q0:q0 + n], v[q0:q0 + n], 0.1, seen(n, n, 100, 4, cuda_device))
            check(out[q0:q0 + n], want, allow)
            q0 += n

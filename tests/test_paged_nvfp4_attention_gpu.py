"""ops.paged_attention_nvfp4, and the window of ops.paged_attention, against attention in 64 bits on what the cache holds."""
import pytest
import torch

from nvfp4_cache_reference import attend, groups, held, pack, quantise, seen
from paged_reference import check, deal_pages

pytestmark = pytest.mark.gpu

WEIGHT = 2.0 ** -11            # half a step of fp16


def _ints(x, device):
    return torch.tensor(x, dtype=torch.int32, device=device)


def _no_error():
    from turbopi_b200 import _lib
    assert _lib.load().tpb200_device_error(0) == 0


class _Problem:
    """Pages dealt in no order; rows behind a sequence's end hold NaN, pages of nobody too."""

    def __init__(self, lens, hq, hk, D, page, dtype, device, bits=4, seed=0, width=None, poison=True):
        g = torch.Generator(device=device).manual_seed(seed)
        self.lens, self.page, self.D, self.bits, self.dtype, self.device = lens, page, D, bits, dtype, device
        self.rows, pool = deal_pages(lens, page, seed, width=width)
        x = torch.randn((2, pool, page, hk, D), generator=g, device=device, dtype=dtype)
        used = torch.zeros(pool, page, dtype=torch.bool, device=device)
        for row, n in zip(self.rows, lens):
            ids = torch.tensor(row[:-(-n // page)], dtype=torch.long, device=device)
            flat = used[ids].flatten()
            flat[:n] = True
            used[ids] = flat.view(-1, page) | used[ids]
        self.q = torch.randn((len(lens), hq, D), generator=g, device=device, dtype=dtype)
        if bits == 4:
            packed = []
            for side in x:
                code, byte = quantise(side.transpose(1, 2))
                if poison:
                    byte[~used[:, None].expand(-1, hk, -1)] = 127
                packed.append(pack(code, byte))
            self.pages = packed
            self.full = [held(p, D) for p in packed]
        else:
            if poison:
                x[:, ~used] = float("nan")
            self.pages = self.full = list(x)
        self.table, self.lengths = _ints(self.rows, device), _ints(lens, device)

    def run(self, scale, **kw):
        from turbopi_b200 import ops
        call = ops.paged_attention_nvfp4 if self.bits == 4 else ops.paged_attention
        return call(self.q, *self.pages, self.table, self.lengths, scale, **kw)

    def check(self, out, scale, window=None, sinks=0, k_scale=1.0, v_scale=1.0):
        for i, n in enumerate(self.lens):
            ids = torch.tensor(self.rows[i][:-(-n // self.page)], dtype=torch.long, device=self.device)
            k, v = (x[ids].flatten(0, 1)[:n].double() * f for x, f in zip(self.full, (k_scale, v_scale)))
            want, allow = attend(self.q[i:i + 1], k, v, scale, seen(1, n, window, sinks, self.device), WEIGHT if self.bits == 4 else None)
            check(out[i:i + 1], want, allow)
        _no_error()


HEADS = [(8, 1, 256), (32, 8, 128), (16, 16, 64), (6, 2, 72), (5, 1, 8), (2, 2, 200), (16, 1, 96), (17, 1, 64), (40, 1, 128), (12, 1, 256), (3, 3, 32)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,hk,D", HEADS)
def test_heads_and_types(cuda_device, hq, hk, D, dtype):
    p = _Problem([1, 0, 15, 16, 17, 63, 64, 65, 129, 300, 1001], hq, hk, D, 16, dtype, cuda_device, seed=D)
    out = p.run(D ** -0.5)
    p.check(out, D ** -0.5)
    assert bool((out[1] == 0).all())


@pytest.mark.parametrize("page", [16, 32, 48, 128, 1024])
def test_page_sizes(cuda_device, page):
    p = _Problem([page, page + 1, 2 * page - 1, 333, 7], 8, 2, 128, page, torch.bfloat16, cuda_device, seed=page)
    p.check(p.run(0.1), 0.1)


@pytest.mark.parametrize("lens", [[1], [50000], [0], [0, 0, 3, 0], [20000, 1, 1, 1], [1] * 700, [37] * 300, [1] * 1100, [4095, 0, 4097]])
def test_how_the_work_is_cut(cuda_device, lens):
    p = _Problem(lens, 8, 1, 64 if len(lens) > 500 else 256, 16, torch.bfloat16, cuda_device, seed=len(lens))
    p.check(p.run(1 / 16), 1 / 16)


def test_same_bits_every_time(cuda_device):
    p = _Problem([3000, 5, 700], 8, 1, 256, 16, torch.float16, cuda_device)
    first = p.run(1 / 16)
    for _ in range(5):
        assert torch.equal(first, p.run(1 / 16))


WINDOWS = [(1, 0), (1, 1), (2, 3), (15, 4), (16, 16), (17, 0), (64, 4), (100, 33), (128, 130), (500, 4), (1000, 64), (10 ** 9, 0), (5, 10 ** 9)]


@pytest.mark.parametrize("bits,hq,hk,D,page", [(4, 8, 1, 256, 16), (4, 8, 2, 128, 32), (4, 16, 1, 128, 16), (4, 4, 4, 64, 48), (4, 6, 2, 72, 16),
                                               (16, 8, 1, 256, 16), (16, 8, 2, 128, 24), (16, 4, 4, 64, 32), (16, 4, 4, 64, 5), (16, 6, 2, 72, 1),
                                               (16, 24, 1, 128, 16)])
def test_windows(cuda_device, bits, hq, hk, D, page):
    p = _Problem([1, 0, 16, 17, 64, 65, 100, 129, 300, 513, 2000], hq, hk, D, page, torch.bfloat16 if D != 128 else torch.float16, cuda_device, bits, seed=D + page)
    for window, sinks in WINDOWS:
        p.check(p.run(D ** -0.5, window=window, sinks=sinks), D ** -0.5, window, sinks)


@pytest.mark.parametrize("bits,D,page", [(4, 128, 16), (4, 256, 64), (4, 64, 16), (16, 128, 16), (16, 64, 24), (16, 256, 7)])
def test_what_a_window_hides_is_not_read(cuda_device, bits, D, page):
    """Pages without a visible key may be absent; hidden rows of the others, infinite or NaN, change nothing."""
    from turbopi_b200 import _lib
    window, sinks = 100, 4
    p = _Problem([1, 90, 104, 105, 400, 3000, 30000], 8, 2, D, page, torch.bfloat16, cuda_device, bits, seed=page)
    clean = p.run(0.1, window=window, sinks=sinks)
    p.check(clean, 0.1, window, sinks)
    for i, n in enumerate(p.lens):
        for j in range(-(-n // page)):
            keys = [x for x in range(j * page, min(n, (j + 1) * page)) if x < sinks or x >= n - window]
            if not keys:
                p.table[i, j] = (-1, 10 ** 6)[j % 2]
    if bits == 16:
        for i, n in enumerate(p.lens):
            for x in list(range(sinks, min(n - window, sinks + page))) + list(range(max(sinks, n - window - page), n - window)):
                for side in p.pages:
                    side[p.rows[i][x // page], x % page] = (float("nan"), float("inf"))[x % 2]
    else:
        g = groups(D)
        for i, n in enumerate(p.lens):
            for x in list(range(sinks, min(n - window, sinks + page))) + list(range(max(sinks, n - window - page), n - window)):
                for side in p.pages:
                    r = x % page
                    side[p.rows[i][x // page], :, r // 16, 256 * g + r % 16 * 2 * g:256 * g + (r % 16 + 1) * 2 * g] = 127
    assert torch.equal(p.run(0.1, window=window, sinks=sinks), clean)
    _no_error()
    # a visible page that is absent is left out, and reported
    lib = _lib.load()
    p.table[5, p.lens[5] // page - 1] = -1
    out = p.run(0.1, window=window, sinks=sinks)
    assert lib.tpb200_device_error(1) == 501
    assert torch.equal(out[:5], clean[:5]) and torch.equal(out[6:], clean[6:]) and bool(out[5].isfinite().all())


def test_pages_that_are_absent(cuda_device):
    """Without a window: their keys are left out, one after the other, and all of them."""
    from turbopi_b200 import _lib
    lib = _lib.load()
    p = _Problem([100, 333, 700, 60, 2000, 15, 130], 8, 2, 128, 16, torch.bfloat16, cuda_device, seed=3)
    gone = [[0], [20], [21], range(4), range(0, 125, 2), range(1), range(3, 6)]
    keep = []
    for i, (n, which) in enumerate(zip(p.lens, gone)):
        keep.append([x for x in range(n) if x // 16 not in list(which)])
        for j in which:
            p.table[i, j] = (-1, 2 ** 30, -2 ** 31)[j % 3]
    assert lib.tpb200_device_error(1) == 0
    out = p.run(0.1)
    assert lib.tpb200_device_error(1) == 501
    for i, at in enumerate(keep):
        where = torch.tensor(at, dtype=torch.long, device=cuda_device)
        ids = torch.tensor(p.rows[i], device=cuda_device)[where // 16]
        k, v = (x[ids, where % 16] for x in p.full)
        want, allow = attend(p.q[i:i + 1], k, v, 0.1, torch.ones(1, len(at), dtype=torch.bool, device=cuda_device), WEIGHT)
        check(out[i:i + 1], want, allow)
    assert bool((out[3] == 0).all()) and bool((out[5] == 0).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_factors_and_large_queries(cuda_device, dtype):
    """Powers of two in front of keys and values; queries of very different sizes, past what fp16 holds; a negative scale."""
    p = _Problem([300, 77, 1000], 8, 2, 128, 16, dtype, cuda_device, seed=9)
    for k_scale, v_scale in ((2.0 ** -6, 2.0 ** 5), (2.0 ** 4, 2.0 ** -9)):
        p.check(p.run(0.1 / k_scale, k_scale=k_scale, v_scale=v_scale), 0.1 / k_scale, k_scale=k_scale, v_scale=v_scale)
    p.check(p.run(-0.07), -0.07)
    p.q[:, 1] *= 1e-3
    p.q[:, 2, ::7] *= 100
    p.q[1] = 0
    p.check(p.run(0.1), 0.1)
    if dtype == torch.bfloat16:
        p.q[:, 3] *= 1e30
        p.q[:, 4] *= 1e-30
        out = p.run(1e-30)
        p.check(out, 1e-30)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_scales_and_queries_of_nothing(cuda_device, dtype):
    """A scale of zero, the least one, queries of zero and subnormal ones: the mean of what is seen, under masks too."""
    p = _Problem([300, 17, 1000, 1], 8, 2, 64, 16, dtype, cuda_device, seed=11)
    p.q[0] = 0
    p.q[1] *= torch.finfo(dtype).smallest_normal / 8
    for scale in (0.0, 1e-38, -1e-38, 1e-42, 0.1, -0.1):
        p.check(p.run(scale), scale)
        p.check(p.run(scale, window=20, sinks=3), scale, 20, 3)


def test_values_that_are_not_numbers(cuda_device):
    """A block of values with a NaN scale that is visible reaches its 16 columns, in its head and sequence alone; keys their whole head."""
    p = _Problem([300, 200], 4, 2, 128, 16, torch.bfloat16, cuda_device, seed=4)
    clean = p.run(0.1)
    for side in (0, 1):
        keep = p.pages[side].clone()
        at = 250
        p.pages[side][p.rows[0][at // 16], 1, 0, 256 * 4 + at % 16 * 8 + 3] = 127
        out = p.run(0.1)
        assert torch.equal(out[1], clean[1]) and torch.equal(out[0, :2], clean[0, :2])
        if side == 0:
            assert bool(out[0, 2:].isnan().all())
        else:
            assert bool(out[0, 2:, 48:64].isnan().all()) and torch.equal(out[0, 2:, :48], clean[0, 2:, :48]) and torch.equal(out[0, 2:, 64:], clean[0, 2:, 64:])
        p.pages[side].copy_(keep)


def test_strides_and_outputs(cuda_device):
    """Queries as columns of a fused projection, an output among other columns, out on q, pages with heads in front."""
    from turbopi_b200 import ops
    p = _Problem([40, 333, 5], 8, 2, 128, 32, torch.bfloat16, cuda_device, seed=2)
    want = p.run(0.1)
    wide = torch.randn((3, 12, 128), device=cuda_device, dtype=torch.bfloat16)
    wide[:, :8] = p.q
    out = torch.zeros((3, 16, 128), device=cuda_device, dtype=torch.bfloat16)
    got = ops.paged_attention_nvfp4(wide[:, :8], *p.pages, p.table, p.lengths, 0.1, out=out[:, 4:12])
    assert torch.equal(got, want) and bool((out[:, :4] == 0).all()) and bool((out[:, 12:] == 0).all())
    pages = [x.transpose(0, 1).contiguous().transpose(0, 1) for x in p.pages]
    assert torch.equal(ops.paged_attention_nvfp4(p.q, *pages, p.table, p.lengths, 0.1), want)
    q = p.q.clone()
    assert ops.paged_attention_nvfp4(q, *p.pages, p.table, p.lengths, 0.1, out=q) is q and torch.equal(q, want)


@pytest.mark.parametrize("bits", [4, 16])
def test_a_graph_follows_lengths_and_tables(cuda_device, bits):
    """One capture, one workspace; replayed for other lengths, with calls on another stream and workspace between."""
    from turbopi_b200 import ops
    p = _Problem([700, 64, 300], 8, 1, 256, 16, torch.bfloat16, cuda_device, bits, seed=6)
    make = ops.paged_attention_nvfp4_workspace if bits == 4 else ops.paged_attention_workspace
    ws, other = (make(8, 1, 256, cuda_device) for _ in range(2))
    out = torch.empty_like(p.q)
    graph = torch.cuda.CUDAGraph()
    p.run(1 / 16, window=200, sinks=4)
    with torch.cuda.graph(graph):
        p.run(1 / 16, out=out, workspace=ws, window=200, sinks=4)
    stream = torch.cuda.Stream(cuda_device)
    for lens in ([700, 64, 300], [1, 0, 299], [205, 10, 204]):
        p.lens = lens
        p.lengths.copy_(_ints(lens, cuda_device))
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            beside = p.run(1 / 16, workspace=other)
        graph.replay()
        torch.cuda.synchronize()
        p.check(out, 1 / 16, 200, 4)
        p.check(beside, 1 / 16)


def test_a_longest_cache(cuda_device):
    """More than 2^32 bytes in a pool of 4-bit pages: the last pages."""
    from turbopi_b200 import ops
    D, page = 256, 1024
    tile = 288 * groups(D)
    P = 2 ** 32 // (page // 16 * tile) + 8
    pages = torch.zeros((P, 1, page // 16, tile), dtype=torch.uint8, device=cuda_device)
    g = torch.Generator(device=cuda_device).manual_seed(0)
    x = torch.randn((3000, 1, D), generator=g, device=cuda_device, dtype=torch.bfloat16)
    v_pages = torch.zeros_like(pages)
    table = _ints([[P - 1, 0, P - 2]], cuda_device)
    lengths, cu = _ints([3000], cuda_device), _ints([0, 3000], cuda_device)
    ops.paged_append_nvfp4(x, x, pages, v_pages, table, cu, lengths)
    k, v = ops.paged_read_nvfp4(pages, v_pages, table, cu, lengths, D, 3000)
    from nvfp4_cache_reference import values
    want = values(*quantise(x), D)
    assert torch.equal(k.double(), want) and torch.equal(v.double(), want)
    q = torch.randn((1, 8, D), generator=g, device=cuda_device, dtype=torch.bfloat16)
    out = ops.paged_attention_nvfp4(q, pages, v_pages, table, lengths, 1 / 16)
    o, allow = attend(q, want, want, 1 / 16, torch.ones(1, 3000, dtype=torch.bool, device=cuda_device), WEIGHT)
    check(out, o, allow)
    _no_error()

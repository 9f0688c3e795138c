"""ops.paged_attention against attention in 64 bits: lengths of zero and one, pages that end inside a tile, odd sizes, strides,
what stands in rows that belong to nobody, graphs, streams."""
import pytest
import torch

from paged_reference import attend, check, deal_pages, gather

pytestmark = pytest.mark.gpu


def _problem(lens, hq, hk, D, page, dtype, device, seed=0, width=None, poison=True):
    g = torch.Generator(device=device).manual_seed(seed)
    rows, pool = deal_pages(lens, page, seed, width=width)
    cache = torch.randn((2, pool, page, hk, D), generator=g, device=device, dtype=dtype)
    if poison:                                  # rows behind a sequence's end and pages of nobody
        used = torch.zeros(pool, page, dtype=torch.bool, device=device)
        for row, n in zip(rows, lens):
            for j in range(n):
                used[row[j // page], j % page] = True
        cache[:, ~used] = float("nan")
    q = torch.randn((len(lens), hq, D), generator=g, device=device, dtype=dtype)
    table = torch.tensor(rows, dtype=torch.int32, device=device)
    return q, cache[0], cache[1], table, torch.tensor(lens, dtype=torch.int32, device=device), rows


def _check(out, q, k, v, rows, lens, scale):
    for i, n in enumerate(lens):
        want, allow = attend(q[i:i + 1], gather(k, rows[i], n), gather(v, rows[i], n), scale)
        check(out[i:i + 1], want, allow)


def _no_error():
    from turbopi_b200 import _lib
    assert _lib.load().tpb200_device_error(0) == 0


HEADS = [(8, 1, 256), (32, 8, 128), (16, 16, 64), (6, 2, 72), (5, 1, 8), (2, 2, 200), (16, 1, 96), (17, 1, 64), (40, 1, 128)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,hk,D", HEADS)
def test_heads_and_types(cuda_device, hq, hk, D, dtype):
    from turbopi_b200 import ops
    lens = [1, 0, 15, 16, 17, 63, 64, 65, 129, 300, 1001]
    q, k, v, table, lengths, rows = _problem(lens, hq, hk, D, 16, dtype, cuda_device, seed=D)
    out = ops.paged_attention(q, k, v, table, lengths, D ** -0.5)
    _check(out, q, k, v, rows, lens, D ** -0.5)
    assert bool((out[1] == 0).all())
    _no_error()


@pytest.mark.parametrize("page", [1, 3, 16, 24, 100, 128])
def test_page_sizes(cuda_device, page):
    from turbopi_b200 import ops
    lens = [page, page + 1, 2 * page - 1, 333, 7]
    q, k, v, table, lengths, rows = _problem(lens, 8, 2, 128, page, torch.bfloat16, cuda_device, seed=page)
    _check(ops.paged_attention(q, k, v, table, lengths, 0.1), q, k, v, rows, lens, 0.1)
    _no_error()


@pytest.mark.parametrize("lens", [[1], [50000], [0], [0, 0, 3, 0], [20000, 1, 1, 1], [1] * 700, [37] * 300, [4095, 0, 4097]])
def test_how_the_work_is_cut(cuda_device, lens):
    """One long sequence over every CTA, hundreds of short ones, empty ones between."""
    from turbopi_b200 import ops
    q, k, v, table, lengths, rows = _problem(lens, 8, 1, 256, 16, torch.bfloat16, cuda_device, seed=len(lens), poison=sum(lens) < 30000)
    out = ops.paged_attention(q, k, v, table, lengths, 1 / 16)
    _check(out, q, k, v, rows, lens, 1 / 16)
    _no_error()


def test_same_bits_every_time_and_alone(cuda_device):
    """The order in which CTAs finish changes nothing, nor does a NaN in another sequence."""
    from turbopi_b200 import ops
    lens = [3000, 5, 700]
    q, k, v, table, lengths, rows = _problem(lens, 8, 1, 256, 16, torch.float16, cuda_device)
    first = ops.paged_attention(q, k, v, table, lengths, 1 / 16)
    for _ in range(5):
        assert torch.equal(first, ops.paged_attention(q, k, v, table, lengths, 1 / 16))
    v[rows[1][0], 2] = float("nan")
    k[rows[1][0], 3] = float("inf")
    out = ops.paged_attention(q, k, v, table, lengths, 1 / 16)
    assert torch.equal(out[0], first[0]) and torch.equal(out[2], first[2]) and bool(out[1].isnan().all())


def test_large_and_small_scores(cuda_device):
    """Maxima that move by hundreds from tile to tile, a scale of zero, a negative one."""
    from turbopi_b200 import ops
    lens = [900, 130]
    q, k, v, table, lengths, rows = _problem(lens, 4, 2, 64, 16, torch.bfloat16, cuda_device)
    for scale in (20.0, 0.0, -3.0):
        _check(ops.paged_attention(q, k, v, table, lengths, scale), q, k, v, rows, lens, scale)


def test_strides(cuda_device):
    """A layer of a cache, heads outside the page, queries inside the fused projection's rows, an output of other strides, a
    table that is wider than it is read."""
    from turbopi_b200 import ops
    lens, hq, hk, D, page = [100, 33, 257], 8, 4, 128, 16
    g = torch.Generator(device=cuda_device).manual_seed(3)
    rows, pool = deal_pages(lens, page, 3, width=40)
    cache = torch.randn((3, 2, pool, hk, page, D), generator=g, device=cuda_device, dtype=torch.bfloat16)
    k, v = cache[1, 0].transpose(1, 2), cache[1, 1].transpose(1, 2)
    qkv = torch.randn((3, hq + 2 * hk, D), generator=g, device=cuda_device, dtype=torch.bfloat16)
    table = torch.tensor(rows, dtype=torch.int32, device=cuda_device)[:, :30]
    out = torch.full((3, 2 * hq, D), 7.0, device=cuda_device, dtype=torch.bfloat16)
    lengths = torch.tensor(lens, dtype=torch.int32, device=cuda_device)
    ops.paged_attention(qkv[:, :hq], k, v, table, lengths, 0.09, out=out[:, ::2])
    _check(out[:, ::2], qkv[:, :hq], k, v, rows, lens, 0.09)
    assert bool((out[:, 1::2] == 7).all())


def test_offsets_beyond_32_bits(cuda_device):
    """Pages whose elements lie beyond 2^31 of the pool."""
    from turbopi_b200 import ops
    page, D, hk = 64, 128, 8
    pool = (2 ** 31) // (page * D * hk) + 40
    k = torch.empty((pool, page, hk, D), dtype=torch.bfloat16, device=cuda_device)
    v = torch.empty_like(k)
    ids = [pool - 1, 3, pool - 20, pool - 7]
    for i in ids:
        k[i].normal_()
        v[i].normal_()
    q = torch.randn((1, 16, D), device=cuda_device).to(torch.bfloat16)
    lens = [4 * page - 5]
    out = ops.paged_attention(q, k, v, torch.tensor([ids], dtype=torch.int32, device=cuda_device),
                              torch.tensor(lens, dtype=torch.int32, device=cuda_device), 0.09)
    _check(out, q, k, v, [ids], lens, 0.09)


def test_a_captured_call_follows_lengths_and_table(cuda_device):
    from turbopi_b200 import ops
    lens = [300, 20, 1500]
    q, k, v, table, lengths, rows = _problem(lens, 8, 1, 256, 16, torch.bfloat16, cuda_device, poison=False)
    ws = ops.paged_attention_workspace(8, 1, 256, cuda_device)
    out = torch.empty_like(q)
    ops.paged_attention(q, k, v, table, lengths, 1 / 16, out=out, workspace=ws)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.paged_attention(q, k, v, table, lengths, 1 / 16, out=out, workspace=ws)
    for now in ([300, 20, 1500], [1, 0, 1499], [250, 3, 5]):
        lengths.copy_(torch.tensor(now, dtype=torch.int32))
        q.normal_()
        graph.replay()
        torch.cuda.synchronize()
        _check(out, q, k, v, rows, now, 1 / 16)
    table.copy_(table.flip(1))                                   # pages in another order (whole ones only are read)
    flipped = [list(reversed(r)) for r in rows]
    lengths.copy_(torch.tensor([0, 0, 1500], dtype=torch.int32))
    graph.replay()
    torch.cuda.synchronize()
    if -1 not in flipped[2]:
        _check(out, q, k, v, flipped, [0, 0, 1500], 1 / 16)


def test_two_streams_with_a_workspace_each(cuda_device):
    from turbopi_b200 import ops
    made = [_problem([2000, 31, 7], 8, 1, 256, 16, torch.bfloat16, cuda_device, seed=s) for s in (1, 2)]
    want = [ops.paged_attention(*p[:5], 1 / 16) for p in made]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in made]
    spaces = [ops.paged_attention_workspace(8, 1, 256, cuda_device) for _ in made]
    got = [torch.empty_like(w) for w in want]
    torch.cuda.synchronize()
    for _ in range(50):
        for st, p, ws, out in zip(streams, made, spaces, got):
            with torch.cuda.stream(st):
                ops.paged_attention(*p[:5], 1 / 16, out=out, workspace=ws)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_dependent_launches(cuda_device):
    """A chain of calls with programmatic dependent launch, each on the one before it."""
    from turbopi_b200 import ops
    q, k, v, table, lengths, rows = _problem([900, 40], 8, 1, 256, 16, torch.bfloat16, cuda_device)
    ws = ops.paged_attention_workspace(8, 1, 256, cuda_device)
    want = q
    for _ in range(6):
        want = ops.paged_attention(want, k, v, table, lengths, 1 / 16, workspace=ws)
    got = q
    with ops.launch_flags(ops.FLAG_PDL):
        for _ in range(6):
            got = ops.paged_attention(got, k, v, table, lengths, 1 / 16, workspace=ws)
    assert torch.equal(want, got)


def test_what_the_table_must_not_hold_is_reported(cuda_device):
    """Page ids outside the pool and lengths beyond the table are errors, not addresses; other sequences are not touched."""
    from turbopi_b200 import _lib, ops
    lib = _lib.load()
    lens = [100, 60]
    q, k, v, table, lengths, rows = _problem(lens, 8, 2, 128, 16, torch.bfloat16, cuda_device)
    want = ops.paged_attention(q, k, v, table, lengths, 0.1)
    assert lib.tpb200_device_error(1) == 0
    for bad in (k.shape[0], 2 ** 30, -5):
        t = table.clone()
        t[0, 2] = bad
        out = ops.paged_attention(q, k, v, t, lengths, 0.1)
        assert lib.tpb200_device_error(1) == 501
        assert torch.equal(out[1], want[1])
    n = lengths.clone()
    n[1] = table.shape[1] * 16 + 1
    out = ops.paged_attention(q, k, v, table, n, 0.1)
    assert lib.tpb200_device_error(1) == 501
    # all lengths decide where the work is cut, and so the order of a sequence's sums: right within the bound, not bit by bit
    _check(out[:1], q[:1], k, v, rows[:1], lens[:1], 0.1)
    n[1] = -3                                                    # no keys
    assert bool((ops.paged_attention(q, k, v, table, n, 0.1)[1] == 0).all())
    assert lib.tpb200_device_error(1) == 0


def test_more_sequences_than_lengths_are_staged(cuda_device):
    """1500 sequences: their lengths are read where they lie."""
    from turbopi_b200 import ops
    lens = [(i * 7) % 40 for i in range(1500)]
    q, k, v, table, lengths, rows = _problem(lens, 4, 2, 64, 16, torch.float16, cuda_device, seed=9, poison=False)
    out = ops.paged_attention(q, k, v, table, lengths, 0.125)
    for i in list(range(0, 1500, 37)) + [1499]:
        want, allow = attend(q[i:i + 1], gather(k, rows[i], lens[i]), gather(v, rows[i], lens[i]), 0.125)
        check(out[i:i + 1], want, allow)
    _no_error()


@pytest.mark.parametrize("hq", [1, 8, 9, 16])
@pytest.mark.parametrize("n", [1, 15, 16, 31, 32, 33, 47, 48, 49, 63, 64, 65, 80, 129, 192, 193, 1000])
def test_lines_of_few_slots(cuda_device, n, hq):
    """Lines too short to give every warp a slot, CTAs inside one item, items that end where a CTA does."""
    from turbopi_b200 import ops
    for D in (64, 256):
        q, k, v, table, lengths, rows = _problem([n], hq, 1, D, 16, torch.bfloat16, cuda_device, seed=n)
        _check(ops.paged_attention(q, k, v, table, lengths, D ** -0.5), q, k, v, rows, [n], D ** -0.5)
    _no_error()


@pytest.mark.parametrize("seed", range(6))
def test_drawn_lengths(cuda_device, seed):
    import random

    from turbopi_b200 import ops
    rng = random.Random(seed)
    hq, hk, D = rng.choice([(8, 1, 256), (8, 2, 128), (16, 16, 64), (12, 4, 128), (16, 2, 96)])
    lens = [rng.choice([0, 1, rng.randint(1, 60), rng.randint(1, 700), rng.randint(1, 4000)]) for _ in range(rng.randint(1, 60))]
    q, k, v, table, lengths, rows = _problem(lens, hq, hk, D, rng.choice([16, 24, 64]), torch.bfloat16, cuda_device, seed=seed, poison=False)
    _check(ops.paged_attention(q, k, v, table, lengths, D ** -0.5), q, k, v, rows, lens, D ** -0.5)
    _no_error()


def test_output_in_place_of_the_queries(cuda_device):
    from turbopi_b200 import ops
    q, k, v, table, lengths, rows = _problem([3000, 5, 700, 64], 16, 1, 128, 16, torch.bfloat16, cuda_device)
    want = ops.paged_attention(q, k, v, table, lengths, 0.1)
    assert ops.paged_attention(q, k, v, table, lengths, 0.1, out=q) is q and torch.equal(q, want)

"""ops.packed_attention against attention in 64 bits: lengths around the tiles' edges, queries behind cached keys and with fewer keys
than queries, groups that are no power of two, what stands in masked places, strides, graphs, streams."""
import pytest
import torch

from paged_reference import attend, check

pytestmark = pytest.mark.gpu


def _offsets(lens, device):
    return torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device=device)


def _problem(lens, klens, hq, hk, D, dtype, device, seed=0, behind=0):
    """Queries, keys, values with `behind` rows of NaN after the last sequence."""
    g = torch.Generator(device=device).manual_seed(seed)
    q = torch.randn((sum(lens) + behind, hq, D), generator=g, device=device, dtype=dtype)
    k, v = torch.randn((2, sum(klens) + behind, hk, D), generator=g, device=device, dtype=dtype)
    for t, n in ((q, sum(lens)), (k, sum(klens)), (v, sum(klens))):
        t[n:] = float("nan")
    return q, k, v


def _check(out, q, k, v, lens, klens, scale, causal):
    q0 = k0 = 0
    for n, m in zip(lens, klens):
        want, allow = attend(q[q0:q0 + n], k[k0:k0 + m], v[k0:k0 + m], scale, m - n if causal else None)
        check(out[q0:q0 + n], want, allow)
        q0, k0 = q0 + n, k0 + m


def _no_error():
    from turbopi_b200 import _lib
    assert _lib.load().tpb200_device_error(0) == 0


def _run(device, lens, klens, hq, hk, D, dtype, causal, scale=None, seed=0, behind=3):
    from turbopi_b200 import ops
    scale = D ** -0.5 if scale is None else scale
    q, k, v = _problem(lens, klens, hq, hk, D, dtype, device, seed, behind)
    out = torch.full_like(q, 9.0)
    same = lens == klens
    got = ops.packed_attention(q, k, v, _offsets(lens, device), scale, out=out, causal=causal,
                               cu_keys=None if same else _offsets(klens, device))
    assert got is out
    _check(out, q, k, v, lens, klens, scale, causal)
    assert bool((out[sum(lens):] == 9).all())
    _no_error()


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("n", [1, 128, 300])
def test_one_sequence(cuda_device, n, D):
    """The smallest calls first."""
    _run(cuda_device, [n], [n], 1, 1, D, torch.bfloat16, False)
    _run(cuda_device, [n], [n], 1, 1, D, torch.bfloat16, True)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,hk,D", [(8, 1, 256), (32, 8, 128), (16, 4, 64), (16, 16, 64), (6, 2, 72), (3, 1, 8), (2, 2, 200), (16, 1, 96),
                                     (20, 1, 128), (48, 1, 64), (4, 2, 136)])
def test_heads_and_types(cuda_device, hq, hk, D, dtype, causal):
    lens = [1, 0, 127, 128, 129, 15, 33, 300, 64]
    _run(cuda_device, lens, lens, hq, hk, D, dtype, causal, seed=D)


@pytest.mark.parametrize("hq,hk,D", [(8, 1, 256), (8, 2, 128), (4, 4, 64)])
@pytest.mark.parametrize("causal", [True, False])
def test_more_and_fewer_keys_than_queries(cuda_device, hq, hk, D, causal):
    """Cached keys before the queries; sequences whose first queries see nothing; ones without any key."""
    _run(cuda_device, [5, 100, 1, 40, 300, 7, 0], [133, 612, 1000, 40, 130, 0, 50], hq, hk, D, torch.bfloat16, causal, seed=1)


@pytest.mark.parametrize("hq,hk,D", [(8, 1, 256), (8, 2, 128), (2, 1, 64)])
def test_long(cuda_device, hq, hk, D):
    _run(cuda_device, [2500, 1031], [2500, 1031], hq, hk, D, torch.bfloat16, True, seed=2)
    _run(cuda_device, [1031], [4000], hq, hk, D, torch.float16, True, seed=2)


def test_many_short_sequences(cuda_device):
    lens = [(7 * i) % 23 for i in range(200)]
    _run(cuda_device, lens, lens, 8, 2, 64, torch.float16, True)


@pytest.mark.parametrize("D", [64, 256])
@pytest.mark.parametrize("scale", [30.0, 0.0, -2.0, 1e-30])
def test_large_and_small_scores(cuda_device, scale, D):
    """Maxima that move by hundreds from tile to tile (the sums in tensor memory are rescaled), none, a negative scale."""
    _run(cuda_device, [700], [700], 2, 1, D, torch.bfloat16, True, scale=scale, seed=4)


@pytest.mark.parametrize("D", [128, 256])
def test_growing_maxima(cuda_device, D):
    """Keys that grow along the sequence: the reference is raised in every tile."""
    from turbopi_b200 import ops
    q, k, v = _problem([900], [900], 4, 2, D, torch.float16, cuda_device, seed=5)
    k *= torch.linspace(0.05, 8, 900, device=cuda_device).to(k.dtype)[:, None, None]
    out = ops.packed_attention(q, k, v, _offsets([900], cuda_device), 0.3)
    _check(out, q, k, v, [900], [900], 0.3, True)
    _no_error()


@pytest.mark.parametrize("hq,hk,D", [(8, 1, 256), (8, 2, 128), (4, 4, 64)])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
def test_what_stands_in_masked_places_does_not_matter(cuda_device, hq, hk, D, value):
    """A bad key or value reaches the queries that see it and no other, nor another sequence."""
    from turbopi_b200 import ops
    lens, klens = [150, 333, 64], [150, 400, 64]
    cu, cuk = _offsets(lens, cuda_device), _offsets(klens, cuda_device)
    q, k, v = _problem(lens, klens, hq, hk, D, torch.bfloat16, cuda_device, seed=6)
    clean = ops.packed_attention(q, k, v, cu, D ** -0.5, cu_keys=cuk)
    for where in ("k", "v"):
        for at in (0, 100, 66 + 67, 201, 399):                    # positions in the second sequence; the first query sees 67
            k2, v2 = k.clone(), v.clone()
            (k2 if where == "k" else v2)[150 + at, 0, D // 2:] = value
            out = ops.packed_attention(q, k2, v2, cu, D ** -0.5, cu_keys=cuk)
            sees = torch.arange(333, device=cuda_device) + 67 >= at
            assert torch.equal(out[:150], clean[:150]) and torch.equal(out[150 + 333:], clean[150 + 333:])
            assert torch.equal(out[150:150 + 333][~sees], clean[150:150 + 333][~sees])
            if where == "v":                                      # the first key head's queries, the columns that hold it
                bad = out[150:150 + 333][sees][:, :hq // hk, D // 2:]
                assert bool((bad.isnan() if value != value else (bad == value)).all())
                assert torch.equal(out[150:150 + 333, :, :D // 2], clean[150:150 + 333, :, :D // 2])
                assert torch.equal(out[150:150 + 333, hq // hk:], clean[150:150 + 333, hq // hk:])
    _no_error()


def test_strides(cuda_device):
    """Columns of a fused projection, an output between other heads, keys whose heads lie outside the tokens."""
    from turbopi_b200 import ops
    lens, hq, hk, D = [100, 257], 8, 2, 128
    g = torch.Generator(device=cuda_device).manual_seed(7)
    qkv = torch.randn((357, hq + 2 * hk, D), generator=g, device=cuda_device, dtype=torch.bfloat16)
    q, k, v = qkv.split([hq, hk, hk], 1)
    out = torch.full((357, 2 * hq, D), 4.0, device=cuda_device, dtype=torch.bfloat16)
    ops.packed_attention(q, k, v, _offsets(lens, cuda_device), 0.1, out=out[:, 1::2])
    _check(out[:, 1::2], q, k, v, lens, lens, 0.1, True)
    assert bool((out[:, ::2] == 4).all())
    k2, v2 = (t.transpose(0, 1).contiguous().transpose(0, 1) for t in (k, v))
    again = ops.packed_attention(q, k2, v2, _offsets(lens, cuda_device), 0.1)
    assert torch.equal(again, out[:, 1::2])
    _no_error()


def test_same_bits_every_time_and_in_a_graph_that_follows_the_offsets(cuda_device):
    from turbopi_b200 import ops
    lens = [300, 40, 500]
    q, k, v = _problem(lens, lens, 8, 1, 256, torch.bfloat16, cuda_device, seed=8)
    cu = _offsets(lens, cuda_device)
    first = ops.packed_attention(q, k, v, cu, 1 / 16)
    for _ in range(5):
        assert torch.equal(first, ops.packed_attention(q, k, v, cu, 1 / 16))
    out = torch.empty_like(q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.packed_attention(q, k, v, cu, 1 / 16, out=out)
    for now in (lens, [1, 838, 1], [0, 0, 840], [280, 280, 280], [5, 6, 7]):
        cu.copy_(_offsets(now, cuda_device))
        out.fill_(9)
        graph.replay()
        torch.cuda.synchronize()
        _check(out, q, k, v, now, now, 1 / 16, True)
        assert bool((out[sum(now):] == 9).all())
    _no_error()


def test_streams_and_dependent_launches(cuda_device):
    """Two streams at once; a chain in which each call reads the one before it."""
    from turbopi_b200 import ops
    made = [_problem([700, 31], [700, 31], 8, 1, 256, torch.bfloat16, cuda_device, seed=s) for s in (1, 2)]
    cu = _offsets([700, 31], cuda_device)
    want = [ops.packed_attention(*p, cu, 1 / 16) for p in made]
    got = [torch.empty_like(w) for w in want]
    streams = [torch.cuda.Stream() for _ in made]
    torch.cuda.synchronize()
    for _ in range(20):
        for st, p, out in zip(streams, made, got):
            with torch.cuda.stream(st):
                ops.packed_attention(*p, cu, 1 / 16, out=out)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    q, k, v = made[0]
    a = b = q
    for _ in range(5):
        a = ops.packed_attention(a, k, v, cu, 1 / 16)
    with ops.launch_flags(ops.FLAG_PDL):
        for _ in range(5):
            b = ops.packed_attention(b, k, v, cu, 1 / 16)
    assert torch.equal(a, b)
    _no_error()


def test_offsets_outside_the_tensors_are_clamped(cuda_device):
    """Never an address: ends beyond the tokens, a beginning below zero, offsets that fall."""
    from turbopi_b200 import ops
    q, k, v = _problem([200], [200], 2, 1, 64, torch.bfloat16, cuda_device, seed=9)
    want = ops.packed_attention(q, k, v, _offsets([150, 50], cuda_device), 0.125)
    cu = torch.tensor([-70, 150, 2 ** 31 - 1], dtype=torch.int32, device=cuda_device)
    assert torch.equal(ops.packed_attention(q, k, v, cu, 0.125), want)
    cu = torch.tensor([0, 150, 100], dtype=torch.int32, device=cuda_device)      # the second sequence has no tokens
    out = torch.zeros_like(q)
    assert torch.equal(ops.packed_attention(q, k, v, cu, 0.125, out=out)[:150], want[:150])
    assert bool((out[150:] == 0).all())
    _no_error()


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,hk,D", [(8, 2, 128), (16, 4, 64), (3, 1, 72), (4, 4, 64)])
def test_two_row_tiles_per_cta(cuda_device, hq, hk, D, dtype, causal):
    """Sequences long enough on average for the form with two row tiles: ragged ends, a tile of rows on its own, queries without keys,
    short sequences between long ones."""
    lens, klens = [129, 40, 300, 7, 128], [4500, 1300, 130, 3000, 128]
    _run(cuda_device, lens, klens, hq, hk, D, dtype, causal, seed=D)


def test_masked_places_with_two_row_tiles(cuda_device):
    from turbopi_b200 import ops
    lens, klens = [300, 200], [300, 3000]
    cu, cuk = _offsets(lens, cuda_device), _offsets(klens, cuda_device)
    q, k, v = _problem(lens, klens, 8, 2, 128, torch.bfloat16, cuda_device, seed=11)
    clean = ops.packed_attention(q, k, v, cu, 0.09, cu_keys=cuk)
    for value in (float("nan"), float("inf")):
        for at in (2850, 2900, 2999, 10):                        # the first query sees 2801
            v2 = v.clone()
            v2[300 + at, 0, 64:] = value
            out = ops.packed_attention(q, k, v2, cu, 0.09, cu_keys=cuk)
            sees = torch.arange(200, device=cuda_device) + 2800 >= at
            assert torch.equal(out[:300], clean[:300]) and torch.equal(out[300:][~sees], clean[300:][~sees])
            bad = out[300:][sees][:, :4, 64:]
            assert bool((bad.isnan() if value != value else (bad == value)).all())
            assert torch.equal(out[300:, :, :64], clean[300:, :, :64]) and torch.equal(out[300:, 4:], clean[300:, 4:])
    _no_error()


def test_rows_without_keys_beside_rows_with_keys(cuda_device):
    """One row tile of a CTA is done before the CTA's queries have landed where outputs are staged; many launches."""
    from turbopi_b200 import ops
    n, m = 256, 100                                              # 128 rows without keys, then 28 more, then 100 with
    lens, klens = [n] * 40 + [16], [m] * 40 + [90000]            # the long one: two row tiles per CTA
    q, k, v = _problem(lens, klens, 1, 1, 64, torch.bfloat16, cuda_device, seed=12)
    cu, cuk = _offsets(lens, cuda_device), _offsets(klens, cuda_device)
    for _ in range(30):
        out = ops.packed_attention(q, k, v, cu, 0.125, cu_keys=cuk)
        assert bool((out[:n * 40].view(40, n, 64)[:, :n - m] == 0).all())
    _check(out[:n], q, k, v, [n], [m], 0.125, True)
    _no_error()


@pytest.mark.parametrize("seed", range(8))
def test_drawn_batches(cuda_device, seed):
    import random
    rng = random.Random(seed)
    hq, hk, D = rng.choice([(8, 1, 256), (32, 8, 128), (16, 4, 64), (16, 16, 64), (12, 4, 128), (16, 16, 72), (16, 2, 96), (4, 4, 256)])
    lens = [rng.choice([0, 1, rng.randint(1, 130), rng.randint(1, 700)]) for _ in range(rng.randint(1, 20))]
    klens = lens if rng.random() < 0.4 else [max(0, n + rng.choice([0, 5, 300, 2000, -50])) for n in lens]
    _run(cuda_device, lens, klens, hq, hk, D, rng.choice([torch.bfloat16, torch.float16]), rng.random() < 0.7, seed=seed)


def test_output_in_place_of_the_queries(cuda_device):
    from turbopi_b200 import ops
    for D in (64, 256):
        q, k, v = _problem([300, 40, 129], [300, 40, 129], 4, 2, D, torch.bfloat16, cuda_device)
        cu = _offsets([300, 40, 129], cuda_device)
        want = ops.packed_attention(q, k, v, cu, 0.1)
        assert ops.packed_attention(q, k, v, cu, 0.1, out=q) is q and torch.equal(q, want)


def test_tokens_in_front_of_the_first_sequence_are_left_alone(cuda_device):
    from turbopi_b200 import ops
    q, k, v = _problem([50, 200], [50, 200], 2, 1, 128, torch.float16, cuda_device)
    out = torch.full_like(q, 6.0)
    ops.packed_attention(q, k, v, torch.tensor([50, 250], dtype=torch.int32, device=cuda_device), 0.1, out=out)
    assert bool((out[:50] == 6).all())
    _check(out[50:], q[50:], k[50:], v[50:], [200], [200], 0.1, True)


def test_launches_behind_copies_fills_and_another_stream(cuda_device):
    """These launches start while what is before them drains: a host copy, a fill, a wait for another stream, captured too."""
    from turbopi_b200 import ops
    lens = [90, 33]
    q, k, v = _problem(lens, lens, 4, 1, 64, torch.bfloat16, cuda_device)
    want = ops.packed_attention(q, k, v, _offsets(lens, cuda_device), 0.125)
    host = q.cpu().pin_memory()
    side = torch.cuda.Stream()
    q2, k2, cu = torch.zeros_like(q), torch.empty_like(k), _offsets(lens, cuda_device)
    torch.cuda.synchronize()

    def chain(out):
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            k2.copy_(k)
        q2.copy_(host, non_blocking=True)
        out.fill_(3)
        torch.cuda.current_stream().wait_stream(side)
        ops.packed_attention(q2, k2, v, cu, 0.125, out=out)
        q2.zero_()
        k2.zero_()
    for _ in range(50):
        out = torch.empty_like(q)
        chain(out)
        assert torch.equal(out, want)
    graph, out = torch.cuda.CUDAGraph(), torch.empty_like(q)
    with torch.cuda.graph(graph):
        chain(out)
    for _ in range(20):
        graph.replay()
        assert torch.equal(out, want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,hk,D", [(4, 2, 64), (3, 1, 40), (4, 2, 128)])
def test_growing_maxima_with_two_row_tiles(cuda_device, hq, hk, D, dtype):
    """Long sequences, the reference raised in every tile: small heads have the next scores, and the last product, under way meanwhile."""
    from turbopi_b200 import ops
    lens, klens = [1300, 1150], [1300, 1400]
    q, k, v = _problem(lens, klens, hq, hk, D, dtype, cuda_device, seed=9)
    k *= torch.linspace(0.05, 8, sum(klens), device=cuda_device).to(k.dtype)[:, None, None]
    cu, cuk = _offsets(lens, cuda_device), _offsets(klens, cuda_device)
    for causal in (True, False):
        first = ops.packed_attention(q, k, v, cu, 0.3, causal=causal, cu_keys=cuk)
        _check(first, q, k, v, lens, klens, 0.3, causal)
        for _ in range(5):
            assert torch.equal(ops.packed_attention(q, k, v, cu, 0.3, causal=causal, cu_keys=cuk), first)
    _no_error()

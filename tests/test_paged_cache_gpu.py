"""ops.paged_append and ops.copy_pages: every value of the cache afterwards, those that nothing was written to among them."""
import pytest
import torch

from paged_reference import HALF_STEP, deal_pages, rotate

pytestmark = pytest.mark.gpu


def _append_problem(new, before, hq, hk, D, page, dtype, device, seed=0, behind=0):
    g = torch.Generator(device=device).manual_seed(seed)
    ends = [a + b for a, b in zip(new, before)]
    rows, pool = deal_pages(ends, page, seed)
    cache = torch.randn((2, pool, page, hk, D), generator=g, device=device, dtype=dtype)
    T = sum(new) + behind
    qkv = torch.randn((T, hq + 2 * hk, D), generator=g, device=device, dtype=dtype)
    cu = torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32, device=device)
    table = torch.tensor(rows, dtype=torch.int32, device=device)
    return dict(q=qkv[:, :hq], k=qkv[:, hq:hq + hk], v=qkv[:, hq + hk:], cache=cache, table=table, cu=cu, rows=rows,
                lengths=torch.tensor(ends, dtype=torch.int32, device=device), ends=ends)


def _places(new, ends, rows, page):
    return [(rows[s][pos // page], pos % page, pos) for s, n in enumerate(new) for pos in range(ends[s] - n, ends[s])]


def _tables(positions, D, dtype, device):
    a = torch.arange(positions, device=device, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, D, 2, device=device, dtype=torch.float64) / D)
    return a.cos().to(dtype), a.sin().to(dtype)


CASES = [([1] * 5, [0, 1, 15, 16, 300], 8, 1, 256, 16), ([7, 0, 40, 1], [3, 9, 0, 100], 6, 2, 72, 16),
         ([33, 129], [5, 0], 32, 8, 128, 24), ([3], [0], 1, 1, 8, 1), ([700, 1, 900], [0, 20, 31], 4, 4, 64, 32), ([5], [2], 2, 1, 96, 100)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("new,before,hq,hk,D,page", CASES)
def test_plain_append(cuda_device, new, before, hq, hk, D, page, dtype):
    from turbopi_b200 import _lib, ops
    p = _append_problem(new, before, hq, hk, D, page, dtype, cuda_device, behind=2)
    want = p["cache"].clone()
    for t, (i, r, _) in enumerate(_places(new, p["ends"], p["rows"], page)):
        want[0, i, r], want[1, i, r] = p["k"][t], p["v"][t]
    assert ops.paged_append(p["k"], p["v"], p["cache"][0], p["cache"][1], p["table"], p["cu"], p["lengths"]) is None
    assert torch.equal(p["cache"], want)
    assert _lib.load().tpb200_device_error(0) == 0


@pytest.mark.parametrize("table_dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("new,before,hq,hk,D,page", CASES)
def test_append_with_rotation(cuda_device, new, before, hq, hk, D, page, dtype, table_dtype):
    """Two products and a sum in fp32 (each off by at most 2^-24 of the larger terms), one rounding to the type."""
    from turbopi_b200 import ops
    p = _append_problem(new, before, hq, hk, D, page, dtype, cuda_device, seed=D, behind=3)
    places = _places(new, p["ends"], p["rows"], page)
    T = len(places)
    cos, sin = _tables(max(p["ends"]), D, table_dtype, cuda_device)
    pos = torch.tensor([x[2] for x in places], device=cuda_device)
    before_cache = p["cache"].clone()
    q_out = torch.full_like(p["q"], 5.0)
    got = ops.paged_append(p["k"], p["v"], p["cache"][0], p["cache"][1], p["table"], p["cu"], p["lengths"], q=p["q"], cos=cos,
                           sin=sin, q_out=q_out)
    assert got is q_out and bool((q_out[T:] == 5).all())
    ids, slots = (torch.tensor([x[j] for x in places], device=cuda_device) for j in (0, 1))
    u = HALF_STEP[dtype]
    for x, y in ((p["q"][:T], q_out[:T]), (p["k"][:T], p["cache"][0][ids, slots])):
        want = rotate(x, cos[pos], sin[pos])
        size = rotate(x.abs(), cos[pos].abs(), -sin[pos].abs())                       # |a c| + |b s| in the first half ...
        size[..., D // 2:] = rotate(x.abs(), cos[pos].abs(), sin[pos].abs())[..., D // 2:]    # ... and in the second
        tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0                           # half the smallest fp16 step
        assert bool(((y.double() - want).abs() <= u * want.abs() + 3 * 2.0 ** -24 * (1 + u) * size + tiny).all())
    want_v = before_cache[1].clone()
    want_v[ids, slots] = p["v"][:T]
    assert torch.equal(p["cache"][1], want_v)
    rest = before_cache[0].clone()
    rest[ids, slots] = p["cache"][0][ids, slots]
    assert torch.equal(p["cache"][0], rest)


def test_rotation_in_place_and_keys_alone(cuda_device):
    from turbopi_b200 import ops
    p = _append_problem([9, 4], [30, 2], 8, 2, 128, 16, torch.bfloat16, cuda_device)
    cos, sin = _tables(64, 128, torch.float32, cuda_device)
    args = (p["k"], p["v"], p["cache"][0], p["cache"][1], p["table"], p["cu"], p["lengths"])
    out = ops.paged_append(*args, q=p["q"], cos=cos, sin=sin)
    both = p["cache"].clone()
    assert ops.paged_append(*args, cos=cos, sin=sin) is None
    assert torch.equal(p["cache"], both)
    same = ops.paged_append(*args, q=p["q"], cos=cos, sin=sin, q_out=p["q"])
    assert same is p["q"] and torch.equal(same, out)


def test_a_token_without_a_place_writes_nothing(cuda_device):
    """A page id outside the pool, a position outside the table or the rotation's tables, before the sequence's beginning."""
    from turbopi_b200 import _lib, ops
    lib = _lib.load()
    cos, sin = _tables(200, 64, torch.float32, cuda_device)

    def run(change, allowed, **kw):
        p = _append_problem([4, 3], [40, 10], 4, 2, 64, 16, torch.bfloat16, cuda_device)
        change(p)
        before = p["cache"].clone()
        q_out = torch.full_like(p["q"], 3.0)
        ops.paged_append(p["k"], p["v"], p["cache"][0], p["cache"][1], p["table"], p["cu"], p["lengths"], q=p["q"], q_out=q_out,
                         cos=kw.get("cos", cos), sin=kw.get("sin", sin))
        assert lib.tpb200_device_error(1) == 501
        changed = (p["cache"] != before).flatten(3).any(-1).any(0)
        assert int(changed.sum()) == allowed
        assert int((q_out != 3).flatten(1).any(1).sum()) == allowed

    def page(p):
        p["table"][0, 2] = p["cache"].shape[1]

    def length(p):
        p["lengths"][0] = p["table"].shape[1] * 16 + 2           # the first two of four tokens still have a place
    run(page, 3)
    run(length, 5)
    run(lambda p: p["lengths"].__setitem__(1, 2), 6)             # three tokens of a sequence that is two long
    run(lambda p: None, 4, cos=cos[:41].contiguous(), sin=sin[:41].contiguous())    # positions 41..43 lie outside the tables
    run(lambda p: p["table"].fill_(-1), 0)


def test_captured_append(cuda_device):
    from turbopi_b200 import ops
    p = _append_problem([1, 1, 1], [5, 31, 0], 8, 1, 256, 16, torch.bfloat16, cuda_device)
    p["table"][:, 0].clamp_(min=0)
    args = (p["k"], p["v"], p["cache"][0], p["cache"][1], p["table"], p["cu"], p["lengths"])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.paged_append(*args)
    p["lengths"].copy_(torch.tensor([3, 17, 1], dtype=torch.int32))
    want = p["cache"].clone()
    for s, n in enumerate([3, 17, 1]):
        want[0, p["rows"][s][(n - 1) // 16], (n - 1) % 16] = p["k"][s]
        want[1, p["rows"][s][(n - 1) // 16], (n - 1) % 16] = p["v"][s]
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(p["cache"], want)


# ---------------------------------------------------------------------------------------------- copies of pages
@pytest.mark.parametrize("shape,dtype", [((3, 2, 40, 16, 1, 256), torch.bfloat16), ((1200, 2, 1, 8), torch.float16),
                                         ((2, 30, 5, 3, 72), torch.float32), ((7, 50, 24, 2, 8), torch.uint8)])
def test_copies(cuda_device, shape, dtype):
    from turbopi_b200 import ops
    g = torch.Generator().manual_seed(len(shape))
    pages = torch.randint(0, 100, shape, generator=g).to(dtype).to(cuda_device)
    P = shape[-4]
    order = torch.randperm(P, generator=g).tolist()
    n = min(P // 2, 599)
    src, dst = order[:n], order[n:2 * n]
    src[1] = src[0]                                              # the same page to two places
    want = pages.clone()
    want[..., dst, :, :, :] = pages[..., src, :, :, :]
    ops.copy_pages(pages, src, torch.tensor(dst))
    assert torch.equal(pages, want)
    ops.copy_pages(pages, [], [])
    assert torch.equal(pages, want)


def test_copies_beyond_32_bits(cuda_device):
    from turbopi_b200 import ops
    pages = torch.empty((2, 20000, 64, 8, 128), dtype=torch.bfloat16, device=cuda_device)    # 2.6 billion values
    pages[:, 5].normal_()
    pages[:, 19999].normal_()
    ops.copy_pages(pages, [5, 19999], [19998, 7])
    assert torch.equal(pages[:, 19998], pages[:, 5]) and torch.equal(pages[:, 7], pages[:, 19999])


def test_captured_copies(cuda_device):
    """The pairs are part of the launch: a graph moves the same pages whatever the lists hold later."""
    from turbopi_b200 import ops
    pages = torch.randn(2, 1200, 4, 1, 8, device=cuda_device).to(torch.float16)
    src, dst = list(range(500)), list(range(600, 1100))          # more than one launch's worth
    ops.copy_pages(pages, [0], [1199])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.copy_pages(pages, src, dst)
    src[:], dst[:] = dst, src
    pages[:, :600].normal_()
    want = pages.clone()
    want[:, 600:1100] = pages[:, :500]
    graph.replay()
    assert torch.equal(pages, want)


def test_ids_that_would_wrap_are_refused(cuda_device):
    from turbopi_b200 import ops
    from turbopi_b200._lib import TurboPiError
    pages = torch.zeros(4, 2, 1, 8, device=cuda_device)
    for bad in ([2 ** 32], [2 ** 70], [1.0], [True], [None]):
        with pytest.raises(TurboPiError):
            ops.copy_pages(pages, bad, [2])

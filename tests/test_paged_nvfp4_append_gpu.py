"""ops.paged_append_nvfp4, ops.paged_read_nvfp4 and ops.paged_read against their definitions: every code and scale, and every byte that is
not theirs."""
import pytest
import torch

from nvfp4_cache_reference import groups, pack, quantise, unpack, values
from paged_reference import HALF_STEP, deal_pages, rotate

pytestmark = pytest.mark.gpu

HEADS = [(8, 1, 256), (32, 8, 128), (16, 16, 64), (6, 2, 72), (5, 1, 8), (2, 2, 200), (16, 1, 96), (3, 3, 40), (1, 1, 32)]


def _ints(x, device):
    return torch.tensor(x, dtype=torch.int32, device=device)


def _offsets(lens):
    return [sum(lens[:i]) for i in range(len(lens) + 1)]


def _pool(pool, hk, page, D, device, seed):
    """Pages of random bytes, scales among them that are NaN."""
    g = torch.Generator(device=device).manual_seed(seed)
    return torch.randint(0, 256, (2, pool, hk, page // 16, 288 * groups(D)), generator=g, device=device, dtype=torch.uint8)


def _tables(n, D, dtype, device):
    a = torch.arange(n, device=device, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, D, 2, device=device, dtype=torch.float64) / D)
    return a.cos().to(dtype), a.sin().to(dtype)


def _no_error():
    from turbopi_b200 import _lib
    assert _lib.load().tpb200_device_error(0) == 0


def _turned(x, cos, sin):
    """The rotation in 32 bits, each operation rounded, as elementary operations give it."""
    a, b = x.float().chunk(2, -1)
    c, s = cos.float()[:, None], sin.float()[:, None]
    return torch.cat([a * c - b * s, b * c + a * s], -1).to(x.dtype)


def _rows(pages, rows, lens, new, page):
    """The rows of the new tokens, [tokens, H, ...], of something [P, H, page, ...]."""
    out = []
    for row, n, m in zip(rows, lens, new):
        for j in range(n - m, n):
            out.append(pages[row[j // page], :, j % page])
    return torch.stack(out)


def _check_append(device, lens, new, hq, hk, D, page, dtype, rope=None, k_scale=1.0, v_scale=1.0, change=None, strided=False, seed=0):
    from turbopi_b200 import ops
    g = torch.Generator(device=device).manual_seed(seed)
    rows, pool = deal_pages(lens, page, seed)
    T = sum(new)
    pages = _pool(pool, hk, page, D, device, seed)
    if strided:                              # heads ahead of pages, bytes behind each tile
        wide = torch.randint(0, 256, (2, hk, pool, page // 16, 288 * groups(D) + 32), generator=g, device=device, dtype=torch.uint8)
        pages = wide.transpose(1, 2)[..., :288 * groups(D)]
        rest = wide[..., 288 * groups(D):].clone()
    before = pages.clone()
    qkv = torch.randn((T + 3, hq + 2 * hk, D), generator=g, device=device, dtype=dtype)
    if change:
        change(qkv)
    q, k, v = qkv.split([hq, hk, hk], 1)
    cu, lengths, table = _ints(_offsets(new), device), _ints(lens, device), _ints(rows, device)
    kw, kk = {}, k[:T]
    if rope is not None:
        cos, sin = _tables(max(lens), D, rope, device)
        kw = dict(q=q, cos=cos, sin=sin, q_out=torch.full((T + 3, hq, D), 9.0, dtype=dtype, device=device))
        pos = torch.cat([torch.arange(n - m, n, device=device) for n, m in zip(lens, new)])
        kk = _turned(k[:T], cos[pos], sin[pos])
        exact = rotate(k[:T], cos[pos], sin[pos])
        big = (k[:T].double().abs() @ torch.ones(D, 1, dtype=torch.float64, device=device)).clamp(min=1e-30)
        fine = kk.isfinite()
        assert bool(((kk.double() - exact).abs() <= HALF_STEP[dtype] * exact.abs() + 2.0 ** -22 * big + 2.0 ** -24)[fine].all())
    got = ops.paged_append_nvfp4(k, v, pages[0], pages[1], table, cu, lengths, k_scale=k_scale, v_scale=v_scale, **kw)
    for side, x, f in ((0, kk, k_scale), (1, v[:T], v_scale)):
        code, byte = quantise(x, f)
        have_code, have_byte = (_rows(y, rows, lens, new, page) for y in unpack(pages[side], D))
        assert torch.equal(have_byte, byte)
        bad = (byte == 127).repeat_interleave(16, -1)
        assert torch.equal(values(have_code, byte, D).nan_to_num(nan=1e9), values(code, byte, D).nan_to_num(nan=1e9))
        assert bool((have_code[..., D:] == 0).all()) and bool((have_code[bad] == 0).all())
    # nothing else was written: the other rows have their bytes
    code, byte = unpack(pages.flatten(0, 1), D)
    old_code, old_byte = unpack(before.flatten(0, 1), D)
    mine = torch.zeros(pool, page, dtype=torch.bool, device=device)
    for row, n, m in zip(rows, lens, new):
        for j in range(n - m, n):
            mine[row[j // page], j % page] = True
    other = ~mine.repeat(2, 1)
    assert torch.equal(code.transpose(1, 2)[other], old_code.transpose(1, 2)[other])
    assert torch.equal(byte.transpose(1, 2)[other], old_byte.transpose(1, 2)[other])
    if strided:
        assert torch.equal(wide[..., 288 * groups(D):], rest)
    if rope is None:
        assert got is None
    else:
        assert got is kw["q_out"] and bool((got[T:] == 9).all())
        assert torch.equal(got[:T], _turned(q[:T], cos[pos], sin[pos]))         # no operation fused with another
        want = rotate(q[:T], cos[pos], sin[pos])
        big = q[:T].double().abs().sum(-1, keepdim=True)
        assert bool(((got[:T].double() - want).abs() <= HALF_STEP[dtype] * want.abs() + 2.0 ** -22 * big + 2.0 ** -24).all())
    _no_error()
    # and read back: the values, rounded once; a type that holds them (factors of 1: multiples of 2^-10 of up to 7 bits, 2688 at most) has them exactly.
    # With a factor of 2^-60 they are below 2^-48, and fp16's least is 2^-24: zeros.
    pos_k = torch.full((T + 3, hk, D), 7.0, dtype=dtype, device=device)
    pos_v = torch.full((T + 3, hk, D), 7.0, dtype=dtype, device=device)
    a, b = ops.paged_read_nvfp4(pages[0], pages[1], table, cu, lengths, D, T + 3, dtype=dtype, out=(pos_k, pos_v), k_scale=k_scale, v_scale=v_scale)
    assert a is pos_k and b is pos_v
    for have, x, f in ((a, kk, k_scale), (b, v[:T], v_scale)):
        want = values(*quantise(x, f), D)
        assert f != 1.0 or torch.equal(want.to(dtype).double().nan_to_num(nan=1e9), want.nan_to_num(nan=1e9))
        want = (want * f).to(dtype).double()
        assert torch.equal(have[:T].double().nan_to_num(nan=1e9), want.nan_to_num(nan=1e9)) and bool((have[T:] == 7).all())
    _no_error()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,hk,D", HEADS)
def test_heads_and_types(cuda_device, hq, hk, D, dtype):
    lens, new = [5, 33, 16, 100], [5, 1, 0, 40]
    _check_append(cuda_device, lens, new, hq, hk, D, 16, dtype, seed=D)
    _check_append(cuda_device, lens, new, hq, hk, D, 16, dtype, rope=torch.float32, seed=D + 1)


@pytest.mark.parametrize("page", [16, 32, 48, 128, 1024])
def test_page_sizes(cuda_device, page):
    _check_append(cuda_device, [page, page + 1, 2 * page - 1, 333, 7], [page, 1, 30, 333, 7], 8, 2, 64, page, torch.bfloat16, rope=torch.bfloat16, seed=page)


@pytest.mark.parametrize("rope", [torch.float32, torch.float16, torch.bfloat16])
def test_tables(cuda_device, rope):
    _check_append(cuda_device, [40, 300], [40, 9], 4, 4, 72, 16, torch.float16, rope=rope)


def test_strides(cuda_device):
    _check_append(cuda_device, [40, 300], [40, 9], 4, 2, 96, 32, torch.bfloat16, strided=True)


def test_many_tokens(cuda_device):
    """Several tokens to a block, more units than threads."""
    _check_append(cuda_device, [1500, 1, 900], [1500, 1, 800], 16, 8, 128, 32, torch.bfloat16, rope=torch.float32)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_values_at_the_edges(cuda_device, dtype):
    """Ties, zeros, the smallest and the largest, infinities and NaN: a block of 16 each."""
    def change(x):
        T, H, D = x.shape
        tie = torch.tensor([6, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, -0.25, -0.75, -1.25, -1.75, -2.5, -3.5, -5, -6], device=x.device)
        for i, s in enumerate([1.0, 1.125, 1.875, 0.25, 2.0 ** -9, 7 * 2.0 ** -9, 448.0, 2.0 ** -6]):
            x[i, :, :16] = (tie * s).to(x.dtype)
        x[8, :, :16] = 0.0
        x[9, :, :16] = -0.0
        x[10, :, :16] = 2.0 ** -13                                # scale rounds to zero
        x[11, :, :16] = 6 * 2.0 ** -10                            # a tie of the scale with zero
        x[12, :, :16] = torch.finfo(x.dtype).max
        x[13, :, 3] = float("inf")
        x[14, :, 5] = float("nan")
        x[15, :, 17] = float("-inf")
        x[16, :, :16] = torch.finfo(x.dtype).tiny
        x[17, :, :16] = torch.finfo(x.dtype).smallest_normal / 4
        x[18, :, 1:16] *= 1e-3
    _check_append(cuda_device, [40], [40], 2, 2, 64, 16, dtype, change=change)
    _check_append(cuda_device, [40], [40], 2, 2, 64, 16, dtype, change=change, k_scale=2.0 ** 5, v_scale=2.0 ** -8)
    _check_append(cuda_device, [40], [40], 2, 2, 72, 16, dtype, change=change, k_scale=2.0 ** 60, v_scale=2.0 ** -60)


def test_every_tie_and_its_neighbours(cuda_device):
    """For every E4M3 scale the 16-bit values at and beside the seven borders between codes."""
    from turbopi_b200 import ops
    from nvfp4_cache_reference import scale_values
    scales = scale_values(torch.arange(1, 127, device=cuda_device))
    borders = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], dtype=torch.float64, device=cuda_device)
    for dtype in (torch.bfloat16, torch.float16):
        tie = (scales[:, None] * borders).to(dtype)
        rows = [(tie.view(torch.int16) + i).view(dtype) for i in (-1, 0, 1)]             # positive: the next bit pattern is the next value
        x = torch.zeros(3, 126, 1, 16, dtype=dtype, device=cuda_device)
        for i, r in enumerate(rows):
            x[i, :, 0, :7], x[i, :, 0, 7:14], x[i, :, 0, 15] = r, -r, (6 * scales).to(dtype)
        x = x.flatten(0, 1)
        T = x.shape[0]
        pages = torch.zeros(2, 32, 1, 1, 288, dtype=torch.uint8, device=cuda_device)
        table = torch.arange(32, dtype=torch.int32, device=cuda_device)[None]
        ops.paged_append_nvfp4(x, x, pages[0], pages[1], table, _ints([0, T], cuda_device), _ints([T], cuda_device))
        code, byte = quantise(x)
        have_code, have_byte = (y.transpose(1, 2).flatten(0, 1)[:T] for y in unpack(pages[0], 16))
        assert torch.equal(have_byte, byte) and torch.equal(values(have_code, byte, 16), values(code, byte, 16))
        assert torch.equal(pages[0], pages[1])


@pytest.mark.parametrize("hq,hk,D", [(8, 1, 256), (4, 4, 64), (6, 2, 72), (32, 8, 128)])
@pytest.mark.parametrize("page", [1, 16, 24])
def test_read_of_16_bits(cuda_device, hq, hk, D, page):
    from turbopi_b200 import ops
    lens, take = [40, 0, 333, 1, 17], [40, 0, 100, 1, 3]
    for dtype in (torch.bfloat16, torch.float16):
        rows, pool = deal_pages(lens, page, 1)
        g = torch.Generator(device=cuda_device).manual_seed(D)
        pages = torch.randn((2, pool, page, hk, D), generator=g, device=cuda_device, dtype=dtype)
        T = sum(take)
        both = torch.full((T + 5, 2, hk, D), 5.0, dtype=dtype, device=cuda_device)
        k, v = ops.paged_read(pages[0], pages[1], _ints(rows, cuda_device), _ints(_offsets(take), cuda_device), _ints(lens, cuda_device), T + 5,
                              out=(both[:, 0], both[:, 1]))
        for have, side in ((k, pages[0]), (v, pages[1])):
            assert torch.equal(have[:T], _rows(side.transpose(1, 2), rows, lens, take, page)) and bool((have[T:] == 5).all())
        k2, v2 = ops.paged_read(pages[0], pages[1], _ints(rows, cuda_device), _ints(_offsets(take), cuda_device), _ints(lens, cuda_device), T)
        assert torch.equal(k2, k[:T]) and torch.equal(v2, v[:T]) and k2.is_contiguous()
    _no_error()


@pytest.mark.parametrize("bits", [4, 16])
def test_read_of_many_tokens(cuda_device, bits):
    from turbopi_b200 import ops
    lens, page, hk, D = [9000, 1, 3333], 32, 8, 128
    rows, pool = deal_pages(lens, page, 1)
    T, cu, lengths, table = sum(lens), _ints(_offsets(lens), cuda_device), _ints(lens, cuda_device), _ints(rows, cuda_device)
    if bits == 4:
        g = torch.Generator(device=cuda_device).manual_seed(1)
        x = torch.randn((2, pool, hk, page, D), generator=g, device=cuda_device, dtype=torch.bfloat16)
        pages = torch.stack([pack(*quantise(s)) for s in x])
        k, v = ops.paged_read_nvfp4(pages[0], pages[1], table, cu, lengths, D, T, dtype=torch.float16)
        full = [values(*unpack(s, D), D).transpose(1, 2) for s in pages]
    else:
        full = pages = torch.randn((2, pool, page, hk, D), device=cuda_device, dtype=torch.float16)
        k, v = ops.paged_read(pages[0], pages[1], table, cu, lengths, T)
    for have, side in ((k, full[0]), (v, full[1])):
        want = torch.cat([side[_ints(r[:-(-n // page)], cuda_device).long()].flatten(0, 1)[:n] for r, n in zip(rows, lens)])
        assert torch.equal(have.double(), want.double())
    _no_error()


@pytest.mark.parametrize("bits", [4, 16])
def test_rows_without_a_place(cuda_device, bits):
    """Lengths beyond the table, more rows than positions, absent pages: zeros, reported; an append writes nothing there."""
    from turbopi_b200 import _lib, ops
    lib = _lib.load()
    lengths, table = _ints([40, 100, 3], cuda_device), _ints([[0, -1, 2], [3, 4, 5], [6, 99, 0]], cuda_device)
    cu = _ints([0, 40, 60, 68], cuda_device)
    g = torch.Generator(device=cuda_device).manual_seed(1)
    code, byte = torch.randint(0, 16, (7, 1, 16, 64), generator=g, device=cuda_device), torch.randint(1, 100, (7, 1, 16, 4), generator=g, device=cuda_device)
    pages4 = pack(code, byte)
    full = values(code, byte, 64).transpose(1, 2)
    assert lib.tpb200_device_error(1) == 0
    if bits == 4:
        k, v = ops.paged_read_nvfp4(pages4, pages4, table, cu, lengths, 64, 68)
    else:
        p = full.to(torch.bfloat16)
        k, v = ops.paged_read(p, p, table, cu, lengths, 68)
    assert lib.tpb200_device_error(1) == 501
    want = torch.zeros(68, 1, 64, dtype=torch.float64, device=cuda_device)
    want[:16], want[32:40], want[65:68] = full[0], full[2, :8], full[6, :3]
    assert torch.equal(k.double(), want) and torch.equal(v.double(), want)
    # an append of the same tokens
    x = torch.randn((68, 1, 64), device=cuda_device, dtype=torch.bfloat16)
    a, b = pages4.clone(), pages4.clone()
    ops.paged_append_nvfp4(x, x, a, b, table, cu, lengths)
    assert lib.tpb200_device_error(1) == 501
    have = values(*unpack(a, 64), 64).transpose(1, 2)
    want = full.clone()
    for row, page, slot in [(i, 0, i) for i in range(16)] + [(32 + i, 2, i) for i in range(8)] + [(65 + i, 6, i) for i in range(3)]:
        want[page, slot] = values(*quantise(x[row]), 64)
    assert torch.equal(have, want) and torch.equal(a, b)


def test_offsets_that_follow_a_graph(cuda_device):
    """Captured once: tables, lengths and offsets are read when it is replayed; on a stream of its own."""
    from turbopi_b200 import ops
    x = torch.randn((8, 2, 128), device=cuda_device, dtype=torch.bfloat16)
    pages = torch.zeros((2, 6, 2, 1, 1152), dtype=torch.uint8, device=cuda_device)
    table, cu, lengths = _ints([[0, 1], [2, 3]], cuda_device), _ints([0, 4, 8], cuda_device), _ints([4, 4], cuda_device)
    out = torch.zeros(2, 8, 2, 128, dtype=torch.bfloat16, device=cuda_device)
    stream = torch.cuda.Stream(cuda_device)
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()

    def step():
        ops.paged_append_nvfp4(x, -x, pages[0], pages[1], table, cu, lengths)
        ops.paged_read_nvfp4(pages[0], pages[1], table, cu, lengths, 128, 8, out=(out[0], out[1]))
    with torch.cuda.stream(stream):
        step()
        with torch.cuda.graph(graph, stream=stream):
            step()
    torch.cuda.current_stream().wait_stream(stream)
    for lens, offsets in (([20, 4], [0, 7, 8]), ([8, 32], [0, 0, 8])):
        lengths.copy_(_ints(lens, cuda_device))
        cu.copy_(_ints(offsets, cuda_device))
        x.normal_()
        graph.replay()
        want = values(*quantise(x), 128)
        assert torch.equal(out[0].double(), want) and torch.equal(out[1].double(), -want)
    _no_error()

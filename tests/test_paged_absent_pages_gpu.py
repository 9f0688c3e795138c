"""Pages that the table does not have: their keys are left out of the attention, as if the sequence had only the others."""
import pytest
import torch

from paged_reference import attend, check, deal_pages

pytestmark = pytest.mark.gpu


def _problem(lens, hq, hk, D, page, dtype, device, seed=0):
    g = torch.Generator(device=device).manual_seed(seed)
    rows, pool = deal_pages(lens, page, seed)
    k, v = torch.randn((2, pool, page, hk, D), generator=g, device=device, dtype=dtype)
    q = torch.randn((len(lens), hq, D), generator=g, device=device, dtype=dtype)
    return q, k, v, rows, torch.tensor(lens, dtype=torch.int32, device=device)


def _there(pages, row, n):
    """The rows of positions [0, n) whose page is in the pool."""
    P, page = pages.shape[:2]
    at = [(i, r) for j in range(n) for i, r in [(row[j // page], j % page)] if 0 <= i < P]
    ids, slots = (torch.tensor([x[side] for x in at], dtype=torch.long, device=pages.device) for side in (0, 1))
    return pages[ids, slots]


def _check(out, q, k, v, rows, lens, scale):
    for i, n in enumerate(lens):
        want, allow = attend(q[i:i + 1], _there(k, rows[i], n), _there(v, rows[i], n), scale)
        check(out[i:i + 1], want, allow)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,hk,D,page", [(8, 1, 256, 16), (8, 2, 128, 16), (4, 4, 64, 16), (4, 1, 64, 64), (8, 2, 128, 24), (6, 2, 72, 5),
                                          (16, 1, 64, 1), (2, 2, 200, 100), (24, 1, 128, 48), (32, 2, 64, 7)])
def test_keys_of_absent_pages_are_left_out(cuda_device, hq, hk, D, page, dtype):
    """The first page, the last, one in the middle, runs of them, every second one, all of them."""
    from turbopi_b200 import _lib, ops
    lib = _lib.load()
    lens = [100, 333, 700, 60, 2000, 15, 130]
    q, k, v, rows, lengths = _problem(lens, hq, hk, D, page, dtype, cuda_device, seed=D + page)
    assert lib.tpb200_device_error(1) == 0
    bad = [-1, k.shape[0], 2 ** 30, -2 ** 31]
    need = [-(-n // page) for n in lens]
    gone = [[0], [need[1] - 1], [need[2] // 2], range(need[3]), range(0, need[4], 2), range(need[5]), range(need[6] // 3, need[6] // 2 + 1)]
    for s, which in enumerate(gone):
        for x, j in enumerate(which):
            rows[s][j] = bad[(s + x) % len(bad)]
    table = torch.tensor(rows, dtype=torch.int32, device=cuda_device)
    out = ops.paged_attention(q, k, v, table, lengths, D ** -0.5)
    _check(out, q, k, v, rows, lens, D ** -0.5)
    assert bool((out[3] == 0).all()) and bool((out[5] == 0).all())
    assert lib.tpb200_device_error(1) == 501


@pytest.mark.parametrize("length", [20000, 50001])
def test_one_sequence_over_many_parts(cuda_device, length):
    """Parts of which some have no key at all, joined with those that have."""
    from turbopi_b200 import _lib, ops
    q, k, v, rows, lengths = _problem([length], 8, 1, 256, 16, torch.bfloat16, cuda_device, seed=3)
    v += 1                                                       # a mean that does not go out among many keys
    for first, last in ((0, 400), (700, 1000), (len(rows[0]) - 90, len(rows[0]))):
        rows[0][first:last] = [-1] * (last - first)
    table = torch.tensor(rows, dtype=torch.int32, device=cuda_device)
    _check(ops.paged_attention(q, k, v, table, lengths, 1 / 16), q, k, v, rows, [length], 1 / 16)
    table.fill_(-1)
    assert bool((ops.paged_attention(q, k, v, table, lengths, 1 / 16) == 0).all())
    assert _lib.load().tpb200_device_error(1) == 501


@pytest.mark.parametrize("page", [16, 24])
def test_a_length_beyond_the_pages_a_sequence_has(cuda_device, page):
    """The table is -1 behind a sequence's pages: a length that reaches there, or beyond the table, adds no keys."""
    from turbopi_b200 import _lib, ops
    lens = [4 * page, 9 * page, 2 * page]
    q, k, v, rows, _ = _problem(lens, 8, 2, 128, page, torch.float16, cuda_device, seed=4)
    table = torch.tensor(rows, dtype=torch.int32, device=cuda_device)
    longer = torch.tensor([7 * page + 3, 40 * page, 2 * page + 1], dtype=torch.int32, device=cuda_device)
    _check(ops.paged_attention(q, k, v, table, longer, 0.1), q, k, v, rows, lens, 0.1)
    assert _lib.load().tpb200_device_error(1) == 501


@pytest.mark.parametrize("D", [64, 128, 256])
def test_keys_that_are_there_with_scores_of_minus_infinity(cuda_device, D):
    """Not the same as no keys: the mean of nothing but weights of zero is no number, beside absent pages too; a single finite score
    takes all the weight."""
    from turbopi_b200 import _lib, ops
    lens = [40, 40, 200, 3000]
    q, k, v, rows, lengths = _problem(lens, 4, 1, D, 16, torch.bfloat16, cuda_device, seed=5)
    q.abs_().clamp_(min=0.5)
    k.fill_(float("-inf"))
    rows[1][1] = -1
    k[rows[2][7], 3] = 1.0
    table = torch.tensor(rows, dtype=torch.int32, device=cuda_device)
    out = ops.paged_attention(q, k, v, table, lengths, 0.1)
    assert bool(out[[0, 1, 3]].isnan().all())
    assert torch.equal(out[2], v[rows[2][7], 3].expand(4, D))
    assert _lib.load().tpb200_device_error(1) == 501

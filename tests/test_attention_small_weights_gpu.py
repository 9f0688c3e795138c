"""fp16: the weights of many far keys beside one near key keep their sum, and weights above the reference stay finite."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

SCORE = -16.21875                        # exact in fp16; a weight of 2^-23.4


def _keys(n, near, D, device):
    """One key of score 0 and value 0 at position `near`, n - 1 keys of score SCORE and value 1."""
    k = torch.zeros((n, 1, D), dtype=torch.float16, device=device)
    v = torch.ones((n, 1, D), dtype=torch.float16, device=device)
    k[:, 0, 0] = SCORE
    k[near], v[near] = 0, 0
    return k, v


def _allowed(n):
    """(the mean, how far it may be off).  Weights are rounded to fp16 with at least seven bits above the reference's one, in steps of 2^-24:
    by 2^-25 of 2^7 w each; n of them are summed in fp32, above and below the line; the output is rounded once."""
    w = math.exp(SCORE)
    want = (n - 1) * w / (1 + (n - 1) * w)
    return want, want * (2.0 ** -32 / w + 2 * n * 2.0 ** -23 + 2.0 ** -11) * 1.01


@pytest.mark.parametrize("near", [0, 7777, 16383])
@pytest.mark.parametrize("D,page", [(64, 16), (128, 16), (256, 16), (64, 24)])
def test_single_tokens(cuda_device, D, page, near):
    """Enough sequences (on the same pages) that one warp has many of the near key's neighbours."""
    from turbopi_b200 import ops
    n, seqs = 16384, 600
    k, v = _keys(n, near, D, cuda_device)
    pages = -(-n // page)
    pool = torch.zeros((2, pages * page, 1, D), dtype=torch.float16, device=cuda_device)
    pool[0, :n], pool[1, :n] = k, v
    pool = pool.view(2, pages, page, 1, D)
    q = torch.zeros((seqs, 4, D), dtype=torch.float16, device=cuda_device)
    q[..., 0] = 1
    out = ops.paged_attention(q, pool[0], pool[1], torch.arange(pages, dtype=torch.int32, device=cuda_device).expand(seqs, pages),
                              torch.full((seqs,), n, dtype=torch.int32, device=cuda_device), 1.0)
    want, allow = _allowed(n)
    assert float((out.double() - want).abs().max()) <= allow


@pytest.mark.parametrize("near", [0, 2222, 8191])
@pytest.mark.parametrize("D,others", [(64, 0), (64, 40), (128, 0), (128, 60), (256, 0)])
def test_packed_queries(cuda_device, D, others, near):
    """`others` empty sequences: the mean length falls under the border between the two forms."""
    from turbopi_b200 import ops
    n = 8192
    k, v = _keys(n, near, D, cuda_device)
    q = torch.zeros((3, 2, D), dtype=torch.float16, device=cuda_device)
    q[..., 0] = 1
    cu = torch.tensor([0, 3] + [3] * others, dtype=torch.int32, device=cuda_device)
    cu_keys = torch.tensor([0, n] + [n] * others, dtype=torch.int32, device=cuda_device)
    out = ops.packed_attention(q, k, v, cu, 1.0, causal=False, cu_keys=cu_keys)
    want, allow = _allowed(n)
    assert float((out.double() - want).abs().max()) <= allow


def test_weights_above_the_reference(cuda_device):
    """Later scores up to eight bits above the reference do not raise it; their weights and sums stay finite."""
    from turbopi_b200 import ops
    for D in (64, 128, 256):
        n = 1500
        k, v = _keys(n, 0, D, cuda_device)
        k[:600], v[:600] = 0, 0
        k[600:, 0, 0] = 5.5390625                                # 7.991 bits
        v[600:] = 2
        q = torch.zeros((1, 2, D), dtype=torch.float16, device=cuda_device)
        q[..., 0] = 1
        ends = torch.tensor([0, n], dtype=torch.int32, device=cuda_device)
        packed = ops.packed_attention(q, k, v, torch.tensor([0, 1], dtype=torch.int32, device=cuda_device), 1.0, causal=False, cu_keys=ends)
        paged = ops.paged_attention(q, k.view(15, 100, 1, D), v.view(15, 100, 1, D), torch.arange(15, dtype=torch.int32, device=cuda_device)[None],
                                    ends[1:], 1.0)
        far = 900 * math.exp(5.5390625)
        want = 2 * far / (600 + far)
        for out in (packed, paged):      # weights and output rounded by half a step, sums in fp32
            assert float((out.double() - want).abs().max()) <= want * (3 * 2.0 ** -11 + 2 * n * 2.0 ** -23) * 1.01

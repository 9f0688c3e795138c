"""Sequences as long as positions of 32 bits allow, on pages that a table names again and again."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("page,width", [(8176, 262657), (49981, 42966)])      # 2^31 - 16 positions, 2^31 - 2
@pytest.mark.parametrize("D", [8, 72, 136])
def test_the_longest_sequences(cuda_device, page, width, D):
    """All keys score 0 and all values are 1, but for the last row of the last page: with it the output is its value (e^40 against 2^31),
    without it the mean of ones, exactly (counts stay below 2^24 until parts are joined, and then go the same way in both sums)."""
    from turbopi_b200 import _lib, ops
    k = torch.zeros((2, page, 1, D), dtype=torch.bfloat16, device=cuda_device)
    v = torch.ones_like(k)
    k[1, page - 1, 0, 0], v[1, page - 1] = 40, 3
    q = torch.zeros((1, 1, D), dtype=torch.bfloat16, device=cuda_device)
    q[..., 0] = 1
    table = torch.zeros((1, width), dtype=torch.int32, device=cuda_device)
    table[:, width - 1] = 1
    most = page * width
    out = ops.paged_attention(q, k, v, table, torch.tensor([most], dtype=torch.int32, device=cuda_device), 1.0)
    assert bool((out == 3).all())
    out = ops.paged_attention(q, k, v, table, torch.tensor([most - 1], dtype=torch.int32, device=cuda_device), 1.0)
    assert bool((out == 1).all())
    # beyond the table: as long as the table
    if most < 2 ** 31 - 2:
        out = ops.paged_attention(q, k, v, table, torch.tensor([2 ** 31 - 1], dtype=torch.int32, device=cuda_device), 1.0)
        assert bool((out == 3).all()) and _lib.load().tpb200_device_error(1) == 501
    assert _lib.load().tpb200_device_error(1) == 0

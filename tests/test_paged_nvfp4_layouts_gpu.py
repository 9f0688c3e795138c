"""4-bit pools of keys and values that lie among one another: a call on them gives what it gives on pools of their own."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("between", ["pages", "heads", "tiles", "rows"])
@pytest.mark.parametrize("D", [72, 128])
def test_values_among_the_keys(cuda_device, between, D):
    from turbopi_b200 import _lib, ops
    P, H, tiles = 7, 2, 2
    size = ops.nvfp4_page_shape(H, 16 * tiles, D)
    g = torch.Generator(device=cuda_device).manual_seed(0)
    table = torch.tensor([[5, 1, 3], [0, 6, -1]], dtype=torch.int32, device=cuda_device)
    lengths, cu = (torch.tensor(x, dtype=torch.int32, device=cuda_device) for x in ([70, 33], [0, 65, 98]))
    k, v = torch.randn((2, 98, H, D), generator=g, device=cuda_device, dtype=torch.bfloat16)
    q = torch.randn((2, 8, D), generator=g, device=cuda_device, dtype=torch.bfloat16)
    own = torch.zeros((2, P, *size), dtype=torch.uint8, device=cuda_device)
    at = {"pages": 1, "heads": 2, "tiles": 3, "rows": 0}[between]
    whole = torch.zeros((*own.shape[1:at + 1], 2, *own.shape[at + 1:]), dtype=torch.uint8, device=cuda_device)
    among = [whole.select(at, i) for i in range(2)]
    got = []
    for pages in (own, among):
        ops.paged_append_nvfp4(k, v, pages[0], pages[1], table, cu, lengths)
        got.append((*ops.paged_read_nvfp4(pages[0], pages[1], table, cu, lengths, D, 98), ops.paged_attention_nvfp4(q, pages[0], pages[1], table, lengths, 0.1)))
    assert all(torch.equal(a, b) for a, b in zip(*got))
    assert torch.equal(torch.stack(among), own)
    assert _lib.load().tpb200_device_error(0) == 0

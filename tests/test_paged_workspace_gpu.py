"""ops.paged_attention refuses a workspace whose bytes do not lie one behind the other: both forms of the call."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("native", [True, False])
def test_refused(cuda_device, monkeypatch, native):
    from turbopi_b200 import _lib, ops
    from turbopi_b200._lib import TurboPiError
    _lib.native()
    if not native:
        monkeypatch.setattr(_lib, "_native", _lib._PythonForms())
    pages = torch.randn(4, 16, 2, 64, device=cuda_device).to(torch.bfloat16)
    q = torch.randn(1, 8, 64, device=cuda_device).to(torch.bfloat16)
    table, lengths = torch.arange(4, dtype=torch.int32, device=cuda_device)[None], torch.tensor([50], dtype=torch.int32, device=cuda_device)
    ws = ops.paged_attention_workspace(8, 2, 64, cuda_device)
    n = ws.numel()
    want = ops.paged_attention(q, pages, pages, table, lengths, 0.1)
    for bad in (ws[:1].expand(n), ws.new_zeros(2 * n)[::2], ws.new_zeros(n, 2)[:, 0]):
        with pytest.raises(TurboPiError, match="contiguous"):
            ops.paged_attention(q, pages, pages, table, lengths, 0.1, workspace=bad)
    for fine in (ws, ws.new_zeros(n + 512)[256:], ws.new_zeros((n + 3) // 4 * 4).view(torch.float32), ws.new_zeros(2, n)):
        assert torch.equal(ops.paged_attention(q, pages, pages, table, lengths, 0.1, workspace=fine), want)

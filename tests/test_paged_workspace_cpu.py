"""A workspace whose bytes do not lie one behind the other is refused before anything is launched: the Python form, on tensors that claim to
be on a GPU."""
import pytest
import torch

from turbopi_b200 import _lib, ops
from turbopi_b200._lib import TurboPiError


@pytest.mark.parametrize("workspace,fine", [(torch.zeros(1, dtype=torch.uint8).expand(1 << 30), False), (torch.zeros(64, dtype=torch.uint8)[::2], False),
                                            (torch.zeros(64, dtype=torch.uint8), True), (torch.zeros(4, 4), True)])
def test_workspaces(monkeypatch, workspace, fine):
    launched = []
    monkeypatch.setattr(_lib, "_native", _lib._PythonForms())
    monkeypatch.setattr(ops, "_cuda", lambda *tensors: None)
    monkeypatch.setattr(ops, "_run", lambda t, f, args: launched.append(args.workspace_bytes) or 0)
    pages = torch.zeros(4, 16, 2, 64, dtype=torch.bfloat16)
    call = lambda: ops.paged_attention(torch.zeros(1, 8, 64, dtype=torch.bfloat16), pages, pages, torch.zeros(1, 4, dtype=torch.int32),   # noqa: E731
                                       torch.zeros(1, dtype=torch.int32), 0.1, workspace=workspace)
    if fine:
        call()
        assert launched == [64]
    else:
        with pytest.raises(TurboPiError, match="contiguous"):
            call()
        assert not launched

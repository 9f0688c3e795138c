"""ops.paged_append of no tokens at all."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("native", [True, False])
def test_no_tokens(cuda_device, monkeypatch, native):
    """A batch without new tokens, in both forms of the call; with rotation, queries of no tokens come back."""
    from turbopi_b200 import _lib, ops
    from turbopi_b200.paged_cache import PagedCache
    _lib.native()
    if not native:
        monkeypatch.setattr(_lib, "_native", _lib._PythonForms())
    cache = PagedCache(1, 4, 16, 2, 64, 2, device=cuda_device)
    a, b = cache.add(), cache.add()
    batch = cache.batch([a, b])
    before = cache.pages.clone()
    k = torch.empty((0, 2, 64), dtype=torch.bfloat16, device=cuda_device)
    q = torch.empty((0, 8, 64), dtype=torch.bfloat16, device=cuda_device)
    cos = torch.ones((32, 32), device=cuda_device)
    assert cache.append(0, batch, k, k) is None
    out = cache.append(0, batch, k, k, q=q, cos=cos, sin=cos)
    assert out.shape == q.shape
    assert cache.append(0, batch, k, k, q=q, cos=cos, sin=cos, q_out=q) is q
    empty = cache.extend([], [])
    assert cache.append(0, empty, k, k) is None
    assert torch.equal(cache.pages, before) and _lib.load().tpb200_device_error(0) == 0

"""ops.paged_append of no tokens at all, and of as many as 32 bits count."""
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


def test_as_many_tokens_as_32_bits_count(cuda_device):
    """2^31 - 1 tokens (34 GB, keys and values the same ones), of which the last three have a place."""
    from turbopi_b200 import _lib, ops
    n = 2 ** 31 - 1
    kv = torch.empty((n, 1, 8), dtype=torch.bfloat16, device=cuda_device)
    kv[-4:] = torch.arange(32, device=cuda_device, dtype=torch.bfloat16).view(4, 1, 8)
    pages = torch.zeros((2, 2, 16, 1, 8), dtype=torch.bfloat16, device=cuda_device)
    want = pages.clone()
    want[:, 1, 14:, 0], want[:, 0, 0, 0] = kv[-3:-1, 0], kv[-1, 0]
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda_device)      # noqa: E731
    ops.paged_append(kv, kv, pages[0], pages[1], ints([[1, 0]]), ints([n - 3, n]), ints([17]))
    assert torch.equal(pages, want) and _lib.load().tpb200_device_error(0) == 0

"""What ops.copy_pages makes of a pool's shape, with the launch stood in for: the Python form."""
import pytest
import torch

from turbopi_b200 import _lib, ops


@pytest.mark.parametrize("stride", [0, 8, 12345])
def test_a_pool_of_one_page(monkeypatch, stride):
    """The stride of a dimension of one page says nothing about its bytes."""
    calls = []
    monkeypatch.setattr(_lib, "_native", _lib._PythonForms())
    monkeypatch.setattr(ops, "_cuda", lambda *tensors: None)
    monkeypatch.setattr(ops, "_run", lambda t, f, base, slab, slabs, page, *rest: calls.append((slab, slabs, page, rest[0])) or 0)
    for lead in ((), (3, 2)):
        shape = (*lead, 1, 4, 1, 64)
        pages = torch.ones(shape, dtype=torch.bfloat16)
        strides = list(pages.stride())
        strides[-4] = stride
        pages = pages.as_strided(shape, strides)
        assert pages.is_contiguous()
        ops.copy_pages(pages, [0], [0])
    assert calls == [(512, 1, 512, 1), (512, 6, 512, 1)]

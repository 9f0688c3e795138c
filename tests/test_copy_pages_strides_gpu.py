"""ops.copy_pages on pools of one page, whose stride may be anything: both forms of the call."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("stride", [0, 8, 12345])
def test_a_pool_of_one_page(cuda_device, monkeypatch, native, stride):
    """Nothing can be moved in it: no pairs are fine, a pair is refused (the page would be read and written)."""
    from turbopi_b200 import _lib, ops
    from turbopi_b200._lib import TurboPiError
    _lib.native()
    if not native:
        monkeypatch.setattr(_lib, "_native", _lib._PythonForms())
    pages = torch.ones((1, 4, 1, 64), dtype=torch.bfloat16, device=cuda_device).as_strided((1, 4, 1, 64), (stride, 64, 64, 1))
    assert pages.is_contiguous()
    ops.copy_pages(pages, [], [])
    with pytest.raises(TurboPiError, match="supported range"):
        ops.copy_pages(pages, [0], [0])
    assert bool((pages == 1).all())


@pytest.mark.parametrize("native", [True, False])
def test_layers_of_one_page(cuda_device, monkeypatch, native):
    from turbopi_b200 import _lib, ops
    from turbopi_b200._lib import TurboPiError
    _lib.native()
    if not native:
        monkeypatch.setattr(_lib, "_native", _lib._PythonForms())
    pages = torch.ones((3, 2, 1, 4, 1, 64), dtype=torch.bfloat16, device=cuda_device).as_strided((3, 2, 1, 4, 1, 64), (512, 256, 8, 64, 64, 1))
    assert pages.is_contiguous()
    ops.copy_pages(pages, [], [])
    with pytest.raises(TurboPiError, match="supported range"):
        ops.copy_pages(pages, [0], [0])

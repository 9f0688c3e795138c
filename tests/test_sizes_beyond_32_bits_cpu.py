"""Sizes that do not fit the 32 bits of the C structures are refused by the Python forms, not cut: expanded tensors, nothing launched."""
import pytest
import torch

from turbopi_b200 import _lib, ops
from turbopi_b200._lib import TurboPiError

LARGE = 2 ** 32 + 4                      # would be cut to 4


@pytest.fixture
def launched(monkeypatch):
    calls = []
    monkeypatch.setattr(_lib, "_native", _lib._PythonForms())
    monkeypatch.setattr(ops, "_cuda", lambda *tensors: None)
    monkeypatch.setattr(ops, "_run", lambda *args: calls.append(args) or 0)
    return calls


def _rows(tokens, heads=1):
    return torch.zeros(1, 1, 8, dtype=torch.bfloat16).expand(tokens, heads, 8)


def _ints(n):
    return torch.zeros(n, dtype=torch.int32)


def _cache(pages=2, page=16, heads=1):
    return (torch.zeros(1, 1, 1, 8, dtype=torch.bfloat16).expand(pages, page, heads, 8),) * 2


def test_what_fits_is_launched(launched):
    ops.packed_attention(_rows(4), _rows(4), _rows(4), _ints(2), 1.0)
    ops.paged_append(_rows(4), _rows(4), *_cache(), _ints(6).view(2, 3), _ints(3), _ints(2))
    ops.copy_pages(torch.zeros(2, 4, 1, 8, dtype=torch.bfloat16), [0], [1])
    assert len(launched) == 3


def test_packed_attention(launched):
    for q, k in ((LARGE, 4), (4, LARGE)):
        with pytest.raises(TurboPiError, match="32 bits"):
            ops.packed_attention(_rows(q), _rows(k), _rows(k), _ints(2), 1.0, cu_keys=_ints(2))
    with pytest.raises(TurboPiError, match="32 bits"):
        ops.packed_attention(_rows(4, LARGE), _rows(4), _rows(4), _ints(2), 1.0)
    assert not launched


def test_append(launched):
    with pytest.raises(TurboPiError, match="32 bits"):
        ops.paged_append(_rows(LARGE), _rows(LARGE), *_cache(), _ints(6).view(2, 3), _ints(3), _ints(2))
    assert not launched


@pytest.mark.parametrize("sizes", [dict(pages=LARGE), dict(page=LARGE), dict(heads=LARGE)])
def test_pages(launched, sizes):
    pages, heads = _cache(**sizes), sizes.get("heads", 1)
    with pytest.raises(TurboPiError, match="32 bits"):
        ops.paged_append(_rows(4, heads), _rows(4, heads), *pages, _ints(6).view(2, 3), _ints(3), _ints(2))
    with pytest.raises(TurboPiError, match="32 bits"):
        ops.paged_attention(_rows(2, heads), *pages, _ints(6).view(2, 3), _ints(2), 1.0, out=_rows(2, heads), workspace=_ints(4))
    assert not launched

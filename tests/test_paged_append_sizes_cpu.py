"""Appends without tokens, whose tensors have no memory behind them, are done at once: through the C entry, which follows no pointer here."""
import ctypes

import pytest

from turbopi_b200 import _lib

NULL = -1
Two = ctypes.c_longlong * 2


def _append(tokens, seqs=2, **kw):
    there = 64 if seqs else 0
    cache = _lib.PagedCacheView(k_pages=1024, v_pages=1 << 20, page_stride=128, row_stride=8, head_stride=8, num_pages=8, page_size=16, kv_heads=1,
                                head_dim=8, dtype=_lib.BF16, table=there, table_stride=4, table_width=4, lengths=there, seqs=seqs)
    base = dict(cache=cache, k_stride=Two(8, 8), v_stride=Two(8, 8), cu=64, tokens=tokens)
    return _lib.load().tpb200_paged_append(_lib.PagedAppendArgs(**{**base, **kw}), None)


@pytest.mark.parametrize("seqs", [0, 2])
def test_no_tokens(seqs):
    assert _append(0, seqs) == 0
    assert _append(0, seqs, cos=64, sin=64, rope_positions=4, rope_dtype=_lib.F32, q_heads=3) == 0
    assert _append(3) == NULL

"""Numbers of tokens near 2^31, which round up past 32 bits, are refused before anything else is looked at; pointers are never followed."""
import ctypes

import pytest

from turbopi_b200 import _lib

SHAPE, ALIGN = -2, -3
Two = ctypes.c_longlong * 2
MOST = 2 ** 31 - 1024


def _packed(**kw):
    """With queries that are not aligned, which is what a call of a number of tokens that fits is refused for."""
    base = dict(q=8, k=1 << 44, v=1 << 45, out=1 << 40, q_stride=Two(16, 8), k_stride=Two(16, 8), v_stride=Two(16, 8), o_stride=Two(16, 8), cu=64,
                seqs=1, q_tokens=9, k_tokens=9, q_heads=2, kv_heads=2, head_dim=8, dtype=_lib.BF16, scale=1.0, causal=1)
    return _lib.load().tpb200_packed_attention(_lib.PackedAttentionArgs(**{**base, **kw}), None)


@pytest.mark.parametrize("tokens", [MOST + 1, 2 ** 31 - 128, 2 ** 31 - 1])
def test_packed_attention(tokens):
    assert _packed() == ALIGN and _packed(q_tokens=MOST, k_tokens=MOST) == ALIGN
    assert _packed(q_tokens=tokens) == SHAPE
    assert _packed(k_tokens=tokens) == SHAPE

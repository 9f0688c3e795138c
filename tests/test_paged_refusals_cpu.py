"""What the calls on a paged cache refuse, before anything is launched: the C entry points with pointers they never follow, and
the Python calls on tensors that claim to be on a GPU."""
import ctypes

import pytest
import torch

from turbopi_b200 import _lib, ops
from turbopi_b200._lib import TurboPiError

NULL, SHAPE, ALIGN, ENUM, WORKSPACE = -1, -2, -3, -4, -6
Two = ctypes.c_longlong * 2


def _cache(**kw):
    base = dict(k_pages=1024, v_pages=4096, page_stride=16 * 256, row_stride=256, head_stride=256, num_pages=8, page_size=16, kv_heads=1,
                head_dim=256, dtype=_lib.BF16, table=64, table_stride=4, table_width=4, lengths=64, seqs=2)
    return _lib.PagedCacheView(**{**base, **kw})


BAD_CACHE = [(dict(k_pages=0), NULL), (dict(v_pages=0), NULL), (dict(table=0), NULL), (dict(lengths=0), NULL), (dict(k_pages=8), ALIGN),
             (dict(page_stride=4097), ALIGN), (dict(row_stride=4), ALIGN), (dict(head_stride=-8), SHAPE), (dict(num_pages=0), SHAPE),
             (dict(page_size=0), SHAPE), (dict(head_dim=12), SHAPE), (dict(head_dim=264), SHAPE), (dict(head_dim=0), SHAPE),
             (dict(dtype=_lib.F32), ENUM), (dict(table_width=0), SHAPE), (dict(seqs=-1), SHAPE),
             (dict(page_size=1 << 16, table_width=1 << 15), SHAPE)]


@pytest.mark.parametrize("change,status", BAD_CACHE)
def test_views_of_a_cache(change, status):
    lib = _lib.load()
    attention = _lib.PagedAttentionArgs(cache=_cache(**change), q=64, out=64, q_stride=Two(2048, 256), o_stride=Two(2048, 256), q_heads=8,
                                        scale=1.0, workspace=256, workspace_bytes=1 << 30)
    append = _lib.PagedAppendArgs(cache=_cache(**change), k=64, v=64, k_stride=Two(256, 256), v_stride=Two(256, 256), cu=64, tokens=3)
    assert lib.tpb200_paged_attention(attention, None) == status
    assert lib.tpb200_paged_append(append, None) == status


@pytest.mark.parametrize("change,status", [(dict(q=0), NULL), (dict(out=0), NULL), (dict(q=8), ALIGN), (dict(q_stride=Two(2044, 256)), ALIGN),
                                           (dict(q_heads=0), SHAPE), (dict(flags=4), ENUM)])
def test_attention_arguments(change, status):
    base = dict(cache=_cache(), q=64, out=64, q_stride=Two(2048, 256), o_stride=Two(2048, 256), q_heads=8, scale=1.0, workspace=256,
                workspace_bytes=1 << 30)
    assert _lib.load().tpb200_paged_attention(_lib.PagedAttentionArgs(**{**base, **change}), None) == status


def test_attention_heads_must_divide():
    args = _lib.PagedAttentionArgs(cache=_cache(kv_heads=3), q=64, out=64, q_heads=8, scale=1.0)
    assert _lib.load().tpb200_paged_attention(args, None) == SHAPE


@pytest.mark.parametrize("change,status", [(dict(k=0), NULL), (dict(cu=0), NULL), (dict(v=4), ALIGN), (dict(tokens=-1), SHAPE),
                                           (dict(cos=64), NULL), (dict(cos=64, sin=64), SHAPE), (dict(cos=64, sin=8, rope_positions=4), ALIGN),
                                           (dict(cos=64, sin=64, rope_positions=4, rope_dtype=9), ENUM),
                                           (dict(q=64, q_out=64, q_heads=8), SHAPE),
                                           (dict(q=64, q_heads=8, cos=64, sin=64, rope_positions=4), NULL),
                                           (dict(k_stride=Two(4, 256)), ALIGN), (dict(flags=2), ENUM)])
def test_append_arguments(change, status):
    base = dict(cache=_cache(), k=64, v=64, k_stride=Two(256, 256), v_stride=Two(256, 256), cu=64, tokens=3)
    assert _lib.load().tpb200_paged_append(_lib.PagedAppendArgs(**{**base, **change}), None) == status


def _copy(src, dst, pages=1024, slab=8 * 4096, slabs=4, page=4096, count=8, flags=0):
    a, b = ((ctypes.c_int * len(x))(*x) for x in (src, dst))
    return _lib.load().tpb200_copy_pages(pages, slab, slabs, page, count, a, b, len(src), flags, None)


@pytest.mark.parametrize("src,dst", [([0], [8]), ([8], [0]), ([-1], [0]), ([0], [-1]), ([0, 1], [2, 2]), ([0, 1], [1, 2]), ([3], [3]),
                                     ([0, 1, 2], [5, 6, 0])])
def test_copies_that_would_depend_on_their_order(src, dst):
    assert _copy(src, dst) == SHAPE


def test_copy_arguments():
    assert _copy([0], [1], pages=0) == NULL
    assert _copy([0], [1], pages=1028) == ALIGN
    assert _copy([0], [1], page=4100) == ALIGN
    assert _copy([0], [1], slab=4096) == SHAPE
    assert _copy([0], [1], slabs=0) == SHAPE
    assert _copy([0], [1], flags=8) == ENUM
    assert _copy([], []) == 0


def test_cpu_tensors_are_refused():
    k = torch.zeros(2, 16, 1, 64, dtype=torch.bfloat16)
    table, lengths = torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(TurboPiError, match="CUDA"):
        ops.paged_attention(torch.zeros(1, 1, 64, dtype=torch.bfloat16), k, k, table, lengths, 1.0)
    with pytest.raises(TurboPiError, match="CUDA"):
        ops.paged_append(k[:, 0], k[:, 0], k, k, table, lengths, lengths)
    with pytest.raises(TurboPiError, match="CUDA"):
        ops.copy_pages(k, [0], [1])


@pytest.mark.parametrize("change,status", [(dict(q=0), NULL), (dict(v=0), NULL), (dict(cu=0), NULL), (dict(out=0), NULL), (dict(k=8), ALIGN),
                                           (dict(q_stride=Two(1020, 256)), ALIGN), (dict(k_stride=Two(0, 256)), SHAPE),
                                           (dict(head_dim=260), SHAPE), (dict(head_dim=4), SHAPE), (dict(q_heads=3), SHAPE),
                                           (dict(kv_heads=0), SHAPE), (dict(dtype=_lib.F32), ENUM), (dict(flags=2), ENUM),
                                           (dict(seqs=-1), SHAPE)])
def test_packed_attention_arguments(change, status):
    base = dict(q=64, k=64, v=64, out=64, q_stride=Two(1024, 256), k_stride=Two(512, 256), v_stride=Two(512, 256), o_stride=Two(1024, 256),
                cu=64, seqs=1, q_tokens=9, k_tokens=9, q_heads=4, kv_heads=2, head_dim=256, dtype=_lib.BF16, scale=1.0, causal=1)
    assert _lib.load().tpb200_packed_attention(_lib.PackedAttentionArgs(**{**base, **change}), None) == status


def test_packed_attention_refuses_cpu_tensors():
    q = torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(TurboPiError, match="CUDA"):
        ops.packed_attention(q, q, q, torch.zeros(2, dtype=torch.int32), 1.0)


@pytest.mark.parametrize("scale", [float("nan"), float("inf"), float("-inf")])
def test_scales_that_are_no_numbers(scale):
    lib = _lib.load()
    packed = _lib.PackedAttentionArgs(q=64, k=64, v=64, out=64, q_stride=Two(1024, 256), k_stride=Two(512, 256), v_stride=Two(512, 256),
                                      o_stride=Two(1024, 256), cu=64, seqs=1, q_tokens=9, k_tokens=9, q_heads=4, kv_heads=2, head_dim=256,
                                      dtype=_lib.BF16, scale=scale, causal=1)
    paged = _lib.PagedAttentionArgs(cache=_cache(), q=64, out=64, q_stride=Two(2048, 256), o_stride=Two(2048, 256), q_heads=8, scale=scale,
                                    workspace=256, workspace_bytes=1 << 30)
    assert lib.tpb200_packed_attention(packed, None) == SHAPE and lib.tpb200_paged_attention(paged, None) == SHAPE


def test_outputs_whose_rows_overlap():
    """An expanded output would be written by several heads or sequences at once."""
    lib = _lib.load()
    base = dict(cache=_cache(), q=64, out=64, q_stride=Two(2048, 256), o_stride=Two(2048, 256), q_heads=8, scale=1.0, workspace=256,
                workspace_bytes=1 << 30)
    for o_stride in (Two(0, 256), Two(2048, 0), Two(2048, 128)):
        assert lib.tpb200_paged_attention(_lib.PagedAttentionArgs(**{**base, "o_stride": o_stride}), None) == SHAPE


def test_capacities_whose_plan_would_not_fit():
    """The plan counts in 32 bits, for sequences as long as the table; with larger slots (smaller heads) more of them fit."""
    lib = _lib.load()
    wide = dict(page_size=1024, table_width=1024, table_stride=1024, seqs=40000)
    args = dict(q=64, out=64, q_stride=Two(2048, 256), o_stride=Two(2048, 256), q_heads=8, scale=1.0, workspace=256, workspace_bytes=1 << 30)
    assert lib.tpb200_paged_attention(_lib.PagedAttentionArgs(cache=_cache(page_stride=1024 * 256, **wide), **args), None) == SHAPE


def test_structures_follow_the_header_field_by_field():
    import re
    from pathlib import Path
    header = (Path(__file__).resolve().parent.parent / "include" / "turbopi_b200.h").read_text()
    for name, mirror in {"tpb200_paged_cache": _lib.PagedCacheView, "tpb200_paged_attention_args": _lib.PagedAttentionArgs,
                         "tpb200_paged_append_args": _lib.PagedAppendArgs, "tpb200_packed_attention_args": _lib.PackedAttentionArgs}.items():
        body = re.sub(r"/\*.*?\*/", "", re.search(r"typedef struct\s*\{([^}]*)\}\s*" + name + r"\s*;", header, re.S).group(1), flags=re.S)
        fields = [part.strip().split()[-1].split("[")[0].lstrip("*") for d in body.split(";") if d.strip() for part in d.split(",")]
        assert fields == [f[0] for f in mirror._fields_], name


def _elements(at, stride, tokens, heads, D):
    return [{at // 2 + t * stride[0] + h * stride[1] + d for d in range(D)} for t in range(tokens) for h in range(heads)]


def test_outputs_in_part_where_inputs_lie():
    """Random views around one place, against sets of their elements: an output on its input row on row is fine, one that shares only some of
    its elements, or its own rows, is refused; views with different token strides are refused where their ranges meet."""
    import random
    rng, lib, seen = random.Random(3), _lib.load(), {True: 0, False: 0}
    for _ in range(1500):
        D, tokens, heads = rng.choice([8, 16, 24]), rng.randint(1, 4), rng.randint(1, 4)

        def view():
            return rng.choice([1024, 1024 + 16 * rng.randint(-12, 12)]), (rng.choice([D * heads, D * heads * 2, D + 8 * rng.randint(0, 12)]),
                                                                         rng.choice([D, D, D + 8, 2 * D, D + 8 * rng.randint(0, 12)]))
        q, q_stride = view()
        out, o_stride = (q, q_stride) if rng.random() < 0.2 else view()
        if rng.random() < 0.6:
            o_stride = (q_stride[0], o_stride[1])
        rows, written = _elements(q, q_stride, tokens, heads, D), _elements(out, o_stride, tokens, heads, D)
        a, b = set().union(*rows), set().union(*written)
        ranges = min(a) <= max(b) and min(b) <= max(a)
        crossed = len(b) < len(written) * D
        bad = crossed or (rows != written and (bool(a & b) or (tokens > 1 and q_stride[0] != o_stride[0] and ranges)))
        args = _lib.PagedAttentionArgs(cache=_cache(head_dim=D, seqs=tokens, page_stride=16 * 256), q=q, out=out, q_stride=Two(*q_stride),
                                       o_stride=Two(*o_stride), q_heads=heads, scale=1.0)
        assert (lib.tpb200_paged_attention(args, None) == SHAPE) == bad, (D, tokens, heads, q, q_stride, out, o_stride)
        seen[bad] += 1
    assert min(seen.values()) > 300


@pytest.mark.parametrize("change", [dict(out=64 + 512), dict(k=1 << 20), dict(v=1 << 20), dict(v=(1 << 20) + 1024 * 2 * 9 - 16)])
def test_packed_outputs_where_others_read(change):
    base = dict(q=64, k=1 << 21, v=1 << 22, out=1 << 20, q_stride=Two(1024, 256), k_stride=Two(512, 256), v_stride=Two(512, 256),
                o_stride=Two(1024, 256), cu=64, seqs=1, q_tokens=9, k_tokens=9, q_heads=4, kv_heads=2, head_dim=256, dtype=_lib.BF16, scale=1.0)
    assert _lib.load().tpb200_packed_attention(_lib.PackedAttentionArgs(**{**base, **change}), None) == SHAPE


@pytest.mark.parametrize("change", [dict(q_out=64 + 512), dict(q_out=(1 << 20) - 512), dict(q_out=1 << 21), dict(o_stride=Two(512, 256)),
                                    dict(cache=_cache(v_pages=1024)),
                                    dict(q=64, q_out=64, q_heads=9, k=64 + 8 * 512, q_stride=Two(2560, 256), o_stride=Two(2560, 256),
                                         k_stride=Two(2560, 256), v=64 + 9 * 512, v_stride=Two(2560, 256))])
def test_appends_that_write_where_others_read(change):
    """The last one: queries and keys of a fused projection turned in place together, while the keys are read for their pages."""
    base = dict(cache=_cache(), k=1 << 20, v=1 << 21, k_stride=Two(256, 256), v_stride=Two(256, 256), cu=64, tokens=3, q=64, q_out=1 << 22, q_heads=8,
                q_stride=Two(2048, 256), o_stride=Two(2048, 256), cos=64, sin=64, rope_positions=4, rope_dtype=_lib.F32)
    assert _lib.load().tpb200_paged_append(_lib.PagedAppendArgs(**{**base, **change}), None) == SHAPE


def test_scales_too_large_for_the_exponent():
    base = dict(cache=_cache(), q=64, out=64, q_stride=Two(2048, 256), o_stride=Two(2048, 256), q_heads=8, scale=3e38, workspace=256, workspace_bytes=1 << 30)
    assert _lib.load().tpb200_paged_attention(_lib.PagedAttentionArgs(**base), None) == SHAPE

"""What the calls on a 4-bit paged cache, and those with a window, refuse before anything is launched: the C entry points with pointers
they never follow, and the Python calls on tensors that claim to be on a GPU."""
import ctypes
import math
import re
from pathlib import Path

import pytest
import torch

from turbopi_b200 import _lib, ops
from turbopi_b200._lib import TurboPiError
from turbopi_b200.paged_cache import PagedCache

NULL, SHAPE, ALIGN, ENUM, WORKSPACE = -1, -2, -3, -4, -6
Two = ctypes.c_longlong * 2
TILE = 288 * 8                                   # heads of 256


def _cache(**kw):
    base = dict(k_pages=1024, v_pages=1 << 20, page_stride=TILE, head_stride=TILE, tile_stride=TILE, num_pages=8, page_size=16, kv_heads=1,
                head_dim=256, k_scale=1.0, v_scale=0.5, table=64, table_stride=4, table_width=4, lengths=64, seqs=2)
    return _lib.PagedNvfp4CacheView(**{**base, **kw})


def _attention(cache=None, **kw):
    base = dict(cache=cache or _cache(), q=64, out=64, dtype=_lib.BF16, q_stride=Two(2048, 256), o_stride=Two(2048, 256), q_heads=8, scale=1.0,
                workspace=256, workspace_bytes=1 << 30)
    return _lib.load().tpb200_paged_attention_nvfp4(_lib.PagedAttentionNvfp4Args(**{**base, **kw}), None)


def _append(cache=None, **kw):
    base = dict(cache=cache or _cache(), k=64, v=64, dtype=_lib.BF16, k_stride=Two(256, 256), v_stride=Two(256, 256), cu=64, tokens=3)
    return _lib.load().tpb200_paged_append_nvfp4(_lib.PagedAppendNvfp4Args(**{**base, **kw}), None)


def _read(cache=None, **kw):
    base = dict(k=1 << 30, v=1 << 31, dtype=_lib.BF16, k_stride=Two(256, 256), v_stride=Two(256, 256), cu=64, tokens=3)
    return _lib.load().tpb200_paged_read_nvfp4(cache or _cache(), _lib.PagedRows(**{**base, **kw}), None)


BAD_CACHE = [(dict(k_pages=0), NULL), (dict(v_pages=0), NULL), (dict(table=0), NULL), (dict(lengths=0), NULL), (dict(k_pages=8), ALIGN),
             (dict(page_stride=TILE + 8), ALIGN), (dict(page_stride=TILE - 16), SHAPE), (dict(kv_heads=2, q=8, head_stride=24), ALIGN),
             (dict(kv_heads=2, head_stride=16), SHAPE), (dict(page_size=32, tile_stride=288), SHAPE), (dict(page_size=32, tile_stride=-16), SHAPE),
             (dict(num_pages=0), SHAPE), (dict(page_size=0), SHAPE), (dict(page_size=24), SHAPE), (dict(head_dim=12), SHAPE), (dict(head_dim=264), SHAPE),
             (dict(head_dim=0), SHAPE), (dict(table_width=0), SHAPE), (dict(seqs=-1), SHAPE), (dict(page_size=1 << 16, table_width=1 << 15), SHAPE),
             (dict(k_scale=0.0), SHAPE), (dict(k_scale=3.0), SHAPE), (dict(v_scale=-1.0), SHAPE), (dict(v_scale=math.inf), SHAPE),
             (dict(k_scale=math.nan), SHAPE), (dict(v_scale=2.0 ** 65), SHAPE), (dict(k_scale=2.0 ** -64), SHAPE)]


@pytest.mark.parametrize("change,status", BAD_CACHE)
def test_views_of_a_cache(change, status):
    change = {k: v for k, v in change.items() if k != "q"}
    assert _attention(_cache(**change)) == status
    assert _append(_cache(**change)) == status
    assert _read(_cache(**change)) == status


@pytest.mark.parametrize("change,status", [(dict(q=0), NULL), (dict(out=0), NULL), (dict(q=8), ALIGN), (dict(q_stride=Two(2044, 256)), ALIGN),
                                           (dict(q_heads=0), SHAPE), (dict(flags=4), ENUM), (dict(dtype=_lib.F32), ENUM), (dict(scale=math.inf), SHAPE),
                                           (dict(window=-1), SHAPE), (dict(sinks=1), SHAPE), (dict(window=4, sinks=-1), SHAPE),
                                           (dict(o_stride=Two(256, 256)), SHAPE)])
def test_attention_arguments(change, status):
    assert _attention(**change) == status


def test_attention_heads_must_divide():
    assert _attention(_cache(kv_heads=3, head_stride=TILE)) == SHAPE


@pytest.mark.parametrize("change,status", [(dict(k=0), NULL), (dict(cu=0), NULL), (dict(v=4), ALIGN), (dict(tokens=-1), SHAPE), (dict(dtype=0), ENUM),
                                           (dict(cos=64), NULL), (dict(cos=64, sin=64), SHAPE), (dict(cos=64, sin=8, rope_positions=4), ALIGN),
                                           (dict(cos=64, sin=64, rope_positions=4, rope_dtype=9), ENUM),
                                           (dict(q=64, q_out=64, q_heads=8), SHAPE),
                                           (dict(q=64, q_heads=8, cos=64, sin=64, rope_positions=4), NULL),
                                           (dict(k_stride=Two(4, 256)), ALIGN), (dict(flags=2), ENUM)])
def test_append_arguments(change, status):
    assert _append(**change) == status


def test_append_needs_two_pools():
    assert _append(_cache(v_pages=1024)) == SHAPE


@pytest.mark.parametrize("change,status", [(dict(k=0), NULL), (dict(cu=0), NULL), (dict(v=8), ALIGN), (dict(tokens=-1), SHAPE), (dict(dtype=0), ENUM),
                                           (dict(flags=8), ENUM), (dict(k_stride=Two(4, 256)), ALIGN), (dict(k_stride=Two(128, 256)), SHAPE),
                                           (dict(v=(1 << 30) + 512), SHAPE), (dict(k=1024), SHAPE), (dict(v=(1 << 20) + 7 * TILE), SHAPE),
                                           (dict(k=1024 - 16), SHAPE)])
def test_read_arguments(change, status):
    """Also rows that share memory with one another or with the pages."""
    assert _read(**change) == status


def test_read_of_16_bits():
    def read(cache=None, **kw):
        view = _lib.PagedCacheView(**{**dict(k_pages=1024, v_pages=1 << 20, page_stride=16 * 256, row_stride=256, head_stride=256, num_pages=8,
                                             page_size=16, kv_heads=1, head_dim=256, dtype=_lib.BF16, table=64, table_stride=4, table_width=4,
                                             lengths=64, seqs=2), **(cache or {})})
        base = dict(k=1 << 30, v=1 << 31, dtype=_lib.BF16, k_stride=Two(256, 256), v_stride=Two(256, 256), cu=64, tokens=3)
        return _lib.load().tpb200_paged_read(view, _lib.PagedRows(**{**base, **kw}), None)
    assert read(dtype=_lib.F16) == ENUM
    assert read(cache=dict(page_size=0)) == SHAPE
    assert read(cache=dict(k_pages=0)) == NULL
    assert read(k=1024 + 8 * 16 * 512 - 16) == SHAPE
    assert read(tokens=0, k=0, v=0, cu=0) == 0 and read(cache=dict(seqs=0, table=0, lengths=0)) == 0


def test_nothing_to_do_is_no_error():
    none = _cache(seqs=0, table=0, lengths=0)
    assert _attention(none) == 0 and _append(none) == 0 and _read(none) == 0
    assert _append(tokens=0, k=0, v=0, cu=0) == 0 and _read(tokens=0, k=0, v=0, cu=0) == 0
    assert _lib.load().tpb200_paged_attention_nvfp4(None, None) == NULL and _lib.load().tpb200_paged_append_nvfp4(None, None) == NULL
    assert _lib.load().tpb200_paged_read_nvfp4(None, None, None) == NULL


def test_windows():
    lib = _lib.load()
    view = _lib.PagedCacheView(k_pages=1024, v_pages=4096, page_stride=16 * 256, row_stride=256, head_stride=256, num_pages=8, page_size=16,
                               kv_heads=1, head_dim=256, dtype=_lib.BF16, table=64, table_stride=4, table_width=4, lengths=64, seqs=0)
    paged = _lib.PagedAttentionArgs(cache=view, q=64, out=64, q_stride=Two(2048, 256), o_stride=Two(2048, 256), q_heads=8, scale=1.0,
                                    workspace=256, workspace_bytes=1 << 30)
    packed = _lib.PackedAttentionArgs(q=64, k=64, v=64, out=64, cu=64, seqs=0, q_tokens=1, k_tokens=1, q_heads=1, kv_heads=1, head_dim=64,
                                      dtype=_lib.BF16, scale=1.0, causal=1)
    for window, sinks, status in ((0, 0, SHAPE), (-1, 0, SHAPE), (1, -1, SHAPE), (1, 0, 0), (2 ** 31 - 1, 2 ** 31 - 1, 0)):
        assert lib.tpb200_paged_attention_window(paged, window, sinks, None) == status
        assert lib.tpb200_packed_attention_window(packed, window, sinks, None) == status
    packed.causal = 0
    assert lib.tpb200_packed_attention_window(packed, 4, 0, None) == SHAPE
    assert lib.tpb200_packed_attention_window(None, 4, 0, None) == NULL and lib.tpb200_paged_attention_window(None, 4, 0, None) == NULL


@pytest.mark.parametrize("window,sinks", [(0, 0), (-3, 0), (4, -1), (None, 2), (1.5, 0), ("8", 0), (8, 0.5), (8, None)])
def test_windows_in_python(window, sinks, monkeypatch):
    monkeypatch.setattr(_lib, "_native", _lib._PythonForms())
    x = torch.zeros(1, 1, 64, dtype=torch.bfloat16)
    i = torch.zeros(2, dtype=torch.int32)
    for call in (lambda **kw: ops.packed_attention(x, x, x, i, 1.0, **kw), lambda **kw: ops.paged_attention(x, x[None], x[None], i[None], i[:1], 1.0, **kw),
                 lambda **kw: ops.paged_attention_nvfp4(x, x[None], x[None], i[None], i[:1], 1.0, **kw)):
        with pytest.raises(TurboPiError, match="window"):
            call(window=window, sinks=sinks)


def test_a_window_goes_with_causal_attention(monkeypatch):
    monkeypatch.setattr(_lib, "_native", _lib._PythonForms())
    x = torch.zeros(1, 1, 64, dtype=torch.bfloat16)
    with pytest.raises(TurboPiError, match="causal"):
        ops.packed_attention(x, x, x, torch.zeros(2, dtype=torch.int32), 1.0, causal=False, window=4)


class _Claims(torch.Tensor):
    """A CPU tensor that says it is on a GPU: the checks are reached, and nothing is launched on what they refuse."""
    is_cuda = True


def _claims(t):
    return t.as_subclass(_Claims)


def _good():
    k = _claims(torch.zeros(5, 2, 64, dtype=torch.bfloat16))
    pages = [_claims(torch.zeros(4, 2, 1, 576, dtype=torch.uint8)) for _ in range(2)]
    table, lengths, cu = (_claims(torch.zeros(s, dtype=torch.int32)) for s in ((1, 4), (1,), (2,)))
    return dict(k=k, v=k, pages=pages, table=table, lengths=lengths, cu=cu)


def test_python_refusals(monkeypatch):
    monkeypatch.setattr(_lib, "_native", _lib._PythonForms())
    monkeypatch.setattr(ops, "_run", lambda *a: pytest.fail("launched"))
    g = _good()

    def append(**kw):
        a = {**g, **kw}
        ops.paged_append_nvfp4(a["k"], a["v"], *a["pages"], a["table"], a["cu"], a["lengths"], **{n: kw[n] for n in ("q", "cos", "sin", "q_out") if n in kw})

    def read(head_dim=64, tokens=5, dtype=torch.bfloat16, out=None, **kw):
        a = {**g, **kw}
        ops.paged_read_nvfp4(*a["pages"], a["table"], a["cu"], a["lengths"], head_dim, tokens, dtype=dtype, out=out)

    def attention(q=None, **kw):
        a = {**g, **kw}
        q = _claims(torch.zeros(1, 4, 64, dtype=torch.bfloat16)) if q is None else q
        ops.paged_attention_nvfp4(q, *a["pages"], a["table"], a["lengths"], 1.0, workspace=kw.get("workspace"), out=kw.get("out"))
    wrong = [[_claims(torch.zeros(4, 2, 1, 576, dtype=torch.int8)) for _ in range(2)], [_claims(torch.zeros(4, 2, 1, 575, dtype=torch.uint8)) for _ in range(2)],
             [g["pages"][0], _claims(torch.zeros(3, 2, 1, 576, dtype=torch.uint8))], [_claims(torch.zeros(4, 2, 576, dtype=torch.uint8)) for _ in range(2)],
             [_claims(torch.zeros(4, 2, 576, 1, dtype=torch.uint8).transpose(2, 3)) for _ in range(2)][:1] * 2]
    for pages in wrong[:4]:
        for call in (append, read, attention):
            with pytest.raises(TurboPiError):
                call(pages=pages)
    f32 = _claims(torch.zeros(5, 2, 64))
    for kw in (dict(k=f32), dict(v=f32), dict(k=g["k"][0]), dict(v=g["k"][:4]), dict(cu=g["cu"][:1]), dict(cu=g["cu"].long()), dict(lengths=g["lengths"].long()),
               dict(q=g["k"]), dict(cos=f32[0], sin=None), dict(q_out=g["k"]), dict(q=g["k"], cos=f32[:, 0], sin=f32[:, 0]), dict(k=g["k"][..., :32])):
        with pytest.raises(TurboPiError):
            append(**kw)
    for kw in (dict(head_dim=60), dict(head_dim=96), dict(tokens=-1), dict(tokens=1.5), dict(dtype=torch.float32), dict(out=(g["k"],)),
               dict(out=(g["k"], g["k"][:2])), dict(out=(f32, f32)), dict(out=7 * (g["k"],)), dict(out=(None, g["k"])), dict(out=5), dict(head_dim=64.0), dict(cu=g["cu"][:1]), dict(tokens=2 ** 31)):
        with pytest.raises(TurboPiError):
            read(**kw)
    for kw in (dict(q=f32), dict(q=g["k"][:1, 0]), dict(q=_claims(torch.zeros(1, 3, 64, dtype=torch.bfloat16))), dict(q=_claims(torch.zeros(2, 4, 64, dtype=torch.bfloat16))),
               dict(out=f32), dict(workspace=_claims(torch.zeros(64, 64, dtype=torch.uint8).t()[::2]))):
        with pytest.raises(TurboPiError):
            attention(**kw)
    with pytest.raises(TurboPiError, match="CUDA"):
        ops.paged_append_nvfp4(torch.zeros(1, 1, 64, dtype=torch.bfloat16), *(torch.zeros(1, 1, 64, dtype=torch.bfloat16),), *g["pages"], g["table"], g["cu"], g["lengths"])
    with pytest.raises(TurboPiError, match="CUDA"):
        ops.paged_read(torch.zeros(1, 16, 1, 64, dtype=torch.bfloat16), torch.zeros(1, 16, 1, 64, dtype=torch.bfloat16), g["table"], g["cu"], g["lengths"], 1)


@pytest.mark.parametrize("args", [(0, 16, 64), (1, 24, 64), (1, 0, 64), (1, 16, 12), (1, 16, 264)])
def test_shapes_of_pages(args):
    with pytest.raises(TurboPiError):
        ops.nvfp4_page_shape(*args)
    assert ops.nvfp4_page_shape(4, 48, 72) == (4, 3, 864)


def test_caches():
    for kw in (dict(page_size=24), dict(k_scale=3.0), dict(v_scale=0.0), dict(v_scale=2.0 ** 80), dict(k_scale="x"), dict(dtype="int4"),
               dict(dtype=torch.bfloat16, k_scale=2.0)):
        with pytest.raises(TurboPiError):
            PagedCache(**{**dict(layers=1, num_pages=4, page_size=16, kv_heads=1, head_dim=64, max_pages=4, dtype="nvfp4", device="cpu"), **kw})
    cache = PagedCache(2, 4, 32, 3, 72, 4, dtype="nvfp4", device="cpu")
    assert cache.pages.shape == (2, 2, 4, 3, 2, 864) and cache.pages.dtype == torch.uint8
    s = cache.add()
    batch = cache.extend([s], [5])
    with pytest.raises(TurboPiError, match="rows"):
        cache.append(0, batch, torch.zeros(4, 3, 72), torch.zeros(4, 3, 72))
    with pytest.raises(TurboPiError, match="heads of 72"):
        cache.append(0, batch, torch.zeros(5, 3, 96, dtype=torch.bfloat16), torch.zeros(5, 3, 96, dtype=torch.bfloat16))
    with pytest.raises(TurboPiError, match="heads of 72"):
        cache.attention(0, batch, torch.zeros(1, 3, 96, dtype=torch.bfloat16), 1.0)
    with pytest.raises(TurboPiError, match="rows"):
        cache.prompt_attention(0, batch, torch.zeros(4, 3, 72, dtype=torch.bfloat16), 1.0)
    cache.truncate(s, 2)
    for call in (lambda: cache.read(0, batch), lambda: cache.attention(0, batch, torch.zeros(1, 3, 72), 1.0),
                 lambda: cache.prompt_attention(0, batch, torch.zeros(5, 3, 72, dtype=torch.bfloat16), 1.0)):
        with pytest.raises(TurboPiError, match="truncated"):
            call()


def test_offsets_of_all_tokens():
    cache = PagedCache(1, 20, 16, 1, 64, 8, device="cpu")
    a, b = cache.add(), cache.add()
    cache.extend([a, b], [20, 3])
    batch = cache.extend([b, a], [1, 2])
    assert batch.cu.tolist() == [0, 1, 3] and batch.cu_keys.tolist() == [0, 4, 26] and batch.keys == 26 and batch.tokens == 3
    again = cache.extend([b, a], [0, 5], out=batch)
    assert again is batch and batch.cu_keys.tolist() == [0, 4, 31] and batch.keys == 31 and batch.lengths.tolist() == [4, 27]


CSRC = Path(__file__).resolve().parent.parent / "turbopi_b200" / "csrc"


@pytest.mark.parametrize("source,kernels", [("paged_nvfp4.cu", 3), ("paged_attention_nvfp4.cu", 2), ("paged_attention.cu", 2)])
def test_the_wait_comes_first(source, kernels):
    """They let the next launch in behind their own wait."""
    text = re.sub(r"//[^\n]*", "", (CSRC / source).read_text())
    bodies = re.findall(r"__global__[^{;]*\{\n(.*?)^\}", text, re.S | re.M)
    assert len(bodies) == kernels
    for body in bodies:
        assert body.index("pdl_wait_prior_grids()") < body.index("pdl_launch_dependents()")
        assert not re.search(r"P\.(cu|cache\.\w+|joins|part_\w+|q|k|v)\b[\[.]", body[:body.index("pdl_wait_prior_grids()")])

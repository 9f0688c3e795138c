"""Memory that one thread of a call on 4-bit pages would write and another read or write: refused before anything is launched, by C entry points
that never follow these pointers."""
import ctypes
import random

import pytest
import torch

from turbopi_b200 import _lib

SHAPE = -2
Two = ctypes.c_longlong * 2
TILE = 288 * 8                                   # heads of 256
POOL = 8 * TILE
K, V = 1 << 24, 1 << 25


def _cache(**kw):
    base = dict(k_pages=K, v_pages=V, page_stride=TILE, head_stride=TILE, tile_stride=TILE, num_pages=8, page_size=16, kv_heads=1,
                head_dim=256, k_scale=1.0, v_scale=1.0, table=64, table_stride=4, table_width=4, lengths=64, seqs=2)
    return _lib.PagedNvfp4CacheView(**{**base, **kw})


def _append(cache=None, **kw):
    base = dict(cache=cache or _cache(), k=1 << 26, v=1 << 27, dtype=_lib.BF16, k_stride=Two(256, 256), v_stride=Two(256, 256), cu=64, tokens=3)
    return _lib.load().tpb200_paged_append_nvfp4(_lib.PagedAppendNvfp4Args(**{**base, **kw}), None)


@pytest.mark.parametrize("pool", [K, V])
@pytest.mark.parametrize("at", [0, 16, POOL - 16, -3 * 512 + 16])
def test_new_rows_in_the_pages(pool, at):
    assert _append(k=pool + at) == SHAPE
    assert _append(v=pool + at) == SHAPE


@pytest.mark.parametrize("pool", [K, V])
@pytest.mark.parametrize("at", [0, POOL - 16, -3 * 4096 + 16])
def test_turned_queries_in_the_pages(pool, at):
    rope = dict(cos=1 << 28, sin=1 << 29, rope_positions=64, q_heads=8, o_stride=Two(2048, 256), q_stride=Two(2048, 256))
    assert _append(q=1 << 30, q_out=pool + at, **rope) == SHAPE
    assert _append(q=pool + at, q_out=1 << 30, **rope) == SHAPE
    assert _append(q=pool + at, q_out=pool + at, **rope) == SHAPE


@pytest.mark.parametrize("change", [dict(v_pages=K + TILE), dict(v_pages=K + 16), dict(v_pages=K + POOL - 16), dict(v_pages=K - POOL + 16),
                                    dict(v_pages=K + TILE, page_stride=2 * TILE + 16, kv_heads=2),
                                    dict(v_pages=K + 3 * TILE - 16, page_stride=4 * TILE, kv_heads=2, head_stride=TILE),
                                    # heads in front of pages
                                    dict(v_pages=K + 8 * TILE, page_stride=TILE, kv_heads=2, head_stride=8 * TILE),
                                    dict(v_pages=K + 4 * TILE, page_stride=2 * TILE, page_size=32, kv_heads=2, head_stride=32 * TILE)])
def test_pools_that_share_bytes(change):
    assert _append(_cache(**change)) == SHAPE


@pytest.mark.parametrize("change", [dict(kv_heads=2), dict(page_size=32, kv_heads=2, page_stride=4 * TILE), dict(page_size=32),
                                    dict(kv_heads=3, head_stride=2 * TILE, page_stride=4 * TILE)])
def test_a_pool_whose_tiles_share_bytes(change):
    assert _append(_cache(**change)) == SHAPE


@pytest.mark.parametrize("pool", [K, V])
@pytest.mark.parametrize("at", [0, POOL - 16, -2 * 4096 + 16])
def test_outputs_of_attention_in_the_pages(pool, at):
    args = _lib.PagedAttentionNvfp4Args(cache=_cache(), q=1 << 26, out=pool + at, dtype=_lib.BF16, q_stride=Two(2048, 256), o_stride=Two(2048, 256),
                                        q_heads=8, scale=1.0, workspace=1 << 27, workspace_bytes=1 << 40)
    assert _lib.load().tpb200_paged_attention_nvfp4(args, None) == SHAPE


@pytest.mark.skipif(torch.cuda.is_available(), reason="what is not refused would be launched")
@pytest.mark.parametrize("seed", range(4))
def test_random_layouts(seed):
    """Every layout whose tiles do share bytes is refused, and no layout of a tensor whose tiles do not is."""
    rng = random.Random(seed)
    small = dict(head_dim=32, table_width=1)
    tile, met, apart = 288, 0, 0
    for _ in range(400):
        pages, heads, tiles = rng.randint(1, 4), rng.randint(1, 3), rng.randint(1, 3)
        order = [("page", pages), ("head", heads), ("tile", tiles)]
        rng.shuffle(order)
        # a tensor: dimensions one around the other, the values' own among them at times, rows cut off
        between, stride, strides, step = rng.randrange(4), tile + rng.choice([0, 16, 32]), {}, None
        for i, (name, n) in enumerate(order):
            if i == between:
                step, stride = stride, 2 * stride
            strides[name] = stride
            stride *= n + rng.choice([0, 0, 1])
        values = K + (step or rng.choice([stride, stride + 16]))
        plain = rng.random() < 0.4
        if not plain:                            # moved out of place
            values += 16 * rng.randint(-stride // 16, stride // 16)
            if rng.random() < 0.3:
                strides[rng.choice(list(strides))] = tile + 16 * rng.randint(0, stride // 16)
        places = [i * strides["page"] + j * strides["head"] + x * strides["tile"] for i in range(pages) for j in range(heads) for x in range(tiles)]
        every = sorted([K + p for p in places] + [values + p for p in places])
        meet = any(b - a < tile for a, b in zip(every, every[1:]))
        status = _append(_cache(v_pages=values, page_stride=strides["page"], head_stride=strides["head"], tile_stride=strides["tile"], num_pages=pages,
                                kv_heads=heads, page_size=16 * tiles, **small), k_stride=Two(96, 32), v_stride=Two(96, 32))
        if meet:
            assert status == SHAPE
            met += 1
        elif plain:
            assert status != SHAPE
            apart += 1
    assert met > 50 and apart > 50

"""The work whose speed the 4-bit paged cache and the attention with a sliding window are judged by, as calls of their public entry
points.

`listed()` names the cases, `draw(rng)` gives further ones of the same ranges, `prepare` is what a program holds before a
call, `run` one call: in elementary torch operations, or with `own` through the package.  `exact` restates each case in 64 bits.

Kinds of case:
  append  ops.paged_append_nvfp4: new tokens' keys and values quantised into their pages, queries and keys rotated, and
          ops.paged_read_nvfp4 of these tokens: what the cache now holds of them, as the prompt's attention reads it
  read    ops.paged_read_nvfp4: whole sequences out of a 4-bit cache, packed for a prompt's attention
  decode  ops.paged_attention_nvfp4, or ops.paged_attention on 16-bit pages: one new token per sequence, over all keys or over the
          last `window` and the first `sinks`
  prompt  ops.packed_attention with a window: prompts one behind the other

A 4-bit page is [heads][page / 16] tiles of 16 tokens.  With G = ceil(D / 32), a tile is 16 rows of 16 G bytes, value 2 i in the low and
2 i + 1 in the high half of byte i (E2M1), then 16 rows of 2 G scales (E4M3), one for every 16 values: the values are code * scale.
"""
import math
import random

import torch

own = False
DEV = "cuda"
THETA = 10000.0


def listed():
    return [
        # a decode step's write on Gemma's head shape: one token for each of 64 requests, all latency
        dict(name="append_step", kind="append", seqs=64, longest=1, shortest=1, before=3000, q_heads=8, kv_heads=1, dim=256, page=16,
             dtype="bf16", rope=True, lens_seed=1),
        # the prompts of a batch written at once
        dict(name="append_prompts", kind="append", seqs=6, longest=4000, shortest=300, before=200, q_heads=32, kv_heads=8, dim=128,
             page=32, dtype="bf16", rope=True, lens_seed=2),
        # the cache of one Pi0.5 request with its action rows, read back
        dict(name="read_one", kind="read", seqs=1, longest=762, shortest=762, kv_heads=1, dim=256, page=16, dtype="bf16", lens_seed=3),
        # conversations that go on: their caches read back for the attention of the next prompts
        dict(name="read_ragged", kind="read", seqs=12, longest=9000, shortest=100, kv_heads=8, dim=128, page=32, dtype="fp16",
             lens_seed=4),
        # one token of one request on the cache of a Pi0.5 prompt with its 50 action rows: the smallest call
        dict(name="decode4_one", kind="decode", bits=4, seqs=1, longest=762, shortest=762, q_heads=8, kv_heads=1, dim=256, page=16,
             dtype="bf16", window=0, sinks=0, lens_seed=5),
        # a serving batch, requests at every stage, four query heads to a key head
        dict(name="decode4_ragged", kind="decode", bits=4, seqs=96, longest=8192, shortest=1, q_heads=32, kv_heads=8, dim=128,
             page=16, dtype="bf16", window=0, sinks=0, lens_seed=6),
        # a few very long conversations: the cache's length is all there is to split
        dict(name="decode4_long", kind="decode", bits=4, seqs=5, longest=131071, shortest=60000, q_heads=8, kv_heads=1, dim=256,
             page=64, dtype="fp16", window=0, sinks=0, lens_seed=7),
        # long conversations under a window, small heads, as many key heads as query heads
        dict(name="decode4_window", kind="decode", bits=4, seqs=64, longest=12000, shortest=500, q_heads=16, kv_heads=16, dim=64,
             page=32, dtype="bf16", window=2048, sinks=4, lens_seed=8),
        # the same question on 16-bit pages, whose size is no multiple of 16
        dict(name="decode_window", kind="decode", bits=16, seqs=64, longest=12000, shortest=500, q_heads=32, kv_heads=8, dim=128,
             page=24, dtype="bf16", window=1024, sinks=4, lens_seed=9),
        # one long document at Gemma's head shape
        dict(name="prompt_window", kind="prompt", seqs=1, longest=8191, shortest=8191, q_heads=8, kv_heads=1, dim=256, dtype="bf16",
             window=1024, sinks=4, cached=0, lens_seed=10),
        # short prompts of every length, small heads, a window as long as a tile or two
        dict(name="prompt_window_ragged", kind="prompt", seqs=24, longest=1200, shortest=1, q_heads=16, kv_heads=4, dim=64,
             dtype="fp16", window=200, sinks=16, cached=0, lens_seed=11),
        # the largest batch: queries behind keys that are already there
        dict(name="prompt_window_batch", kind="prompt", seqs=4, longest=4000, shortest=1500, q_heads=32, kv_heads=8, dim=128,
             dtype="bf16", window=1500, sinks=64, cached=500, lens_seed=12),
    ]


def _log_int(rng, lo, hi):
    return int(min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


# (query heads, key heads, head size): Gemma's, and the usual ones; a group of three, sizes that are no power of two
_HEADS = [(8, 1, 256), (8, 1, 256), (32, 8, 128), (16, 4, 64), (16, 16, 64), (8, 2, 128), (12, 4, 128), (4, 4, 256), (16, 16, 72),
          (16, 2, 96)]


def draw(rng):
    kind = rng.choice(["append", "append", "read", "decode", "decode", "decode", "prompt", "prompt"])
    hq, hk, d = rng.choice(_HEADS)
    base = dict(kind=kind, q_heads=hq, kv_heads=hk, dim=d, dtype=rng.choice(["bf16", "fp16"]), lens_seed=rng.randint(0, 10 ** 6))
    page4 = rng.choice([16, 16, 32, 48, 64, 128])
    if kind == "append":
        longest = _log_int(rng, 1, 4000)
        return dict(base, seqs=_log_int(rng, 1, max(1, min(128, 12000 // longest))), longest=longest,
                    shortest=rng.choice([1, longest]), before=rng.randint(0, 3000), page=page4, rope=rng.random() < 0.7)
    if kind == "read":
        del base["q_heads"]
        longest = _log_int(rng, 16, 30000)
        most = max(1, min(64, int(4e7 / (longest * hk * d))))
        return dict(base, seqs=_log_int(rng, 1, most), longest=longest, shortest=rng.choice([1, longest // 2 + 1, longest]),
                    page=page4)
    if kind == "decode":
        bits = rng.choice([4, 4, 16])
        longest = _log_int(rng, 16, 131072)
        window = rng.choice([0, _log_int(rng, 16, 4096)]) if bits == 4 else _log_int(rng, 16, 4096)
        most = max(1, min(256, int(1e9 / (longest * hk * d * 4))))
        return dict(base, bits=bits, seqs=_log_int(rng, 1, most), longest=longest,
                    shortest=rng.choice([1, longest // 2 + 1, longest]), page=page4 if bits == 4 else rng.choice([16, 24, 32, 64]),
                    window=window, sinks=rng.choice([0, 4, 16, 130]) if window else 0)
    longest, cached, window = _log_int(rng, 16, 8000), rng.choice([0, 0, rng.randint(1, 600)]), _log_int(rng, 16, 4096)
    sinks = rng.choice([0, 4, 16, 130])
    most = int(min(2e9 / (hq * longest * (longest + cached)), 2e11 / (4 * hq * d * longest * min(longest + cached, window + sinks))))
    return dict(base, seqs=_log_int(rng, 1, max(1, min(32, most))), longest=longest,
                shortest=rng.choice([1, longest // 2 + 1, longest]), cached=cached, window=window, sinks=sinks)


# ------------------------------------------------------------------------------------------ sizes
def _lengths(case):
    """The sequences' lengths: one of the longest, the others spread over the logarithm of the range."""
    rng = random.Random(case["lens_seed"])
    lens = [_log_int(rng, case["shortest"], case["longest"]) for _ in range(case["seqs"])]
    lens[rng.randrange(len(lens))] = case["longest"]
    return lens


def _before(case):
    """Tokens that an append finds in each sequence."""
    rng = random.Random(case["lens_seed"] + 1)
    return [rng.randint(0, case["before"]) for _ in range(case["seqs"])]


def _groups(dim):
    return (dim + 31) // 32


def _visible(n, window, sinks):
    """Keys of n that the last one's query sees."""
    return n if not window else min(n, sinks + window)


def _pairs(case, n):
    """Pairs of a query and a key it attends to, in a prompt of n queries."""
    c, w, s = case["cached"], case["window"], case["sinks"]
    free = max(0, min(n, w + s - c))             # queries that see every key before them
    return free * c + free * (free + 1) // 2 + (n - free) * (w + s)


def work(case):
    size, row, held = 2, case["kv_heads"] * case["dim"], case["kv_heads"] * 18 * _groups(case["dim"])
    lens = _lengths(case)
    total = sum(lens)
    if case["kind"] == "read":
        return {"bytes": 2 * total * (held + row * size), "flops": 0}
    qrow = case["q_heads"] * case["dim"]
    if case["kind"] == "append":
        tables = 2 * total * (case["dim"] // 2) * 4 if case["rope"] else 0
        return {"bytes": 4 * total * (row * size + held) + (2 * total * qrow * size if case["rope"] else 0) + tables,
                "flops": 3 * total * (qrow + row) if case["rope"] else 0}
    if case["kind"] == "decode":
        seen = sum(_visible(n, case["window"], case["sinks"]) for n in lens)
        return {"bytes": 2 * seen * (held if case["bits"] == 4 else row * size) + 2 * len(lens) * qrow * size,
                "flops": 4 * seen * qrow}
    keys = total + case["cached"] * len(lens)
    return {"bytes": 2 * total * qrow * size + 2 * keys * row * size, "flops": 4 * qrow * sum(_pairs(case, n) for n in lens)}


# ------------------------------------------------------------------------------------------ inputs
def _dtype(case):
    return {"fp16": torch.float16, "bf16": torch.bfloat16}[case["dtype"]]


def _normal(seed, index, shape, dtype):
    g = torch.Generator(device=DEV).manual_seed((int(seed) * 1000003 + index) % (2 ** 62))
    return torch.randn(shape, generator=g, device=DEV, dtype=dtype)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _offsets(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


def _table(lens, page, seed):
    """Pages dealt to the sequences in no order, a few left over: (table, pages of the pool)."""
    rng = random.Random(int(seed) * 7919 + 17)
    need = [-(-n // page) for n in lens]
    pool = list(range(sum(need) + 3))
    rng.shuffle(pool)
    rows, at = [], 0
    for n in need:
        rows.append(pool[at:at + n] + [-1] * (max(need) - n))
        at += n
    return rows, len(pool)


def _rope_tables(positions, dim):
    inv = THETA ** (-torch.arange(0, dim, 2, dtype=torch.float64, device=DEV) / dim)
    angle = torch.arange(positions, dtype=torch.float64, device=DEV)[:, None] * inv
    return angle.cos().float().contiguous(), angle.sin().float().contiguous()


def _pages(seed, index, case, pool):
    """A layer's pages, filled: keys as a projection leaves them, a few columns larger than the others, or values."""
    h, d, page = case["kv_heads"], case["dim"], case["page"]
    if case.get("bits", 4) == 16:
        return _normal(seed, index, (pool, page, h, d), _dtype(case))
    x = _normal(seed, index, (pool, h, page // 16, 16, d), _dtype(case))
    x[..., ::37] *= 3
    codes, scales = _quantise(x.float())
    return torch.cat([codes.flatten(-2), scales.view(torch.uint8).flatten(-2)], -1)


def prepare(case, seed):
    kind, dt = case["kind"], _dtype(case)
    hk, d = case["kv_heads"], case["dim"]
    s = dict(case=case, kind=kind, scale=d ** -0.5)
    lens = s["lens"] = _lengths(case)
    if kind == "prompt":
        hq, total, cached = case["q_heads"], sum(lens), case["cached"]
        if cached:                   # the keys of the cached tokens stand before the prompt's own
            klens = s["klens"] = [n + cached for n in lens]
            s["q"] = _normal(seed, 0, (total, hq, d), dt)
            s["k"], s["v"] = _normal(seed, 1, (2, sum(klens), hk, d), dt)
            s["cu_keys"] = _ints(_offsets(klens))
        else:                        # as the fused projection leaves them: columns of one row
            qkv = _normal(seed, 0, (total, hq + 2 * hk, d), dt)
            s["q"], s["k"], s["v"] = qkv.split([hq, hk, hk], 1)
            s["klens"], s["cu_keys"] = lens, None
        s["cu"] = _ints(_offsets(lens))
        return s
    before = _before(case) if kind == "append" else [0] * len(lens)
    ends = [n + b for n, b in zip(lens, before)]
    rows, pool = _table(ends, case["page"], seed)
    s["k_pages"], s["v_pages"] = _pages(seed, 0, case, pool), _pages(seed, 1, case, pool)
    s["rows"], s["table"], s["ends"], s["lengths"] = rows, _ints(rows), ends, _ints(ends)
    if kind == "decode":
        s["q"] = _normal(seed, 2, (len(lens), case["q_heads"], d), dt)
        if own:
            from turbopi_b200 import ops
            make = ops.paged_attention_nvfp4_workspace if case["bits"] == 4 else ops.paged_attention_workspace
            s["workspace"] = make(case["q_heads"], hk, d, DEV)
        return s
    s["cu"] = _ints(_offsets(lens))
    if kind == "read":
        return s
    hq = case["q_heads"]
    qkv = _normal(seed, 2, (sum(lens), hq + 2 * hk, d), dt)
    s["q"], s["k"], s["v"] = qkv.split([hq, hk, hk], 1)
    s["cos"], s["sin"] = _rope_tables(max(ends), d) if case["rope"] else (None, None)
    return s


# ------------------------------------------------------------------------------------------ one pass
def _quantise(x):
    """[..., D] fp32 -> (codes uint8 [..., 16 G], scales E4M3 [..., 2 G]): per 16 values the scale is max / 6, rounded to E4M3, and the
    codes are the values over it, rounded to the nearest E2M1, ties to the even code."""
    d = x.shape[-1]
    x = torch.nn.functional.pad(x, (0, 32 * _groups(d) - d)).unflatten(-1, (-1, 16))
    scales = (x.abs().amax(-1) / 6).clamp(max=448).to(torch.float8_e4m3fn)
    q = x / scales.float()[..., None]
    a = q.abs()
    code = torch.zeros_like(x, dtype=torch.uint8)
    code += a > 0.25
    code += a >= 0.75
    code += a > 1.25
    code += a >= 1.75
    code += a > 2.5
    code += a >= 3.5
    code += a > 5
    code += 8 * (q < 0)
    code = code.flatten(-2)
    return code[..., ::2] | (code[..., 1::2] << 4), scales


def _values(codes, scales, d):
    """What codes uint8 [..., 16 G] and scales uint8 [..., 2 G] stand for: fp32 [..., D]."""
    e2m1 = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, 0, -0.5, -1, -1.5, -2, -3, -4, -6], device=codes.device)
    x = e2m1[torch.stack([codes & 15, codes >> 4], -1).flatten(-2).int()]
    s = scales.contiguous().view(torch.float8_e4m3fn).float()
    return (x.unflatten(-1, (-1, 16)) * s[..., None]).flatten(-2)[..., :d]


def _parts(pages, d):
    """Views of 4-bit pages [P, H, tiles, bytes]: codes [P, H, tiles, 16, 16 G], scales [P, H, tiles, 16, 2 G]."""
    g = _groups(d)
    return pages[..., :256 * g].unflatten(-1, (16, 16 * g)), pages[..., 256 * g:].unflatten(-1, (16, 2 * g))


def _places(s):
    """Of every packed token: its page, and its row there."""
    cu, page = s["cu"].long(), s["case"]["page"]
    total = sum(s["lens"])
    seq = torch.repeat_interleave(torch.arange(len(s["lens"]), device=DEV), cu[1:] - cu[:-1], output_size=total)
    pos = torch.arange(total, device=DEV) - cu[1:][seq] + s["lengths"].long()[seq]
    return s["table"].long()[seq, pos // page], pos % page, pos


def _read(s, pages, ids, row):
    codes, scales = _parts(pages, s["case"]["dim"])
    return _values(codes[ids, :, row // 16, row % 16], scales[ids, :, row // 16, row % 16], s["case"]["dim"]).to(_dtype(s["case"]))


def _rotate(x, cos, sin):
    a, b = x.float().chunk(2, -1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1).to(x.dtype)


def _softmax_rows(scores, seen):
    scores = scores.masked_fill(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    w = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    return w / w.sum(-1, keepdim=True).clamp(min=1e-30)


def _decode(s):
    case, page, d = s["case"], s["case"]["page"], s["case"]["dim"]
    length = s["lengths"].long()[:, None]
    window = case["window"] or max(s["lens"])
    # the pages a query sees: the first ones, for the sinks, then those of the window
    first = -(-case["sinks"] // page)
    behind = torch.clamp((length - window) // page, min=first)
    count = min(window // page + 2, s["table"].shape[1])
    at = torch.cat([torch.arange(first, device=DEV).expand(len(s["lens"]), -1), behind + torch.arange(count, device=DEV)], 1)
    pos = (at[..., None] * page + torch.arange(page, device=DEV)).flatten(1)
    seen = (pos < length) & ((pos < case["sinks"]) | (pos >= length - window))
    ids = s["table"].long().gather(1, at.clamp(max=s["table"].shape[1] - 1)).clamp(min=0)
    kv = []
    for pages in (s["k_pages"], s["v_pages"]):
        if case["bits"] == 4:
            codes, scales = _parts(pages, d)
            kv.append(_values(codes[ids], scales[ids], d).transpose(1, 2).flatten(2, 4))      # [S, H, keys, D]
        else:
            kv.append(pages[ids].flatten(1, 2).transpose(1, 2).float())
    k, v = kv
    q = s["q"].float().unflatten(1, (case["kv_heads"], -1)) * s["scale"]
    w = _softmax_rows(q @ k.transpose(-1, -2), seen[:, None, None])
    return (w @ torch.where(seen[:, None, :, None], v, 0.0)).flatten(1, 2).to(s["q"].dtype)


def _padded(x, cu, lens):
    """[tokens, H, D] -> fp32 [S, H, longest, D]."""
    at = cu.long()[:-1, None] + torch.arange(max(lens), device=DEV)
    return x[at.clamp(max=x.shape[0] - 1)].transpose(1, 2).float()


def _prompt(s):
    case, cu, cu_keys = s["case"], s["cu"], s["cu"] if s["cu_keys"] is None else s["cu_keys"]
    g = case["q_heads"] // case["kv_heads"]
    q, k, v = _padded(s["q"], cu, s["lens"]), _padded(s["k"], cu_keys, s["klens"]), _padded(s["v"], cu_keys, s["klens"])
    i = torch.arange(q.shape[2], device=DEV)[:, None] + case["cached"]
    j = torch.arange(k.shape[2], device=DEV)
    seen = (j <= i) & ((j < case["sinks"]) | (j > i - case["window"]))
    q = q.unflatten(1, (case["kv_heads"], g)) * s["scale"]
    o = (_softmax_rows(q @ k[:, :, None].transpose(-1, -2), seen) @ v[:, :, None]).flatten(1, 2).transpose(1, 2)
    n = cu.long()[1:] - cu.long()[:-1]
    return o[torch.arange(q.shape[3], device=DEV) < n[:, None]].to(s["q"].dtype)


def _plain(s):
    kind = s["kind"]
    if kind == "prompt":
        return _prompt(s)
    if kind == "decode":
        return _decode(s)
    ids, row, pos = _places(s)
    if kind == "read":
        return [_read(s, s["k_pages"], ids, row), _read(s, s["v_pages"], ids, row)]
    q, k = None, s["k"]
    if s["cos"] is not None:
        cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]
        q, k = _rotate(s["q"], cos, sin), _rotate(k, cos, sin)
    for x, pages in ((k, s["k_pages"]), (s["v"], s["v_pages"])):
        codes, scales = _parts(pages, s["case"]["dim"])
        c, f = _quantise(x.float())
        codes[ids, :, row // 16, row % 16] = c
        scales[ids, :, row // 16, row % 16] = f.view(torch.uint8)
    return [q, _read(s, s["k_pages"], ids, row), _read(s, s["v_pages"], ids, row)]


def run(s):
    if not own:
        return _plain(s)
    from turbopi_b200 import ops
    case, kind = s["case"], s["kind"]
    if kind == "prompt":
        return ops.packed_attention(s["q"], s["k"], s["v"], s["cu"], s["scale"], cu_keys=s["cu_keys"], window=case["window"],
                                    sinks=case["sinks"])
    if kind == "decode":
        call = ops.paged_attention_nvfp4 if case["bits"] == 4 else ops.paged_attention
        return call(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lengths"], s["scale"], workspace=s["workspace"],
                    window=case["window"] or None, sinks=case["sinks"])
    tokens, dt = sum(s["lens"]), _dtype(case)
    if kind == "read":
        return list(ops.paged_read_nvfp4(s["k_pages"], s["v_pages"], s["table"], s["cu"], s["lengths"], case["dim"], tokens, dtype=dt))
    q = ops.paged_append_nvfp4(s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["cu"], s["lengths"],
                               q=s["q"] if s["cos"] is not None else None, cos=s["cos"], sin=s["sin"])
    k, v = ops.paged_read_nvfp4(s["k_pages"], s["v_pages"], s["table"], s["cu"], s["lengths"], case["dim"], tokens, dtype=dt)
    return [q, k, v]


# ------------------------------------------------------------------------------------------ the definition in 64 bits
_LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _held(x):
    """What the cache holds of rows [T, H, D] of a 16-bit type: for each 16 values the nearest multiples of their scale."""
    t, h, d = x.shape
    pad = -d % 16
    y = torch.cat([x.double(), x.new_zeros((t, h, pad), dtype=torch.float64)], -1).reshape(t, h, -1, 16)
    scale = (y.abs().amax(-1, keepdim=True).float() / 6).clamp(max=448).to(torch.float8_e4m3fn).double()
    ratio = torch.where(scale > 0, y.abs() / scale.clamp(min=2.0 ** -9), 0.0)
    best, at = torch.full_like(ratio, 9.0), torch.zeros_like(ratio)
    for i in (0, 2, 4, 6, 1, 3, 5, 7):           # even codes first: they win a tie
        off = (ratio - _LEVELS[i]).abs()
        at = torch.where(off < best, _LEVELS[i], at)
        best = torch.minimum(best, off)
    return (at * scale * y.sign()).reshape(t, h, -1)[..., :d]


def _stored(s, pages, seq, positions):
    """Rows [n, H, D] in 64 bits of positions of a sequence."""
    case = s["case"]
    d, page = case["dim"], case["page"]
    ids = torch.tensor(s["rows"][seq], device=DEV)[positions // page]
    r = positions % page
    if case.get("bits", 4) == 16:
        return pages[ids, r].double()
    g = _groups(d)
    tiles = pages[ids, :, r // 16]                                            # [n, H, bytes]
    n, h = tiles.shape[:2]
    at = (r % 16)[:, None, None]
    col = torch.arange(16 * g, device=DEV)
    code = tiles.gather(2, (at * 16 * g + col).expand(n, h, -1)).int()
    byte = tiles.gather(2, (256 * g + at * 2 * g + col[:2 * g]).expand(n, h, -1)).int()
    e, m = (byte >> 3) & 15, (byte & 7).double()                             # E4M3 without its sign
    scale = torch.where(e == 0, m * 2.0 ** -9, (1 + m / 8) * torch.exp2(e.double() - 7))
    x = torch.stack([code % 16, code // 16], -1).reshape(n, h, -1)
    level = torch.tensor(_LEVELS, dtype=torch.float64, device=DEV)[x % 8] * (1.0 - 2.0 * (x // 8))
    return (level.reshape(n, h, 2 * g, 16) * scale[..., None]).reshape(n, h, -1)[..., :d]


def _mean(scores, values):
    """Rows of scores (-inf where not allowed) -> the weighted mean of the values."""
    top = scores.max(-1, keepdim=True).values
    w = (scores - top).exp()
    return torch.einsum("...k,kd->...d", w, values) / w.sum(-1, keepdim=True)


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "prompt":
        g, out = case["q_heads"] // case["kv_heads"], torch.empty(s["q"].shape, dtype=torch.float64, device=DEV)
        q0, k0 = 0, 0
        for n, m in zip(s["lens"], s["klens"]):
            for lo in range(0, n, 512):
                hi = min(n, lo + 512)
                last = m - n + hi
                i = torch.arange(lo, hi, device=DEV)[:, None] + (m - n)
                j = torch.arange(last, device=DEV)[None, :]
                hidden = (j > i) | ((j >= case["sinks"]) & (j <= i - case["window"]))
                for h in range(case["q_heads"]):
                    sc = s["scale"] * (s["q"][q0 + lo:q0 + hi, h].double() @ s["k"][k0:k0 + last, h // g].double().T)
                    out[q0 + lo:q0 + hi, h] = _mean(torch.where(hidden, -math.inf, sc), s["v"][k0:k0 + last, h // g].double())
            q0, k0 = q0 + n, k0 + m
        return out
    if kind == "decode":
        g, out = case["q_heads"] // case["kv_heads"], torch.empty(s["q"].shape, dtype=torch.float64, device=DEV)
        for i, n in enumerate(s["lens"]):
            keep = torch.arange(n, device=DEV)
            if case["window"]:
                keep = keep[(keep < case["sinks"]) | (keep >= n - case["window"])]
            k, v = _stored(s, s["k_pages"], i, keep), _stored(s, s["v_pages"], i, keep)
            for h in range(case["kv_heads"]):
                q = s["q"][i, h * g:h * g + g].double()
                out[i, h * g:h * g + g] = _mean(s["scale"] * q @ k[:, h].T, v[:, h])
        return out
    if kind == "read":
        out = [[], []]
        for i, n in enumerate(s["lens"]):
            for x, pages in zip(out, (s["k_pages"], s["v_pages"])):
                x.append(_stored(s, pages, i, torch.arange(n, device=DEV)))
        return [torch.cat(x) for x in out]
    q, k = None, s["k"].double()
    if case["rope"]:
        pos = torch.cat([torch.arange(end - n, end, device=DEV) for n, end in zip(s["lens"], s["ends"])])
        turn = torch.complex(s["cos"][pos].double(), s["sin"][pos].double())[:, None]
        half = case["dim"] // 2

        def rotated(x):
            z = torch.complex(x[..., :half].double().contiguous(), x[..., half:].double().contiguous()) * turn
            return torch.cat([z.real, z.imag], -1)
        q, k = rotated(s["q"]), rotated(s["k"])
    return [q, _held(k.to(_dtype(case))), _held(s["v"])]

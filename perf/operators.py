"""The work whose speed the paged KV cache and the packed attention are judged by, as calls of their public entry points.

`listed()` names the cases, `draw(rng)` gives further ones of the same ranges, `prepare` is what a program holds before a
call, `run` one call: in elementary torch operations, or with `own` through the package.  `exact` restates each case in 64 bits.

Kinds of case:
  prompt  ops.packed_attention: causal attention over the prompts of a batch, one behind the other
  decode  ops.paged_attention: one new token per sequence on a cache of pages
  append  ops.paged_append: new tokens' keys and values into their pages, queries and keys rotated
  copy    ops.copy_pages: pages of every layer moved for a fork or a compaction
"""
import math
import random

import torch

own = False
DEV = "cuda"
THETA = 10000.0


def listed():
    return [
        # one token of one request on the cache of a Pi0.5 prompt with its 50 action rows: the smallest call, all latency
        dict(name="decode_one", kind="decode", seqs=1, longest=762, shortest=762, q_heads=8, kv_heads=1, dim=256, page=16,
             dtype="bf16", lens_seed=1),
        # a serving batch, requests at every stage, four query heads to a key head
        dict(name="decode_ragged", kind="decode", seqs=48, longest=4096, shortest=1, q_heads=32, kv_heads=8, dim=128, page=16,
             dtype="bf16", lens_seed=2),
        # a few very long conversations: the cache's length is all there is to split
        dict(name="decode_long", kind="decode", seqs=3, longest=131071, shortest=40000, q_heads=8, kv_heads=1, dim=256, page=64,
             dtype="fp16", lens_seed=3),
        # as many key heads as query heads: the largest cache per token
        dict(name="decode_heads", kind="decode", seqs=128, longest=2000, shortest=16, q_heads=16, kv_heads=16, dim=64, page=32,
             dtype="fp16", lens_seed=4),
        # the text of a Pi0.5 prompt on its own
        dict(name="prompt_one", kind="prompt", seqs=1, longest=200, shortest=200, q_heads=8, kv_heads=1, dim=256, dtype="bf16",
             causal=True, cached=0, lens_seed=5),
        # a batch of short prompts of every length, small heads
        dict(name="prompt_ragged", kind="prompt", seqs=24, longest=1200, shortest=1, q_heads=16, kv_heads=4, dim=64, dtype="fp16",
             causal=True, cached=0, lens_seed=6),
        # one long document at Gemma's head shape
        dict(name="prompt_long", kind="prompt", seqs=1, longest=8191, shortest=8191, q_heads=8, kv_heads=1, dim=256, dtype="bf16",
             causal=True, cached=0, lens_seed=7),
        # the largest batch: long prompts side by side, the queries behind keys that are already there
        dict(name="prompt_batch", kind="prompt", seqs=4, longest=9000, shortest=1500, q_heads=32, kv_heads=8, dim=128,
             dtype="bf16", causal=True, cached=500, lens_seed=8),
        # a decode step's write: one token for each of 64 requests
        dict(name="append_step", kind="append", seqs=64, longest=1, shortest=1, before=3000, q_heads=8, kv_heads=1, dim=256,
             page=16, dtype="bf16", rope=True, lens_seed=9),
        # the prompts of a batch written at once
        dict(name="append_prompts", kind="append", seqs=6, longest=4000, shortest=300, before=200, q_heads=32, kv_heads=8, dim=128,
             page=32, dtype="bf16", rope=True, lens_seed=10),
        # a fork: the last, half-filled page of a few sequences, in every layer
        dict(name="copy_fork", kind="copy", layers=18, pages=600, moves=5, kv_heads=1, dim=256, page=16, dtype="bf16"),
        # a compaction of a fragmented cache
        dict(name="copy_compact", kind="copy", layers=18, pages=2000, moves=900, kv_heads=1, dim=256, page=16, dtype="bf16"),
    ]


def _log_int(rng, lo, hi):
    return int(min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


# (query heads, key heads, head size): Gemma's, and the usual ones; a group of three, sizes that are no power of two
_HEADS = [(8, 1, 256), (8, 1, 256), (32, 8, 128), (16, 4, 64), (16, 16, 64), (8, 2, 128), (12, 4, 128), (4, 4, 256), (16, 16, 72),
          (16, 2, 96)]


def draw(rng):
    kind = rng.choice(["prompt", "prompt", "prompt", "decode", "decode", "decode", "append", "copy"])
    hq, hk, d = rng.choice(_HEADS)
    base = dict(kind=kind, q_heads=hq, kv_heads=hk, dim=d, dtype=rng.choice(["bf16", "fp16"]), lens_seed=rng.randint(0, 10 ** 6))
    if kind == "prompt":
        longest = _log_int(rng, 16, 8000)
        return dict(base, seqs=_log_int(rng, 1, max(1, min(32, 16000 // longest))), longest=longest,
                    shortest=rng.choice([1, longest // 2 + 1, longest]), causal=rng.random() < 0.8,
                    cached=rng.choice([0, 0, rng.randint(1, 600)]))
    if kind == "decode":
        longest = _log_int(rng, 16, 131072)
        most = max(1, min(256, int(5e8 / (longest * hk * d * 4))))
        return dict(base, seqs=_log_int(rng, 1, most), longest=longest, shortest=rng.choice([1, longest // 2 + 1, longest]),
                    page=rng.choice([16, 16, 24, 32, 64, 128]))
    if kind == "append":
        longest = _log_int(rng, 1, 4000)
        return dict(base, seqs=_log_int(rng, 1, max(1, min(128, 12000 // longest))), longest=longest,
                    shortest=rng.choice([1, longest]), before=rng.randint(0, 3000), page=rng.choice([16, 16, 24, 32, 64, 128]),
                    rope=rng.random() < 0.7)
    page = rng.choice([16, 16, 24, 32, 64])
    layers = rng.randint(1, 18)
    most = int(5e8 / (layers * 2 * page * hk * d * 2))
    pages = _log_int(rng, 16, max(16, min(4000, most)))
    return dict(kind=kind, layers=layers, pages=pages, moves=_log_int(rng, 1, pages // 2), kv_heads=hk, dim=d, page=page,
                dtype=base["dtype"])


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


def _pairs(case, n):
    """Pairs of a query and a key it attends to, in a prompt of n queries."""
    m = n + case["cached"]
    return n * m - n * (n - 1) // 2 if case["causal"] else n * m


def work(case):
    size, row = 2, case["kv_heads"] * case["dim"]
    if case["kind"] == "copy":
        return {"bytes": 2 * case["layers"] * 2 * case["moves"] * case["page"] * row * size, "flops": 0}
    lens, qrow = _lengths(case), case["q_heads"] * case["dim"]
    total = sum(lens)
    if case["kind"] == "decode":
        return {"bytes": 2 * total * row * size + 2 * len(lens) * qrow * size, "flops": 4 * total * qrow}
    if case["kind"] == "append":
        tables = 2 * total * (case["dim"] // 2) * 4 if case["rope"] else 0
        return {"bytes": 2 * total * (2 * row + (qrow if case["rope"] else 0)) * size + tables,
                "flops": 3 * total * (qrow + row) if case["rope"] else 0}
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
    """Pages dealt to the sequences in no order, a few left over: (table, the same on the host, pages of the pool)."""
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


def prepare(case, seed):
    kind, dt = case["kind"], _dtype(case)
    hk, d = case["kv_heads"], case["dim"]
    s = dict(case=case, kind=kind, scale=d ** -0.5)
    if kind == "copy":
        s["pages"] = _normal(seed, 0, (case["layers"], 2, case["pages"], case["page"], hk, d), dt)
        ids = list(range(case["pages"]))
        random.Random(int(seed) * 7919 + 5).shuffle(ids)
        s["src"], s["dst"] = ids[:case["moves"]], ids[case["moves"]:2 * case["moves"]]
        return s
    hq = case["q_heads"]
    lens = s["lens"] = _lengths(case)
    if kind == "prompt":
        total, cached = sum(lens), case["cached"]
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
    s["k_pages"], s["v_pages"] = _normal(seed, 0, (2, pool, case["page"], hk, d), dt)
    s["rows"], s["table"], s["ends"], s["lengths"] = rows, _ints(rows), ends, _ints(ends)
    if kind == "decode":
        s["q"] = _normal(seed, 1, (len(lens), hq, d), dt)
        if own:
            from turbopi_b200 import ops
            s["workspace"] = ops.paged_attention_workspace(hq, hk, d, DEV)
        return s
    qkv = _normal(seed, 1, (sum(lens), hq + 2 * hk, d), dt)
    s["q"], s["k"], s["v"] = qkv.split([hq, hk, hk], 1)
    s["cu"] = _ints(_offsets(lens))
    s["cos"], s["sin"] = _rope_tables(max(ends), d) if case["rope"] else (None, None)
    return s


# ------------------------------------------------------------------------------------------ one pass
def _attend(q, k, v, scale, first):
    """softmax(scale q k^T) v in fp32 for [n, Hq, D] on [m, Hk, D]; query i sees keys up to first + i (all with None)."""
    n, hq, d = q.shape
    m, hk = k.shape[0], k.shape[1]
    g = hq // hk
    out = torch.empty_like(q)
    masked = None
    if first is not None:
        masked = torch.arange(m, device=q.device)[None, :] > torch.arange(n, device=q.device)[:, None] + first
    for h in range(hq):
        s = (q[:, h].float() * scale) @ k[:, h // g].float().t()
        if masked is not None:
            s.masked_fill_(masked, -math.inf)
        s = torch.exp(s - s.amax(1, keepdim=True))
        out[:, h] = ((s @ v[:, h // g].float()) / s.sum(1, keepdim=True)).to(q.dtype)
    return out


def _rotate(x, cos, sin):
    a, b = x.float().chunk(2, -1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1).to(x.dtype)


def _plain(s):
    kind = s["kind"]
    if kind == "copy":
        src, dst = (torch.tensor(x, device=DEV) for x in (s["src"], s["dst"]))
        s["pages"][:, :, dst] = s["pages"][:, :, src]
        return s["pages"]
    if kind == "prompt":
        out, q0, k0 = [], 0, 0
        for n, m in zip(s["lens"], s["klens"]):
            out.append(_attend(s["q"][q0:q0 + n], s["k"][k0:k0 + m], s["v"][k0:k0 + m], s["scale"],
                               m - n if s["case"]["causal"] else None))
            q0, k0 = q0 + n, k0 + m
        return torch.cat(out)
    page, table = s["case"]["page"], s["table"].long()
    if kind == "decode":
        out = torch.empty_like(s["q"])
        for i, n in enumerate(s["lens"]):
            ids = table[i, :-(-n // page)]
            k, v = (p[ids].flatten(0, 1)[:n] for p in (s["k_pages"], s["v_pages"]))
            hk, d = k.shape[1:]
            q = s["q"][i].float().view(hk, -1, d) * s["scale"]
            w = q @ k.float().permute(1, 2, 0)
            w = torch.exp(w - w.amax(-1, keepdim=True))
            out[i] = ((w @ v.float().transpose(0, 1)) / w.sum(-1, keepdim=True)).to(out.dtype).flatten(0, 1)
        return out
    cu, ends = s["cu"].long(), s["lengths"].long()
    seq = torch.repeat_interleave(torch.arange(len(s["lens"]), device=DEV), cu[1:] - cu[:-1], output_size=s["q"].shape[0])
    pos = torch.arange(s["q"].shape[0], device=DEV) - cu[1:][seq] + ends[seq]
    ids, slot = table[seq, pos // page], pos % page
    q, k = None, s["k"]
    if s["cos"] is not None:
        cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]
        q, k = _rotate(s["q"], cos, sin), _rotate(k, cos, sin)
    s["k_pages"][ids, slot] = k
    s["v_pages"][ids, slot] = s["v"]
    return [q, s["k_pages"], s["v_pages"]]


def run(s):
    if not own:
        return _plain(s)
    from turbopi_b200 import ops
    kind = s["kind"]
    if kind == "copy":
        ops.copy_pages(s["pages"], s["src"], s["dst"])
        return s["pages"]
    if kind == "prompt":
        return ops.packed_attention(s["q"], s["k"], s["v"], s["cu"], s["scale"], causal=s["case"]["causal"],
                                    cu_keys=s["cu_keys"])
    if kind == "decode":
        return ops.paged_attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lengths"], s["scale"],
                                   workspace=s["workspace"])
    q = ops.paged_append(s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["cu"], s["lengths"],
                         q=s["q"] if s["cos"] is not None else None, cos=s["cos"], sin=s["sin"])
    return [q, s["k_pages"], s["v_pages"]]


# ------------------------------------------------------------------------------------------ the definition in 64 bits
def _softmax_mean(scores, values):
    """Rows of scores (-inf where not allowed) -> the weighted mean of the values."""
    top = scores.max(-1, keepdim=True).values
    w = (scores - top).exp()
    return torch.einsum("...k,kd->...d", w, values) / w.sum(-1, keepdim=True)


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "copy":
        out = s["pages"].double()
        for a, b in zip(s["src"], s["dst"]):
            out[:, :, b] = s["pages"][:, :, a].double()
        return out
    g, scale = case["q_heads"] // case["kv_heads"], s["scale"]
    if kind == "prompt":
        out = torch.empty(s["q"].shape, dtype=torch.float64, device=DEV)
        q0, k0 = 0, 0
        for n, m in zip(s["lens"], s["klens"]):
            for h in range(case["kv_heads"]):
                keys, values = s["k"][k0:k0 + m, h].double(), s["v"][k0:k0 + m, h].double()
                for lo in range(0, n, 1024):
                    hi = min(n, lo + 1024)
                    last = m - n + hi if case["causal"] else m
                    for head in range(h * g, h * g + g):
                        sc = scale * (s["q"][q0 + lo:q0 + hi, head].double() @ keys[:last].T)
                        if case["causal"]:
                            row = torch.arange(lo, hi, device=DEV)[:, None] + (m - n)
                            sc = torch.where(torch.arange(last, device=DEV)[None, :] <= row, sc, -math.inf)
                        out[q0 + lo:q0 + hi, head] = _softmax_mean(sc, values[:last])
            q0, k0 = q0 + n, k0 + m
        return out
    page = case["page"]

    def place(i, positions):
        """Rows of the flattened pool where positions of sequence i stand."""
        ids = torch.tensor(s["rows"][i], device=DEV)
        return ids[positions // page] * page + positions % page

    if kind == "decode":
        out = torch.empty(s["q"].shape, dtype=torch.float64, device=DEV)
        kf, vf = (p.reshape(-1, *p.shape[2:]) for p in (s["k_pages"], s["v_pages"]))
        for i, n in enumerate(s["lens"]):
            at = place(i, torch.arange(n, device=DEV))
            for h in range(case["kv_heads"]):
                q = s["q"][i, h * g:h * g + g].double()
                out[i, h * g:h * g + g] = _softmax_mean(scale * q @ kf[at, h].double().T, vf[at, h].double())
        return out
    kf, vf = (p.double().flatten(0, 1) for p in (s["k_pages"], s["v_pages"]))
    half = case["dim"] // 2
    turned = torch.empty(s["q"].shape, dtype=torch.float64, device=DEV) if case["rope"] else None
    t0 = 0
    for i, (n, end) in enumerate(zip(s["lens"], s["ends"])):
        pos = torch.arange(end - n, end, device=DEV)
        at, k = place(i, pos), s["k"][t0:t0 + n].double()
        if case["rope"]:
            turn = torch.complex(s["cos"][pos].double(), s["sin"][pos].double())[:, None]

            def rotated(x):
                z = torch.complex(x[..., :half].contiguous(), x[..., half:].contiguous()) * turn
                return torch.cat([z.real, z.imag], -1)
            k = rotated(k)
            turned[t0:t0 + n] = rotated(s["q"][t0:t0 + n].double())
        kf[at], vf[at] = k, s["v"][t0:t0 + n].double()
        t0 += n
    return [turned, kf.view(s["k_pages"].shape), vf.view(s["v_pages"].shape)]

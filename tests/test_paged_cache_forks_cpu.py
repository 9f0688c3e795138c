"""Forks of sequences whose newest tokens have room but are not written yet: a copy of their page would lack them."""
import pytest
import torch

from turbopi_b200 import ops
from turbopi_b200._lib import TurboPiError
from turbopi_b200.paged_cache import PagedCache


@pytest.fixture
def cache(monkeypatch):
    monkeypatch.setattr(ops, "copy_pages", lambda pages, src, dst: None)
    monkeypatch.setattr(ops, "paged_append", lambda *a, **k: "appended")
    monkeypatch.setattr(ops, "paged_attention", lambda *a, **k: "attended")
    return PagedCache(2, 20, 4, 1, 8, 6, dtype=torch.float16, device="cpu")


KV = torch.zeros(2, 1, 8)


def _append(cache, batch, layer=0):
    kv = torch.zeros(batch.tokens, 1, 8)
    return cache.append(layer, batch, kv, kv)


def test_tokens_written_after_their_page_was_copied_are_refused(cache):
    a = cache.add()
    old = cache.extend([a], [9])
    assert _append(cache, old) == "appended"
    late = cache.extend([a], [2])                                # positions 9 and 10 of the third page
    b = cache.fork(a)
    assert _append(cache, late) == "appended"                    # the page is shared: both have them, in this layer
    cache.extend([b], [1])                                       # b's copy is made
    for layer in (1, -1):
        with pytest.raises(TurboPiError, match=f"copied to sequence {b}"):
            _append(cache, late, layer)
        with pytest.raises(TurboPiError, match="copied"):        # its ninth token lies in that page
            _append(cache, old, layer)
    assert _append(cache, late) == _append(cache, old) == _append(cache, late, -2) == "appended"      # what was written before the copy
    # the pages are a's as before: attention goes on, and so do new batches
    assert cache.attention(0, late, KV[:1], 1.0) == "attended"
    assert _append(cache, cache.extend([a], [1])) == "appended"
    assert cache.extend([a], [1], out=late) is late and _append(cache, late, 1) == "appended"
    with pytest.raises(IndexError):
        _append(cache, late, 2)


def test_both_extended_in_one_call(cache):
    """The first gets the copy and its batches are refused as before; the other one's own tokens are where they were."""
    a = cache.add()
    late = cache.extend([a], [2])
    b = cache.fork(a)
    both = cache.extend([a, b], [1, 1])
    with pytest.raises(TurboPiError, match="copied"):
        _append(cache, late)
    assert _append(cache, both) == "appended"


def test_tokens_that_no_copy_needs(cache):
    """In other pages, or behind where the copying sequence ends."""
    a = cache.add()
    first = cache.extend([a], [4])                               # a whole page, which is shared and never copied
    late = cache.extend([a], [3])                                # positions 4 to 6
    b, c = cache.fork(a), cache.fork(a)
    cache.truncate(c, 4)
    cache.extend([c], [2])                                       # a page of its own
    assert _append(cache, first) == _append(cache, late, 1) == "appended"
    cache.truncate(b, 5)
    more = cache.extend([a], [0])
    alone = cache.extend([cache.add()], [2])
    cache.extend([b], [1])                                       # copies the page for position 4 alone
    assert _append(cache, first) == _append(cache, more) == _append(cache, alone) == "appended"
    with pytest.raises(TurboPiError, match="copied"):
        _append(cache, late)
    d = cache.fork(a)
    last = cache.extend([a], [1])                                # a copies: position 7 is a's alone
    cache.extend([d], [1])
    assert _append(cache, last) == "appended"


def test_truncated_below_the_reserved_tokens(cache):
    a = cache.add()
    _append(cache, cache.extend([a], [2]))
    late = cache.extend([a], [1])
    b = cache.fork(a)
    cache.truncate(b, 2)
    cache.extend([b], [1])                                       # its copy needs positions 0 and 1, not 2
    assert _append(cache, late) == "appended"


@pytest.mark.parametrize("seed", range(20))
def test_random_histories(monkeypatch, seed):
    """Appends that come late, or never: what was appended without a refusal is what every sequence with those tokens reads."""
    import random
    rng, layers = random.Random(seed), 2
    cache = PagedCache(layers, 14, 4, 1, 8, 5, dtype=torch.float16, device="cpu")
    monkeypatch.setattr(ops, "copy_pages", lambda pages, src, dst: pages.index_copy_(2, torch.tensor(dst), pages[:, :, src].clone()))

    def write(k, v, k_pages, v_pages, table, cu, lengths, **kw):
        cu, lengths = cu.tolist(), lengths.tolist()
        for s, row in enumerate(table.tolist()):
            for t in range(cu[s], cu[s + 1]):
                pos = lengths[s] - cu[s + 1] + t
                k_pages[row[pos // 4], pos % 4] = k[t]
    monkeypatch.setattr(ops, "paged_append", write)
    want, open_batches, written, stamp, refused = {}, [], [set() for _ in range(layers)], 0, 0
    for _ in range(400):
        what = rng.choice(["add", "extend", "extend", "extend", "append", "append", "append", "fork", "fork", "free", "truncate", "compact"])
        if what == "add" and len(want) < 5:
            want[cache.add()] = []
        elif what == "extend" and want:
            seqs = rng.sample(sorted(want), rng.randint(1, len(want)))
            new = [rng.choice([0, 1, 1, 2, 5]) for _ in seqs]
            try:
                batch = cache.extend(seqs, new)
            except TurboPiError:
                continue
            tokens = [float(stamp + i) for i in range(sum(new))]
            stamp += len(tokens)
            open_batches.append((batch, tokens))
            for s, n in zip(seqs, new):
                want[s] = want[s] + tokens[:n]
                tokens = tokens[n:]
        elif what == "append" and open_batches:
            batch, tokens = rng.choice(open_batches[-4:])
            layer = rng.randrange(layers)
            kv = torch.tensor(tokens).view(-1, 1, 1).expand(-1, 1, 8)
            if layer in batch._layers:
                continue
            try:
                cache.append(layer, batch, kv, kv)
                written[layer].update(tokens)
            except TurboPiError:
                refused += 1
        elif what == "fork" and want and len(want) < 5:
            s = rng.choice(sorted(want))
            want[cache.fork(s)] = list(want[s])
        elif what == "free" and len(want) > 2:
            s = rng.choice(sorted(want))
            cache.free(s)
            del want[s]
        elif what == "truncate" and want:
            s = rng.choice(sorted(want))
            n = rng.randint(len(want[s]) // 2, len(want[s]))
            cache.truncate(s, n)
            want[s] = want[s][:n]
        elif what == "compact":
            cache.compact()
        for s, tokens in want.items():
            pages = cache.page_ids(s)
            for layer in range(layers):
                for pos, token in enumerate(tokens):
                    if token in written[layer]:
                        assert float(cache.pages[layer, 0, pages[pos // 4], pos % 4, 0, 0]) == token
    assert refused and sum(map(len, written)) > 20

"""PagedCache's bookkeeping: pages on the CPU, the moves of bytes stood in for, every token of every sequence compared after random calls."""
import random

import pytest
import torch

from turbopi_b200 import ops
from turbopi_b200._lib import TurboPiError
from turbopi_b200.paged_cache import PagedCache


@pytest.fixture
def cpu_copies(monkeypatch):
    calls = []

    def copy_pages(pages, src, dst):
        assert not set(src) & set(dst) and len(set(dst)) == len(dst) and len(src) == len(dst) > 0
        assert all(0 <= p < pages.shape[-4] for p in src + dst)
        pages[..., dst, :, :, :] = pages[..., src, :, :, :].clone()
        calls.append(len(src))
    monkeypatch.setattr(ops, "copy_pages", copy_pages)
    return calls


def _cache(num_pages=12, page_size=4, max_pages=6):
    return PagedCache(2, num_pages, page_size, 1, 8, max_pages, dtype=torch.float16, device="cpu")


def _write(cache, batch, tokens):
    """What `append` does with the batch: `tokens` one number per new token, in both layers."""
    cu, lengths = batch.cu.tolist(), batch.lengths.tolist()
    for s, row in enumerate(batch.table.tolist()):
        n = cu[s + 1] - cu[s]
        for i in range(n):
            pos = lengths[s] - n + i
            assert row[pos // cache.page_size] >= 0
            cache.pages[:, :, row[pos // cache.page_size], pos % cache.page_size] = tokens[cu[s] + i]


def _read(cache, seq):
    return [float(cache.pages[1, 0, p, r, 0, 0]) for p in cache.page_ids(seq) for r in range(cache.page_size)][:cache.length(seq)]


def _consistent(cache):
    held = [p for e in cache._seqs.values() for p in e[0]]
    assert all(cache._refs[p] == held.count(p) for p in range(cache.num_pages))
    assert sorted(cache._free) == [p for p in range(cache.num_pages) if p not in held]
    for e in cache._seqs.values():
        assert len(e[0]) == -(-e[1] // cache.page_size) and len(set(e[0])) == len(e[0])


@pytest.mark.parametrize("seed", range(12))
def test_random_calls(cpu_copies, seed):
    rng = random.Random(seed)
    cache, want, stamp = _cache(), {}, 0
    for _ in range(300):
        what = rng.choice(["add", "extend", "extend", "extend", "fork", "free", "truncate", "compact"])
        if what == "add" and len(want) < 5:
            want[cache.add()] = []
        elif what == "extend" and want:
            seqs = rng.sample(sorted(want), rng.randint(1, len(want)))
            new = [rng.choice([0, 1, 1, 3, 4, 9]) for _ in seqs]
            before = {s: (cache.page_ids(s), cache.length(s)) for s in want}, cache.free_pages
            try:
                batch = cache.extend(seqs, new)
            except TurboPiError as e:
                assert "need" in str(e)
                assert before == ({s: (cache.page_ids(s), cache.length(s)) for s in want}, cache.free_pages)
                continue
            tokens = [float((stamp + i) % 2000) for i in range(sum(new))]
            stamp += len(tokens)
            assert batch.tokens == len(tokens) and batch.lengths.tolist() == [cache.length(s) for s in seqs]
            _write(cache, batch, tokens)
            for s, n in zip(seqs, new):
                want[s] = want[s] + tokens[:n]
                tokens = tokens[n:]
        elif what == "fork" and want and len(want) < 5:
            s = rng.choice(sorted(want))
            want[cache.fork(s)] = list(want[s])
        elif what == "free" and want:
            s = rng.choice(sorted(want))
            cache.free(s)
            del want[s]
        elif what == "truncate" and want:
            s = rng.choice(sorted(want))
            n = rng.randint(0, len(want[s]))
            cache.truncate(s, n)
            want[s] = want[s][:n]
        elif what == "compact":
            used = cache.compact()
            assert used == cache.num_pages - cache.free_pages and all(p < used for s in want for p in cache.page_ids(s))
        _consistent(cache)
        assert all(_read(cache, s) == tokens for s, tokens in want.items())
    assert cpu_copies


def test_truncated_forks_do_not_write_into_each_other(cpu_copies):
    """A whole shared page becomes a half-filled one by truncation; extending copies it then."""
    cache = _cache()
    a = cache.add()
    _write(cache, cache.extend([a], [8]), [float(i) for i in range(8)])
    b = cache.fork(a)
    cache.truncate(b, 6)
    _write(cache, cache.extend([b], [2]), [60.0, 70.0])
    assert _read(cache, a) == [float(i) for i in range(8)] and _read(cache, b) == [0, 1, 2, 3, 4, 5, 60, 70]


def test_both_halves_of_a_fork_in_one_batch(cpu_copies):
    """Only the first copies: the page is the second's alone then."""
    cache = _cache()
    a = cache.add()
    _write(cache, cache.extend([a], [5]), [float(i) for i in range(5)])
    b = cache.fork(a)
    _write(cache, cache.extend([a, b], [1, 1]), [10.0, 20.0])
    assert cpu_copies == [1]
    assert _read(cache, a)[5:] == [10.0] and _read(cache, b)[5:] == [20.0]


def test_refusals():
    cache = _cache()
    a = cache.add()
    for call in (lambda: cache.extend([a, a], [1, 1]), lambda: cache.extend([a], [-1]), lambda: cache.extend([a], [1, 2]),
                 lambda: cache.extend([a], [25]), lambda: cache.free(99), lambda: cache.fork([a]), lambda: cache.truncate(a, 1),
                 lambda: cache.length(None), lambda: PagedCache(1, 4, 4, 1, 12, 4, device="cpu"), lambda: PagedCache(0, 4, 4, 1, 8, 4, device="cpu"),
                 lambda: PagedCache(1, 4, 2 ** 20, 1, 8, 2 ** 11, device="cpu"), lambda: PagedCache(1, 4, 4, 1, 8, 4, dtype=torch.float32, device="cpu")):
        with pytest.raises(TurboPiError):
            call()
    b = cache.add()
    with pytest.raises(TurboPiError, match="13 pages needed, 12 free"):
        cache.extend([a, b, cache.add()], [24, 24, 1])
    assert cache.free_pages == 12 and cache.length(a) == 0
    batch = cache.extend([a], [3])
    with pytest.raises(TurboPiError, match="2 rows for 3"):
        cache.append(0, batch, torch.zeros(2, 1, 8), torch.zeros(2, 1, 8))


def test_batches_are_refused_after_pages_have_moved(cpu_copies):
    cache = _cache()
    a, b = cache.add(), cache.add()
    cache.extend([a], [8])
    batch = cache.extend([b], [3])
    cache.free(a)
    assert cache.compact() == 1
    with pytest.raises(TurboPiError, match="moved"):
        cache.attention(0, batch, torch.zeros(1, 1, 8), 1.0)
    again = cache.extend([b], [0], out=batch)
    assert again is batch and batch.table[0, 0] == 0
    cache._current(batch)


@pytest.mark.parametrize("what", ["freed", "truncated", "copied"])
def test_a_batch_whose_pages_may_be_others_is_refused(cpu_copies, monkeypatch, what):
    monkeypatch.setattr(ops, "paged_append", lambda *a, **k: "appended")
    monkeypatch.setattr(ops, "paged_attention", lambda *a, **k: "attended")
    cache = _cache()
    a, other = cache.add(), cache.add()
    batch, kv = cache.extend([a, other], [5, 2]), torch.zeros(7, 1, 8)
    alone = cache.extend([other], [1])
    # what leaves the pages of the batch with their sequences leaves the batch as it is
    cache.extend([a], [1])
    fork = cache.fork(a)
    assert cache.append(0, batch, kv, kv) == "appended" and cache.attention(0, batch, kv, 1.0) == "attended"
    if what == "freed":
        cache.free(a)
    elif what == "truncated":
        cache.truncate(a, 3)
    else:
        cache.extend([a], [1])
    for call in (lambda: cache.append(0, batch, kv, kv), lambda: cache.attention(0, batch, kv, 1.0)):
        with pytest.raises(TurboPiError, match=what):
            call()
    assert cache.attention(0, alone, kv, 1.0) == "attended"
    cache.extend([fork, other], [1, 1], out=batch)           # written anew, it holds again, and for these sequences
    assert cache.append(0, batch, kv[:2], kv[:2]) == "appended"
    if what != "freed":
        cache.free(a)
        assert cache.attention(0, batch, kv, 1.0) == "attended"
    cache.free(fork)
    with pytest.raises(TurboPiError, match="freed"):
        cache.attention(0, batch, kv, 1.0)


def test_a_batch_of_another_cache_is_refused(cpu_copies):
    one, two = _cache(), _cache()
    batch, seq = one.extend([one.add()], [1]), two.add()
    kv = torch.zeros(1, 1, 8)
    for call in (lambda: two.append(0, batch, kv, kv), lambda: two.attention(0, batch, kv, 1.0), lambda: two.extend([seq], [1], out=batch)):
        with pytest.raises(TurboPiError, match="another cache"):
            call()
    assert two.length(seq) == 0 and two.free_pages == two.num_pages

"""What PagedCache does when a call of it fails: arguments of the wrong kind, a launch or an upload that does not come about."""
import pytest
import torch

from turbopi_b200 import ops
from turbopi_b200._lib import TurboPiError
from turbopi_b200.paged_cache import PagedCache


def _cache(num_pages=12, page_size=4, max_pages=6):
    return PagedCache(2, num_pages, page_size, 1, 8, max_pages, dtype=torch.float16, device="cpu")


def _state(cache):
    return {s: (list(e[0]), e[1], len(e[2])) for s, e in cache._seqs.items()}, list(cache._refs), sorted(cache._free)


@pytest.mark.parametrize("seqs,new", [([[1]], [1]), ([{}], [1]), ([None], [1]), (None, [1]), (1, [1]), ([1], None), ([1], [None]), ([1], ["x"]),
                                      ([1], [1.5]), ([1], [float("nan")]), ([1], [2 ** 70])])
def test_arguments_of_the_wrong_kind(seqs, new):
    cache = _cache()
    cache.extend([cache.add()], [3])
    before = _state(cache)
    with pytest.raises(TurboPiError):
        cache.extend(seqs, new)
    assert _state(cache) == before


def test_batches_and_lengths_of_the_wrong_kind():
    cache = _cache()
    a = cache.add()
    cache.extend([a], [6])
    before = _state(cache)
    for call in (lambda: cache.batch(None), lambda: cache.batch(a), lambda: cache.batch([[a]]), lambda: cache.truncate(a, None),
                 lambda: cache.truncate(a, 1.5), lambda: cache.truncate(a, "2"), lambda: cache.truncate([a], 2)):
        with pytest.raises(TurboPiError):
            call()
    assert _state(cache) == before
    cache.truncate(a, 2.0)
    assert cache.length(a) == 2 and len(cache.page_ids(a)) == 1


def test_arguments_of_other_kinds_that_are_fine():
    cache = _cache()
    a, b = cache.add(), cache.add()
    assert cache.extend((a, b), torch.tensor([2, 0])).lengths.tolist() == [2, 0]
    assert cache.extend(iter([b]), (3.0,)).lengths.tolist() == [3]


def _pages(cache):
    return {s: (cache.page_ids(s), cache.length(s)) for s in cache._seqs}, list(cache._refs), sorted(cache._free)


def _shared(cache):
    """Two sequences on one half-filled page, a third beside them, and a batch of each."""
    a, c = cache.add(), cache.add()
    cache.extend([a, c], [6, 5])
    b = cache.fork(a)
    return a, b, c, [cache.batch([s]) for s in (a, b, c)]


@pytest.mark.parametrize("out", [False, True])
@pytest.mark.parametrize("what", ["copy", "upload"])
def test_extend_changes_nothing_when_a_step_of_it_fails(monkeypatch, what, out):
    """The copy of a shared page, or the upload of the tables: pages, lengths and batches are as they were, and the next call works."""
    cache = _cache()
    a, b, c, batches = _shared(cache)
    before, tables = _pages(cache), [x.table.clone() for x in batches]

    def fail(*args):
        raise TurboPiError("this step fails")
    with monkeypatch.context() as m:
        m.setattr(*((ops, "copy_pages", fail) if what == "copy" else (cache, "_upload", fail)))
        if what == "upload":
            m.setattr(ops, "copy_pages", lambda *args: None)
        with pytest.raises(TurboPiError, match="this step fails"):
            cache.extend([a, c, b], [7, 4, 1], out=cache.batch([a, c, b]) if out and what == "copy" else None)
    assert _pages(cache) == before
    for batch, table in zip(batches, tables):
        cache._current(batch)
        assert torch.equal(batch.table, table)
    copied = []
    monkeypatch.setattr(ops, "copy_pages", lambda pages, src, dst: copied.append((src, dst)))
    last = cache.page_ids(a)[1]
    batch = cache.extend([a, c, b], [7, 4, 1])
    assert batch.lengths.tolist() == [13, 9, 7]
    assert copied == [([last], [cache.page_ids(a)[1]])] and cache.page_ids(b)[1] == last
    # the copied page's sequence has to have its batches made again, the others hold
    with pytest.raises(TurboPiError, match="copied"):
        cache._current(batches[0])
    cache._current(batches[1])
    cache._current(batches[2])


def test_compaction_changes_nothing_when_its_copy_fails(monkeypatch):
    cache = _cache()
    a, b, c, batches = _shared(cache)
    cache.free(a)
    cache.free(b)
    before = _state(cache)

    def fail(*args):
        raise TurboPiError("this step fails")
    with monkeypatch.context() as m:
        m.setattr(ops, "copy_pages", fail)
        with pytest.raises(TurboPiError, match="this step fails"):
            cache.compact()
    assert _state(cache) == before
    cache._current(batches[2])

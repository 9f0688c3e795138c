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

"""PagedBatch objects made by hand, with the five arguments that they have always taken, as `out` of PagedCache.extend."""
import torch

from turbopi_b200.paged_cache import PagedBatch, PagedCache


def test_a_batch_made_by_hand_is_written():
    cache = PagedCache(1, 20, 16, 1, 64, 8, device="cpu")
    seqs = [cache.add(), cache.add()]
    cache.extend(seqs, [20, 3])
    table, lengths, cu = (torch.zeros(s, dtype=torch.int32) for s in ((2, 8), (2,), (3,)))
    mine = PagedBatch(table, lengths, cu, 0, cache)
    batch = cache.extend(seqs, [1, 2], out=mine)
    assert batch is mine and batch.table is table and batch.lengths is lengths and batch.cu is cu
    assert lengths.tolist() == [21, 5] and cu.tolist() == [0, 1, 3] and batch.tokens == 3
    assert batch.cu_keys.tolist() == [0, 21, 26] and batch.keys == 26
    kept = batch.cu_keys
    cache.extend(seqs, [0, 4], out=mine)
    assert batch.cu_keys is kept and kept.tolist() == [0, 21, 30] and batch.keys == 30
    assert [cache.length(s) for s in seqs] == [21, 9]

"""A KV cache of pages that many sequences share.

The pages of every layer lie in one tensor [layers, 2, pages, page_size, kv_heads, head_dim]; a sequence is a list of page ids
and a length.  Which page belongs to whom is kept on the host (reference counts, lowest free page first, so the same calls give the
same pages); the bytes are moved by `ops.copy_pages`, written by `ops.paged_append` and read by `ops.paged_attention`.

    cache = PagedCache(layers=18, num_pages=4096, page_size=16, kv_heads=1, head_dim=256, max_pages=64, device="cuda")
    a = cache.add()
    batch = cache.extend([a], [len(prompt)])            # room for the prompt: table, lengths and offsets on the device
    for l in range(18):                                 # per layer: q, k, v of the prompt's tokens [T, heads, head_dim]
        q = cache.append(l, batch, k, v, q=q, cos=cos, sin=sin)
        ...
    b = cache.fork(a)                                   # shares every page; the half-filled last one is copied by whoever writes first
    batch = cache.extend([a, b], [1, 1])                # one decode step of both
    for l in range(18):
        q = cache.append(l, batch, k, v, q=q, cos=cos, sin=sin)
        out = cache.attention(l, batch, q, scale)

A batch holds for its cache until one of its sequences is freed, truncated or had a shared page copied, or pages have moved (compact);
then `append` and `attention` refuse it, since its table may name pages of others.  `append` also refuses tokens whose page has been copied
to a fork, which would lack them: write a batch's tokens before extending a fork of its sequences.  Calls that move or write pages enqueue on the
current stream; use one stream per cache, or order them yourself.
"""
import heapq
import weakref

import torch

from . import ops
from ._lib import TurboPiError


class PagedBatch:
    """What the kernels read of some sequences: table int32 [S, max_pages], lengths int32 [S] (the new tokens among them) and cu int32
    [S + 1], the offsets of the new tokens; `tokens` is their number."""

    def __init__(self, table, lengths, cu, tokens, cache):
        self.table, self.lengths, self.cu, self.tokens = table, lengths, cu, tokens
        # _new: sequence -> [first, last + 1) of its new tokens' positions; _stale: why it no longer holds, _late: why its tokens can
        # no longer be written in a layer that is not among _layers, the ones where `append` wrote them
        self._cache, self._new, self._stale, self._late, self._layers = weakref.ref(cache), {}, None, None, set()


def _whole(x):
    n = int(x)
    if n != x:
        raise ValueError(f"{x} is no whole number")
    return n


class PagedCache:
    def __init__(self, layers, num_pages, page_size, kv_heads, head_dim, max_pages, dtype=torch.bfloat16, device="cuda"):
        if min(layers, num_pages, page_size, kv_heads, max_pages) < 1 or not 8 <= head_dim <= 256 or head_dim % 8:
            raise TurboPiError("PagedCache: sizes must be positive, head_dim a multiple of 8 up to 256")
        if page_size * max_pages >= 2 ** 31:
            raise TurboPiError("PagedCache: positions are 32 bits wide")
        if dtype not in (torch.bfloat16, torch.float16):
            raise TurboPiError("PagedCache: bf16 or fp16")
        self.page_size, self.max_pages, self.num_pages = page_size, max_pages, num_pages
        self.device = torch.device(device)
        # zeroed once: rows of a page that no token has reached are masked, not left out of the copies
        self.pages = torch.zeros((layers, 2, num_pages, page_size, kv_heads, head_dim), dtype=dtype, device=self.device)
        self._free = list(range(num_pages))           # a heap
        self._refs = [0] * num_pages
        self._seqs = {}                               # id -> [page ids, length, batches that name its pages]
        self._next = 0

    # ------------------------------------------------------------------ sequences
    def _get(self, seq):
        try:
            return self._seqs[seq]
        except (KeyError, TypeError):
            raise TurboPiError(f"PagedCache: no sequence {seq!r}") from None

    def add(self):
        """A new sequence without tokens; returns its id."""
        self._next += 1
        self._seqs[self._next] = [[], 0, weakref.WeakSet()]
        return self._next

    def length(self, seq):
        return self._get(seq)[1]

    def page_ids(self, seq):
        return list(self._get(seq)[0])

    @property
    def free_pages(self):
        return len(self._free)

    def _release(self, page):
        self._refs[page] -= 1
        if self._refs[page] == 0:
            heapq.heappush(self._free, page)

    def free(self, seq):
        """Gives the sequence up; pages that no other one shares are free again."""
        entry = self._get(seq)
        for page in entry[0]:
            self._release(page)
        self._outdate(entry, f"sequence {seq} was freed")
        del self._seqs[seq]

    def fork(self, seq):
        """A second sequence with the same tokens, on the same pages; returns its id.  Nothing is copied until one of them is extended
        within the page they share last.  By then tokens that a batch has made room for there must be written, in every layer: the copy
        lacks later ones, and `append` refuses to write them.  (A captured graph that writes them is not seen here.)"""
        pages, length, _ = self._get(seq)
        for page in pages:
            self._refs[page] += 1
        self._next += 1
        self._seqs[self._next] = [list(pages), length, weakref.WeakSet()]
        return self._next

    def truncate(self, seq, length):
        """Forgets the tokens from position `length` on."""
        entry = self._get(seq)
        try:
            length = _whole(length)
        except (TypeError, ValueError, OverflowError):
            raise TurboPiError(f"PagedCache: cannot truncate to {length!r} tokens") from None
        if not 0 <= length <= entry[1]:
            raise TurboPiError(f"PagedCache: cannot truncate {entry[1]} tokens to {length}")
        keep = -(-length // self.page_size)
        for page in entry[0][keep:]:
            self._release(page)
        if length < entry[1]:
            self._outdate(entry, f"sequence {seq} was truncated")
        entry[0], entry[1] = entry[0][:keep], length

    @staticmethod
    def _outdate(entry, why):
        for batch in entry[2]:
            batch._stale = why
        entry[2].clear()

    # ------------------------------------------------------------------ room for tokens
    def extend(self, seqs, new, out=None):
        """Room for new[i] >= 0 more tokens of sequence seqs[i]; returns the PagedBatch for `append` and `attention`.  Pages are
        allocated, and a half-filled last page that another sequence shares is copied first (every layer).  All or nothing: where pages
        run out, or a step fails, nothing has changed.  `out`: a PagedBatch of as many sequences whose tensors are written (a captured graph
        reads them)."""
        try:
            seqs, new = list(seqs), [_whole(n) for n in new]
            fine = len(seqs) == len(new) and len(set(seqs)) == len(seqs) and all(n >= 0 for n in new)
        except (TypeError, ValueError, OverflowError):
            fine = False
        if not fine:
            raise TurboPiError("PagedCache: extend takes different sequences and a number of new tokens >= 0 for each")
        if out is not None and (out._cache() is not self or out.lengths.shape[0] != len(seqs)):
            raise TurboPiError("PagedCache: `out` is a batch of another cache or number of sequences")
        page, plan, taken = self.page_size, [], 0
        refs = {}                                     # of shared last pages, as the plan leaves them
        for seq, n in zip(seqs, new):
            pages, length, _ = self._get(seq)
            total = -(-(length + n) // page)
            if total > self.max_pages:
                raise TurboPiError(f"PagedCache: {length + n} tokens need more than {self.max_pages} pages")
            copied = False
            if n > 0 and length % page:
                last = pages[-1]
                count = refs.get(last, self._refs[last])
                copied = count > 1
                refs[last] = count - copied
            plan.append((copied, total - len(pages)))
            taken += copied + total - len(pages)
        if taken > len(self._free):
            raise TurboPiError(f"PagedCache: {taken} pages needed, {len(self._free)} free")
        fresh = [heapq.heappop(self._free) for _ in range(taken)]
        try:                                          # what may fail comes before anything is changed
            take, held, src, dst = iter(fresh), [], [], []
            for seq, (copied, more) in zip(seqs, plan):
                pages = list(self._seqs[seq][0])
                if copied:
                    src.append(pages[-1])
                    pages[-1] = next(take)
                    dst.append(pages[-1])
                pages.extend(next(take) for _ in range(more))
                held.append(pages)
            if src:
                ops.copy_pages(self.pages, src, dst)
            tensors = self._tensors(held, [self._seqs[seq][1] + n for seq, n in zip(seqs, new)], new)
        except BaseException:
            for p in fresh:
                heapq.heappush(self._free, p)
            raise
        if src:
            self._copied([(seq, *self._seqs[seq][:2]) for seq, (copied, _) in zip(seqs, plan) if copied])
        for p in fresh:
            self._refs[p] = 1
        for seq, n, pages, (copied, _) in zip(seqs, new, held, plan):
            entry = self._seqs[seq]
            if copied:
                self._release(entry[0][-1])
                self._outdate(entry, f"a shared page of sequence {seq} was copied")
            entry[0] = pages
            entry[1] += n
        return self._batch(seqs, new, tensors, out)

    def _copied(self, copies):
        """The last pages of some sequences, (sequence, page ids, length) each, were copied for them: tokens that others were still to
        write there, below that length, are not in the copy."""
        page, where = self.page_size, {}
        for seq, pages, length in copies:                        # a page has the same place in all that share it
            where.setdefault((len(pages) - 1, pages[-1]), []).append((seq, length))
        low, high = min(i for i, _ in where), max(i for i, _ in where)
        for other, (held, _, batches) in self._seqs.items():
            for batch in batches:
                first, last = batch._new.get(other, (0, 0))
                for i in range(max(low, first // page), min(high + 1, len(held), -(-last // page))):
                    for seq, length in where.get((i, held[i]), ()):
                        if other != seq and max(first, i * page) < min(last, length):
                            batch._late = f"a page with new tokens of sequence {other} was copied to sequence {seq}"

    def batch(self, seqs):
        """The PagedBatch of sequences as they are, without new tokens."""
        try:
            seqs = list(seqs)
        except TypeError:
            raise TurboPiError("PagedCache: batch takes sequences") from None
        return self.extend(seqs, [0] * len(seqs))

    def _upload(self, values, shape):
        t = torch.tensor(values, dtype=torch.int32).reshape(shape)
        return t.pin_memory().to(self.device, non_blocking=True) if self.device.type == "cuda" else t

    def _tensors(self, held, lengths, new):
        """Tables, lengths and offsets in one copy to the device."""
        S, W = len(held), self.max_pages
        rows, cu = [], [0]
        for pages, n in zip(held, new):
            rows += pages + [-1] * (W - len(pages))
            cu.append(cu[-1] + n)
        flat = self._upload(rows + lengths + cu, (-1,))
        return flat[:S * W].view(S, W), flat[S * W:S * W + S], flat[S * W + S:]

    def _batch(self, seqs, new, tensors, out):
        table, lengths, offsets = tensors
        if out is None:
            out = PagedBatch(table, lengths, offsets, sum(new), self)
        else:
            for seq in out._new:
                if seq in self._seqs:
                    self._seqs[seq][2].discard(out)
            out.table.copy_(table)
            out.lengths.copy_(lengths)
            out.cu.copy_(offsets)
            out.tokens, out._stale, out._late, out._layers = sum(new), None, None, set()
        out._new = {seq: (self._seqs[seq][1] - n, self._seqs[seq][1]) for seq, n in zip(seqs, new)}
        for seq in seqs:
            self._seqs[seq][2].add(out)
        return out

    # ------------------------------------------------------------------ the device side
    def layer(self, layer):
        """(key pages, value pages) of a layer, views [pages, page_size, kv_heads, head_dim]."""
        return self.pages[layer, 0], self.pages[layer, 1]

    def _current(self, batch):
        if batch._cache() is not self:
            raise TurboPiError("PagedCache: a batch of another cache")
        if batch._stale:
            raise TurboPiError(f"PagedCache: {batch._stale} since this batch was made; make it again")

    def append(self, layer, batch, k, v, q=None, cos=None, sin=None, q_out=None):
        """ops.paged_append of the batch's new tokens: k, v (and q) [batch.tokens, heads, head_dim], sequence by sequence."""
        self._current(batch)
        layer = range(self.pages.shape[0])[layer]
        if batch._late and layer not in batch._layers:
            raise TurboPiError(f"PagedCache: {batch._late} before this append; append in every layer before a fork is extended")
        if k.shape[0] != batch.tokens:
            raise TurboPiError(f"PagedCache: {k.shape[0]} rows for {batch.tokens} new tokens")
        out = ops.paged_append(k, v, *self.layer(layer), batch.table, batch.cu, batch.lengths, q=q, cos=cos, sin=sin, q_out=q_out)
        batch._layers.add(layer)
        return out

    def attention(self, layer, batch, q, scale, out=None, workspace=None):
        """ops.paged_attention of one query row per sequence of the batch, over all its tokens."""
        self._current(batch)
        return ops.paged_attention(q, *self.layer(layer), batch.table, batch.lengths, scale, out=out, workspace=workspace)

    def compact(self):
        """Moves pages so that those in use are the lowest ids, each at most once; returns how many are in use.  Batches made before
        are refused afterwards; a captured graph needs its batch written anew (`extend(out=)`)."""
        used = self.num_pages - len(self._free)
        low = sorted(p for p in self._free if p < used)
        high = [p for p in range(used, self.num_pages) if self._refs[p] > 0]
        if not high:
            return used
        ops.copy_pages(self.pages, high, low)
        to = dict(zip(high, low))
        for entry in self._seqs.values():
            entry[0] = [to.get(p, p) for p in entry[0]]
            self._outdate(entry, "pages have moved (compact)")
        for a, b in to.items():
            self._refs[b], self._refs[a] = self._refs[a], 0
        self._free = list(range(used, self.num_pages))          # sorted, which is a heap
        return used

"""The operators as a server uses them: a batch of prompts through packed attention into the cache, forks, decode steps on the pages,
freed and compacted pages, a decode step replayed as a graph; every output against attention in 64 bits on the tokens written."""
import pytest
import torch

from paged_reference import attend, check, rotate

pytestmark = pytest.mark.gpu


class _Model:
    """Per layer random queries, keys and values for tokens; remembers the (rotated, rounded) keys and values of each sequence."""

    def __init__(self, cache, layers, hq, hk, D, dtype, device, rope):
        self.cache, self.layers, self.hq, self.hk, self.D, self.dtype, self.device = cache, layers, hq, hk, D, dtype, device
        self.g = torch.Generator(device=device).manual_seed(0)
        a = torch.arange(600, device=device, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, D, 2, device=device, dtype=torch.float64) / D)
        self.cos, self.sin = (a.cos().float(), a.sin().float()) if rope else (None, None)
        self.seen = {}
        self.scale = D ** -0.5

    def rows(self, n):
        return torch.randn((n, self.hq + 2 * self.hk, self.D), generator=self.g, device=self.device, dtype=self.dtype).split([self.hq, self.hk, self.hk], 1)

    def _keep(self, seqs, new, k, v, layer):
        at = 0
        for s, n in zip(seqs, new):
            old = self.seen.setdefault(s, [None] * self.layers)
            kk = k[at:at + n].double()
            if self.cos is not None:
                pos = torch.arange(self.cache.length(s) - n, self.cache.length(s), device=self.device)
                kk = rotate(kk, self.cos[pos], self.sin[pos])
            kk = kk.to(self.dtype)
            old[layer] = (kk, v[at:at + n]) if old[layer] is None else (torch.cat([old[layer][0], kk]), torch.cat([old[layer][1], v[at:at + n]]))
            at += n

    def fork(self, s):
        t = self.cache.fork(s)
        self.seen[t] = list(self.seen[s])
        return t

    def step(self, seqs, new, prompt, pdl=False):
        """All layers of a batch: prompts are attended to among themselves, single tokens on the cache."""
        from turbopi_b200 import ops
        batch = self.cache.extend(seqs, new)
        for layer in range(self.layers):
            q, k, v = self.rows(sum(new))
            kw = dict(q=q, cos=self.cos, sin=self.sin) if self.cos is not None else {}
            with ops.launch_flags(ops.FLAG_PDL if pdl else ops.FLAG_NONE):
                turned = self.cache.append(layer, batch, k, v, **kw)
                turned = q if turned is None else turned
                if prompt:
                    keys, values = (torch.cat([self._read(layer, s)[i] for s in seqs]) for i in (0, 1))
                    out = ops.packed_attention(turned, keys, values, batch.cu, self.scale)
                else:
                    out = self.cache.attention(layer, batch, turned, self.scale)
            self._keep(seqs, new, k, v, layer)
            at = 0
            for s, n in zip(seqs, new):
                keys, values = self.seen[s][layer]
                got = self._read(layer, s)
                assert torch.equal(got[1], values)
                assert bool(((got[0].double() - keys.double()).abs() <= 2.0 ** -7 * keys.double().abs() + 1e-6).all())   # rounded twice at most
                want, allow = attend(turned[at:at + n], got[0], got[1], self.scale, keys.shape[0] - n)
                check(out[at:at + n], want, allow)
                at += n

    def _read(self, layer, s):
        ids = torch.tensor(self.cache.page_ids(s), device=self.device)
        return [p[ids].flatten(0, 1)[:self.cache.length(s)] for p in self.cache.layer(layer)]


@pytest.mark.parametrize("hq,hk,D,dtype,page,rope", [(8, 1, 256, torch.bfloat16, 16, True), (8, 2, 128, torch.float16, 24, False),
                                                     (4, 4, 64, torch.bfloat16, 32, True)])
def test_a_served_batch(cuda_device, hq, hk, D, dtype, page, rope):
    from turbopi_b200 import _lib
    from turbopi_b200.paged_cache import PagedCache
    layers = 2
    cache = PagedCache(layers, 80, page, hk, D, 24, dtype=dtype, device=cuda_device)
    m = _Model(cache, layers, hq, hk, D, dtype, cuda_device, rope)
    a, b, c = cache.add(), cache.add(), cache.add()
    m.step([a, b, c], [133, 1, 260], prompt=True)
    for i in range(3):
        m.step([c, a, b], [1, 1, 1], prompt=False, pdl=i > 0)
    d, e = m.fork(a), m.fork(a)
    for _ in range(2):
        m.step([a, b, d, e], [1, 1, 1, 1], prompt=False)         # a, d, e go apart inside a page
    cache.free(a)
    cache.free(b)
    f = cache.add()
    m.step([f], [70], prompt=True)                               # on freed pages, among what was there before
    cache.free(c)
    used = cache.compact()
    assert used == cache.num_pages - cache.free_pages and max(p for s in (d, e, f) for p in cache.page_ids(s)) < used
    cache.pages[:, :, used:] = float("nan")                      # what lies above belongs to nobody
    for _ in range(page + 1):
        m.step([d, f, e], [1, 1, 1], prompt=False)
    assert _lib.load().tpb200_device_error(0) == 0


def test_a_decode_step_as_a_graph(cuda_device):
    """One captured step for batches written anew: append, attention, the next append on its output, on the same addresses."""
    from turbopi_b200 import ops
    from turbopi_b200.paged_cache import PagedCache
    cache = PagedCache(1, 40, 16, 1, 256, 12, device=cuda_device)
    m = _Model(cache, 1, 8, 1, 256, torch.bfloat16, cuda_device, False)
    seqs = [cache.add(), cache.add()]
    m.step(seqs, [50, 31], prompt=True)
    batch = cache.extend(seqs, [1, 1])
    q, k, v = (t.contiguous() for t in m.rows(2))
    out, ws = torch.empty_like(q), ops.paged_attention_workspace(8, 1, 256, cuda_device)

    def step():
        cache.append(0, batch, k, v)
        cache.attention(0, batch, q, m.scale, out=out, workspace=ws)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(20):
        if i:
            batch = cache.extend(seqs, [1, 1], out=batch)
        for t, fresh in zip((q, k, v), m.rows(2)):
            t.copy_(fresh)
        graph.replay()
        m._keep(seqs, [1, 1], k.clone(), v.clone(), 0)
        for j, s in enumerate(seqs):
            keys, values = m._read(0, s)
            assert torch.equal(keys, m.seen[s][0][0]) and torch.equal(values, m.seen[s][0][1])
            want, allow = attend(q[j:j + 1], keys, values, m.scale)
            check(out[j:j + 1], want, allow)


@pytest.mark.parametrize("hq,hk,D,dtype", [(8, 1, 256, torch.bfloat16), (6, 2, 64, torch.float16)])
def test_prompts_from_a_fused_projection(cuda_device, hq, hk, D, dtype):
    """Queries and keys are neighbouring columns of a projection: rotated together, the keys come back packed, as they lie in the pages."""
    from turbopi_b200 import ops
    from turbopi_b200.paged_cache import PagedCache
    cache = PagedCache(1, 40, 16, hk, D, 12, dtype=dtype, device=cuda_device)
    g = torch.Generator(device=cuda_device).manual_seed(5)
    lens = [37, 1, 150]
    seqs = [cache.add() for _ in lens]
    qkv = torch.randn((sum(lens), hq + 2 * hk, D), generator=g, device=cuda_device, dtype=dtype)
    cos, sin = ops.rope_tables(160, D, device=cuda_device)
    batch, v = cache.extend(seqs, lens), qkv[:, hq + hk:]
    turned = cache.append(0, batch, qkv[:, hq:hq + hk], v, q=qkv[:, :hq + hk], cos=cos, sin=sin)
    out = ops.packed_attention(turned[:, :hq], turned[:, hq:], v, batch.cu, D ** -0.5)
    at = 0
    for s, n in zip(seqs, lens):
        ids = torch.tensor(cache.page_ids(s), device=cuda_device)
        keys, values = (p[ids].flatten(0, 1)[:n] for p in cache.layer(0))
        assert torch.equal(keys, turned[at:at + n, hq:]) and torch.equal(values, v[at:at + n])
        pos = torch.arange(n, device=cuda_device)
        wanted = rotate(qkv[at:at + n, :hq].double(), cos[pos], sin[pos])
        # rounded once, the rotation itself in fp32: half a step, and three roundings of 2^-24 of the pair's largest product
        half, size = torch.finfo(dtype).eps / 2, qkv[at:at + n, :hq].double().abs().amax(-1, keepdim=True)
        assert bool(((turned[at:at + n, :hq].double() - wanted).abs() <= half * wanted.abs() + 8 * 2.0 ** -24 * size + torch.finfo(dtype).tiny).all())
        want, allow = attend(turned[at:at + n, :hq], keys, values, D ** -0.5, 0)
        check(out[at:at + n], want, allow)
        at += n

"""A 4-bit PagedCache as a server uses it: prompts behind cached tokens, forks, decode steps, freed and compacted pages, windows, a decode step
replayed as a graph; every output against attention in 64 bits on what the cache holds, and that against what was written."""
import pytest
import torch

from nvfp4_cache_reference import attend, held, quantise, seen, values
from paged_reference import check, rotate

pytestmark = pytest.mark.gpu

WEIGHT = 2.0 ** -11


def _no_error():
    from turbopi_b200 import _lib
    assert _lib.load().tpb200_device_error(0) == 0


class _Model:
    def __init__(self, cache, layers, hq, hk, D, dtype, device, rope, window=None, sinks=0):
        self.cache, self.layers, self.hq, self.hk, self.D, self.dtype, self.device = cache, layers, hq, hk, D, dtype, device
        self.g = torch.Generator(device=device).manual_seed(0)
        a = torch.arange(900, device=device, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, D, 2, device=device, dtype=torch.float64) / D)
        self.cos, self.sin = (a.cos().float(), a.sin().float()) if rope else (None, None)
        self.window, self.sinks, self.scale, self.seen = window, sinks, D ** -0.5, {}

    def rows(self, n):
        return torch.randn((n, self.hq + 2 * self.hk, self.D), generator=self.g, device=self.device, dtype=self.dtype).split([self.hq, self.hk, self.hk], 1)

    def fork(self, s):
        t = self.cache.fork(s)
        self.seen[t] = [x for x in self.seen[s]]
        return t

    def held(self, layer, s):
        """(keys, values) of a sequence in 64 bits."""
        ids = torch.tensor(self.cache.page_ids(s), device=self.device, dtype=torch.long)
        return [held(p[ids], self.D).flatten(0, 1)[:self.cache.length(s)] for p in self.cache.layer(layer)]

    def step(self, seqs, new, prompt):
        from turbopi_b200 import ops
        batch = self.cache.extend(seqs, new)
        assert batch.keys == sum(self.cache.length(s) for s in seqs)
        for layer in range(self.layers):
            q, k, v = self.rows(sum(new))
            kw = dict(q=q, cos=self.cos, sin=self.sin) if self.cos is not None else {}
            with ops.launch_flags(ops.FLAG_PDL):
                turned = self.cache.append(layer, batch, k, v, **kw)
                turned = q if turned is None else turned
                call = self.cache.prompt_attention if prompt else self.cache.attention
                out = call(layer, batch, turned, self.scale, window=self.window, sinks=self.sinks)
                kk, vv = self.cache.read(layer, batch, dtype=self.dtype)
            at = key = 0
            for s, n in zip(seqs, new):
                m = self.cache.length(s)
                have = self.held(layer, s)
                assert torch.equal(kk[key:key + m].double(), have[0]) and torch.equal(vv[key:key + m].double(), have[1])
                # values as their definition has them; keys within what a rotation's two roundings move them, a level at most where those cross a border
                assert torch.equal(have[1][m - n:], values(*quantise(v[at:at + n]), self.D))
                x = k[at:at + n].double()
                if self.cos is not None:
                    x = rotate(x, self.cos[m - n:m], self.sin[m - n:m])
                top = torch.nn.functional.pad(x.abs(), (0, -self.D % 16)).unflatten(-1, (-1, 16)).amax(-1).repeat_interleave(16, -1)[..., :self.D]
                # half a level is a sixth of the largest at most, the scale is off by 2^-4 and the rounding to 16 bits by 2^-8
                assert bool(((have[0][m - n:] - x).abs() <= top * (1 / 6 + 2.0 ** -4 + 2.0 ** -7)).all())
                old = self.seen.setdefault(s, [None] * self.layers)
                if old[layer] is not None:       # what was there is there
                    assert all(torch.equal(a, b[:m - n]) for a, b in zip(old[layer], have))
                old[layer] = have
                want, allow = attend(turned[at:at + n], *have, self.scale, seen(n, m, self.window, self.sinks, self.device), None if prompt else WEIGHT)
                check(out[at:at + n], want, allow)
                at, key = at + n, key + m


@pytest.mark.parametrize("hq,hk,D,dtype,page,rope,window,sinks", [(8, 1, 256, torch.bfloat16, 16, True, None, 0), (8, 2, 128, torch.float16, 32, False, 40, 4),
                                                                  (4, 4, 64, torch.bfloat16, 16, True, 100, 20), (6, 2, 72, torch.bfloat16, 48, True, None, 0)])
def test_a_served_batch(cuda_device, hq, hk, D, dtype, page, rope, window, sinks):
    from turbopi_b200.paged_cache import PagedCache
    layers = 2
    cache = PagedCache(layers, 120, page, hk, D, 40, dtype="nvfp4", device=cuda_device)
    m = _Model(cache, layers, hq, hk, D, dtype, cuda_device, rope, window, sinks)
    a, b, c = cache.add(), cache.add(), cache.add()
    m.step([a, b, c], [133, 1, 260], prompt=True)
    for _ in range(3):
        m.step([c, a, b], [1, 1, 1], prompt=False)
    m.step([b, a], [70, 5], prompt=True)                         # a turn of the conversation: prompts behind cached tokens
    d, e = m.fork(a), m.fork(a)
    for _ in range(2):
        m.step([a, b, d, e], [1, 1, 1, 1], prompt=False)         # a, d, e go apart inside a page
    cache.free(a)
    cache.free(b)
    f = cache.add()
    m.step([f], [70], prompt=True)                               # on freed pages, among what was there before
    cache.free(c)
    used = cache.compact()
    cache.pages[:, :, used:] = 127                               # what lies above belongs to nobody
    for _ in range(page + 1):
        m.step([d, f, e], [1, 1, 1], prompt=False)
    _no_error()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_prompts_behind_a_cache_in_16_bits(cuda_device, dtype):
    """PagedCache.read and prompt_attention on 16-bit pages."""
    from turbopi_b200.paged_cache import PagedCache
    cache = PagedCache(1, 60, 24, 2, 128, 20, dtype=dtype, device=cuda_device)
    g = torch.Generator(device=cuda_device).manual_seed(0)
    a, b = cache.add(), cache.add()
    kept = {a: [], b: []}
    for new in ([100, 30], [1, 0], [50, 200]):
        batch = cache.extend([a, b], new)
        q = torch.randn((sum(new), 4, 128), generator=g, device=cuda_device, dtype=dtype)
        k, v = torch.randn((2, sum(new), 2, 128), generator=g, device=cuda_device, dtype=dtype)
        cache.append(0, batch, k, v)
        kept[a].append((k[:new[0]], v[:new[0]]))
        kept[b].append((k[new[0]:], v[new[0]:]))
        all_k, all_v = (torch.cat([x[i] for s in (a, b) for x in kept[s]]) for i in (0, 1))
        kk, vv = cache.read(0, batch)
        assert kk.dtype == dtype and torch.equal(kk, all_k) and torch.equal(vv, all_v)
        for window, sinks in ((None, 0), (60, 4)):
            out = cache.prompt_attention(0, batch, q, 0.09, window=window, sinks=sinks)
            q0 = k0 = 0
            for s, n in zip((a, b), new):
                m = cache.length(s)
                want, allow = attend(q[q0:q0 + n], kk[k0:k0 + m], vv[k0:k0 + m], 0.09, seen(n, m, window, sinks, cuda_device))
                check(out[q0:q0 + n], want, allow)
                q0, k0 = q0 + n, k0 + m
    _no_error()


def test_a_decode_step_as_a_graph(cuda_device):
    from turbopi_b200 import ops
    from turbopi_b200.paged_cache import PagedCache
    cache = PagedCache(1, 40, 16, 1, 256, 12, dtype="nvfp4", device=cuda_device, k_scale=2.0, v_scale=0.5)
    seqs = [cache.add(), cache.add()]
    g = torch.Generator(device=cuda_device).manual_seed(0)
    k, v = torch.randn((2, 81, 1, 256), generator=g, device=cuda_device, dtype=torch.bfloat16)
    cache.append(0, cache.extend(seqs, [50, 31]), k, v)
    batch = cache.extend(seqs, [1, 1])
    q, k, v = (torch.randn((2, h, 256), generator=g, device=cuda_device, dtype=torch.bfloat16) for h in (8, 1, 1))
    out, ws = torch.empty_like(q), ops.paged_attention_nvfp4_workspace(8, 1, 256, cuda_device)

    def step():
        cache.append(0, batch, k, v)
        cache.attention(0, batch, q, 1 / 16, out=out, workspace=ws)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(20):
        if i:
            cache.extend(seqs, [1, 1], out=batch)
        for t in (q, k, v):
            t.normal_(generator=g)
        graph.replay()
        for j, s in enumerate(seqs):
            n = cache.length(s)
            ids = torch.tensor(cache.page_ids(s), device=cuda_device)
            kk, vv = (held(p[ids], 256).flatten(0, 1)[:n] * f for p, f in zip(cache.layer(0), (2.0, 0.5)))
            assert torch.equal(vv[n - 1], values(*quantise(v[j], 0.5), 256) * 0.5)
            want, allow = attend(q[j:j + 1], kk, vv, 1 / 16, seen(1, n, None, 0, cuda_device), WEIGHT)
            check(out[j:j + 1], want, allow)
    _no_error()


class _Recorder:
    def __init__(self, native):
        self._native, self.taken = native, []

    def __getattr__(self, name):
        def call(*args):
            done = getattr(self._native, name)(*args)
            self.taken.append((name, done is not None))
            return done
        return call


def _calls(device):
    from turbopi_b200 import ops
    g = torch.Generator(device=device).manual_seed(0)

    def t(*shape):
        return torch.randn(shape, generator=g, device=device).to(torch.bfloat16)
    q, k, v, cache = t(40, 8, 64), t(40, 2, 64), t(40, 2, 64), t(2, 9, 16, 2, 64)
    pages = torch.zeros(2, 9, 2, 1, 576, dtype=torch.uint8, device=device)
    cu = torch.tensor([0, 30, 40], dtype=torch.int32, device=device)
    table = torch.tensor([[4, 1, 0], [2, 8, -1]], dtype=torch.int32, device=device)
    lengths = torch.tensor([33, 20], dtype=torch.int32, device=device)
    cos, sin = torch.rand(64, 32, device=device), torch.rand(64, 32, device=device)
    ws = ops.paged_attention_nvfp4_workspace(8, 2, 64, device)
    rows = [torch.zeros(40, 2, 64, dtype=torch.float16, device=device) for _ in range(2)]

    def append(**kw):
        c = pages.clone()
        return ops.paged_append_nvfp4(k, v, c[0], c[1], table, cu, lengths, k_scale=2, **kw), c
    full = append()[1]
    return {"packed_attention_window": lambda: ops.packed_attention(q, k, v, cu, 0.1, window=9, sinks=2),
            "paged_attention_window": lambda: ops.paged_attention(q[:2], cache[0], cache[1], table, lengths, 0.1, window=9, sinks=2),
            "paged_attention_nvfp4": lambda: (ops.paged_attention_nvfp4(q[:2], full[0], full[1], table, lengths, 0.1),
                                              ops.paged_attention_nvfp4(q[:2], full[0], full[1], table, lengths, 0.1, workspace=ws, window=9, sinks=2, v_scale=4.0)),
            "paged_append_nvfp4": lambda: (append(), append(q=q, cos=cos, sin=sin)),
            "paged_read": lambda: ops.paged_read(cache[0], cache[1], table, cu, lengths, 40),
            "paged_read_nvfp4": lambda: (ops.paged_read_nvfp4(full[0], full[1], table, cu, lengths, 64, 40),
                                         tuple(x.clone() for x in ops.paged_read_nvfp4(full[0], full[1], table, cu, lengths, 64, 40, dtype=torch.float16, out=rows)))}


def _flat(x):
    if isinstance(x, (tuple, list)):
        return [z for y in x for z in _flat(y)]
    return [] if x is None else [x]


def test_the_native_forms_are_taken_and_agree(cuda_device, monkeypatch):
    from turbopi_b200 import _lib
    r = _Recorder(_lib.native())
    monkeypatch.setattr(_lib, "_native", r)
    calls = _calls(cuda_device)
    got = {}
    for name, call in calls.items():
        r.taken.clear()
        got[name] = [x.clone() for x in _flat(call())]
        assert r.taken and all(t == (name, True) for t in r.taken), (name, r.taken)
    monkeypatch.setattr(_lib, "_native", _lib._PythonForms())
    for name, call in calls.items():
        for a, b in zip(got[name], _flat(call()), strict=True):
            assert torch.equal(a, b), name
    _no_error()


def test_refusals_on_the_gpu(cuda_device):
    """The native forms leave to the Python forms what those refuse; small or missing workspaces."""
    from turbopi_b200 import ops
    from turbopi_b200._lib import TurboPiError
    x = torch.zeros(2, 4, 64, dtype=torch.bfloat16, device=cuda_device)
    k = torch.zeros(2, 2, 64, dtype=torch.bfloat16, device=cuda_device)
    pages = torch.zeros(2, 3, 2, 1, 576, dtype=torch.uint8, device=cuda_device)
    table, lengths, cu = (torch.zeros(s, dtype=torch.int32, device=cuda_device) for s in ((2, 3), (2,), (3,)))
    ws = ops.paged_attention_nvfp4_workspace(4, 2, 64, cuda_device)
    for bad in (lambda: ops.paged_attention_nvfp4(x, pages[0], pages[1], table, lengths, 1.0, workspace=ws[:-1]),
                lambda: ops.paged_attention_nvfp4(x, pages[0], pages[1], table, lengths, 1.0, workspace=ws[8:]),
                lambda: ops.paged_attention_nvfp4(x, pages[0], pages[1], table, lengths, 1.0, k_scale=3.0),
                lambda: ops.paged_attention_nvfp4(x.float(), pages[0], pages[1], table, lengths, 1.0),
                lambda: ops.paged_attention_nvfp4(x[..., :60], pages[0], pages[1], table, lengths, 1.0),
                lambda: ops.paged_append_nvfp4(k, k, pages[0], pages[0], table, cu, lengths),
                lambda: ops.paged_append_nvfp4(k, k, pages[0], pages[1], table.long(), cu, lengths),
                lambda: ops.paged_append_nvfp4(k, k, pages[0], pages[1], table, cu, lengths, v_scale=float("nan")),
                lambda: ops.paged_read_nvfp4(pages[0], pages[1], table, cu, lengths, 64, 2, out=(k, k)),
                lambda: ops.paged_read_nvfp4(pages[0], pages[1], table, cu, lengths, 64, -1),
                lambda: ops.paged_read_nvfp4(pages[0], pages[1], table, cu.cpu(), lengths, 64, 2),
                lambda: ops.paged_attention_nvfp4_workspace(4, 3, 64, cuda_device)):
        with pytest.raises(TurboPiError):
            bad()

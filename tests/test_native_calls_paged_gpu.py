"""The calls on packed prompts and paged caches take their C++ forms in the plain case; the Python forms give the same bits and say
what the C++ forms leave to them."""
import pytest
import torch

pytestmark = pytest.mark.gpu


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
    cu = torch.tensor([0, 30, 40], dtype=torch.int32, device=device)
    table = torch.tensor([[4, 1, 0], [2, 8, -1]], dtype=torch.int32, device=device)
    lengths = torch.tensor([33, 20], dtype=torch.int32, device=device)
    cos, sin = torch.rand(64, 32, device=device), torch.rand(64, 32, device=device)
    ws = ops.paged_attention_workspace(8, 2, 64, device)

    def append(**kw):
        c = cache.clone()
        return ops.paged_append(k, v, c[0], c[1], table, cu, lengths, **kw), c

    def copy(src, dst):
        c = cache.clone()
        ops.copy_pages(c, src, dst)
        return c
    return {"packed_attention": lambda: ops.packed_attention(q, k, v, cu, 0.1),
            "paged_attention": lambda: (ops.paged_attention(q[:2], cache[0], cache[1], table, lengths, 0.1),
                                        ops.paged_attention(q[:2], cache[0], cache[1], table, lengths, 0.1, workspace=ws)),
            "paged_append": lambda: (append(), append(q=q, cos=cos, sin=sin)), "copy_pages": lambda: copy([3, 1], [0, 7])}


def _flat(x):
    if isinstance(x, (tuple, list)):
        return [z for y in x for z in _flat(y)]
    return [x]


@pytest.mark.parametrize("name", ["packed_attention", "paged_attention", "paged_append", "copy_pages"])
def test_both_forms(cuda_device, monkeypatch, name):
    from turbopi_b200 import _lib
    call = _calls(cuda_device)[name]
    r = _Recorder(_lib.native())
    monkeypatch.setattr(_lib, "_native", r)
    got = _flat(call())
    assert r.taken and all(taken and n == name for n, taken in r.taken)
    monkeypatch.setattr(_lib, "_native", _lib._PythonForms())
    want = _flat(call())
    assert len(got) == len(want)
    for a, b in zip(got, want):
        assert (a is None and b is None) or torch.equal(a, b)


def test_refusals(cuda_device):
    """One wrong argument each, on tensors of the GPU."""
    from turbopi_b200 import ops
    from turbopi_b200._lib import TurboPiError

    def bad(match, f, *a, **kw):
        with pytest.raises(TurboPiError, match=match):
            f(*a, **kw)
    q = torch.zeros(4, 8, 64, dtype=torch.bfloat16, device=cuda_device)
    k = torch.zeros(4, 2, 64, dtype=torch.bfloat16, device=cuda_device)
    cu = torch.tensor([0, 4], dtype=torch.int32, device=cuda_device)
    bad("bf16 or fp16", ops.packed_attention, q.float(), k.float(), k.float(), cu, 1.0)
    bad("v must be", ops.packed_attention, q, k, k[:3], cu, 1.0)
    bad("k must be", ops.packed_attention, q, k.half(), k, cu, 1.0)
    bad("out must be", ops.packed_attention, q, k, k, cu, 1.0, out=q[:, :4])
    bad("contiguous last", ops.packed_attention, q.transpose(1, 2).contiguous().transpose(1, 2), k, k, cu, 1.0)
    bad("int32", ops.packed_attention, q, k, k, cu.long(), 1.0)
    bad("need cu_keys", ops.packed_attention, q, k[:3], k[:3], cu, 1.0)
    bad("int32", ops.packed_attention, q, k, k, cu, 1.0, cu_keys=cu[:1])
    bad("supported range", ops.packed_attention, q, k[:, :1].expand(4, 3, 64).contiguous(), k[:, :1].expand(4, 3, 64).contiguous(), cu, 1.0)
    bad("supported range", ops.packed_attention, q, k[:, :1].expand(4, 2, 64), k[:, :1].expand(4, 2, 64), cu, 1.0)     # overlapping heads
    bad("16-byte", ops.packed_attention, torch.zeros(4, 8, 68, dtype=torch.bfloat16, device=cuda_device)[..., 4:], k, k, cu, 1.0)
    pages = torch.zeros(5, 16, 2, 64, dtype=torch.bfloat16, device=cuda_device)
    table, lengths = torch.zeros(4, 2, dtype=torch.int32, device=cuda_device), torch.zeros(4, dtype=torch.int32, device=cuda_device)
    bad("of one shape", ops.paged_attention, q, pages, pages[:4], table, lengths, 1.0)
    bad("same strides", ops.paged_attention, q, pages, pages.transpose(1, 2).contiguous().transpose(1, 2), table, lengths, 1.0)
    bad("int32", ops.paged_attention, q, pages, pages, table.long(), lengths, 1.0)
    bad("per row of the table", ops.paged_attention, q, pages, pages, table, lengths[:3], 1.0)
    bad("q must be", ops.paged_attention, q[:3], pages, pages, table, lengths, 1.0)
    bad("query heads", ops.paged_attention, q[:, :7], pages, pages, table, lengths, 1.0)
    bad("workspace", ops.paged_attention, q, pages, pages, table, lengths, 1.0, workspace=torch.zeros(64, dtype=torch.uint8, device=cuda_device))
    cu5 = torch.zeros(5, dtype=torch.int32, device=cuda_device)
    cos = torch.zeros(9, 32, device=cuda_device)
    bad("cu must be", ops.paged_append, k, k, pages, pages, table, cu, lengths)
    bad("go together", ops.paged_append, k, k, pages, pages, table, cu5, lengths, cos=cos)
    bad("go together", ops.paged_append, k, k, pages, pages, table, cu5, lengths, q=q)
    bad("cos and sin", ops.paged_append, k, k, pages, pages, table, cu5, lengths, cos=cos[:, :16], sin=cos[:, :16])
    bad("v must be", ops.paged_append, k, k[:2], pages, pages, table, cu5, lengths)
    bad("supported range", ops.copy_pages, pages, [0], [5])
    bad("supported range", ops.copy_pages, pages, [0, 1], [2, 2])
    bad("supported range", ops.copy_pages, pages, [0, 1], [1, 2])
    bad("supported range", ops.copy_pages, pages, [-1], [2])
    bad("differ in length", ops.copy_pages, pages, [0], [1, 2])
    bad("on the CPU", ops.copy_pages, pages, table[0], [1, 2])
    bad("contiguous", ops.copy_pages, pages.transpose(0, 1), [0], [1])

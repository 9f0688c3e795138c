"""Attention, appends and page tables in 64 bits for the tests, and how far a kernel may be off."""
import random

import torch

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}     # a rounding's largest relative error


def attend(q, k, v, scale, first=None):
    """softmax(scale q k^T) v in 64 bits, [n, Hq, D] on [m, Hk, D]; query i sees keys up to first + i (None: all).  A query
    without keys gives zeros.  Returns (out, allowance): the bound of a kernel's error per output.

    With u half a step of the type, A = sum w |v| / sum w: weights are rounded (the sum is that of the rounded ones): 2 u A; the
    output is: u |o| <= u A.  The scores carry an error of (D + 8) 2^-23 of sum |q k| scale, ds, which moves weights
    by a factor exp(+-ds), in numerator and denominator: 2 ds A.  Sums over m keys: 2 m 2^-23 A.  fp16 weights below 2^-14 are
    off by 2^-25 each, against a sum of at least one for the largest weight: 2 m 2^-25 max |v|."""
    n, hq, D = q.shape
    m, hk = k.shape[:2]
    dtype = q.dtype
    u = HALF_STEP[dtype]
    q, k, v = q.double(), k.double(), v.double()
    out, allow = torch.zeros_like(q), torch.zeros_like(q)
    if m == 0 or n == 0:
        return out, allow
    seen = torch.ones(n, m, dtype=torch.bool, device=q.device)
    if first is not None:
        seen = torch.arange(m, device=q.device)[None] <= torch.arange(n, device=q.device)[:, None] + first
    some = seen.any(1)
    for h in range(hq):
        kh, vh = k[:, h // (hq // hk)], v[:, h // (hq // hk)]
        s = (scale * q[:, h] @ kh.T).masked_fill(~seen, -torch.inf)[some]
        w = torch.softmax(s, 1)
        out[some, h] = w @ vh
        A = w @ vh.abs()
        ds = (D + 8) * 2.0 ** -23 * abs(scale) * float((q[:, h].abs() @ kh.abs().T).max())
        allow[some, h] = A * (3 * u + 2 * ds + 2 * m * 2.0 ** -23)
        if dtype == torch.float16:
            allow[some, h] += 2 * m * 2.0 ** -25 * float(vh.abs().max()) + 2.0 ** -25
    return out, allow * 1.01          # second-order terms


def check(got, want, allow):
    assert got.shape == want.shape
    off = (got.double() - want).abs() - allow
    assert bool((off <= 0).all()), f"off by {float(off.max()):.3e} beyond the allowance, {float((off > 0).double().mean()):.2%} of the values"


def deal_pages(lens, page, seed, spare=2, width=None):
    """(table rows with -1 behind a sequence's pages, pages of the pool), pages in no order."""
    need = [-(-n // page) for n in lens]
    ids = list(range(sum(need) + spare))
    random.Random(seed).shuffle(ids)
    width = max([1, *need]) if width is None else width
    rows, at = [], 0
    for n in need:
        rows.append(ids[at:at + n] + [-1] * (width - n))
        at += n
    return rows, len(ids)


def gather(pages, row, n):
    """The first n rows of a sequence, [n, heads, D]."""
    page = pages.shape[1]
    if n == 0:
        return pages[0, :0]
    ids = torch.tensor(row[:-(-n // page)], device=pages.device)
    return pages[ids].flatten(0, 1)[:n]


def rotate(x, cos, sin):
    """Rotate-half in 64 bits, [T, heads, D] with tables [T, D / 2]."""
    a, b = x.double().chunk(2, -1)
    c, s = cos.double()[:, None], sin.double()[:, None]
    return torch.cat([a * c - b * s, b * c + a * s], -1)

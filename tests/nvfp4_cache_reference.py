"""A 4-bit paged cache and attention with a window restated for the tests, in 64 bits where numbers are computed."""
import torch

from paged_reference import HALF_STEP

LEVELS = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def groups(D):
    return -(-D // 32)


def scale_values(byte):
    """E4M3 bytes in 64 bits; 0x7f is NaN."""
    byte = byte.long()
    e, m = (byte >> 3) & 15, (byte & 7).double()
    x = torch.where(e == 0, m * 2.0 ** -9, (1 + m / 8) * torch.exp2((e - 7).double()))
    return torch.where((byte & 127) == 127, torch.nan, x)


def quantise(x, factor=1.0):
    """Rows [..., D] of a 16-bit type -> (codes [..., 32 G] of 0 to 15, scale bytes [..., 2 G]), by their definition: the scale is the E4M3
    nearest to max / 6 (ties to even), the codes the nearest levels (ties to the even one)."""
    D = x.shape[-1]
    y = torch.zeros((*x.shape[:-1], 32 * groups(D)), dtype=torch.float64, device=x.device)
    y[..., :D] = x.double() / factor
    y = y.unflatten(-1, (-1, 16))
    bad = ~y.isfinite().all(-1)
    y = torch.where(bad[..., None], 0.0, y)
    table = scale_values(torch.arange(127, device=x.device))                    # ascending: the index is the byte
    want = (y.abs().amax(-1) / 6).clamp(max=448)
    hi = torch.searchsorted(table, want.contiguous()).clamp(max=126)
    lo = (hi - 1).clamp(min=0)
    up, down = table[hi] - want, want - table[lo]
    byte = torch.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    s = table[byte][..., None]
    ratio = torch.where(s > 0, y.abs() / s.clamp(min=2.0 ** -9), 0.0).clamp(max=6)
    off = (ratio[..., None] - LEVELS.to(x.device)).abs()
    off = off + torch.tensor([0, 1e-9] * 4, dtype=torch.float64, device=x.device)          # ties to even: ratios are no nearer than that
    code = off.argmin(-1) + 8 * ((y < 0) & (s > 0))
    code = torch.where(bad[..., None], 0, code)
    return code.flatten(-2), torch.where(bad, 127, byte)


def values(code, byte, D):
    """[..., D] in 64 bits (without the cache's factor)."""
    x = LEVELS.to(code.device)[code % 8] * torch.where(code >= 8, -1.0, 1.0)
    return (x.unflatten(-1, (-1, 16)) * scale_values(byte)[..., None]).flatten(-2)[..., :D]


def unpack(pages, D):
    """uint8 [P, H, tiles, 288 G] -> (codes [P, H, 16 tiles, 32 G], scale bytes [P, H, 16 tiles, 2 G])."""
    g = groups(D)
    c = pages[..., :256 * g].unflatten(-1, (16, 16 * g)).flatten(2, 3)
    s = pages[..., 256 * g:].unflatten(-1, (16, 2 * g)).flatten(2, 3)
    return torch.stack([c & 15, c >> 4], -1).flatten(-2).long(), s.long()


def pack(code, byte):
    """The inverse of unpack: uint8 [P, H, tiles, 288 G]."""
    c = (code[..., ::2] | (code[..., 1::2] << 4)).to(torch.uint8).unflatten(2, (-1, 16)).flatten(-2)
    return torch.cat([c, byte.to(torch.uint8).unflatten(2, (-1, 16)).flatten(-2)], -1).contiguous()


def held(pages, D):
    """Every row of the pool, [P, page, H, D] in 64 bits."""
    return values(*unpack(pages, D), D).transpose(1, 2)


def seen(n, m, window, sinks, device, first=None):
    """[n, m]: whether query i, which stands at key first + i (m - n + i), sees key j."""
    i = torch.arange(n, device=device)[:, None] + (m - n if first is None else first)
    j = torch.arange(m, device=device)[None]
    return (j <= i) & ((j < sinks) | (j > i - window)) if window else j <= i


def attend(q, k, v, scale, mask, weight_step=None):
    """softmax(scale q k^T) v in 64 bits under a mask [n, m]: (out, allowance).  q [n, Hq, D] of a 16-bit type, k and v [m, Hk, D], masked rows
    of v may hold anything.

    With u half a step of the output's type, u_w of the weights' and A = sum w |v| / sum w: weights are rounded, 2 u_w A, and so is the output,
    u |o|.  The scores carry an error ds of (D + 8) 2^-23 of sum |q k| scale from sums in 32 bits, and 2^-24 max |q| sum |k| scale where small
    queries are divided by their head's largest (half a step 2^-25 against a largest below 2); it moves weights by exp(+-ds), in numerator and denominator: 2 ds A.  Sums over m
    keys: 2 m 2^-23 A.  fp16 weights below 2^-14 are off by 2^-25 each, against a sum of at least one for the largest weight: 2 m 2^-25 max |v|;
    an fp16 output below 2^-14 is off by 2^-25."""
    n, hq, D = q.shape
    m, hk = k.shape[:2]
    u = HALF_STEP[q.dtype]
    uw = u if weight_step is None else weight_step
    half_weights = q.dtype == torch.float16 or weight_step is not None
    half_out = q.dtype == torch.float16
    q, k, v = q.double(), k.double(), v.double()
    out, allow = torch.zeros_like(q), torch.zeros_like(q)
    some = mask.any(1)
    if m == 0 or n == 0 or not bool(some.any()):
        return out, allow
    used = mask.any(0)
    k, v = (torch.where(used[:, None, None], x, 0.0) for x in (k, v))
    for h in range(hq):
        kh, vh = k[:, h // (hq // hk)], v[:, h // (hq // hk)]
        s = (scale * q[:, h] @ kh.T).masked_fill(~mask, -torch.inf)[some]
        w = torch.softmax(s, 1)
        out[some, h] = w @ vh
        A = w @ vh.abs()
        ds = (D + 8) * 2.0 ** -23 * abs(scale) * float((q[:, h].abs() @ kh.abs().T).max())
        ds += 2.0 ** -24 * abs(scale) * float(q[:, h].abs().max() * kh.abs().sum(1).max())
        allow[some, h] = A * (2 * uw + u + 2 * ds + 2 * m * 2.0 ** -23)
        if half_weights:
            allow[some, h] += 2 * m * 2.0 ** -25 * float(vh.abs().max())
        if half_out:
            allow[some, h] += 2.0 ** -25
    return out, allow * 1.01          # second-order terms

"""Attention of single tokens on long caches whose every stretch of keys shows in the result: the values of a stretch have one column of their own, so that a
lost or doubled part changes that column by its share of the stretch, and the allowance grows with what is added up one after the other, not with the cache."""
import torch

from paged_reference import HALF_STEP


def stretches(n, D, dtype, generator, device):
    """Values [n, 1, D] of 0.75 to 1.25 in the column of their stretch, n / D keys long, zeros elsewhere."""
    v = torch.zeros(n, D, dtype=dtype, device=device)
    size = 0.75 + 0.5 * torch.rand(n, generator=generator, device=device)
    j = torch.arange(n, device=device)
    v[j, j * D // max(n, 1)] = size.to(dtype)
    return v[:, None]


def roundings(keys, workers):
    """On the way of a key into the result: the keys of all items are dealt evenly to `workers` warps at least, a slot of 64 more or less at either end; a
    product adds 16 keys in as many roundings at most, their weights are added up besides; then come lanes, warps and parts, 64 at most after one
    another."""
    return 2 * (-(-keys // workers) + 128) + 64


def attend_long(q, k, v, scale, seen, weight_step, steps):
    """softmax(scale q k^T) v in 64 bits over the keys that are seen [m], and the allowance.  q [Hq, D] of a 16-bit type, k and v [m, Hk, D].

    With u half a step of the output's type, u_w of the weights' and A = sum w |v| / sum w over these keys: rounded weights 2 u_w A; the output u |o|; scores are
    off by ds = (D + 8) 2^-23 of the largest scale sum |q k| for their sums in 32 bits, and 2^-24 max |q| sum |k| scale where queries are divided by their head's
    largest: 2 ds A; `steps` roundings of a sum: 2 steps 2^-23 A.  fp16 weights are held 2^7 times larger, eleven bits down to 2^-21 and 2^-32 off
    below, against a sum S of weights over the largest one, which the reference does not pass: n 2^-32 max |v| / S.  fp16 outputs below 2^-14: 2^-25."""
    hq, D = q.shape
    hk = k.shape[1]
    u = HALF_STEP[q.dtype]
    half_out = q.dtype == torch.float16
    k, v, q = k[seen].double(), v[seen].double(), q.double()
    out, allow = torch.zeros_like(q), torch.zeros_like(q)
    n = k.shape[0]
    if n == 0:
        return out, allow
    for h in range(hq):
        kh, vh = k[:, h // (hq // hk)], v[:, h // (hq // hk)]
        s = scale * kh @ q[h]
        w = torch.exp(s - s.max())
        total = w.sum()
        out[h] = w @ vh / total
        A = w @ vh.abs() / total
        ds = abs(scale) * ((D + 8) * 2.0 ** -23 * (kh.abs() @ q[h].abs()).max() + 2.0 ** -24 * q[h].abs().max() * kh.abs().sum(1).max())
        allow[h] = A * (2 * weight_step + 2 * ds + 2 * steps * 2.0 ** -23) + out[h].abs() * u
        if weight_step == HALF_STEP[torch.float16]:
            allow[h] += n * 2.0 ** -32 * vh.abs().max() / total
        if half_out:
            allow[h] += 2.0 ** -25
    return out, allow * 1.01          # second-order terms

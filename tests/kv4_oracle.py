"""Plain float64 forms of the 4-bit cache and of attention over it, for the tests of its kernels."""

import torch


def values64(codes, scales):
    """Rows [..., D / 2] uint8 and [..., groups, 2] by value, value by value from the definition."""
    D = codes.shape[-1] * 2
    d = torch.arange(D, device=codes.device)
    word, nibble = d % (D // 8), (d // (D // 4)) + 4 * (d // (D // 8) % 2)
    n = (codes[..., word * 4 + nibble // 2].long() >> (4 * (nibble % 2))) & 15
    s = scales.double()
    g = d * scales.shape[-2] // D
    return n.double() * s[..., g, 0] + s[..., g, 1]


def context64(cache, scales, table, n):
    """[KVH, n, D] of the first n positions of a block table."""
    BS = cache.shape[2]
    at = table[: -(-n // BS)].long()
    return values64(cache[at], scales[at]).transpose(0, 1).flatten(1, 2)[:, :n]


def attention64(q, k, v, ks, vs, tables, lens, scale):
    """(result, bound): softmax attention of rows q [B, H, D] in 64 bits, and how far a kernel may be off.

    A kernel multiplies fp16(p step) with whole numbers: 2^-11 of each term (a rounding is off by half of 2^-10), so of A = sum of
    p (step n + |least|). The scores are fp32 sums of 128 terms: off by 130 * 2^-24 of the sum C of their magnitudes at
    most, as are the exponentials, over and under the line. The result's rounding to bf16 is off by 2^-8 of it (half of 2^-7),
    and sums of fp32 over the keys by 2^-16 of A, generously."""
    B, H, D = q.shape
    KVH = k.shape[1]
    out, off = torch.zeros(B, H, D, dtype=torch.float64), torch.zeros(B, H, D, dtype=torch.float64)
    for b in range(B):
        n = int(lens[b])
        if n == 0:
            continue
        kk, vv = context64(k, ks, tables[b], n), context64(v, vs, tables[b], n)
        least = context64(torch.zeros_like(v), vs, tables[b], n)
        rows = q[b].double().view(KVH, H // KVH, D)
        p = torch.softmax(rows @ kk.transpose(1, 2) * scale, -1)
        C = (rows.abs() @ (kk.abs() + 2 * context64(torch.zeros_like(k), ks, tables[b], n).abs()).transpose(1, 2)).amax() * abs(scale)
        A = p @ ((vv - least).abs() + least.abs())
        out[b] = (p @ vv).view(H, D)
        off[b] = (2 ** -8 * (p @ vv).abs() + A * (2 ** -11 + 2 ** -16 + 2 * 130 * 2 ** -24 * float(C))).view(H, D)
    return out, off + 1e-30


def prompts64(q, k, v, ks, vs, tables, lens, scale):
    """attention64 of the rows of prompt portions, with what a kernel may be off that makes fp16 of keys and values.

    Values: a power of 2^16, u, is taken out of a group, 1 where the larger exponent e of its least value and of 16 steps is -10 to
    12, else such that e lies there. Then |x| < 2^14 u. Least value and step have 8 bits: they are whole multiples of 2^-24 u (fp16's least) or
    off by half of that; the step counts up to 15 times. Their sum is rounded once: 2^-11 of it (half of fp16's 2^-10), or half of
    2^-24 u. So a value is off by a = 2^-11 |x| + 17 * 2^-25 u at most.
    Scores: D = |scale| sum |q| a of the key that is furthest off, so that weights are off by exp(2 D) - 1 of themselves, over
    and under the line; and as in attention64 by 130 * 2^-24 of C, twice.
    P: 2^-11 of a weight, or half of 2^-24 of the largest one, to which the sum of all is at least one.
    Sums over keys in fp32, and of a group with u the products of two bf16 parts of each side (2^-16 of either): 2^-14 of sum p |v|,
    generously. The result's rounding: 2^-8 of it."""
    def values(cache, scales, table, n):
        x = context64(cache, scales, table, n)
        s, least = scales.double()[..., 0], scales.double()[..., 1]
        e = torch.frexp(torch.maximum(least.abs(), 16 * s)).exponent - 1
        c = torch.where(e > 12, (e - 13).div(16, rounding_mode="floor") + 1, -(-11 - e).div(16, rounding_mode="floor") - 1).clamp(min=-7)
        u = torch.where((e >= -10) & (e <= 12) | (least == 0) & (s == 0), 0, c) * 16
        at = table[: -(-n // cache.shape[2])].long()
        u = torch.ldexp(torch.ones((), dtype=torch.float64), u)[at].transpose(0, 1).flatten(1, 2)[:, :n].repeat_interleave(cache.shape[3] * 2 // s.shape[-1], -1)
        return x, 2 ** -11 * x.abs() + 17 * 2 ** -25 * u

    B, H, D = q.shape
    KVH = k.shape[1]
    out, off = torch.zeros(B, H, D, dtype=torch.float64), torch.zeros(B, H, D, dtype=torch.float64)
    for b in range(B):
        n = int(lens[b])
        (kk, ka), (vv, va) = values(k, ks, tables[b], n), values(v, vs, tables[b], n)
        rows = q[b].double().view(KVH, H // KVH, D)
        p = torch.softmax(rows @ kk.transpose(1, 2) * scale, -1)
        C = (rows.abs() @ kk.abs().transpose(1, 2)).amax() * abs(scale)
        far = (rows.abs() @ ka.transpose(1, 2)).amax(-1, keepdim=True) * abs(scale)
        out[b] = (p @ vv).view(H, D)
        off[b] = (2 ** -8 * (p @ vv).abs() + (p @ vv.abs()) * (torch.expm1(2 * far) + 2 ** -11 + 2 ** -14 + 2 * 130 * 2 ** -24 * float(C))
                  + p @ va + 2 ** -25 * vv.abs().sum(1, keepdim=True)).view(H, D)
    return out, off + 1e-30

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

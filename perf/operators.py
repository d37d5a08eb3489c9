"""Performance cases of the operators that serve a model in fewer bits.

A key/value cache held in 4 bits with the attention that reads it, and products of activations in 8-bit integers (a
scale for each token) with weights in 8-bit integers (a scale for each output channel). Each case is one call that a
decode step or a prompt of a served model makes; ``run`` computes it with elementary tensor operations in 32 bits, or,
where ``own`` is true, with the package's kernels.

``op`` of a case:

  store    new keys and values of ``tokens`` rows go into the paged 4-bit cache, and the rows are read back
  decode   one query row for each of ``streams`` against its paged context
  segment  rows of ``segments`` prompt portions, each behind a cached prefix, against the paged cache
  linear   rows of bf16 activations times a weight matrix: bf16 [rows, out]; ``gated``: silu(gate) * up of a fused
           [gate; up] matrix, bf16 [rows, out / 2]

The 4-bit cache: 64 neighbouring values of a row are a group with its least value and its step, bf16 both, step = (most -
least) / 15; a value is stored as the whole number of steps above the least one. ``k`` and ``v`` [blocks, kv heads, block,
64] uint8 hold the numbers of a row of 128 values as 16 little-endian words of 32 bits: nibble p of word n is that of value
32 (p mod 4) + 16 (p div 4) + n. The ``scales`` [blocks, kv heads, block, 2, 2] bf16 hold (step, least) of both groups.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DEVICE = "cuda:0"
HEAD = 128
GROUP = 64
F32, F64, BF16 = torch.float32, torch.float64, torch.bfloat16


def listed():
    return [
        # a decode step's new rows for the benchmark's batch: 24 requests of n=5
        dict(name="store-120", op="store", tokens=120, kv_heads=8, block=16),
        # a long document's rows, an odd length
        dict(name="store-7777", op="store", tokens=7777, kv_heads=8, block=16),
        # the smallest call: one plain chat stream of a small model
        dict(name="decode-1", op="decode", streams=1, fan=1, heads=16, kv_heads=4, block=16, shortest=150, longest=150, prompt=0),
        # the benchmark's batch: prompts of 512 tokens, each shared by five streams
        dict(name="decode-120", op="decode", streams=120, fan=5, heads=32, kv_heads=8, block=16, shortest=520, longest=577, prompt=512),
        # long documents, one answer each
        dict(name="decode-16-long", op="decode", streams=16, fan=1, heads=32, kv_heads=8, block=16, shortest=4500, longest=7777,
             prompt=0),
        # one very long context of a large model, eight query heads to a kv head
        dict(name="decode-1-131071", op="decode", streams=1, fan=1, heads=64, kv_heads=8, block=16, shortest=131071,
             longest=131071, prompt=0),
        # eight requests behind a system prompt that is already in the cache
        dict(name="segment-8x150", op="segment", segments=8, rows=150, behind=1536, heads=32, kv_heads=8, block=16),
        # a long document behind another one
        dict(name="segment-1x2100", op="segment", segments=1, rows=2100, behind=7777, heads=32, kv_heads=8, block=16),
        # one request's streams through the fused projection of queries, keys and values
        dict(name="linear-5", op="linear", rows=5, inner=4096, out=6144, gated=False, bias=False),
        # the benchmark's batch through gate and up
        dict(name="linear-120-gated", op="linear", rows=120, inner=4096, out=28672, gated=True, bias=False),
        # a short prompt, the biased projection of another model
        dict(name="linear-333-bias", op="linear", rows=333, inner=3584, out=4608, gated=False, bias=True),
        # a long prompt through gate and up
        dict(name="linear-7777-gated", op="linear", rows=7777, inner=4096, out=28672, gated=True, bias=False),
    ]


def _log(rng, lo, hi):
    """A whole number from lo to hi, spread evenly over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng: random.Random):
    op = rng.choice(["store", "decode", "decode", "segment", "linear", "linear"])
    kv_heads, group = rng.choice([1, 2, 4, 8, 8]), rng.choice([1, 2, 4, 4, 8])
    block = rng.choice([16, 16, 16, 32, 8, 5])
    if op == "store":
        return dict(op=op, tokens=_log(rng, 1, 12000), kv_heads=kv_heads, block=block)
    if op == "decode":
        streams = _log(rng, 1, 200)
        longest = _log(rng, 1, max(2, 1000000 // (streams * kv_heads)))
        longest = min(longest, 131071)
        fan = rng.choice([1, 1, 3, 5, 8])
        prompt = rng.randint(0, longest - 1) if fan > 1 else 0
        return dict(op=op, streams=streams, fan=fan, heads=kv_heads * group, kv_heads=kv_heads, block=block,
                    shortest=rng.randint(prompt, longest), longest=longest, prompt=prompt)
    if op == "segment":
        segments = _log(rng, 1, 16)
        return dict(op=op, segments=segments, rows=_log(rng, 2, 2000 // segments), behind=rng.choice([0, _log(rng, 1, 8000)]),
                    heads=kv_heads * group, kv_heads=kv_heads, block=block)
    gated = rng.random() < 0.4
    return dict(op=op, rows=_log(rng, 1, 7000), inner=128 * _log(rng, 2, 112), out=64 * _log(rng, 4, 440), gated=gated,
                bias=not gated and rng.random() < 0.4)


# --- inputs -----------------------------------------------------------------------


def _quantized(x):
    """(whole numbers [..., groups, 64], step, least) of rows, in 32 bits; step and least are bf16 values."""
    x = x.to(F32).unflatten(-1, (-1, GROUP))
    least, most = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    step = ((most - least) / 15).to(BF16).to(F32)
    n = torch.where(step > 0, torch.round((x - least) / step), 0.0)
    return n.clamp(0, 15), step, least


def _packed(n):
    """Whole numbers [..., 128] of rows as the cache's bytes [..., 64]."""
    n = n.to(torch.uint8).unflatten(-1, (4, 2, 16))              # value 32 a + 16 h + word
    n = n.movedim(-1, -3).transpose(-1, -2).flatten(-2)          # [word, nibble 4 h + a]
    return (n[..., 0::2] | (n[..., 1::2] << 4)).flatten(-2)


def _unpacked(b):
    """Bytes [..., 64] as whole numbers [..., 128] in 32 bits."""
    n = torch.stack((b & 15, b >> 4), -1).unflatten(-2, (16, 4)).flatten(-2)       # [word, nibble]
    return n.unflatten(-1, (2, 4)).movedim(-3, -1).transpose(-2, -3).flatten(-3).to(F32)


def _values(codes, scales):
    """What rows of the cache stand for, in 32 bits."""
    s = scales.to(F32)
    return (_unpacked(codes).unflatten(-1, (-1, GROUP)) * s[..., :1] + s[..., 1:]).flatten(-2)


def _activations(g, *shape):
    """Rows as layers give them: a few channels are much larger than the others."""
    x = torch.randn(*shape, generator=g, device=DEVICE)
    wide = torch.rand(shape[1:], generator=g, device=DEVICE) < 0.02
    return (x * torch.where(wide, 6.0, 1.0)).to(BF16)


def _cache(g, blocks, case):
    """(codes, scales) of keys or values that were stored before."""
    n, step, least = _quantized(_activations(g, blocks * case["block"], case["kv_heads"], HEAD))
    at = (blocks, case["block"], case["kv_heads"])
    codes = _packed(n.flatten(-2)).view(*at, HEAD // 2).transpose(1, 2).contiguous()
    scales = torch.cat((step, least), -1).to(BF16).view(*at, 2, 2).transpose(1, 2).contiguous()
    return codes, scales


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    rng = random.Random(seed)
    op = case["op"]
    if op == "linear":
        w = torch.randn(case["out"], case["inner"], generator=g, device=DEVICE) * 0.02
        most = w.abs().amax(-1, keepdim=True)
        state = dict(x=_activations(g, case["rows"], case["inner"]), w=torch.round(127 * w / most).to(torch.int8),
                     w_scale=(most / 127).squeeze(-1), bias=None)
        if case["bias"]:
            state["bias"] = torch.randn(case["out"], generator=g, device=DEVICE).to(BF16)
        return {"case": case, **state}
    block, kv_heads = case["block"], case["kv_heads"]
    if op == "store":
        tokens = case["tokens"]
        blocks = -(-tokens // block) + 8
        k, k_scale = _cache(g, blocks, case)
        v, v_scale = _cache(g, blocks, case)
        fresh = _activations(g, tokens, 2 * kv_heads, HEAD)      # the rows of a fused projection
        return dict(case=case, k=k, v=v, k_scale=k_scale, v_scale=v_scale, k_new=fresh[:, :kv_heads], v_new=fresh[:, kv_heads:],
                    slots=torch.randperm(blocks * block, generator=g, device=DEVICE)[:tokens])
    if op == "decode":
        streams, fan = case["streams"], case["fan"]
        lens = [rng.randint(case["shortest"], case["longest"]) for _ in range(streams)]
        lens[rng.randrange(streams)] = case["longest"]
        width = -(-case["longest"] // block)
        whole = case["prompt"] // block                          # blocks that a request's streams share
        request = torch.arange(streams, device=DEVICE) // fan
        column = torch.arange(width, device=DEVICE)
        table = torch.where(column < whole, (request * fan)[:, None], torch.arange(streams, device=DEVICE)[:, None])
        blocks = streams * width
        table = torch.randperm(blocks, generator=g, device=DEVICE)[table * width + column].to(torch.int32)
        k, k_scale = _cache(g, blocks, case)
        v, v_scale = _cache(g, blocks, case)
        return dict(case=case, k=k, v=v, k_scale=k_scale, v_scale=v_scale, tables=table,
                    lens=torch.tensor(lens, dtype=torch.int32, device=DEVICE),
                    q=_activations(g, streams, case["heads"], HEAD))
    # segments: (position of the first row, rows); how many rows there are is the case's
    ragged = random.Random(case["rows"])
    segs = [(rng.randint(case["behind"] - case["behind"] // 8, case["behind"]),
             ragged.randint(case["rows"] - case["rows"] // 8, case["rows"])) for _ in range(case["segments"])]
    width = max(-(-(p + n) // block) for p, n in segs)
    blocks = len(segs) * width
    seg_tables = torch.randperm(blocks, generator=g, device=DEVICE).view(len(segs), width).to(torch.int32)
    rows = torch.tensor([n for _, n in segs], device=DEVICE)
    start = torch.tensor([p for p, _ in segs], dtype=torch.int32, device=DEVICE)
    seg = torch.repeat_interleave(torch.arange(len(segs), device=DEVICE), rows)
    at = torch.arange(len(seg), device=DEVICE) - (rows.cumsum(0) - rows)[seg]
    k, k_scale = _cache(g, blocks, case)
    v, v_scale = _cache(g, blocks, case)
    state = dict(case=case, k=k, v=v, k_scale=k_scale, v_scale=v_scale, seg_tables=seg_tables, seg_start=start, seg=seg, at=at,
                 most=max(n for _, n in segs), segs=segs, q=_activations(g, len(seg), case["heads"], HEAD),
                 tables=seg_tables[seg], lens=(start[seg] + at + 1).to(torch.int32), plan=None)
    if own:
        from kllms_amd import ops

        # made once for all layers of a pass
        state["plan"] = ops.paged_plan(segs, case["heads"], kv_heads, DEVICE, k.dtype)
    return state


# --- one pass -----------------------------------------------------------------------


def _weighted(q, k, v, seen):
    """softmax(q k^T / sqrt(d)) v of the keys that ``seen`` admits: q [n, kv heads, rows, d], k and v [n, kv heads, keys, d],
    seen [n, 1, rows, keys]. Rows that see nothing are zero."""
    score = (q @ k.transpose(-1, -2)) / math.sqrt(HEAD)
    score = torch.where(seen, score, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top > -math.inf, top, 0.0))
    total = p.sum(-1, keepdim=True)
    return torch.where(total > 0, (p @ v) / total, 0.0)


def _context(state, name, tables, dtype=F32):
    """Keys or values [n, kv heads, width * block, d] of the blocks of each table row."""
    at = tables.long()
    rows = _values(state[name][at], state[name + "_scale"][at])
    return rows.transpose(1, 2).flatten(2, 3)


def _plain_decode(state):
    q = state["q"].to(F32)
    n, heads, _ = q.shape
    kv_heads = state["case"]["kv_heads"]
    k, v = (_context(state, name, state["tables"]) for name in "kv")
    seen = torch.arange(k.shape[2], device=DEVICE) < state["lens"][:, None, None, None]
    o = _weighted(q.view(n, kv_heads, heads // kv_heads, HEAD), k, v, seen)
    return o.reshape(n, heads, HEAD).to(BF16)


def _plain_segments(state):
    seg, at, heads, kv_heads = state["seg"], state["at"], state["case"]["heads"], state["case"]["kv_heads"]
    n, most, group = len(state["seg_start"]), state["most"], heads // kv_heads
    q = torch.zeros(n, most, heads, HEAD, device=DEVICE)
    q[seg, at] = state["q"].to(F32)
    k, v = (_context(state, name, state["seg_tables"]) for name in "kv")
    last = state["seg_start"][:, None] + torch.arange(most, device=DEVICE)        # the last key that a row sees
    seen = torch.arange(k.shape[2], device=DEVICE) <= last.repeat(1, group)[:, None, :, None]
    q = q.view(n, most, kv_heads, group, HEAD).permute(0, 2, 3, 1, 4).flatten(2, 3)
    o = _weighted(q, k, v, seen).view(n, kv_heads, group, most, HEAD)
    return o.permute(0, 3, 1, 2, 4).flatten(2, 3)[seg, at].to(BF16)


def _plain_store(state):
    block, slots = state["case"]["block"], state["slots"]
    blk, off = slots // block, slots % block
    out = []
    for name in "kv":
        n, step, least = _quantized(state[name + "_new"])
        state[name][blk, :, off] = _packed(n.flatten(-2))
        state[name + "_scale"][blk, :, off] = torch.cat((step, least), -1).to(BF16)
        out.append(_values(state[name][blk, :, off], state[name + "_scale"][blk, :, off]).to(BF16))
    return tuple(out)


def _plain_linear(state):
    x = state["x"].to(F32)
    most = x.abs().amax(-1, keepdim=True)
    codes = torch.where(most > 0, torch.round(127 * x / most), 0.0)
    y = (codes @ state["w"].to(F32).t()) * (most / 127) * state["w_scale"]
    if state["bias"] is not None:
        y = y + state["bias"].to(F32)
    if state["case"]["gated"]:
        gate, up = y.chunk(2, -1)
        y = gate / (1 + torch.exp(-gate)) * up
    return y.to(BF16)


def run(state):
    case = state["case"]
    if own:
        from kllms_amd import ops

        if case["op"] == "linear":
            if case["gated"]:
                return ops.linear_silu_int8(state["x"], state["w"], state["w_scale"])
            return ops.linear_int8(state["x"], state["w"], state["w_scale"], state["bias"])
        cache = (state["k"], state["v"])
        scales = (state["k_scale"], state["v_scale"])
        if case["op"] == "store":
            ops.store_kv(state["k_new"], state["v_new"], *cache, state["slots"], *scales)
            return ops.load_kv(*cache, state["slots"], *scales)
        if case["op"] == "decode":
            return ops.attn_decode_paged(state["q"], *cache, state["tables"], state["lens"], HEAD ** -0.5, *scales)
        plan, short = state["plan"]
        return ops.attn_segments_paged(state["q"], *cache, state["tables"], state["lens"], HEAD ** -0.5, plan, short,
                                       state["seg_tables"], state["seg_start"], *scales)
    return {"store": _plain_store, "decode": _plain_decode, "segment": _plain_segments, "linear": _plain_linear}[case["op"]](state)


def work(case):
    op = case["op"]
    if op == "linear":
        rows, inner, out = case["rows"], case["inner"], case["out"]
        kept = out // 2 if case["gated"] else out
        return {"bytes": 2 * rows * inner + out * inner + 4 * out + 2 * rows * kept, "flops": 2 * rows * inner * out}
    kv_heads = case["kv_heads"]
    row = 2 * (HEAD // 2 + 8) * kv_heads                         # a position's keys and values
    if op == "store":
        # rows in, rows into the cache and out of it, what they stand for
        return {"bytes": case["tokens"] * (2 * 4 * HEAD * kv_heads + 2 * row + 8), "flops": 10 * 2 * case["tokens"] * kv_heads * HEAD}
    if op == "decode":
        mean, whole = (case["shortest"] + case["longest"]) / 2, case["prompt"] // case["block"] * case["block"]
        keys = case["streams"] * (mean - whole) + -(-case["streams"] // case["fan"]) * whole
        return {"bytes": keys * row + 4 * case["streams"] * case["heads"] * HEAD,
                "flops": 4 * case["streams"] * case["heads"] * HEAD * mean}
    n, behind = case["rows"] * 15 / 16, case["behind"] * 15 / 16
    return {"bytes": case["segments"] * ((behind + n) * row + 4 * n * case["heads"] * HEAD),
            "flops": 4 * case["segments"] * case["heads"] * HEAD * n * (behind + n / 2)}


# --- what the definitions give in 64 bits ------------------------------------------------


def _exact_rows(codes, scales):
    """Rows [..., 64 bytes] of the cache by value: number * step + least."""
    d = torch.arange(HEAD, device=DEVICE)
    word, nibble = d % 16, (d // 32) + 4 * (d // 16 % 2)
    number = (codes[..., word * 4 + nibble // 2].to(torch.int64) >> (4 * (nibble % 2))) & 15
    s = scales.to(F64)
    return number.to(F64) * s[..., d // GROUP, 0] + s[..., d // GROUP, 1]


def _exact_attention(q, keys, values, last):
    """Rows q [rows, heads, d] against keys and values [kv heads, keys, d]; row i sees those up to last[i]."""
    heads, kv_heads = q.shape[1], keys.shape[0]
    out = torch.zeros(q.shape, dtype=F64, device=DEVICE)
    for h in range(heads):
        if keys.shape[1] == 0:
            continue
        s = q[:, h].to(F64) @ keys[h // (heads // kv_heads)].t() / math.sqrt(HEAD)
        s = s.masked_fill(torch.arange(keys.shape[1], device=DEVICE) > last[:, None], -math.inf)
        out[:, h] = torch.softmax(s, -1) @ values[h // (heads // kv_heads)]
    return out


def exact(case, seed):
    state = prepare(case, seed)
    op = case["op"]
    if op == "linear":
        x, w = state["x"].to(F64), state["w"].to(F64)
        most = x.abs().max(dim=-1).values
        unit = torch.where(most > 0, most / 127, 1.0)
        # 127 x is exact and its quotient rounded once: halves are halves
        y = torch.round(127 * x / torch.where(most > 0, most, 1.0)[:, None])
        y = (y @ w.t()) * unit[:, None] * state["w_scale"].to(F64)
        if state["bias"] is not None:
            y = y + state["bias"].to(F64)
        if case["gated"]:
            half = case["out"] // 2
            y = y[:, :half] * torch.sigmoid(y[:, :half]) * y[:, half:]
        return y
    if op == "store":
        got = []
        for name in ("k_new", "v_new"):
            x = state[name].to(F64).reshape(case["tokens"], case["kv_heads"], 2, GROUP)
            low, high = x.min(-1, keepdim=True).values, x.max(-1, keepdim=True).values
            step = ((high - low) / 15).to(BF16).to(F64)
            n = torch.floor((x - low) / torch.where(step > 0, step, 1.0))
            rest = (x - low) / torch.where(step > 0, step, 1.0) - n
            n = n + ((rest > 0.5) | ((rest == 0.5) & (n % 2 == 1))).to(F64)
            got.append((low + torch.clamp(n, max=15) * step).reshape(case["tokens"], case["kv_heads"], HEAD))
        return tuple(got)
    if op == "decode":
        out = []
        for b in range(case["streams"]):
            n = int(state["lens"][b])
            at = state["tables"][b, : -(-n // case["block"])].long()
            rows = [_exact_rows(state[x][at], state[x + "_scale"][at]).transpose(0, 1).flatten(1, 2)[:, :n] for x in "kv"]
            out.append(_exact_attention(state["q"][b : b + 1], *rows, torch.tensor([n - 1], device=DEVICE)))
        return torch.cat(out)
    out, row = [], 0
    for i, (p, n) in enumerate(state["segs"]):
        at = state["seg_tables"][i, : -(-(p + n) // case["block"])].long()
        rows = [_exact_rows(state[x][at], state[x + "_scale"][at]).transpose(0, 1).flatten(1, 2)[:, : p + n] for x in "kv"]
        out.append(_exact_attention(state["q"][row : row + n], *rows, torch.arange(p, p + n, device=DEVICE)))
        row += n
    return torch.cat(out)

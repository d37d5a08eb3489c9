"""Kernels of the 4-bit cache against float64."""

import pytest
import torch

from kllms_amd import ops
from kllms_amd.ops import torch_ref

from kv4_oracle import attention64, prompts64, values64

pytestmark = pytest.mark.gpu
DEV = "cuda"
D = 128


def rows(*shape, seed=0, spread=0.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(*shape, generator=g)
    if spread:
        x = x * torch.exp2(torch.randn(*shape[:-1], 1, generator=g) * spread)
    return x.bfloat16()


def special_rows(T, G, seed):
    x = rows(T, G, D, seed=seed, spread=4.0)
    if T >= 6:
        x[0] = 1.5
        x[1, 0, 3] = float("nan")
        x[2, 0, 100] = float("-inf")
        x[3, 0, :64] = 0
        x[4, 0, 1], x[4, 0, 2] = 3e38, -3e38
        x[5] = x[5] * 1e-39
    return x


@pytest.mark.parametrize("T,G,BS", [(1, 1, 1), (7, 3, 5), (120, 8, 16), (2049, 2, 32)])
def test_store_and_load(T, G, BS):
    NB = -(-T // BS) + 3
    k, v = special_rows(T, G, 1), special_rows(T, G, 2)
    wide = torch.cat((k, v, k), 1).to(DEV)                        # rows of a fused projection
    slots = torch.randperm(NB * BS)[:T]
    g = torch.Generator().manual_seed(3)
    caches = [torch.randint(0, 256, (NB, G, BS, D // 2), dtype=torch.uint8, generator=g) for _ in range(2)]
    scales = [torch.randn(NB, G, BS, 2, 2, generator=g).bfloat16() for _ in range(2)]
    dev = [t.to(DEV) for t in caches + scales]
    ops.store_kv(wide[:, :G], wide[:, G:2 * G], dev[0], dev[1], slots.to(DEV), dev[2], dev[3])
    torch_ref.store_kv(k, v, *caches, slots, *scales)
    for got, want in zip(dev, caches + scales):                   # also the rows that nobody wrote
        assert torch.equal(got.cpu().view(torch.uint8), want.view(torch.uint8)) if got.dtype == torch.uint8 else \
            torch.equal(got.cpu().float().nan_to_num(7e37), want.float().nan_to_num(7e37))
    slots[0] = NB * BS                                            # outside: loads NaN
    for got, want in zip(ops.load_kv(*dev[:2], slots.to(DEV), *dev[2:]), torch_ref.load_kv(*caches, slots, *scales)):
        assert torch.equal(got.cpu().float().nan_to_num(7e37), want.float().nan_to_num(7e37))


def test_rows_for_no_slot_go_nowhere_and_odd_rows_are_taken():
    T, G, BS, NB = 5, 2, 4, 3
    base = torch.randn(T, 3 * G * D + 1).bfloat16().to(DEV)
    k = base[:, 1:1 + G * D].unflatten(1, (G, D))                 # rows off 16 bytes, an odd stride
    v = torch.randn(T, G, D).bfloat16().to(DEV)
    kc, vc = (torch.zeros(NB, G, BS, D // 2, dtype=torch.uint8, device=DEV) for _ in range(2))
    ks, vs = (torch.zeros(NB, G, BS, 2, 2, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    slots = torch.tensor([2, -1, NB * BS, 7, 1 << 40], device=DEV)
    ops.store_kv(k, v, kc, vc, slots, ks, vs)
    a, b = ops.load_kv(kc, vc, slots, ks, vs)
    for got, x in ((a, k), (b, v)):
        assert torch.equal(got[[0, 3]].cpu(), torch_ref.kv4_values(*torch_ref.kv4_quantize(x.cpu()[[0, 3]])).bfloat16())
    assert int((ks != 0).sum()) == 2 * G * 4 and int((kc.view(NB, G, BS, -1) != 0).any(-1).sum()) == 2 * G


@pytest.mark.parametrize("T,H,G,BS", [(1, 4, 1, 16), (33, 32, 8, 16), (300, 8, 4, 5)])
def test_rope_store(T, H, G, BS):
    NB = -(-T // BS) + 2
    qkv = special_rows(T, H + 2 * G, 5).to(DEV)
    qkv[:, :H] = rows(T, H, D, seed=6).to(DEV)
    qkv[:, H:H + G] = rows(T, G, D, seed=7).to(DEV)               # what is turned is finite; values are what they are
    cos_sin = torch_ref.build_cos_sin_cache(D, 4096, 1e4, "cpu").to(DEV)
    pos = torch.randint(0, 4096, (T,), device=DEV)
    slots = torch.randperm(NB * BS, device=DEV)[:T]

    def caches():
        return [torch.zeros(NB, G, BS, D // 2, dtype=torch.uint8, device=DEV) for _ in range(2)] + \
            [torch.zeros(NB, G, BS, 2, 2, dtype=torch.bfloat16, device=DEV) for _ in range(2)]

    def same(x, y):
        return all(torch.equal(s.float().nan_to_num(7e37), t.float().nan_to_num(7e37)) for s, t in zip(x, y))

    for at in (pos, pos * 0):
        one, two = qkv.clone(), qkv.clone()
        a, b = caches(), caches()
        ops.rope_store(*one.split([H, G, G], 1), at, cos_sin, a[0], a[1], slots, a[2], a[3])
        torch_ref.rope_inplace(two[:, :H], two[:, H:H + G], at, cos_sin)
        # a product and a sum of it rounded to bf16 from fp32: of neighbouring values at most, where one lies between
        assert torch.allclose(one.float(), two.float(), rtol=2 ** -7, atol=2 ** -20, equal_nan=True)
        ops.store_kv(one[:, H:H + G], one[:, H + G:], b[0], b[1], slots, b[2], b[3])
        assert same(a, b)
    # a decode step's form, from sums in two shares; at position 0, where turning rounds nothing
    c = caches()
    flat = qkv.view(1, T, -1).float()
    part = torch.cat((flat * 0.5, flat * 0.5)).contiguous()
    got = ops.rope_store_rows(part, None, H, pos * 0, cos_sin, c[0], c[1], slots, c[2], c[3])
    assert torch.equal(got, one[:, :H]) and same(a, c)


def case(ctx, gqa, KVH, BS, seed=0, width=None, shared=0, spread=0.0, behind=True):
    """q, caches, scales, tables, lengths; what lies behind a context is another's: any codes, scales that are none."""
    g = torch.Generator().manual_seed(seed)
    B = len(ctx)
    need = [max(1, -(-c // BS)) for c in ctx]
    NB = sum(need) + 2
    perm = torch.randperm(NB, generator=g).tolist()
    tables = torch.zeros(B, width or max(need), dtype=torch.int32)
    kc, vc = (torch.randint(0, 256, (NB, KVH, BS, D // 2), dtype=torch.uint8, generator=g) for _ in range(2))
    ks, vs = (torch.full((NB, KVH, BS, 2, 2), float("nan") if behind else 0.0).bfloat16() for _ in range(2))
    if behind:
        ks[::2], vs[::2] = float("inf"), 3e38
    for b in range(B):
        own = [perm.pop() for _ in range(need[b])]
        if b and shared:
            n = min(shared, min(ctx[0], ctx[b]) // BS)
            own[:n] = tables[0, :n].tolist()
        tables[b, :need[b]] = torch.tensor(own, dtype=torch.int32)
    for b in range(B):
        at = torch.arange(ctx[b])
        blk, off = tables[b].long()[at // BS], at % BS
        for i, (cache, scale) in enumerate(((kc, ks), (vc, vs))):
            cache[blk, :, off], scale[blk, :, off] = torch_ref.kv4_quantize(rows(ctx[b], KVH, D, seed=seed * 7 + 2 * b + i, spread=spread))
    return rows(B, KVH * gqa, D, seed=seed + 99), kc, vc, ks, vs, tables, torch.tensor(ctx, dtype=torch.int32)


def check(outs, q, kc, vc, ks, vs, tables, n, scale):
    want, off = attention64(q, kc, vc, ks, vs, tables, n, scale)
    for out in outs:
        far = (out.double().cpu() - want).abs()
        assert bool((far <= off).all()), f"{float((far / off).max())} of what is allowed, at {torch.nonzero(far > off)[:3].tolist()}"


def both(q, kc, vc, ks, vs, tables, n, scale):
    """The results without counters and with them, whose shares are added up in another order."""
    dev = [t.to(DEV) for t in (q, kc, vc, tables, n, ks, vs)]
    q, kc, vc, tables, n, ks, vs = dev
    out = ops.attn_decode_paged(q, kc, vc, tables, n, scale, ks, vs)
    arrived = torch.zeros(q.shape[0] * kc.shape[1] * ops.ATTN_COUNTER_GAP, dtype=torch.int32, device=DEV)
    joined = ops.attn_decode_paged(q, kc, vc, tables, n, scale, ks, vs, arrived)
    assert torch.equal(ops.attn_decode_paged(q, kc, vc, tables, n, scale, ks, vs, arrived).nan_to_num(7e37), joined.nan_to_num(7e37))
    assert not bool(arrived.any())
    return out, joined


@pytest.mark.parametrize("gqa,KVH,BS", [(1, 2, 16), (2, 1, 8), (4, 8, 16), (8, 2, 32), (4, 3, 5), (1, 1, 1), (2, 2, 48), (8, 1, 7)])
@pytest.mark.parametrize("ctx,width", [
    ([1], None), ([0, 1, 15, 16, 17], None), ([63, 64, 65, 0], None), ([255, 256, 257, 1000], None),
    ([1, 1000, 300, 17], 256),                        # a table much wider than the contexts
    ([700 - 13 * i for i in range(30)], None),        # several tiles for a wave
])
def test_decode(gqa, KVH, BS, ctx, width):
    args = case(ctx, gqa, KVH, BS, seed=gqa + BS + len(ctx), width=width and width * 16 // BS + 1, shared=3)
    check(both(*args, D ** -0.5), *args, D ** -0.5)


@pytest.mark.parametrize("gqa,KVH,BS", [(4, 8, 16), (8, 1, 16), (1, 2, 6), (2, 1, 32)])
def test_long_contexts_in_shares(gqa, KVH, BS):
    args = case([9000, 5], gqa, KVH, BS, seed=gqa)
    check(both(*args, D ** -0.5), *args, D ** -0.5)


@pytest.mark.parametrize("ctx", [[40000, 3, 0], [9000, 30000], [0, 20000], [17000] + [40] * 20, [100] * 70 + [9000], [300 + 7 * i for i in range(200)],
                                 [5] * 300, [0, 0, 0, 700]])
@pytest.mark.parametrize("KVH,BS", [(1, 16), (4, 6)])
def test_one_context_much_longer_than_the_others(ctx, KVH, BS):
    args = case(ctx, 4, KVH, BS, seed=len(ctx))
    check(both(*args, D ** -0.5), *args, D ** -0.5)


@pytest.mark.parametrize("ctx", [[520] * 24, [1000] * 16, [2000] * 16, [640, 641] * 3, [900 + 60 * i for i in range(12)]])
def test_contexts_that_nearly_fill_the_chip(ctx):
    """Where shares of a context are one, two or four by how many contexts there are."""
    args = case(ctx, 4, 8, 16, seed=len(ctx), shared=3)
    check(both(*args, D ** -0.5), *args, D ** -0.5)


@pytest.mark.parametrize("gqa", [1, 2, 4, 8])
@pytest.mark.parametrize("spread", [3.0, 20.0])
def test_steps_and_scores_of_very_different_sizes(gqa, spread):
    """Rows of 2^-60 to 2^60: the running max and the steps' common power are renewed again and again."""
    q, kc, vc, ks, vs, tables, n = case([500, 129, 64], gqa, 2, 16, seed=gqa, spread=spread)
    scale = 2.0 ** (-3.5 - spread)
    check(both(q, kc, vc, ks, vs, tables, n, scale), q, kc, vc, ks, vs, tables, n, scale)


@pytest.mark.parametrize("gqa", [1, 4])
def test_rising_scores_and_rising_steps(gqa):
    q, kc, vc, ks, vs, tables, n = case([640], gqa, 1, 16, seed=3)
    at = torch.arange(640)
    blk, off = tables[0].long()[at // 16], at % 16
    up = torch.exp2(at / 40.0)[:, None, None]
    kc[blk, :, off], ks[blk, :, off] = torch_ref.kv4_quantize(q[0, :1].float() * up / 2048)
    vc[blk, :, off], vs[blk, :, off] = torch_ref.kv4_quantize(rows(640, 1, D, seed=5).float() * up)
    check(both(q, kc, vc, ks, vs, tables, n, 0.1), q, kc, vc, ks, vs, tables, n, 0.1)


def test_queries_of_any_size_scales_of_any_sign():
    q, kc, vc, ks, vs, tables, n = case([100, 100, 100, 100], 4, 2, 16, seed=11)
    q[0] = 0
    q[1] = (q[1].float() * 2.0 ** 100).bfloat16()
    q[2] = (q[2].float() * 2.0 ** -100).bfloat16()
    scale = torch.tensor([1.0, 2.0 ** -104, 2.0 ** 96, -0.2])
    for b in range(4):
        one = (q[b:b + 1], kc, vc, ks, vs, tables[b:b + 1], n[b:b + 1])
        check(both(*one, float(scale[b])), *one, float(scale[b]))


def test_a_row_that_is_no_number_is_its_groups_alone():
    q, kc, vc, ks, vs, tables, n = case([70, 200], 4, 2, 16, seed=12)
    blk, off = int(tables[1, 3]), 5
    vs[blk, 1, off, 1] = float("nan")                 # of kv head 1, values 64 to 127
    for out in both(q, kc, vc, ks, vs, tables, n, 0.1):
        bad = torch.isnan(out)
        assert bool(bad[1, 4:, 64:].all()) and int(bad.sum()) == 4 * 64
    ks[blk, 0, off, 0] = float("nan")                 # a key: all of its heads
    for out in both(q, kc, vc, ks, vs, tables, n, 0.1):
        assert bool(torch.isnan(out[1, :4]).all()) and int(torch.isnan(out).sum()) == 4 * 64 + 4 * 128


def test_strided_queries_and_empty_calls():
    q, kc, vc, ks, vs, tables, n = (t.to(DEV) for t in case([33, 65, 7], 4, 2, 16, seed=13))
    want = ops.attn_decode_paged(q, kc, vc, tables, n, 0.1, ks, vs)
    wide = torch.cat((q, q), 1)
    assert torch.equal(ops.attn_decode_paged(wide[:, 8:], kc, vc, tables, n, 0.1, ks, vs), want)
    odd = torch.empty(3 * 8 * D + 1, dtype=torch.bfloat16, device=DEV)[1:].view(3, 8, D).copy_(q)
    assert torch.equal(ops.attn_decode_paged(odd, kc, vc, tables, n, 0.1, ks, vs), want)
    assert ops.attn_decode_paged(q[:0], kc, vc, tables[:0], n[:0], 0.1, ks, vs).shape == (0, 8, D)
    assert not bool(ops.attn_decode_paged(q, kc, vc, tables[:, :0].contiguous(), n * 0, 0.1, ks, vs).any())
    assert not bool(ops.attn_decode_paged(q, kc, vc, tables, n * 0, 0.1, ks, vs).any())


def test_caches_of_more_than_2_gb():
    KVH, BS, NB = 8, 16, 300000                       # 2.5 GB of codes
    q, kc, vc, ks, vs, tables, n = case([300], 4, KVH, BS, seed=14)
    big = [torch.zeros(NB, *t.shape[1:], dtype=t.dtype, device=DEV) for t in (kc, vc, ks, vs)]
    far = torch.arange(NB - kc.shape[0], NB)
    for t, small in zip(big, (kc, vc, ks, vs)):
        t[far[0]:] = small.to(DEV)
    moved = (tables.long() + far[0]).int()
    want = both(q, kc, vc, ks, vs, tables, n, 0.1)[0]
    out = ops.attn_decode_paged(q.to(DEV), big[0], big[1], moved.to(DEV), n.to(DEV), 0.1, big[2], big[3])
    assert torch.equal(out, want)
    slots = torch.tensor([NB * BS - 1, (NB - 5) * BS], device=DEV)
    new = rows(2, KVH, D, seed=15).to(DEV)
    ops.store_kv(new, new, big[0], big[1], slots, big[2], big[3])
    a, b = ops.load_kv(big[0], big[1], slots, big[2], big[3])
    assert torch.equal(a, b) and torch.equal(a.cpu(), torch_ref.kv4_values(*torch_ref.kv4_quantize(new.cpu())).bfloat16())


@torch.inference_mode()                  # as the engine captures: torch's own state is of one kind for all captures
def test_replayed_and_on_another_stream():
    """Captured with the store, replayed with other work between; two graphs of one cache."""
    q, kc, vc, ks, vs, tables, n = (t.to(DEV) for t in case([700, 20], 4, 2, 16, seed=16))
    k_new, v_new = rows(2, 2, D, seed=17).to(DEV), rows(2, 2, D, seed=18).to(DEV)
    slots = torch.stack([tables[b, (n[b] - 1) // 16].long() * 16 + (n[b] - 1) % 16 for b in range(2)])
    arrived = torch.zeros(4, dtype=torch.int32, device=DEV)

    def step():
        ops.store_kv(k_new, v_new, kc, vc, slots, ks, vs)
        return ops.attn_decode_paged(q, kc, vc, tables, n, 0.1, ks, vs, arrived)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        graphs.append((g, out))
    for i in range(4):
        k_new.copy_(rows(2, 2, D, seed=20 + i))
        q.copy_(rows(2, 8, D, seed=40 + i))
        want = step().clone()
        for g, out in graphs:
            out.zero_()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want)


def test_refusals():
    q, kc, vc, ks, vs, tables, n = (t.to(DEV) for t in case([20], 4, 2, 16, seed=21))
    call = lambda **o: ops.attn_decode_paged(*[o.get(k, v) for k, v in dict(q=q, kc=kc, vc=vc, tables=tables, n=n, scale=0.1, ks=ks, vs=vs).items()])
    call()
    for bad in (dict(ks=ks.float()), dict(vs=vs[:, :, :, :1].contiguous()), dict(kc=kc[..., :32].contiguous()), dict(tables=tables.long()),
                dict(n=n.long()), dict(q=q.float()), dict(q=q[:, :6].contiguous()), dict(q=q[:, :, :64].contiguous()),
                dict(kc=kc.transpose(1, 2)), dict(tables=tables.cpu()), dict(n=torch.cat((n, n))), dict(vc=vc[:1])):
        with pytest.raises(RuntimeError):
            call(**bad)
    new, slots = rows(1, 2, D).to(DEV), torch.zeros(1, dtype=torch.long, device=DEV)
    for bad in (dict(slots=slots.int()), dict(k=new.float()), dict(k=new[:, :1]), dict(ks=ks.float()),
                dict(slots=torch.zeros(2, dtype=torch.long, device=DEV))):
        with pytest.raises(RuntimeError):
            ops.store_kv(bad.get("k", new), new, kc, vc, bad.get("slots", slots), bad.get("ks", ks), vs)


def segments(segs, gqa, KVH, BS, seed=0, spread=0.0):
    """q rows of segments [(start, rows)], caches and tables; every position up to a segment's last row is stored."""
    q, kc, vc, ks, vs, tables, n = case([p + r for p, r in segs], gqa, KVH, BS, seed=seed, spread=spread)
    rows_of = torch.tensor([r for _, r in segs])
    start = torch.tensor([p for p, _ in segs], dtype=torch.int32)
    seg = torch.repeat_interleave(torch.arange(len(segs)), rows_of)
    at = torch.arange(len(seg)) - (rows_of.cumsum(0) - rows_of)[seg]
    q = rows(len(seg), KVH * gqa, D, seed=seed + 5)
    return q, kc, vc, ks, vs, tables, start, tables[seg].contiguous(), (start[seg] + at + 1).int()


def attend(q, kc, vc, ks, vs, seg_tables, start, tables, lens, scale, segs, plan=None):
    plan, short = plan or ops.kv4_plan(segs, q.shape[1], kc.shape[1], DEV)
    return ops.attn_segments_paged(*(t.to(DEV) for t in (q, kc, vc, tables, lens)), scale, plan, short, seg_tables.to(DEV),
                                   start.to(DEV), ks.to(DEV), vs.to(DEV))


SEGMENTS = [[(0, 8)], [(5, 31), (0, 33)], [(300, 40), (0, 3), (77, 64), (1, 1), (500, 8)], [(1000, 150)], [(0, 700)],
            [(16, 257), (128, 128), (0, 1)], [(3, 7), (2, 6)], [(40, 300), (0, 0), (41, 20)]]


@pytest.mark.parametrize("segs", SEGMENTS)
@pytest.mark.parametrize("gqa,KVH,BS", [(4, 2, 16), (1, 3, 16), (2, 1, 5), (8, 1, 32), (4, 1, 1)])
def test_segments(segs, gqa, KVH, BS):
    args = segments(segs, gqa, KVH, BS, seed=gqa + BS)
    q, kc, vc, ks, vs, seg_tables, start, tables, lens = args
    out = attend(*args, D ** -0.5, segs)
    check([out], q, kc, vc, ks, vs, tables, lens, D ** -0.5)


@pytest.mark.parametrize("gqa,KVH", [(4, 2), (1, 1), (8, 1)])
def test_segments_whose_keys_are_cut(gqa, KVH):
    segs = [(2500, 40), (700, 9), (3000, 8)]
    args = segments(segs, gqa, KVH, 16, seed=3)
    q, kc, vc, ks, vs, seg_tables, start, tables, lens = args
    plan, _ = ops.kv4_plan(segs, gqa * KVH, KVH, DEV)
    assert plan.parts > 0
    check([attend(*args, 0.1, segs)], q, kc, vc, ks, vs, tables, lens, 0.1)


@pytest.mark.parametrize("segs,least", [([(0, 1), (64, 1), (300, 2), (7, 5)], 1), ([(40, 30), (9, 9), (0, 12), (3, 2)], 10),
                                        ([(40, 30), (9, 9)], 100)])
def test_segments_together_and_row_by_row(segs, least):
    args = segments(segs, 4, 2, 16, seed=12)
    q, kc, vc, ks, vs, seg_tables, start, tables, lens = args
    plan, short = ops.kv4_plan(segs, 8, 2, DEV, least)
    alone = sum(n for _, n in segs if n < least)
    assert sum(n for _, n in short) == alone and (plan is None) == (alone == len(q))
    check([attend(*args, 0.1, segs, (plan, short))], q, kc, vc, ks, vs, tables, lens, 0.1)


def test_plan_goes_row_by_row_where_there_is_little():
    assert ops.paged_plan([(500, 32)], 32, 8, DEV, torch.uint8) == (None, [(0, 32)])
    plan, short = ops.paged_plan([(4000, 16), (4000, 9), (4000, 40)], 32, 8, DEV, torch.uint8)
    assert plan is not None and short == [(16, 9)]


@pytest.mark.parametrize("spread", [3.0, 20.0])
def test_segments_with_rows_of_very_different_sizes(spread):
    """Rows of 2^-60 to 2^60: each slab has a power of its own, sums are put back."""
    segs = [(200, 70), (0, 40)]
    args = segments(segs, 4, 2, 16, seed=4, spread=spread)
    q, kc, vc, ks, vs, seg_tables, start, tables, lens = args
    scale = 2.0 ** (-3.5 - spread)
    check([attend(*args, scale, segs)], q, kc, vc, ks, vs, tables, lens, scale)


def test_segments_see_what_rows_see_alone():
    """Keys behind a row, of its own segment too, are not its own: one that is no number does not reach it."""
    segs = [(50, 100), (20, 64)]
    q, kc, vc, ks, vs, seg_tables, start, tables, lens = segments(segs, 4, 1, 16, seed=6)
    blk, off = int(seg_tables[0, 90 // 16]), 90 % 16              # position 90: rows 40 and on of the first segment
    for t in (ks, vs):
        held = t[blk, 0, off].clone()
        t[blk, 0, off, 1] = float("nan")
        out = attend(q, kc, vc, ks, vs, seg_tables, start, tables, lens, 0.1, segs).cpu()
        bad = torch.isnan(out)
        assert not bool(bad[:40].any()) and not bool(bad[100:].any()) and bool(bad[40:100, :, 64:].all())
        keep = list(range(40)) + list(range(100, 164))
        check([out[keep]], q[keep], kc, vc, ks, vs, tables[keep], lens[keep], 0.1)
        t[blk, 0, off] = held


def test_segments_of_any_queries_and_scales():
    segs = [(100, 40)]
    args = list(segments(segs, 4, 2, 16, seed=7))
    args[0][3] = 0
    args[0][5] = (args[0][5].float() * 2.0 ** 90).bfloat16()
    args[0][6] = (args[0][6].float() * 2.0 ** -90).bfloat16()
    for scale in (-0.2, 0.05):
        out = attend(*args, scale, segs).cpu()
        keep = [r for r in range(40) if r != 5]
        check([out[keep]], args[0][keep], *args[1:5], args[7][keep], args[8][keep], scale)
        assert bool(torch.isfinite(out[5]).all())               # one key alone


def test_segments_in_strided_rows_and_empty():
    segs = [(30, 40), (0, 2)]
    q, kc, vc, ks, vs, seg_tables, start, tables, lens = segments(segs, 4, 2, 16, seed=8)
    rest = (kc, vc, ks, vs, seg_tables, start, tables, lens, 0.1, segs)
    want = attend(q, *rest)
    wide = torch.cat((q, q), 1)
    plan = ops.kv4_plan(segs, 8, 2, DEV)
    got = ops.attn_segments_paged(wide.to(DEV)[:, 8:], kc.to(DEV), vc.to(DEV), tables.to(DEV), lens.to(DEV), 0.1, *plan,
                                  seg_tables.to(DEV), start.to(DEV), ks.to(DEV), vs.to(DEV))
    assert torch.equal(got, want)
    assert ops.paged_plan([], 8, 2, DEV, kc.dtype) == (None, []) and ops.paged_plan([(5, 0)], 8, 2, DEV, kc.dtype) == (None, [])


@torch.inference_mode()                  # as the engine captures: torch's own state is of one kind for all captures
def test_segments_replayed():
    segs = [(900, 70), (100, 30)]
    args = [t.to(DEV) for t in segments(segs, 4, 2, 16, seed=9)]
    q = args[0]
    plan = ops.kv4_plan(segs, 8, 2, DEV)
    step = lambda: attend(*args, 0.1, segs, plan)
    step()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    for i in range(3):
        q.copy_(rows(*q.shape, seed=60 + i))
        want = step().clone()
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


@pytest.mark.parametrize("B", [65535, 65536, 65839])              # one launch, a second of one row, a second of more rows than are dealt out
def test_more_decode_rows_than_a_grid_has_in_y(B):
    """A row for each token of long prompt portions, against the same rows in two calls: contexts of up to ten tiles, the
    first rows' and the second launch's among them, of which fewer rows would be given several workgroups."""
    q, kc, vc, ks, vs, tables, _ = case([640] * 8, 4, 1, 16, seed=31)
    g = torch.Generator().manual_seed(B)
    own = torch.randint(0, 8, (B,), generator=g)
    n = torch.randint(0, 641, (B,), generator=g).int()
    n[:4], n[-4:] = 640, 640
    q = torch.randn(B, 4, D, generator=g).bfloat16()
    q, kc, vc, ks, vs, tables, n = (t.to(DEV) for t in (q, kc, vc, ks, vs, tables[own], n))
    call = lambda a, b: ops.attn_decode_paged(q[a:b], kc, vc, tables[a:b], n[a:b], 0.1, ks, vs)
    out = call(0, B)
    assert torch.equal(out, torch.cat([call(0, 40000), call(40000, B)]))
    some = torch.tensor([0, 3, 255, 256, 65534, B - 1])
    check([out[some]], *(t.cpu() for t in (q[some], kc, vc, ks, vs, tables[some], n[some])), 0.1)


def test_turned_rows_for_no_slot_go_nowhere():
    """rope_store of aligned rows, of rows off 16 bytes and of a decode step's sums: a slot in front of the cache, the first one
    behind it and far ones. Rows of other memory lie on both sides, so that what went there would be seen."""
    T, H, G, BS, NB, off = 7, 4, 2, 4, 3, 2
    inside, slots = torch.tensor([0, 3, 6]), torch.tensor([2, -1, NB * BS, 7, -BS, 1 << 40, NB * BS - 1], device=DEV)
    qkv = rows(T, H + 2 * G, D, seed=33).to(DEV)
    pos = torch.zeros(T, dtype=torch.long, device=DEV)           # where turning rounds nothing: all forms have the same rows
    cos_sin = torch_ref.build_cos_sin_cache(D, 64, 1e4, "cpu").to(DEV)
    shapes = [(G, BS, D // 2), (G, BS, D // 2), (G, BS, 2, 2), (G, BS, 2, 2)]

    def caches():                                 # blocks off.. off + NB of larger ones
        big = [torch.zeros(NB + 2 * off, *s, dtype=torch.uint8 if len(s) == 3 else torch.bfloat16, device=DEV) for s in shapes]
        return big, [t[off:off + NB] for t in big]

    odd = torch.empty(qkv.numel() + 1, dtype=torch.bfloat16, device=DEV)[1:].view(qkv.shape)
    stored = []
    for rows_at in (torch.empty_like(qkv), odd):
        rows_at.copy_(qkv)
        big, c = caches()
        ops.rope_store(*rows_at.split([H, G, G], 1), pos, cos_sin, c[0], c[1], slots, c[2], c[3])
        stored.append((big, c, rows_at.clone()))
    big, c = caches()
    got = ops.rope_store_rows(qkv.view(1, T, -1).float().contiguous(), None, H, pos, cos_sin, c[0], c[1], slots, c[2], c[3])
    stored.append((big, c, torch.cat((got, stored[0][2][:, H:]), 1)))
    for big, c, turned in stored:
        assert torch.equal(turned, stored[0][2])                  # of all rows
        want = [torch.zeros(NB + 2 * off, *s, dtype=t.dtype) for s, t in zip(shapes, big)]
        inner = [t[off:off + NB] for t in want]
        torch_ref.store_kv(turned[:, H:H + G].cpu()[inside], turned[:, H + G:].cpu()[inside], inner[0], inner[1], slots.cpu()[inside], inner[2], inner[3])
        assert all(torch.equal(t.cpu().float(), w.float()) for t, w in zip(big, want))


def grouped(x, sizes):
    """Rows [..., 128] with values 0..63 and 64..127 in sizes of their own [..., 2]."""
    return (x.float().unflatten(-1, (2, 64)) * sizes[..., None]).flatten(-2).bfloat16()


def check_prompts(out, q, kc, vc, ks, vs, tables, n, scale):
    want, off = prompts64(q, kc, vc, ks, vs, tables, n, scale)
    far = (out.double().cpu() - want).abs()
    assert bool((far <= off).all()), f"{float((far / off).max())} of what is allowed, at {torch.nonzero(far > off)[:3].tolist()}"


def restore(cache, scales, table, at, x):
    BS = cache.shape[2]
    blk, off = table.long()[at // BS], at % BS
    cache[blk, :, off], scales[blk, :, off] = torch_ref.kv4_quantize(x)


@pytest.mark.parametrize("gqa,KVH", [(4, 2), (1, 1), (8, 1)])
@pytest.mark.parametrize("segs", [[(200, 70), (0, 40)], [(2500, 40)]])
@pytest.mark.parametrize("low", [-9, -16, -20, -24, -60])
def test_segments_whose_groups_differ_in_size(segs, gqa, KVH, low):
    """Values 64..127 of keys and values 2^low of the others; what q has there is as much larger (up to 2^20), so that both groups
    say which keys count."""
    q, kc, vc, ks, vs, seg_tables, start, tables, lens = segments(segs, gqa, KVH, 16, seed=low + 100)
    sizes = torch.tensor([1.0, 2.0 ** low])
    for i, (p, r) in enumerate(segs):
        at = torch.arange(p + r)
        restore(kc, ks, seg_tables[i], at, grouped(rows(p + r, KVH, D, seed=i + 40), sizes))
        restore(vc, vs, seg_tables[i], at, grouped(rows(p + r, KVH, D, seed=i + 50), sizes))
    q = grouped(q, torch.tensor([1.0, 2.0 ** min(-low, 20)]))
    out = attend(q, kc, vc, ks, vs, seg_tables, start, tables, lens, D ** -0.5, segs)
    check_prompts(out, q, kc, vc, ks, vs, tables, lens, D ** -0.5)


@pytest.mark.parametrize("gqa", [1, 4])
def test_segments_whose_groups_have_any_size(gqa):
    segs = [(300, 70), (10, 40), (2100, 12)]
    q, kc, vc, ks, vs, seg_tables, start, tables, lens = segments(segs, gqa, 2, 16, seed=71)
    g = torch.Generator().manual_seed(72)
    for i, (p, r) in enumerate(segs):
        for cache, scales, spread in ((kc, ks, 5.0), (vc, vs, 15.0)):
            x = grouped(rows(p + r, 2, D, seed=i + 60), torch.exp2(torch.randn(p + r, 2, 2, generator=g) * spread))
            restore(cache, scales, seg_tables[i], torch.arange(p + r), x)
    scale = 2.0 ** -18
    check_prompts(attend(q, kc, vc, ks, vs, seg_tables, start, tables, lens, scale, segs), q, kc, vc, ks, vs, tables, lens, scale)


def test_one_group_of_another_size_in_a_cut_segment():
    """One key's and another's value's second group, in one of the items of a segment: the others go on as they were."""
    segs = [(2500, 40)]
    q, kc, vc, ks, vs, seg_tables, start, tables, lens = segments(segs, 4, 2, 16, seed=73)
    for cache, scales, at, size in ((kc, ks, 1300, 2.0 ** 18), (vc, vs, 1301, 2.0 ** -40), (vc, vs, 77, 2.0 ** 30)):
        restore(cache, scales, seg_tables[0], torch.tensor([at]), grouped(rows(1, 2, D, seed=at), torch.tensor([1.0, size])))
    q = grouped(q, torch.tensor([1.0, 2.0 ** -16]))
    assert ops.kv4_plan(segs, 8, 2, DEV)[0].parts > 1
    out = attend(q, kc, vc, ks, vs, seg_tables, start, tables, lens, 0.1, segs)
    check_prompts(out, q, kc, vc, ks, vs, tables, lens, 0.1)


@pytest.mark.parametrize("segs", SEGMENTS)
def test_segments_are_as_far_off_as_their_roundings(segs):
    q, kc, vc, ks, vs, seg_tables, start, tables, lens = segments(segs, 4, 2, 16, seed=74)
    out = attend(q, kc, vc, ks, vs, seg_tables, start, tables, lens, D ** -0.5, segs)
    check_prompts(out, q, kc, vc, ks, vs, tables, lens, D ** -0.5)


@pytest.mark.parametrize("planned", [[(2500, 40), (100, 33)], [(0, 40), (4000, 33)], [(1300, 40), (0, 33)]])
def test_segments_at_other_starts_than_the_plans(planned):
    """The starts on the device say which keys a row sees: more than the plan was made of, fewer, or none of a cut piece."""
    segs = [(1300, 40), (700, 33)]
    q, kc, vc, ks, vs, seg_tables, start, tables, lens = segments(segs, 4, 2, 16, seed=75)
    plan = ops.kv4_plan(planned, 8, 2, DEV)
    out = attend(q, kc, vc, ks, vs, seg_tables, start, tables, lens, 0.1, segs, plan)
    check_prompts(out, q, kc, vc, ks, vs, tables, lens, 0.1)


def test_segments_of_tables_without_blocks_are_zeros():
    segs = [(0, 40), (0, 12)]
    q, kc, vc, ks, vs, seg_tables, start, tables, lens = segments(segs, 4, 2, 16, seed=76)
    plan = ops.kv4_plan(segs, 8, 2, DEV)
    for cut in (dict(tables=slice(0, 0)), dict(blocks=0)):
        full = torch.full(q.shape, 7.0, dtype=torch.bfloat16, device=DEV)      # its memory is the next result's
        del full
        if "tables" in cut:
            out = attend(q, kc, vc, ks, vs, seg_tables[:, :0].contiguous(), start, tables[:, :0].contiguous(), lens * 0, 0.1, segs, plan)
        else:
            out = attend(q, kc[:0], vc[:0], ks[:0], vs[:0], seg_tables * 0, start, tables * 0, lens * 0, 0.1, segs, plan)
        assert not bool(out.any())

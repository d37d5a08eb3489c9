"""The 4-bit cache on the CPU: its form, its bounds, its refusals, the engine with it."""

import pytest
import torch

from kllms_amd import ops
from kllms_amd.ops import torch_ref

from kv4_oracle import attention64, values64


@pytest.mark.parametrize("D", [8, 16, 24, 64, 128, 256])
def test_half_a_step_off_at_most(D):
    x = (torch.randn(9, 3, D) * torch.exp(torch.randn(9, 3, 1) * 3)).bfloat16()
    codes, scales = torch_ref.kv4_quantize(x)
    assert codes.shape == (9, 3, D // 2) and scales.shape == (9, 3, torch_ref.kv4_groups(D), 2)
    got = values64(codes, scales)
    step = scales[..., 0].double()
    far = (got - x.double()).abs().view(9, 3, step.shape[-1], -1).amax(-1)
    # half a step, and at the far end what the step's rounding to bf16 (2^-8 of it, half of 2^-7) makes of fifteen
    assert bool((far <= step * (0.5 + 15 * 2 ** -8)).all())
    assert torch.equal(torch_ref.kv4_values(codes, scales).double(), got.float().double())


def test_rows_that_are_constant_or_not_finite():
    x = torch.randn(6, 1, 128).bfloat16()
    x[0] = 3.25
    x[1, :, :64] = 0
    x[2, 0, 5] = float("nan")
    x[3, 0, 70] = float("inf")
    x[4, 0, 1], x[4, 0, 2] = 3e38, -3e38                  # a range that fp32 does not hold
    x[5] = x[5] * 1e-39                                   # a step below the normal numbers
    codes, scales = torch_ref.kv4_quantize(x)
    v = values64(codes, scales)[:, 0]
    assert torch.equal(v[0], x[0, 0].double()) and bool((v[1, :64] == 0).all())
    nan = torch.isnan(v)
    want = torch.zeros_like(nan)
    want[2, :64] = want[3, 64:] = want[4, :64] = True
    assert torch.equal(nan, want)
    assert bool((v[5] - x[5, 0].double()).abs().max() < 1e-37)


def test_head_sizes_that_have_no_form():
    for D in (4, 12, 96, 100):
        with pytest.raises(ValueError, match="4-bit cache"):
            torch_ref.kv4_quantize(torch.zeros(1, D))


def caches(NB, KVH, BS, D=128):
    kc, vc = (torch.randint(0, 256, (NB, KVH, BS, D // 2), dtype=torch.uint8) for _ in range(2))
    ks, vs = (torch.randn(NB, KVH, BS, torch_ref.kv4_groups(D), 2).abs().bfloat16() for _ in range(2))
    return kc, vc, ks, vs


def test_store_and_load_leave_other_rows_alone():
    kc, vc, ks, vs = caches(4, 2, 8)
    before = [t.clone() for t in (kc, vc, ks, vs)]
    k, v = torch.randn(3, 2, 128).bfloat16(), torch.randn(3, 2, 128).bfloat16()
    slots = torch.tensor([31, -1, 9])
    ops.store_kv(k, v, kc, vc, slots, ks, vs)
    a, b = ops.load_kv(kc, vc, slots, ks, vs)
    assert bool(torch.isnan(a[1]).all() and torch.isnan(b[1]).all())
    for got, x in ((a, k), (b, v)):
        want = torch_ref.kv4_values(*torch_ref.kv4_quantize(x)).bfloat16()
        assert torch.equal(got[[0, 2]], want[[0, 2]])
    touched = torch.zeros(4, 8, dtype=torch.bool)
    touched.view(-1)[[31, 9]] = True
    for t, old in zip((kc, vc, ks, vs), before):
        assert torch.equal(t.transpose(1, 2)[~touched], old.transpose(1, 2)[~touched])


def test_refusals():
    kc, vc, ks, vs = caches(2, 1, 4)
    k, slots = torch.zeros(1, 1, 128), torch.zeros(1, dtype=torch.long)
    tables, lens = torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    for call in (lambda: ops.store_kv(k, k, kc, vc, slots), lambda: ops.load_kv(kc, vc, slots, ks, None),
                 lambda: ops.attn_decode_paged(k, kc, vc, tables, lens, 1.0),
                 lambda: ops.rope_store(k, k, k, slots, torch.ones(1, 128), kc, vc, slots),
                 lambda: ops.attn_segments_paged(k, kc, vc, tables, lens, 1.0, None, [], tables, lens)):
        with pytest.raises(ValueError, match="4-bit cache needs"):
            call()
    with pytest.raises(ValueError, match="load_kv reads 4-bit"):
        ops.load_kv(torch.zeros(2, 1, 4, 128), torch.zeros(2, 1, 4, 128), slots, ks, vs)


@pytest.mark.parametrize("D,gqa", [(128, 4), (16, 1), (64, 2)])
def test_decode_against_64_bits(D, gqa):
    KVH, BS, lens = 2, 4, [1, 9, 0, 30]
    kc, vc, ks, vs = caches(40, KVH, BS, D)
    tables = torch.randperm(40)[:32].view(4, 8).int()
    n = torch.tensor(lens, dtype=torch.int32)
    q = torch.randn(4, KVH * gqa, D).bfloat16()
    out = ops.attn_decode_paged(q, kc, vc, tables, n, D ** -0.5, ks, vs)
    want, off = attention64(q, kc, vc, ks, vs, tables, n, D ** -0.5)
    assert bool(((out.double() - want).abs() <= off).all())


def engine(**more):
    from kllms_amd.engine.config import EngineConfig
    from kllms_amd.engine.engine import LLMEngine

    return LLMEngine(EngineConfig(**{**dict(model="tiny-llama", max_kv_blocks=256, use_hip_graphs=False, device="cpu", seed=0,
                                            kv_cache_dtype="int4"), **more}))


def greedy(n):
    from kllms_amd.engine.sampling import SamplingParams

    return SamplingParams(temperature=0.0, max_new_tokens=n)


@pytest.mark.parametrize("model", ["tiny-llama", "tiny-mixtral"])
def test_engine_generates(model):
    from kllms_amd.engine.engine import GenRequest

    eng = engine(model=model)
    assert eng.kv.k_all.dtype == torch.uint8 and eng.kv.k_all.shape[-1] * 2 == eng.arch.head_dim_
    outs = eng.generate([GenRequest(prompt_ids=list(range(1, 30)), n=3, sampling=greedy(8)),
                         GenRequest(prompt_ids=[5], n=1, sampling=greedy(4))])
    first = outs[0].streams[0].token_ids
    assert len(first) >= 1 and all(s.token_ids == first for s in outs[0].streams)      # one prompt, no drawing: all alike


def test_step_logits_are_those_of_the_values_the_cache_holds():
    """A decode step over the 4-bit cache equals one over a plain cache that holds the same values."""
    from kllms_amd.engine.engine import GenRequest

    eng, plain = engine(), engine(kv_cache_dtype="bf16")
    ids = list(range(1, 40))
    outs = {}
    for name, e in (("int4", eng), ("bf16", plain)):
        seqs, streams = [], []
        with torch.inference_mode():
            e.begin_requests([GenRequest(prompt_ids=ids, n=1, sampling=greedy(4))], seqs, streams)
        outs[name] = streams[0]
    a, b = outs["int4"].seq, outs["bf16"].seq
    assert a.blocks == b.blocks
    for layer in range(eng.kv.num_layers):
        for c4, s4, c in ((eng.kv.k_caches, eng.kv.k_scale_all, plain.kv.k_caches), (eng.kv.v_caches, eng.kv.v_scale_all, plain.kv.v_caches)):
            held = torch_ref.kv4_values(c4[layer][a.blocks], s4[layer][a.blocks])
            had = c[layer][a.blocks].bfloat16().float()
            step = s4[layer][a.blocks][..., 0].float().amax()
            assert bool(((held - had).abs() <= 0.53 * step).all())
            c[layer][a.blocks] = held
    from kllms_amd.models.llama import ForwardBatch

    def step(e, seq):
        slot = e.kv.append_slot(seq)
        n = seq.num_tokens
        batch = ForwardBatch(mode="decode", positions=torch.tensor([n - 1]), slot_mapping=torch.tensor([slot]),
                             kv_caches=e.kv.layer_caches(), block_tables=torch.tensor([seq.blocks], dtype=torch.int32),
                             context_lens=torch.tensor([n], dtype=torch.int32))
        with torch.inference_mode():
            return e.model.forward_decode(torch.tensor([7]), batch)

    got, want = step(eng, a), step(plain, b)
    # one position of 40 is rounded to 4 bits in one of them: the logits move by a small part of their spread
    assert float((got - want).abs().max()) < 0.1 * float(want.std())


def test_a_copied_block_takes_its_scales_along():
    eng = engine()
    kv = eng.kv
    src = kv.allocator.alloc()
    for t in (kv.k_all, kv.v_all):
        t[:, src] = torch.randint(0, 256, t[:, src].shape, dtype=torch.uint8)
    for t in (kv.k_scale_all, kv.v_scale_all):
        t[:, src] = torch.randn(t[:, src].shape).bfloat16()
    dst = kv._copy_block(src)
    for t in (kv.k_all, kv.v_all, kv.k_scale_all, kv.v_scale_all):
        assert torch.equal(t[:, src], t[:, dst]) and dst != src
    assert all(len(c) == 4 and c[2].dtype == torch.bfloat16 for c in kv.layer_caches())


def test_models_with_states_are_refused():
    with pytest.raises(ValueError, match="int4"):
        engine(model="tiny-zutalix")


def test_a_plan_of_other_rows_is_refused():
    segs = [(40, 20), (0, 12)]
    plan, short = ops.kv4_plan(segs, 8, 2, "cpu")
    assert (plan.rows, plan.segments, plan.heads) == (32, 2, 4)
    q, cache = torch.zeros(32, 8, 128, dtype=torch.bfloat16), torch.zeros(4, 2, 16, 64, dtype=torch.uint8)
    scales, tables, start = torch.zeros(4, 2, 16, 2, 2, dtype=torch.bfloat16), torch.zeros(2, 4, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    lens = torch.zeros(32, dtype=torch.int32)
    for bad in (dict(q=q[:31]), dict(seg_tables=tables[:1]), dict(q=torch.zeros(32, 4, 128, dtype=torch.bfloat16))):
        args = {**dict(q=q, k_cache=cache, v_cache=cache, block_tables=tables, context_lens=lens, scale=0.1, plan=plan, short=short, seg_tables=tables,
                       seg_start=start, k_scale=scales, v_scale=scales), **bad}
        with pytest.raises(ValueError, match="a plan of 32 rows in 2 segments"):
            ops.attn_segments_paged(**args)


def test_a_plan_of_fewer_rows_than_there_are_is_refused():
    """The rows behind the plan's would be nobody's: their results were left as the memory had them."""
    plan, short = ops.kv4_plan([(40, 20), (0, 12)], 8, 2, "cpu")
    cache = torch.zeros(4, 2, 16, 64, dtype=torch.uint8)
    scales, tables, start = torch.zeros(4, 2, 16, 2, 2, dtype=torch.bfloat16), torch.zeros(2, 4, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    call = lambda rows, plan, short: ops.attn_segments_paged(torch.zeros(rows, 8, 128, dtype=torch.bfloat16), cache, cache, torch.zeros(rows, 4, dtype=torch.int32),
                                                             torch.zeros(rows, dtype=torch.int32), 0.1, plan, short, tables, start, scales, scales)
    with pytest.raises(ValueError, match="a plan of 32 rows in 2 segments"):
        call(33, plan, short)
    for rows, short in ((33, [(0, 32)]), (5, [(0, 2), (2, 2)]), (1, [])):
        with pytest.raises(ValueError, match="row by row"):
            call(rows, None, short)

"""The engine on the GPU with weights in 8-bit integers and a 4-bit cache: whole runs of the operators together."""

import pytest
import torch

from kllms_amd import ops
from kllms_amd.engine.config import EngineConfig
from kllms_amd.engine.engine import GenRequest, LLMEngine
from kllms_amd.engine.sampling import SamplingParams
from kllms_amd.models.llama import ForwardBatch
from kllms_amd.ops import torch_ref

pytestmark = pytest.mark.gpu


def engine(**more):
    return LLMEngine(EngineConfig(**{**dict(model="mid-llama", max_kv_blocks=512, use_hip_graphs=False, device="cuda:0", seed=0), **more}))


def requests(n=3, tokens=12):
    g = torch.Generator().manual_seed(0)
    return [GenRequest(prompt_ids=torch.randint(1, 400, (k,), generator=g).tolist(), n=n,
                       sampling=SamplingParams(temperature=0.0, max_new_tokens=tokens)) for k in (40, 3, 170)]


@pytest.mark.parametrize("weight,cache", [("bf16", "int4"), ("int8", "bf16"), ("int8", "fp8_e4m3"), ("int8", "int4")])
@pytest.mark.parametrize("model", ["mid-llama", "mid-mixtral"])
def test_graphs_give_what_eager_steps_give(model, weight, cache):
    runs = []
    for graphs in (False, True):
        eng = engine(model=model, weight_dtype=weight, kv_cache_dtype=cache, use_hip_graphs=graphs, hip_graph_batch_sizes=[9, 16])
        runs.append([[s.token_ids for s in o.streams] for o in eng.generate(requests())])
        if graphs:
            assert eng._graph_runner._enabled and eng._graph_runner.graphs
    assert runs[0] == runs[1]
    assert all(len(t) > 0 for o in runs[0] for t in o)


@pytest.mark.parametrize("B", [5, 24])
def test_a_step_on_the_few_row_kernels_is_one_of_the_modules(B):
    """The step's sums in shares against the layers' own calls: the same whole numbers, rounded at other places."""
    eng = engine(weight_dtype="int8", kv_cache_dtype="int4")
    model, kv = eng.model, eng.kv
    ctx = 70
    g = torch.Generator().manual_seed(1)
    per = -(-ctx // 16)
    tables = torch.arange(B * per, dtype=torch.int32).view(B, per).cuda()
    slots = torch.arange(B * per * 16).view(B, -1)[:, :ctx].reshape(-1).cuda()
    for k, v, ks, vs in kv.layer_caches():
        rows = torch.randn(2, B * ctx, k.shape[1], 128, generator=g).bfloat16().cuda()
        ops.store_kv(rows[0], rows[1], k, v, slots, ks, vs)
    batch = ForwardBatch(mode="decode", positions=torch.full((B,), ctx - 1, device="cuda"), kv_caches=kv.layer_caches(), block_tables=tables,
                         slot_mapping=slots.view(B, ctx)[:, -1].contiguous(), context_lens=torch.full((B,), ctx, dtype=torch.int32, device="cuda"))
    ids = torch.arange(3, 3 + B, device="cuda")
    with torch.inference_mode():
        assert model._takes_rows(ids, batch)
        got = model.forward_hidden(ids, batch).float()
        hidden, residual = model.embed_tokens(ids), None
        for layer in model.layers:
            hidden, residual = layer(hidden, residual, batch, model.cos_sin)
        want = ops.fused_add_rmsnorm(hidden, residual, model.norm.weight, model.norm.eps)[0].float()
    # a bf16 rounding that falls differently moves a row's codes by one of 127 steps here and there
    assert float((got - want).norm()) < 0.03 * float(want.norm())


@pytest.mark.parametrize("cache", ["int4"])
def test_prompts_behind_a_cached_prefix(cache):
    """Whole prompts, then others with the same head, whose tails attend over the 4-bit cache."""
    eng = engine(kv_cache_dtype=cache, weight_dtype="int8", prefix_cache_min_tokens=32, max_seq_len=1024)
    head = list(range(5, 5 + 160))
    first = [GenRequest(prompt_ids=head + [7] * 40, n=1, sampling=SamplingParams(temperature=0.0, max_new_tokens=4))]
    eng.generate(first)
    g = torch.Generator().manual_seed(2)
    tails = [GenRequest(prompt_ids=head + torch.randint(1, 400, (k,), generator=g).tolist(), n=2,
                        sampling=SamplingParams(temperature=0.0, max_new_tokens=5)) for k in (1, 33, 90, 300)]
    outs = eng.generate(tails)
    alone = [eng.generate([t])[0] for t in tails]
    for o, a in zip(outs, alone):
        assert o.streams[0].token_ids == o.streams[1].token_ids and len(o.streams[0].token_ids) > 0
        assert len(a.streams[0].token_ids) > 0


def test_int8_weights_hold_half_the_bytes():
    eng = engine(weight_dtype="int8")
    at = eng.model.layers[0].self_attn
    assert at.qkv_proj.weight.dtype == torch.int8 and at.qkv_proj.weight.is_cuda
    codes, scales = torch_ref.quantize_weights(at.qkv_proj.weight.float().cpu() * at.qkv_proj.weight_scale.cpu()[:, None])
    assert torch.equal(codes, at.qkv_proj.weight.cpu())


def step_operands(device, G=2, M=3, H=4):
    g = torch.Generator().manual_seed(3)
    sizes = dict(part=torch.randn(2, M, (H + 2 * G) * 128, generator=g), bias=torch.randn((H + 2 * G) * 128, generator=g).bfloat16(), num_heads=H,
                 positions=torch.arange(M), cos_sin=torch_ref.build_cos_sin_cache(128, 64, 1e4, "cpu"), k_cache=torch.zeros(2, G, 16, 64, dtype=torch.uint8),
                 v_cache=torch.zeros(2, G, 16, 64, dtype=torch.uint8), slot_mapping=torch.arange(M), k_scale=torch.zeros(2, G, 16, 2, 2).bfloat16(),
                 v_scale=torch.zeros(2, G, 16, 2, 2).bfloat16())
    return {k: t.to(device) if isinstance(t, torch.Tensor) else t for k, t in sizes.items()}


def test_operands_on_another_device_are_refused():
    args = step_operands("cuda:0")
    ops.rope_store_rows(**args)
    for name, t in args.items():
        if isinstance(t, torch.Tensor):
            with pytest.raises(RuntimeError):
                ops.rope_store_rows(**{**args, name: t.cpu()})
    rows = torch.randn(3, 8, 128, device="cuda:0").bfloat16()
    q, k, v = rows.split([4, 2, 2], 1)
    more = [args[n] for n in ("positions", "cos_sin", "k_cache", "v_cache", "slot_mapping", "k_scale", "v_scale")]
    ops.rope_store(q, k, v, *more)
    for i in range(len(more)):
        with pytest.raises(RuntimeError):
            ops.rope_store(q, k, v, *more[:i], more[i].cpu(), *more[i + 1:])
    part, residual, weight = torch.zeros(2, 3, 256), torch.zeros(3, 256).bfloat16(), torch.ones(256).bfloat16()
    for away in range(3):
        with pytest.raises(RuntimeError):
            ops.add_norm_rows_int8(*(t if i == away else t.cuda() for i, t in enumerate((part, residual, weight))), 1e-5)


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_a_steps_operators_on_a_device_that_is_not_the_current_one():
    def step(device):
        args = step_operands(device)
        q = ops.rope_store_rows(**args)
        residual = torch.ones(3, 1024, device=device).bfloat16()
        codes, scales = ops.add_norm_rows_int8(args["part"].contiguous(), residual, residual[0].contiguous(), 1e-5)
        torch.cuda.synchronize(device)
        return [t.cpu() for t in (q, args["k_cache"], args["v_scale"], residual, codes, scales)]

    with torch.cuda.device(0):
        assert all(torch.equal(a, b) for a, b in zip(step("cuda:0"), step("cuda:1")))


def test_tails_behind_a_cached_prefix_attend_to_what_the_cache_holds(monkeypatch):
    """Each layer's attention of tails that share a cached head against 64 bits over the cache's values, for rows of each tail
    (positions and blocks of rows, where the kernel has those of segments); and the model's rows against the same passes row by row."""
    from kv4_oracle import prompts64

    head = list(range(5, 5 + 160))
    g = torch.Generator().manual_seed(2)
    sizes = (1, 33, 90, 400)
    tails = [GenRequest(prompt_ids=head + torch.randint(1, 400, (k,), generator=g).tolist(), n=2,
                        sampling=SamplingParams(temperature=0.0, max_new_tokens=5)) for k in sizes]
    first = [GenRequest(prompt_ids=head + [7] * 40, n=1, sampling=SamplingParams(temperature=0.0, max_new_tokens=4))]
    together, plan_of = ops.attn_segments_paged, ops.paged_plan
    seen = []

    def watched(q, k, v, tables, lens, scale, plan, short, seg_tables, seg_start, ks=None, vs=None):
        out = together(q, k, v, tables, lens, scale, plan, short, seg_tables, seg_start, ks, vs)
        ends = torch.tensor([r for r in range(len(lens)) if r + 1 == len(lens) or int(lens[r + 1]) != int(lens[r]) + 1])
        starts = torch.cat((torch.zeros(1, dtype=torch.long), ends[:-1] + 1))
        some = torch.cat((starts, (starts + ends) // 2, ends)).unique()
        want, off = prompts64(*(t.cpu() for t in (q[some], k, v, ks, vs, tables[some], lens[some])), scale)
        assert bool(((out[some].double().cpu() - want).abs() <= off).all())
        seen.append((plan is not None, (lens[starts] - 1).tolist(), (ends - starts + 1).tolist()))
        return out

    runs = []
    for rows_alone in (False, True):
        eng = engine(kv_cache_dtype="int4", weight_dtype="int8", prefix_cache_min_tokens=32, max_seq_len=1024)
        eng.generate(first)
        hidden, forward = [], eng.model.forward_hidden
        with monkeypatch.context() as m:
            m.setattr(eng.model, "forward_hidden", lambda *a: hidden.append(forward(*a)) or hidden[-1])
            if rows_alone:
                m.setattr(ops, "paged_plan", lambda segs, *a: (None, [(0, sum(n for _, n in segs))]))
            else:
                m.setattr(ops, "attn_segments_paged", watched)
            saved = eng.prefix_cache.tokens_saved
            outs = eng.generate(tails)
        assert eng.prefix_cache.tokens_saved - saved == 160 * len(tails)
        assert all(len(s.token_ids) > 0 for o in outs for s in o.streams)
        runs.append(hidden[0].float())
    assert seen == [(True, [160] * 4, list(sizes))] * eng.kv.num_layers
    assert ops.paged_plan is plan_of and runs[0].shape == runs[1].shape == (sum(sizes), eng.arch.hidden_size)
    # a bf16 rounding that falls differently moves a row's codes by one of 127 steps here and there
    assert float((runs[0] - runs[1]).norm()) < 0.03 * float(runs[1].norm())

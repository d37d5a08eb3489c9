"""Weights in 8-bit integers and the 4-bit cache in shards: two ranks over gloo against one process that adds the shards up."""

import multiprocessing as mp
import os
import socket

import pytest
import torch

from kllms_amd import ops

IDS = list(range(1, 33))
MODELS = ["tiny-llama", "tiny-qwen", "tiny-mixtral"]               # plain, with biases, with experts


def engine(model, world=1, ctx=None):
    from kllms_amd.engine.config import EngineConfig
    from kllms_amd.engine.engine import LLMEngine

    return LLMEngine(EngineConfig(model=model, tp_size=world, max_kv_blocks=64, use_hip_graphs=False, device="cpu", seed=0, weight_dtype="int8",
                                  kv_cache_dtype="int4"), parallel_ctx=ctx)


def biases_(model, world=1, rank=0):
    """Biases that differ from row to row, sharded as the weights are."""
    for m in model.modules():
        if getattr(m, "partition_sizes", None) and m.bias is not None:
            full = torch.randn(sum(m.partition_sizes), generator=torch.Generator().manual_seed(len(m.bias) * world)) * 0.1
            m.bias.data.copy_(torch.cat([p.chunk(world)[rank] for p in full.split(m.partition_sizes)]))


def logits_and_tokens(eng):
    """Logits of a prompt's last row and of a step behind it, which attends over the cache; greedy tokens."""
    from kllms_amd.engine.engine import GenRequest
    from kllms_amd.engine.sampling import SamplingParams
    from kllms_amd.models.llama import ForwardBatch

    seq = eng.kv.alloc_sequence(len(IDS))
    with torch.inference_mode():
        first = eng.model.forward_prefill(torch.tensor(IDS), ForwardBatch(
            mode="prefill", positions=torch.arange(len(IDS)), slot_mapping=torch.tensor(eng.kv.prefill_slot_mapping(seq)),
            kv_caches=eng.kv.layer_caches(), cu_seqlens=torch.tensor([0, len(IDS)], dtype=torch.int32)))
        slot = eng.kv.append_slot(seq)
        n = seq.num_tokens
        step = eng.model.forward_decode(torch.tensor([7]), ForwardBatch(
            mode="decode", positions=torch.tensor([n - 1]), slot_mapping=torch.tensor([slot]), kv_caches=eng.kv.layer_caches(),
            block_tables=torch.tensor([seq.blocks], dtype=torch.int32), context_lens=torch.tensor([n], dtype=torch.int32)))
    eng.kv.free_sequence(seq)
    out = eng.generate([GenRequest(prompt_ids=IDS, n=2, sampling=SamplingParams(temperature=0.0, max_new_tokens=6))])[0]
    return torch.cat((first.view(1, -1), step.view(1, -1))).clone(), [s.token_ids for s in out.streams]


def worker(rank, world, port, q):
    import torch.distributed as dist

    from kllms_amd.parallel.tp import ParallelContext

    torch.set_num_threads(1)             # two ranks' many small products otherwise wait for each other's threads
    os.environ["MASTER_ADDR"], os.environ["MASTER_PORT"] = "127.0.0.1", str(port)
    dist.init_process_group("gloo", rank=rank, world_size=world)
    try:
        results = []
        for model in MODELS:
            eng = engine(model, world, ParallelContext(world_size=world, rank=rank))
            biases_(eng.model, world, rank)
            held = {n: p.detach().numpy() for n, p in eng.model.named_parameters() if n.endswith(("proj.weight", "weight_scale"))}
            logits, tokens = logits_and_tokens(eng)
            results.append((held, logits.numpy(), tokens))
        q.put((rank, results))
    finally:
        dist.destroy_process_group()


@pytest.fixture(scope="module")
def ranks():
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    procs = [ctx.Process(target=worker, args=(r, 2, port, q)) for r in range(2)]
    for p in procs:
        p.start()
    got = dict(q.get(timeout=240) for _ in procs)
    for p in procs:
        p.join(timeout=60)
    return [got[0], got[1]]


@pytest.mark.timeout(300)
@pytest.mark.parametrize("i", range(len(MODELS)), ids=MODELS)
def test_two_ranks_are_one_process_that_adds_the_shards_up(ranks, i, monkeypatch):
    from kllms_amd.engine.engine import LLMEngine
    from kllms_amd.parallel.tp import ColumnParallelLinear, RowParallelLinear

    (held0, logits0, tokens0), (held1, logits1, tokens1) = ranks[0][i], ranks[1][i]
    assert tokens0 == tokens1 and tokens0[0] == tokens0[1] and len(tokens0[0]) >= 1
    assert torch.equal(torch.from_numpy(logits0), torch.from_numpy(logits1))      # the head is whole on each

    # the plain weights of one process, in the shards' form
    monkeypatch.setattr("kllms_amd.models.llama.LlamaForCausalLM.quantize_weights_", lambda self: None)
    eng = engine(MODELS[i])
    biases_(eng.model)
    assert isinstance(eng, LLMEngine)
    seen = set()
    for name, m in eng.model.named_modules():
        if not isinstance(m, (ColumnParallelLinear, RowParallelLinear)):
            continue
        if isinstance(m, ColumnParallelLinear):
            parts = [[p.chunk(2)[r] for p in m.weight.split(m.partition_sizes)] for r in range(2)]
            shards = [torch.cat(p) for p in parts]
        else:
            shards = list(m.weight.chunk(2, 1))
        shards = [ops.quantize_weights(w) for w in shards]
        for (codes, scales), held in zip(shards, (held0, held1)):
            assert torch.equal(codes, torch.from_numpy(held[name + ".weight"])) and torch.equal(scales, torch.from_numpy(held[name + ".weight_scale"]))
            seen.add(name)
        if isinstance(m, ColumnParallelLinear):
            def forward(x, m=m, shards=shards):
                sizes = [p // 2 for p in m.partition_sizes]
                each = [ops.linear_int8(x, *s).split(sizes, -1) for s in shards]
                y = torch.cat([t for pair in zip(*each) for t in pair], -1)
                return y if m.bias is None else y + m.bias
        else:
            def forward(x, shards=shards):
                return sum(ops.linear_int8(part, *s) for part, s in zip(x.chunk(2, -1), shards))
        monkeypatch.setattr(m, "forward", forward)
    assert len(seen) == len({n[: -len(".weight_scale")] for n in held0 if n.endswith("weight_scale")})
    want, tokens = logits_and_tokens(eng)
    got = torch.from_numpy(logits0)
    # fp32 sums in another order may move a value over the border between two codes of 255, or of 16 in the cache: a
    # change of 1/127 of a row's largest value at most in the former, of a step of one value among 64 in the latter
    for row in range(2):
        assert float((got[row] - want[row]).norm()) < 0.02 * float(want[row].norm())

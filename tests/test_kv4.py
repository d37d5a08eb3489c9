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

"""Kernels of products in 8-bit integers: codes to the last bit, products against float64."""

import pytest
import torch

from kllms_amd import ops
from kllms_amd.ops import torch_ref

pytestmark = pytest.mark.gpu
DEV = "cuda"


def rows(M, K, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(M, K, generator=g) * torch.exp(torch.randn(M, 1, generator=g) * 2)
    x[:, ::37] *= 8
    return x.bfloat16()


def weights(N, K, seed=1):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(-127, 128, (N, K), generator=g, dtype=torch.int8), torch.rand(N, generator=g) * 1e-3 + 1e-5


def check(got, x, w, ws, bias=None, gated=False):
    """Sums are exact; fp32 products with both scales and the bias are three roundings of 2^-24, bf16 is half of 2^-7. Of
    silu(g) u with g off by e |g|: its slope is at most 1.1, and the exponential is off by 2^-20."""
    xc, xs = torch_ref.quantize_rows(x)
    dev = x.shape[0] * w.shape[0] * w.shape[1] > 1 << 28       # larger ones on the GPU, in 64 bits as well
    put = (lambda t: t.to(DEV)) if dev else (lambda t: t)
    y = (put(xc).double() @ put(w).double().t()) * put(xs).double()[:, None] * put(ws).double()
    fine = 2 ** -22
    if gated:
        g, u = y.chunk(2, -1)
        y = torch.sigmoid(g) * g * u
        off = 2 ** -8 * y.abs() + (fine * g.abs() + 2 ** -20 * (torch.sigmoid(g) * g).abs()) * u.abs() * 1.2
    else:
        off = y.abs() * fine
        if bias is not None:
            y = y + put(bias).double()
            off = off + put(bias).double().abs() * fine
        off = off + 2 ** -8 * y.abs()
    far = (got.to(y.device).double() - y).abs()
    assert bool((far <= off + 1e-30).all()), f"{float((far / (off + 1e-30)).max())} of what is allowed"


@pytest.mark.parametrize("M", [1, 3, 4, 5, 130])
@pytest.mark.parametrize("K", [16, 112, 512, 528, 1024, 2048, 3584, 4096, 8208, 14336, 16384, 18944, 131072])
def test_codes(M, K):
    x = rows(M, K, seed=K)
    if M >= 3:
        x[0] = 0
        x[1, 5], x[2, K - 1] = float("nan"), float("-inf")
    if M >= 5:
        x[3] = (x[3].float() * 2.0 ** -128).bfloat16()
        x[4, 0] = 3.3e38
    codes, scales = ops.quantize_rows(x.to(DEV))
    want, want_scales = torch_ref.quantize_rows(x)
    sound = ~torch.isnan(want_scales)
    assert torch.equal(torch.isnan(scales).cpu(), ~sound)
    assert torch.equal(codes.cpu()[sound], want[sound]) and torch.equal(scales.cpu()[sound], want_scales[sound])


SIZES = [(16, 16), (48, 32), (64, 128), (272, 144), (512, 1024), (1040, 528), (4608, 3584), (6144, 4096)]


@pytest.mark.parametrize("M", [1, 5, 32, 33, 64, 97, 128, 129, 200, 333])
@pytest.mark.parametrize("N,K", SIZES)
def test_product(M, N, K):
    x, (w, ws) = rows(M, K, seed=M), weights(N, K, seed=N)
    bias = torch.randn(N, generator=torch.Generator().manual_seed(2)).bfloat16() if (M + N) % 3 else None
    got = ops.linear_int8(x.to(DEV), w.to(DEV), ws.to(DEV), None if bias is None else bias.to(DEV))
    check(got, x, w, ws, bias)


@pytest.mark.parametrize("M", [1, 5, 64, 120, 129, 300])
@pytest.mark.parametrize("N,K", [(32, 16), (96, 64), (544, 144), (2048, 512), (16384, 2048), (28672, 4096)])
def test_gated_product(M, N, K):
    x, (w, ws) = rows(M, K, seed=M), weights(N, K, seed=N)
    ws = ws * 0.05
    got = ops.linear_silu_int8(x.to(DEV), w.to(DEV), ws.to(DEV))
    check(got, x, w, ws, gated=True)


@pytest.mark.parametrize("M,N,K", [(1000, 4096, 14336), (2100, 2048, 8192), (777, 512, 131072), (4097, 1040, 528), (8200, 256, 128)])
def test_many_rows(M, N, K):
    x, (w, ws) = rows(M, K, seed=M), weights(N, K, seed=N)
    args = [t.to(DEV) for t in (x, w, ws)]
    got = ops.linear_int8(*args)
    check(got, x, w, ws)
    assert torch.equal(ops.linear_int8(*args), got)          # sums of whole numbers: whoever is last
    if N % 32 == 0:
        check(ops.linear_silu_int8(args[0], args[1], args[2] * 0.02), x, w, ws * 0.02, gated=True)


@pytest.mark.parametrize("M", [1, 7, 40, 128])
@pytest.mark.parametrize("N,K", [(16, 16), (768, 512), (6144, 4096), (4096, 14336)])
def test_sums_in_shares(M, N, K):
    x, (w, ws) = rows(M, K, seed=M), weights(N, K, seed=N)
    part = ops.linear_part_int8(x.to(DEV), w.to(DEV), ws.to(DEV))
    xc, xs = torch_ref.quantize_rows(x)
    y = (xc.double() @ w.double().t()) * xs.double()[:, None] * ws.double()
    size = (xc.double().abs() @ w.double().abs().t()) * xs.double()[:, None] * ws.double()
    assert part.shape[1:] == (M, N)
    assert bool(((part.double().sum(0).cpu() - y).abs() <= 2 ** -22 * size + 1e-30).all())


@pytest.mark.parametrize("M", [1, 7, 40, 129, 400])
@pytest.mark.parametrize("N,K", [(64, 16), (544, 144), (2048, 1024), (6144, 4096)])
def test_products_of_codes_are_those_of_rows(M, N, K):
    x, (w, ws) = rows(M, K, seed=M + N), weights(N, K, seed=N)
    bias = torch.randn(N, generator=torch.Generator().manual_seed(2)).bfloat16().to(DEV)
    x, w, ws = (t.to(DEV) for t in (x, w, ws))
    small = ws * 0.05
    codes = ops.quantize_rows(x)
    assert isinstance(codes, ops.Int8Rows)
    packed = ops.Int8Rows(codes.codes.contiguous(), codes.scales)
    behind = torch.randint(-127, 128, (M, K + 160), dtype=torch.int8, device=DEV)        # rows of a wider matrix, others' codes behind
    behind[:, 16:16 + K] = codes.codes
    for c in (codes, packed, ops.Int8Rows(behind[:, 16:16 + K], codes.scales)):
        assert torch.equal(ops.linear_int8(c, w, ws, bias), ops.linear_int8(x, w, ws, bias))
        assert torch.equal(ops.linear_silu_int8(c, w, small), ops.linear_silu_int8(x, w, small))
        if M <= 128:
            # 3 roundings of 2^-24 of each share's size either way, whose sizes add up to the products' at most
            size = (codes.codes.double().abs() @ w.double().abs().t()) * codes.scales.double()[:, None] * ws.double()
            far = (ops.linear_part_int8(c, w, ws).double().sum(0) - ops.linear_part_int8(x, w, ws).double().sum(0)).abs()
            assert bool((far <= 2 ** -21 * size + 1e-30).all())


@pytest.mark.parametrize("M", [1, 9, 128])
@pytest.mark.parametrize("n", [128, 1024, 4096, 8192, 16384])
def test_norm_that_leaves_codes(M, n):
    g = torch.Generator().manual_seed(n + M)
    part = (torch.randn(2, M, n, generator=g) * 3).to(DEV)
    residual, weight = torch.randn(M, n, generator=g).bfloat16().to(DEV), torch.randn(n, generator=g).bfloat16().to(DEV)
    if M > 2:
        part[0, 1, 5] = float("nan")
        residual[2] = 0
        part[:, 2] = 0
    two = residual.clone()
    want = ops.quantize_rows(ops.add_norm_rows(part, residual, weight, 1e-5))
    got = ops.add_norm_rows_int8(part, two, weight, 1e-5)
    sound = ~torch.isnan(want.scales)
    assert torch.equal(sound, ~torch.isnan(got.scales)) and int((~sound).sum()) == (M > 2)
    assert torch.equal(got.codes[sound], want.codes[sound]) and torch.equal(got.scales[sound], want.scales[sound])
    assert torch.equal(two[sound], residual[sound])


def test_refusals_of_codes():
    x, (w, ws) = rows(20, 256).to(DEV), weights(64, 256)
    w, ws = w.to(DEV), ws.to(DEV)
    c = ops.quantize_rows(x)
    for bad in (ops.Int8Rows(x, c.scales), ops.Int8Rows(c.codes, c.scales.half()), ops.Int8Rows(c.codes, c.scales[:3]),
                ops.Int8Rows(c.codes[:, :128], c.scales)):
        with pytest.raises(ValueError):
            ops.linear_int8(bad, w, ws)
    for bad in (ops.Int8Rows(c.codes, c.scales.cpu()), ops.Int8Rows(c.codes, torch.cat((c.scales, c.scales))[::2])):
        with pytest.raises(RuntimeError):
            ops.linear_int8(bad, w, ws)
    with pytest.raises(RuntimeError, match="multiple of 128"):
        ops.add_norm_rows_int8(torch.zeros(1, 2, 96, device=DEV), torch.zeros(2, 96, device=DEV).bfloat16(), torch.ones(96, device=DEV).bfloat16(), 1e-5)


@pytest.mark.parametrize("M", [1, 2, 3, 4, 5, 6, 7, 8, 9])
@pytest.mark.parametrize("N,K", [(32, 16), (64, 144), (4096, 1040), (4128, 2064), (8224, 4112), (544, 8208), (256, 16384), (128, 16400), (512, 8192),
                                 (1040, 4096), (4608, 4096)])
def test_few_rows(M, N, K):
    """Codes made on the way: stages that end inside K, waves without a stage, an odd number of tiles, all forms."""
    x, (w, ws) = rows(M, K, seed=M + K), weights(N, K, seed=N)
    bias = torch.randn(N, generator=torch.Generator().manual_seed(2)).bfloat16()
    if M > 2:
        x[1] = 0
    args = [t.to(DEV) for t in (x, w, ws)]
    check(ops.linear_int8(*args), x, w, ws)
    check(ops.linear_int8(*args, bias.to(DEV), once=True), x, w, ws, bias)
    small = ws * (0.05 * 64 / K ** 0.5)
    if N % 32 == 0:
        check(ops.linear_silu_int8(args[0], args[1], small.to(DEV)), x, w, small, gated=True)
    part = ops.linear_part_int8(*args)
    # each share's exact sum is rounded by 2^-24 as it becomes fp32 and at both scales, 3 * 2^-24 < 2^-22 of its own size; the
    # shares' sizes add up to no more than the products' do, and may cancel
    xc, xs = torch_ref.quantize_rows(x)
    y = (xc.double() @ w.double().t()) * xs.double()[:, None] * ws.double()
    size = (xc.double().abs() @ w.double().abs().t()) * xs.double()[:, None] * ws.double()
    assert bool(((part.double().sum(0).cpu() - y).abs() <= 2 ** -22 * size + 1e-30).all())


@pytest.mark.parametrize("M", [1, 8])
def test_few_rows_the_last_of_memory(M):
    """Rows of x and W that end where their storage does, and rows of x far apart."""
    N, K = 48, 1040
    x, (w, ws) = rows(M, K, seed=9), weights(N, K, seed=4)
    apart = torch.full((M, 1 << 21), float("nan"), dtype=torch.bfloat16, device=DEV)
    apart[:, -K:] = x.to(DEV)
    want = ops.linear_int8(x.to(DEV), w.to(DEV), ws.to(DEV))
    check(want, x, w, ws)
    assert torch.equal(ops.linear_int8(apart[:, -K:], w.to(DEV), ws.to(DEV)), want)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("at", [0, 1023, 4095])
def test_few_rows_that_are_no_numbers(bad, at):
    x, (w, ws) = rows(5, 4096, seed=6), weights(6144, 4096)
    x[2, at] = bad
    got = ops.linear_int8(x.to(DEV), w.to(DEV), ws.to(DEV)).cpu()
    assert bool(torch.isnan(got[2]).all())
    keep = [0, 1, 3, 4]
    check(got[keep], x[keep], w, ws)


def test_rows_that_are_no_numbers_are_their_own_alone():
    x, (w, ws) = rows(6, 256), weights(64, 256)
    x[1, 3], x[4, 200] = float("nan"), float("inf")
    got = ops.linear_int8(x.to(DEV), w.to(DEV), ws.to(DEV)).cpu()
    bad = torch.isnan(got)
    assert bool(bad[[1, 4]].all()) and int(bad.sum()) == 2 * 64
    keep = [0, 2, 3, 5]
    check(got[keep], x[keep], w, ws)


def test_largest_sums_fit():
    K = 131072
    x = torch.full((2, K), -3.0).bfloat16()
    x[1] = 3.0
    w = torch.full((16, K), 127, dtype=torch.int8)
    ws = torch.ones(16)
    check(ops.linear_int8(x.to(DEV), w.to(DEV), ws.to(DEV)), x, w, ws)


@pytest.mark.parametrize("M", [1, 5, 200])
def test_views_and_empty_calls(M):
    x, (w, ws) = rows(M, 256, seed=3), weights(64, 256)
    w, ws = w.to(DEV), ws.to(DEV)
    want = ops.linear_int8(x.to(DEV), w, ws)
    wide = torch.randn(M, 1000).bfloat16().to(DEV)
    wide[:, 8:264] = x.to(DEV)
    assert torch.equal(ops.linear_int8(wide[:, 8:264], w, ws), want)         # rows on 16 bytes, another stride
    wide[:, 3:259] = x.to(DEV)
    assert torch.equal(ops.linear_int8(wide[:, 3:259], w, ws), want)         # off 16 bytes
    assert torch.equal(ops.linear_int8(x.t().contiguous().t().to(DEV), w, ws), want)
    one = x[:1].to(DEV).expand(M, 256)                                       # one row for all
    assert torch.equal(ops.linear_int8(one, w, ws), want[:1].expand(M, 64))
    off = torch.randn(65).bfloat16().to(DEV)[1:]
    assert torch.equal(ops.linear_int8(x.to(DEV), w, ws, off), ops.linear_int8(x.to(DEV), w, ws, off.clone()))
    assert ops.linear_int8(x.to(DEV)[:0], w, ws).shape == (0, 64)
    assert ops.linear_silu_int8(x.to(DEV)[:0], w, ws).shape == (0, 32) and ops.quantize_rows(x.to(DEV)[:0])[0].shape == (0, 256)


def test_weights_of_more_than_2_gb():
    N, K = 18000, 131072                                     # 2.4 GB
    w = torch.zeros(N, K, dtype=torch.int8, device=DEV)
    ws = torch.full((N,), 1e-3, device=DEV)
    x = rows(200, K, seed=8)
    part, _ = weights(16, K, seed=9)
    w[-16:] = part.to(DEV)
    for M in (5, 200):
        got = ops.linear_int8(x[:M].to(DEV), w, ws)
        assert not bool(got[:, :-16].any())
        check(got[:, -16:], x[:M], part, ws[-16:].cpu())


@torch.inference_mode()                  # as the engine captures: torch's own state is of one kind for all captures
def test_replayed():
    x, (w, ws) = rows(5, 4096), weights(6144, 4096)
    long, (w2, ws2) = rows(333, 3584), weights(4608, 3584)
    x, w, ws, long, w2, ws2 = (t.to(DEV) for t in (x, w, ws, long, w2, ws2))

    def step():
        return ops.linear_int8(x, w, ws), ops.linear_int8(long, w2, ws2), ops.linear_silu_int8(x, w, ws)

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
        x.copy_(rows(5, 4096, seed=10 + i))
        long.copy_(rows(333, 3584, seed=20 + i))
        want = [t.clone() for t in step()]
        for g, out in graphs:
            for t in out:
                t.zero_()
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_refusals():
    x, (w, ws) = rows(3, 256), weights(64, 256)
    x, w, ws = x.to(DEV), w.to(DEV), ws.to(DEV)
    ops.linear_int8(x, w, ws)
    wide = torch.zeros(3, 264, dtype=torch.bfloat16, device=DEV)
    for call in (lambda: ops.linear_int8(x.float(), w, ws), lambda: ops.linear_int8(x, w, ws[:32]), lambda: ops.linear_int8(x, w, ws.double()),
                 lambda: ops.linear_int8(x, w[:60], ws[:60]), lambda: ops.linear_silu_int8(x, w[:48], ws[:48]), lambda: ops.linear_int8(x, w.cpu(), ws),
                 lambda: ops.linear_int8(wide, torch.zeros(64, 264, dtype=torch.int8, device=DEV), ws),
                 lambda: ops.linear_int8(x, w, ws, ws), lambda: ops.linear_int8(x, torch.zeros(256, 64, dtype=torch.int8, device=DEV).t(), ws),
                 lambda: ops.quantize_rows(x.half()), lambda: ops.linear_part_int8(x[:0], w, ws),
                 lambda: ops.quantize_rows(torch.zeros(1, 131088, dtype=torch.bfloat16, device=DEV))):
        with pytest.raises(RuntimeError):
            call()

"""8-bit integer rows, products and linears. Every bit is defined: the quotients and sums are exact, two fp32
products and one rounding follow, so results are compared for equality with the oracle's."""
import math

import pytest
import torch

from flint_amd import _lib, quantize
from oracle import scoring

pytestmark = pytest.mark.gpu


def rows_of(m, k, seed, kind="normal"):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(m, k, generator=g)
    if kind == "outliers":
        x[:, torch.randint(0, k, (max(1, k // 100),), generator=g)] *= 30.0
    if kind == "ties":  # every value a multiple of half a scale step: max = 127 / 128
        x = torch.randint(-254, 255, (m, k), generator=g).float() / 256.0
        x[:, 0] = 254.0 / 256.0
    if kind == "halves":  # the largest value halved again and again
        x = x.abs().amax(1, keepdim=True) * 2.0 ** -torch.randint(0, 9, (m, k), generator=g).float()
        x[:, 0] *= 2.0
    if kind == "tiny":
        x = x * 2.0 ** -torch.randint(120, 134, (m, 1), generator=g).float()
    if kind == "huge":
        x = x.sign() * torch.rand(m, k, generator=g) * 3.3e38
    return x.to(torch.bfloat16)


def same(a, b):
    a, b = a.cpu(), b.cpu()
    return a.dtype == b.dtype and torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(), b.nan_to_num())


@pytest.mark.parametrize("kind", ["normal", "outliers", "ties", "halves", "tiny", "huge"])
@pytest.mark.parametrize("m,k", [(1, 16), (5, 48), (3, 2560), (2, 8192), (2, 8208), (1, 65536)])
def test_quantized_rows_are_the_oracles(dev, m, k, kind):
    x = rows_of(m, k, 7 * m + k, kind)
    q, s = quantize.quantize_int8(x.to(dev))
    qr, sr = scoring.quantize_rows(x)
    assert torch.equal(s.cpu(), sr)
    assert torch.equal(q.cpu(), qr)
    # half a step, and the half ulp that the scale may be off, of 127 steps
    live = sr > 2.0 ** -100
    off = (q.cpu().double() * sr.double()[:, None] - x.double()).abs().amax(1)
    assert bool((off[live] <= sr.double()[live] * (0.5 + 127 * 2.0 ** -22)).all())


def test_quantized_rows_at_every_mantissa_and_quotient(dev):
    """All bf16 mantissas as the row's maximum, against every smaller bf16 value of nine octaves."""
    top = torch.arange(128, 256).float()
    small = torch.cat([torch.arange(128, 256).float() * 2.0 ** -e for e in range(1, 10)])
    small = torch.cat([small, -small, top, -top])
    x = small.repeat(128, 1)
    x = torch.where(x.abs() > top[:, None], torch.zeros(()), x)
    x = torch.cat([top[:, None], x, torch.zeros(128, (-(x.shape[1] + 1)) % 16)], 1).to(torch.bfloat16)
    q, s = quantize.quantize_int8(x.to(dev))
    qr, sr = scoring.quantize_rows(x)
    assert torch.equal(s.cpu(), sr) and torch.equal(q.cpu(), qr)


def test_rows_of_zeros_nan_and_infinities(dev):
    x = rows_of(6, 96, 3)
    x[1] = 0.0
    x[2, 95] = math.nan
    x[3, 0] = -math.inf
    x[4] = -0.0
    q, s = quantize.quantize_int8(x.to(dev))
    qr, sr = scoring.quantize_rows(x)
    assert torch.equal(q.cpu(), qr) and same(s, sr)
    assert s[1] == 0 and s[4] == 0 and s[2].isnan() and s[3].isnan()
    w = quantize.DynamicInt8Linear.from_float(rows_of(40, 96, 4).to(dev))
    y, clean = w(x.to(dev)).cpu(), w(rows_of(6, 96, 3).to(dev)).cpu()
    assert bool(y[2].isnan().all()) and bool(y[3].isnan().all()) and bool((y[1] == 0).all())
    for r in (0, 5):  # the other rows are what they were
        assert torch.equal(y[r], clean[r])


M_SIZES = [1, 2, 3, 5, 8, 15, 16, 17, 31, 32, 33, 47, 48, 63, 64, 65, 96, 127, 128, 129, 200, 256, 257, 333, 520]
SHAPES = [(1, 16), (17, 48), (70, 64), (64, 128), (129, 144), (257, 272), (500, 1040), (2570, 2560), (96, 8192)]


def ints(m, k, seed, extreme=False):
    g = torch.Generator().manual_seed(seed)
    if extreme:
        return torch.where(torch.rand(m, k, generator=g) < 0.97, -128, 127).to(torch.int8)
    return torch.randint(-128, 128, (m, k), generator=g).to(torch.int8)


@pytest.mark.parametrize("n,k", SHAPES)
def test_products_are_exact(dev, n, k):
    wq = ints(n, k, n + k)
    ws = torch.rand(n, generator=torch.Generator().manual_seed(k)) * 1e-3
    wd, sd = wq.to(dev), ws.to(dev)
    xq = ints(max(M_SIZES), k, n)
    xs = torch.rand(max(M_SIZES), generator=torch.Generator().manual_seed(n)) * 0.05
    ref = scoring.product(xq, xs, wq, ws)
    for m in M_SIZES:
        y = quantize.gemm_int8(xq[:m].to(dev), xs[:m].to(dev), wd, sd, out_dtype=torch.float32)
        assert torch.equal(y.cpu(), ref[:m]), m
        y = quantize.gemm_int8(xq[:m].to(dev), xs[:m].to(dev), wd, sd)
        assert torch.equal(y.cpu(), ref[:m].to(torch.bfloat16)), m


@pytest.mark.parametrize("m", [1, 16, 40, 130, 300])
def test_sums_of_the_largest_values(dev, m):
    n, k = 72, 65536  # 128 * 128 * 65536 = 2^30
    xq, wq = ints(m, k, 1, True), ints(n, k, 2, True)
    one = torch.ones(max(m, n))
    y = quantize.gemm_int8(xq.to(dev), one[:m].to(dev), wq.to(dev), one[:n].to(dev), out_dtype=torch.float32)
    ref = scoring.product(xq, one[:m], wq, one[:n])
    assert float(ref.abs().max()) > 2.0 ** 29
    assert torch.equal(y.cpu(), ref)


@pytest.mark.parametrize("m,n,k", [(1, 2560, 2560), (4, 3584, 2560), (12, 5003, 1408), (20, 16384, 2560), (32, 2560, 8192),
                                   (33, 2560, 8192), (100, 1000, 4112), (1024, 3584, 2560), (300, 16384, 2560),
                                   (1, 49152, 2560), (7, 49152, 2560)])
def test_linear_is_quantising_and_the_product(dev, m, n, k):
    w, x = rows_of(n, k, m), rows_of(m, k, n, "outliers")
    lin = quantize.DynamicInt8Linear.from_float(w.to(dev))
    wq, ws = lin.weight.cpu(), lin.scales.cpu()
    xq, xs = scoring.quantize_rows(x)
    ref = scoring.product(xq, xs, wq, ws)
    assert torch.equal(lin(x.to(dev)).cpu(), ref.to(torch.bfloat16))
    y = quantize.linear_int8(x.to(dev), lin.weight, lin.scales, out_dtype=torch.float32)
    assert torch.equal(y.cpu(), ref)
    # a row alone gives the bits that it gives in the batch
    for r in {0, m // 2, m - 1}:
        assert torch.equal(quantize.linear_int8(x[r:r + 1].to(dev), lin.weight, lin.scales, torch.float32).cpu(),
                           ref[r:r + 1])


def test_linear_takes_the_inputs_that_linears_take(dev):
    lin = quantize.DynamicInt8Linear.from_float(rows_of(48, 64, 1).to(dev))
    x = rows_of(6, 64, 2).to(dev)
    y = lin(x)
    assert torch.equal(lin(x.view(2, 3, 64)), y.view(2, 3, 48))
    assert torch.equal(lin(x[0]), y[0])
    assert torch.equal(lin(x.float()), y)
    wide = torch.zeros(6, 80, dtype=torch.bfloat16, device=dev)
    wide[:, :64] = x
    assert torch.equal(lin(wide[:, :64]), y)                      # strided rows
    assert torch.equal(lin(x.t().contiguous().t()), y)            # another order
    shifted = torch.zeros(6 * 64 + 1, dtype=torch.bfloat16, device=dev)[1:].view(6, 64)
    shifted.copy_(x)
    assert shifted.data_ptr() % 16 and torch.equal(lin(shifted), y)
    w2 = torch.zeros(48 * 64 + 1, dtype=torch.int8, device=dev)[1:].view(48, 64)
    w2.copy_(lin.weight)
    assert torch.equal(quantize.linear_int8(x, w2, lin.scales), y)
    xq, xs = quantize.quantize_int8(x)
    q2 = torch.zeros(6 * 64 + 1, dtype=torch.int8, device=dev)[1:].view(6, 64)
    q2.copy_(xq)
    assert torch.equal(quantize.gemm_int8(q2, xs, lin.weight, lin.scales), y)
    assert lin(x[:0]).shape == (0, 48) and lin(x.view(2, 3, 64)[:, :0]).shape == (2, 0, 48)
    assert quantize.gemm_int8(xq[:0], xs[:0], lin.weight, lin.scales).shape == (0, 48)
    assert not lin(x.detach().requires_grad_()).requires_grad


def test_refusals(dev):
    lin = quantize.DynamicInt8Linear.from_float(rows_of(48, 64, 1).to(dev))
    x = rows_of(6, 64, 2).to(dev)
    xq, xs = quantize.quantize_int8(x)
    w, s = lin.weight, lin.scales
    for bad in (lambda: quantize.linear_int8(x.float(), w, s), lambda: quantize.linear_int8(x[:, :48], w, s),
                lambda: quantize.linear_int8(x, w.t(), s), lambda: quantize.linear_int8(x, w, s[:40]),
                lambda: quantize.linear_int8(x, w, s.double()), lambda: quantize.linear_int8(x, w, s, torch.float16),
                lambda: quantize.linear_int8(x, w.cpu(), s), lambda: quantize.gemm_int8(xq, xs[:5], w, s),
                lambda: quantize.gemm_int8(x, xs, w, s), lambda: quantize.gemm_int8(xq[:, :48], xs, w, s),
                lambda: quantize.quantize_int8(x[:, :40].contiguous()), lambda: quantize.quantize_int8(x.float()),
                lambda: quantize.quantize_int8(x, q=xq[:5]), lambda: quantize.quantize_int8(x, scale=xs[:5])):
        with pytest.raises(ValueError):
            bad()


@pytest.mark.parametrize("m,n,k", [(1, 33, 80), (7, 100, 2560), (40, 77, 208), (130, 131, 336), (300, 259, 272)])
@pytest.mark.parametrize("f32", [False, True])
def test_writes_its_outputs_and_nothing_else(dev, m, n, k, f32):
    xq, wq = ints(m, k, 1).to(dev), ints(n, k, 2).to(dev)
    xs, ws = torch.rand(m, device=dev), torch.rand(n, device=dev)
    y = torch.full((m * n + 4096,), -7.0, dtype=torch.float32 if f32 else torch.bfloat16, device=dev)
    need = _lib.ctypes.c_int64()
    _lib.call("fl_gemm_int8_workspace", m, n, k, _lib.ctypes.byref(need))
    work = torch.full((need.value + 4096,), 0x5A, dtype=torch.uint8, device=dev)
    _lib.call("fl_gemm_int8", _lib.ptr(xq), _lib.ptr(xs), _lib.ptr(wq), _lib.ptr(ws), _lib.ptr(y), int(f32),
              _lib.ptr(work), m, n, k, _lib.stream_ptr())
    ref = scoring.product(xq.cpu(), xs.cpu(), wq.cpu(), ws.cpu()).to(y.dtype)
    assert torch.equal(y[:m * n].view(m, n).cpu(), ref)
    assert bool((y[m * n:] == -7.0).all()) and bool((work[need.value:] == 0x5A).all())


@pytest.mark.parametrize("m", [1, 9, 40, 100, 400])
def test_captured_and_replayed(dev, m):
    n, k = 520, 1296
    lin = quantize.DynamicInt8Linear.from_float(rows_of(n, k, 1).to(dev))
    x = torch.zeros(m, k, dtype=torch.bfloat16, device=dev)
    lin(x)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):  # two graphs, each with workspaces of its own
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = lin(x)
        graphs.append((g, y))
    for seed in range(4):
        new = rows_of(m, k, seed)
        x.copy_(new)
        for g, y in graphs:
            g.replay()
            assert torch.equal(y.cpu(), lin(x).cpu())
            torch.cuda.synchronize()
        xq, xs = scoring.quantize_rows(new)
        ref = scoring.product(xq, xs, lin.weight.cpu(), lin.scales.cpu()).to(torch.bfloat16)
        assert torch.equal(graphs[0][1].cpu(), ref)


def test_two_streams_at_once(dev):
    lin = quantize.DynamicInt8Linear.from_float(rows_of(2560, 2560, 1).to(dev))
    xs = [rows_of(m, 2560, m).to(dev) for m in (1, 16, 64, 300)]
    ref = [lin(x).cpu() for x in xs]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in xs], []
    for _ in range(3):
        for s, x in zip(streams, xs):
            with torch.cuda.stream(s):
                got.append(lin(x))
    torch.cuda.synchronize()
    for i, y in enumerate(got):
        assert torch.equal(y.cpu(), ref[i % len(xs)])


@pytest.mark.parametrize("m,n,k", [
    (33, 90, 4112), (70, 1003, 4112), (64, 1000, 8208),        # few tiles of 64: K in parts, joined
    (333, 2571, 1104), (64, 2570, 16),                         # up to 256 tiles of 64
    (600, 2571, 272), (333, 4003, 400),                        # more of them
    (1000, 3999, 1104), (1021, 4000, 2064),                    # up to 256 tiles of 128
    (1500, 5003, 1104), (1501, 5000, 144),                     # more of them
    (1900, 8003, 400), (2048, 8192, 528), (2049, 16130, 144),  # tiles of 256
    (19, 1001, 2064), (32, 4095, 1040),                        # up to 32 rows without LDS
    (1, 8195, 9616), (2, 16390, 1040), (9, 8191, 1040),        # up to 16 rows without, of long and of short matrices
    (3, 8209, 1040), (8, 16400, 2576), (16, 9001, 2832), (5, 8209, 9600), (4, 24577, 2576)])  # in LDS, blocks in turn
@pytest.mark.parametrize("f32", [False, True])
def test_every_way_to_cut_a_product(dev, m, n, k, f32):
    """Ragged rows, weights and K; scales that start on 4 bytes only; rows behind the last are left as they were."""
    xq, wq = ints(m, k, m + k), ints(n, k, n)
    g = torch.Generator().manual_seed(k)
    xs, ws = torch.rand(m, generator=g) * 0.05, torch.rand(n, generator=g) * 1e-3
    y = torch.full((m * n + 4096,), -7.0, dtype=torch.float32 if f32 else torch.bfloat16, device=dev)
    need = _lib.ctypes.c_int64()
    _lib.call("fl_gemm_int8_workspace", m, n, k, _lib.ctypes.byref(need))
    work = torch.full((need.value + 4096,), 0x5A, dtype=torch.uint8, device=dev)
    a, b = xq.to(dev), wq.to(dev)
    s = torch.cat([torch.full((1,), math.nan), xs, torch.full((2,), math.nan), ws]).to(dev)
    off = s[1:], s[1 + m + 2:]
    _lib.call("fl_gemm_int8", _lib.ptr(a), _lib.ptr(off[0]), _lib.ptr(b), _lib.ptr(off[1]), _lib.ptr(y), int(f32),
              _lib.ptr(work), m, n, k, _lib.stream_ptr())
    ref = scoring.product(xq, xs, wq, ws).to(y.dtype)
    assert torch.equal(y[:m * n].view(m, n).cpu(), ref)
    assert bool((y[m * n:] == -7.0).all()) and bool((work[need.value:] == 0x5A).all())


@pytest.mark.parametrize("kind", ["normal", "halves", "tiny"])
@pytest.mark.parametrize("m,k", [(1024, 16), (1025, 2560), (1027, 1040), (1030, 2576)])
def test_quantized_rows_of_large_batches(dev, m, k, kind):
    x = rows_of(m, k, m + k, kind)
    x[m - 1] = 0.0
    x[m - 2, k - 1] = math.inf
    q = torch.full((m + 2, k), 99, dtype=torch.int8, device=dev)
    s = torch.full((m + 2,), 99.0, device=dev)
    quantize.quantize_int8(x.to(dev), q[:m], s[:m])
    qr, sr = scoring.quantize_rows(x)
    assert torch.equal(q[:m].cpu(), qr) and same(s[:m], sr)
    assert bool((q[m:] == 99).all()) and bool((s[m:] == 99.0).all())


@pytest.mark.parametrize("m", list(range(1, 18)))
def test_linears_that_quantise_on_the_way(dev, m):
    """As long rows as 16384 values in all allow, one step longer, and short ones; more blocks than workgroups."""
    n = 8225
    for k in {16384 // m // 16 * 16, 16384 // m // 16 * 16 + 16, 528}:
        x = rows_of(m, k, k, "outliers")
        if m > 2:
            x[1] = 0.0
            x[2, k - 1] = math.nan
        wq, ws = ints(n, k, m), torch.rand(n, generator=torch.Generator().manual_seed(m)) * 1e-3
        y = quantize.linear_int8(x.to(dev), wq.to(dev), ws.to(dev), torch.float32)
        assert same(y, scoring.product(*scoring.quantize_rows(x), wq, ws)), k


@pytest.mark.parametrize("m,n,k", [(1, 2577, 32768), (2, 1001, 16384), (3, 2577, 8192), (3, 2577, 8208), (4, 4097, 8192),
                                   (4, 40, 8208), (2, 32767, 512), (2, 32768, 512), (5, 32801, 1040), (8, 32801, 4096),
                                   (8, 33000, 4112), (7, 49152, 2560), (5, 8191, 3264), (8, 8191, 2048), (9, 8191, 1040),
                                   (16, 4095, 1024), (16, 4096, 1024), (15, 77, 1088), (9, 33000, 1040)])
def test_linears_on_both_sides_of_the_rules_lines(dev, m, n, k):
    x = rows_of(m, k, n, "outliers")
    x[m // 2, k // 2:] = 0.0
    wq, ws = ints(n, k, m), torch.rand(n, generator=torch.Generator().manual_seed(m)) * 1e-3
    ref = scoring.product(*scoring.quantize_rows(x), wq, ws)
    assert torch.equal(quantize.linear_int8(x.to(dev), wq.to(dev), ws.to(dev), torch.float32).cpu(), ref)
    assert torch.equal(quantize.linear_int8(x.to(dev), wq.to(dev), ws.to(dev)).cpu(), ref.to(torch.bfloat16))


def scaled_sums(xq, xs, wq, ws):
    """The definition on the device, for a few rows or columns of a large product."""
    acc = xq.double() @ wq.double().T  # whole numbers below 2^53: exact in any order
    return acc.float() * (xs[:, None] * ws[None, :])


@pytest.mark.parametrize("n", [1, 3, 70])
def test_as_many_rows_as_there_may_be(dev, n):
    """2^23 rows of x, and of weights: offsets of the operand beyond 2^31."""
    m, k = 1 << 23, 272
    xq = torch.randint(-128, 128, (m, k), dtype=torch.int8, device=dev)
    xs, ws = torch.rand(m, device=dev), torch.rand(n, device=dev)
    wq = torch.randint(-128, 128, (n, k), dtype=torch.int8, device=dev)
    at = torch.tensor([0, 1, 63, 64, 4095, (1 << 22) + 5, m - 65, m - 2, m - 1], device=dev)
    y = quantize.gemm_int8(xq, xs, wq, ws, torch.float32)
    assert torch.equal(y[at], scaled_sums(xq[at], xs[at], wq, ws))
    y = quantize.gemm_int8(wq, ws, xq, xs, torch.float32)  # the other way round
    assert torch.equal(y[:, at], scaled_sums(wq, ws, xq[at], xs[at]))
    with pytest.raises(ValueError):
        quantize.gemm_int8(xq[:, :264], xs, wq[:, :264], ws)


def test_more_results_than_32_bits_count(dev):
    m, n, k = 1 << 17, 33000, 16
    xq, wq = (torch.randint(-128, 128, (r, k), dtype=torch.int8, device=dev) for r in (m, n))
    xs, ws = torch.rand(m, device=dev), torch.rand(n, device=dev)
    y = quantize.gemm_int8(xq, xs, wq, ws)
    at = torch.tensor([0, 65535, 65536, 130156, 130157, m - 257, m - 1], device=dev)
    assert y.numel() > 2 ** 32 and torch.equal(y[at], scaled_sums(xq[at], xs[at], wq, ws).to(torch.bfloat16))


def test_as_many_rows_quantised_as_there_may_be(dev):
    m = 1 << 23
    x = torch.randn(m, 16, device=dev).to(torch.bfloat16)
    q, s = quantize.quantize_int8(x)
    at = torch.tensor([0, 3, 4, 1 << 22, m - 5, m - 1], device=dev)
    qr, sr = scoring.quantize_rows(x[at].cpu())
    assert torch.equal(q[at].cpu(), qr) and torch.equal(s[at].cpu(), sr)


@pytest.mark.parametrize("m,n,k", [(8, 12288, 2560), (8, 12289, 2560), (5, 12288, 4096), (5, 12288, 4112), (4, 12288, 4080),
                                   (4, 12288, 4096), (4, 12289, 4080), (1, 8192, 8192), (1, 8193, 8192), (16, 8192, 1024),
                                   (16, 8193, 1024), (9, 8192, 1808), (9, 8192, 1824), (7, 4097, 2912), (7, 4097, 2928)])
def test_linears_whose_workgroups_take_blocks_in_turn(dev, m, n, k):
    x = rows_of(m, k, n + k, "outliers")
    wq, ws = ints(n, k, m), torch.rand(n, generator=torch.Generator().manual_seed(m)) * 1e-3
    ref = scoring.product(*scoring.quantize_rows(x), wq, ws)
    assert torch.equal(quantize.linear_int8(x.to(dev), wq.to(dev), ws.to(dev), torch.float32).cpu(), ref)
    assert torch.equal(quantize.linear_int8(x.to(dev), wq.to(dev), ws.to(dev)).cpu(), ref.to(torch.bfloat16))


@pytest.mark.parametrize("m,n,k", [(2, 4096, 4112), (2, 4097, 4112), (2, 4097, 4080), (1, 5003, 65536), (6, 8191, 8000),
                                   (7, 8191, 8000), (11, 4500, 4400), (2, 8192, 4096), (1, 10007, 8208), (3, 8192, 4080)])
def test_few_rows_with_and_without_lds(dev, m, n, k):
    xq, wq = ints(m, k, m + k), ints(n, k, n)
    g = torch.Generator().manual_seed(k)
    xs, ws = torch.rand(m, generator=g) * 0.05, torch.rand(n, generator=g) * 1e-3
    ref = scoring.product(xq, xs, wq, ws)
    d = [t.to(dev) for t in (xq, xs, wq, ws)]
    assert torch.equal(quantize.gemm_int8(*d, out_dtype=torch.float32).cpu(), ref)
    assert torch.equal(quantize.gemm_int8(*d).cpu(), ref.to(torch.bfloat16))


@pytest.mark.parametrize("m,n,k", [(72, 72, 96), (5, 5, 1040), (300, 300, 272)])
def test_both_operands_off_16_bytes(dev, m, n, k):
    """x and weights of one size in views that start on 1, 4 or 8 bytes: each is copied, and both copies have to live."""
    xq, wq = ints(m, k, 1), ints(n, k, 2)
    xs, ws = torch.rand(m), torch.rand(n)
    ref = scoring.product(xq, xs, wq, ws)
    for off in (1, 4, 8):
        packed = torch.zeros(2 * m * k + 16 + off, dtype=torch.int8, device=dev)
        a, b = packed[off:off + m * k].view(m, k), packed[off + 16 + m * k:].view(n, k)
        a.copy_(xq)
        b.copy_(wq)
        assert a.data_ptr() % 16 == off and b.data_ptr() % 16 == off
        y = quantize.gemm_int8(a, xs.to(dev), b, ws.to(dev), out_dtype=torch.float32)
        assert torch.equal(y.cpu(), ref)
        assert torch.equal(packed[:off].cpu(), torch.zeros(off, dtype=torch.int8))


@pytest.mark.parametrize("rows", [128, 1024])
def test_the_scale_is_the_product(dev, rows):
    """Every bf16 significand as the maximum, with its half in the row: the scale is fp32(max fp32(1 / 127)), which torch's
    max / 127 on the device is too, and not always fp32(max / 127); for six significands that makes the half 64."""
    top = torch.arange(128, 256).repeat(rows // 128).float()
    x = torch.zeros(rows, 32)
    x[:, 3], x[:, 17], x[:, 31] = -top, top / 2, -top / 2
    q, s = quantize.quantize_int8(x.to(torch.bfloat16).to(dev))
    product = top.to(dev) * (torch.ones(()) / torch.full((), 127.0)).to(dev)
    assert torch.equal(s, product) and torch.equal(s, top.to(dev) / 127)
    quotient = (top.double() / 127).float()  # the nearest fp32: a quotient of 8 by 7 bits is no half of an ulp in fp64
    six = torch.tensor([143.0, 144.0, 175.0, 207.0, 208.0, 239.0])
    assert torch.equal(top[s.cpu() != quotient].unique(), six)
    low = torch.isin(top, six)
    assert bool((q[:, 3] == -127).all()) and torch.equal(q[:, 17], -q[:, 31])
    assert bool((q.cpu()[low][:, 17] == 64).all())
    ref = torch.round(top.double() / 2 / s.cpu().double())
    assert torch.equal(q[:, 17].cpu().double(), ref)


def test_linear_in_a_model_that_is_cast(dev):
    w, x = rows_of(48, 64, 1), rows_of(6, 64, 2).to(dev)
    lin = quantize.DynamicInt8Linear.from_float(w.to(dev))
    y = lin(x)
    model = torch.nn.Sequential(lin).to(device=dev, dtype=torch.bfloat16)
    assert torch.equal(model(x), y)
    assert torch.equal(model.cpu().to(dev)(x), y)

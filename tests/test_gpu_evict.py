"""Eviction from a cache by gathered weight: the kept slots and every moved row equal the definition's."""
import math

import pytest
import torch

from oracle import cache as oracle

pytestmark = pytest.mark.gpu


def make(lead, slots, dim, dtype=torch.bfloat16, seed=0, kind="plain"):
    g = torch.Generator().manual_seed(seed)
    k = torch.randn(*lead, slots, dim, generator=g).to(dtype)
    v = torch.randn(*lead, slots, dim, generator=g).to(dtype)
    w = torch.rand(*lead, slots, generator=g)
    if kind == "ties":  # few different values
        w = (w * 4).floor() / 4
    elif kind == "odd":
        w[..., ::5] = 0.0
        w[..., 1::5] = -0.0
        w[..., 2::7] = math.inf
        w[..., 3::11] = math.nan
        w[..., 4::6] = -w[..., 4::6]
    return k, v, w


def wanted(w, n, keep, recent, sink):
    flat = w.reshape(-1, w.shape[-1])
    return torch.tensor([oracle.kept_slots(r.tolist(), n, keep, recent, sink) for r in flat]).view(*w.shape[:-1], min(keep, n))


def moved(t, kept):
    return t.gather(t.dim() - 2, kept[..., None].expand(*kept.shape, t.shape[-1]))


CASES = [  # lead, slots, n, keep, recent, sink, dim
    ((8,), 1100, 1100, 512, 64, 4, 64), ((2, 3), 100, 77, 20, 5, 2, 64), ((1,), 70, 64, 63, 0, 0, 128), ((2,), 5000, 4999, 1, 0, 0, 64),
    ((2,), 5000, 4999, 1, 1, 0, 64), ((2,), 5000, 4999, 1, 0, 1, 64), ((1, 2), 3000, 2777, 2776, 100, 3, 64), ((3,), 40, 1, 1, 0, 0, 64),
    ((2,), 9000, 8193, 4097, 4000, 97, 128), ((4,), 2100, 2050, 1025, 1024, 1, 64), ((1,), 40000, 39999, 20001, 7, 0, 64),
]


@pytest.mark.parametrize("kind", ["plain", "ties", "odd"])
@pytest.mark.parametrize("case", CASES)
def test_evict(dev, case, kind):
    from flint_amd.attention import evict
    lead, slots, n, keep, recent, sink, dim = case
    k, v, w = make(lead, slots, dim, seed=n + keep, kind=kind)
    want = wanted(w, n, keep, recent, sink)
    # into another cache
    kd, vd, wd = k.to(dev), v.to(dev), w.to(dev)
    new = keep + 3
    out = (torch.full((*lead, new, dim), 7.0, dtype=k.dtype, device=dev), torch.full((*lead, new, dim), 8.0, dtype=k.dtype, device=dev),
           torch.full((*lead, new), 9.0, device=dev))
    kept = evict(kd, vd, wd, n, keep, recent=recent, sink=sink, out=out)
    assert torch.equal(kept.cpu().long(), want)
    assert torch.equal(out[0][..., :keep, :].cpu(), moved(k, want)) and torch.equal(out[1][..., :keep, :].cpu(), moved(v, want))
    assert torch.equal(out[2][..., :keep].cpu().view(torch.int32), w.gather(-1, want).view(torch.int32))
    assert (out[0][..., keep:, :] == 7).all() and (out[1][..., keep:, :] == 8).all() and (out[2][..., keep:] == 9).all()
    assert torch.equal(kd.cpu(), k) and torch.equal(vd.cpu(), v) and torch.equal(wd.cpu().view(torch.int32), w.view(torch.int32))
    # in place
    kept = evict(kd, vd, wd, n, keep, recent=recent, sink=sink)
    assert torch.equal(kept.cpu().long(), want)
    assert torch.equal(kd[..., :keep, :].cpu(), moved(k, want)) and torch.equal(vd[..., :keep, :].cpu(), moved(v, want))
    assert torch.equal(kd[..., keep:, :].cpu(), k[..., keep:, :]) and torch.equal(vd[..., keep:, :].cpu(), v[..., keep:, :])
    assert torch.equal(wd[..., :keep].cpu().view(torch.int32), w.gather(-1, want).view(torch.int32))
    assert (wd[..., keep:n] == 0).all() and torch.equal(wd[..., n:].cpu().view(torch.int32), w[..., n:].view(torch.int32))


def test_nothing_leaves(dev):
    from flint_amd.attention import evict
    k, v, w = make((2, 2), 50, 64)
    kd, vd, wd = k.to(dev), v.to(dev), w.to(dev)
    for keep in (40, 50, 1000):
        kept = evict(kd, vd, wd, 40, keep, recent=100, sink=100)
        assert torch.equal(kept.cpu().long(), torch.arange(40).expand(2, 2, 40))
        assert torch.equal(kd.cpu(), k) and torch.equal(wd.cpu(), w)
    assert evict(kd, vd, wd, 0, 10).shape == (2, 2, 0)
    assert evict(kd[:0], vd[:0], wd[:0], 10, 5).shape == (0, 2, 5)


@pytest.mark.parametrize("in_place", [False, True])
def test_strides_and_types(dev, in_place):
    """Caches as [L, slots, heads, dim] views; rows of fp32; a window of layers."""
    from flint_amd.attention import evict
    for dtype, dim in ((torch.bfloat16, 64), (torch.float32, 64), (torch.float16, 8), (torch.uint8, 48), (torch.float32, 1024)):
        k, v, w = make((3, 4), 300, dim, torch.float32, seed=dim)
        k, v = (k * 50).to(dtype), (v * 50).to(dtype)
        want = wanted(w, 290, 100, 10, 1)
        kd = k.transpose(1, 2).contiguous().to(dev).transpose(1, 2)
        big = torch.zeros(5, 4, 300, dim, dtype=dtype, device=dev)
        big[1:4] = v.to(dev)
        vd, wd = big[1:4], w.to(dev)
        out = None if in_place else (torch.zeros(3, 100, 4, dim, dtype=dtype, device=dev).transpose(1, 2), torch.zeros(3, 4, 100, dim, dtype=dtype, device=dev))
        kept = evict(kd, vd, wd, 290, 100, 10, 1, out)
        ko, vo = (kd, vd) if in_place else out
        assert torch.equal(kept.cpu().long(), want)
        assert torch.equal(ko[..., :100, :].cpu(), moved(k, want)) and torch.equal(vo[..., :100, :].cpu(), moved(v, want))
        assert (big[0] == 0).all() and (big[4] == 0).all()


def test_long_cache_passes_32_bits(dev):
    """A head's rows more than 4 GiB from the caches' start."""
    from flint_amd.attention import evict, tree_attention
    big = torch.zeros(40, 1, 1 << 20, 64, dtype=torch.bfloat16, device=dev)  # 5.4 GB
    k = big[39:, :, :2000]
    k.copy_(torch.randn(1, 1, 2000, 64))
    first = k.clone()
    w = torch.rand(40, 1, 1 << 20, device=dev)
    view = big[:, :, :2000]
    wv = w[:, :, :2000].contiguous()
    kept = evict(view, view.clone(), wv, 2000, 500)
    assert torch.equal(view[39, 0, :500], first[0, 0][kept[39, 0].long()])
    # attention over slots that lie 4 GiB apart
    far = big.view(1, 1, 40 << 20, 64)[:, :, ::16384]  # slots 2 MB apart, 2560 of them
    q = torch.randn(1, 3, 4, 64, device=dev, dtype=torch.bfloat16)
    far.copy_(torch.randn(far.shape, device=dev))
    near = far.contiguous()
    assert torch.equal(tree_attention(q, far, far, 2500), tree_attention(q, near, near, 2500))


def test_refusals(dev):
    from flint_amd.attention import evict
    k, v, w = (x.to(dev) for x in make((2, 2), 50, 64))
    new = torch.zeros(2, 2, 20, 64, dtype=k.dtype, device=dev)
    for kw in (dict(n=51), dict(n=-1), dict(keep=0), dict(recent=-1), dict(recent=11), dict(sink=6, recent=5), dict(v_cache=v.float()), dict(v_cache=v.cpu()),
               dict(weights=w.half()), dict(weights=w[..., :40]), dict(weights=w.transpose(0, 1)), dict(out=(new,)), dict(out=(new, new[..., :5, :])),
               dict(out=(new[..., :5, :], new[..., :5, :])), dict(out=(k[..., :20, :], new)), dict(out=(new, new.float())), dict(out=(new, new.cpu())),
               dict(out=(new, new.clone(), w[..., :20])), dict(k_cache=k[..., :4], v_cache=v[..., :4])):
        with pytest.raises(ValueError):
            evict(**{**dict(k_cache=k, v_cache=v, weights=w, n=40, keep=10), **kw})


def test_captured_and_replayed(dev):
    from flint_amd.attention import evict
    ins = [[x.to(dev) for x in make((3, 2), 2000, 64, seed=s, kind="ties")] for s in range(3)]
    held = [x.clone() for x in ins[0]]
    out = (torch.zeros(3, 2, 600, 64, dtype=torch.bfloat16, device=dev), torch.zeros(3, 2, 600, 64, dtype=torch.bfloat16, device=dev),
           torch.zeros(3, 2, 600, device=dev))
    want = [(evict(*x, 1900, 600, 50, 4, out).clone(), *[t.clone() for t in out]) for x in ins]
    torch.cuda.synchronize()
    gr, gp = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        kept = evict(*held, 1900, 600, 50, 4, out)
    with torch.cuda.graph(gp):
        in_place = evict(*held, 1900, 600, 50, 4)
    for i in (0, 2, 1, 0):
        for h, x in zip(held, ins[i]):
            h.copy_(x)
        for t in out:
            t.zero_()
        gr.replay()
        torch.cuda.synchronize()
        assert torch.equal(kept, want[i][0]) and all(torch.equal(a, b) for a, b in zip(out, want[i][1:]))
        gp.replay()
        torch.cuda.synchronize()
        assert torch.equal(in_place, want[i][0]) and torch.equal(held[0][..., :600, :], want[i][1])
        assert torch.equal(held[1][..., :600, :], want[i][2]) and (held[2][..., 600:1900] == 0).all()


@pytest.mark.parametrize("n", [1023, 1024, 1025, 2048, 2049, 8192, 8193, 32768, 32769, 70001])
def test_lengths_at_the_seams(dev, n):
    """A lane's keys in registers, two to thirty-two of them, and read again beyond: against a stable sort."""
    from flint_amd.attention import evict
    k, v, w = make((2,), n, 8, seed=n, kind="ties")
    keep = n // 3 + 1
    kept = evict(k.to(dev), v.to(dev), w.to(dev), n, keep, recent=5, sink=3)
    score = w.clone()
    score[:, :3], score[:, n - 5:] = math.inf, math.inf
    want = score.sort(dim=1, descending=True, stable=True).indices[:, :keep].sort(dim=1).values
    assert torch.equal(kept.cpu().long(), want)


def test_shared_rows_are_not_written(dev):
    from flint_amd.attention import evict
    k, v, w = (x.to(dev) for x in make((2, 2), 50, 64))
    new = torch.zeros(2, 2, 20, 64, dtype=k.dtype, device=dev)
    with pytest.raises(ValueError):
        evict(k, k, w, 40, 10)
    with pytest.raises(ValueError):
        evict(k, v, w, 40, 10, out=(new, new))
    wide = k[:1].expand(2, 2, 50, 64)
    with pytest.raises(ValueError):
        evict(wide, v, w, 40, 10)
    with pytest.raises(ValueError):
        evict(k, v, w, 40, 10, out=(new[:1].expand(2, 2, 20, 64), new.clone()))
    # to be read they may be shared
    kept = evict(wide, v, w, 40, 10, out=(new, new.clone()))
    assert torch.equal(new[:, :, :10].cpu(), moved(wide.cpu(), kept.cpu().long()))


def test_more_slots_than_indices_reach(dev):
    from flint_amd.attention import evict
    k, v = (torch.zeros(1, 16, dtype=torch.uint8, device=dev).expand(2 ** 30 + 1, 16) for _ in range(2))
    with pytest.raises(ValueError, match="slots"):
        evict(k, v, torch.zeros(1, device=dev).expand(2 ** 30 + 1), 100, 10)


@pytest.mark.parametrize("low", [-math.inf, -3e38])
@pytest.mark.parametrize("n,keep", [(100, 100), (100, 99), (1100, 1100), (3000, 3000), (3000, 2990), (33000, 33000), (70001, 70001)])
def test_lowest_weights(dev, n, keep, low):
    """Weights whose ordered keys begin with zeros, as empty places' do: the slots kept, and nothing behind them."""
    from flint_amd.attention import evict
    k, v = (torch.randn(2, n, 8, device=dev) for _ in range(2))
    w = torch.full((2, n), low, device=dev)
    w[1, ::7] = 1.0
    kept = evict(k, v, w, n, keep, out=(torch.zeros(2, keep, 8, device=dev), torch.zeros(2, keep, 8, device=dev)))
    for h in range(2):
        assert kept[h].tolist() == oracle.kept_slots(w[h].tolist(), n, keep, 0, 0)


@pytest.mark.parametrize("heads,n", [(2, 49152), (2, 49153), (257, 32769), (257, 40001), (257, 49152), (256, 49152)])
def test_lengths_at_the_last_seams(dev, heads, n):
    """Up to forty-eight keys of a lane in registers, for up to 256 heads: against a stable sort."""
    from flint_amd.attention import evict
    k, v = (torch.zeros(heads, n, 8, dtype=torch.bfloat16, device=dev) for _ in range(2))
    g = torch.Generator(device=dev).manual_seed(n)
    w = (torch.rand(heads, n, generator=g, device=dev) * 50).floor()
    k[..., 0] = w
    keep = n // 3 + 1
    score = w.clone()
    score[:, :3], score[:, n - 5:] = math.inf, math.inf
    want = score.sort(dim=1, descending=True, stable=True).indices[:, :keep].sort(dim=1).values
    kept = evict(k, v, w, n, keep, recent=5, sink=3)
    assert torch.equal(kept.long(), want)
    assert torch.equal(k[:, :keep, 0], w[:, :keep].bfloat16()) and (w[:, keep:] == 0).all()


def test_rows_that_meet_are_not_written(dev):
    """K and V, heads or weights that share a part of their memory; views that only lie between each other go through."""
    from flint_amd.attention import evict
    _, _, w = (x.to(dev) for x in make((2, 2), 50, 64))
    flat = torch.randn(2 * 2 * 50 * 64 + 4096, device=dev).bfloat16()

    def view(start, *strides, slots=50):
        return flat.as_strided((2, 2, slots, 64), (*strides, 1), start)
    k = view(0, 6400, 3200, 64)
    for v in (view(64, 6400, 3200, 64), view(3200, 6400, 3200, 64), view(32, 6400, 3200, 64), view(8, 6400, 3200, 64), view(0, 64, 128, 256)):
        with pytest.raises(ValueError, match="same memory"):
            evict(k, v, w, 40, 10)
    far = torch.randn(2, 2, 50, 64, device=dev).bfloat16()
    for bad in (view(0, 3200, 1600, 64), view(0, 64, 3200, 64), view(0, 8, 3200, 64)):
        with pytest.raises(ValueError, match="share"):
            evict(bad, far, w, 40, 10)
        with pytest.raises(ValueError, match="share"):
            evict(far, far.clone(), w, 40, 10, out=(bad, far.clone()))
    new = torch.zeros(2 * 2 * 20 * 64 + 640, dtype=torch.bfloat16, device=dev)
    a, b = new[:5120].view(2, 2, 20, 64), new[64:5184].view(2, 2, 20, 64)
    with pytest.raises(ValueError, match="same memory"):
        evict(far, far.clone(), w, 40, 10, out=(a, b))
    with pytest.raises(ValueError, match="overlap"):
        evict(far, far.clone(), w, 40, 10, out=(a, torch.zeros_like(a), new[16:176].view(torch.float32).view(2, 2, 20)))
    with pytest.raises(ValueError, match="overlap"):
        evict(far, far.clone(), far.view(-1)[:400].view(torch.float32).view(2, 2, 50), 40, 10)
    # K and V of a slot next to each other, of a head next to each other, of a sequence next to each other
    for shape, dim in (((2, 2, 50, 2, 64), 3), ((2, 2, 2, 50, 64), 2), ((2, 2, 2, 50, 64), 1)):
        both = torch.randn(shape, device=dev).bfloat16()
        kk, vv = both.unbind(dim)
        k0, v0, w0 = kk.clone(), vv.clone(), w.clone()
        want = evict(k0, v0, w0, 40, 10, 2, 1)
        wi = w.clone()
        assert torch.equal(evict(kk, vv, wi, 40, 10, 2, 1), want)
        assert torch.equal(kk, k0) and torch.equal(vv, v0) and torch.equal(wi, w0)
    # slots before heads
    t = [torch.randn(2, 50, 2, 64, device=dev).bfloat16().transpose(1, 2) for _ in range(2)]
    c = [x.clone() for x in t]
    assert torch.equal(evict(*t, w.clone(), 40, 10), evict(*c, w.clone(), 40, 10)) and all(torch.equal(x, y) for x, y in zip(t, c))

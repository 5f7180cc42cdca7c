"""Attention of drafted trees over a cache, and the weight that keys gather, against 64 bits.

Tolerances. q, k, v are 16-bit, so products are exact in fp32 and a score's error is at most dim roundings of its
partial sums: dim 2^-24 sum|q k| scale, plus the exponent's own (2^-22 of its argument). The weights P go through the
matrix cores as two 16-bit terms: 2^-16 relative at most. fp32 sums over n keys: n 2^-24. All of it acts on the
numerator and the denominator of a mean of values no larger than max|v|; the output is rounded once to its type.
"""
import math

import pytest
import torch

from oracle import cache as oracle

pytestmark = pytest.mark.gpu


def tree_mask(g, b, m, empty=False):
    """bool [b, m, m]: ancestors in random trees; with `empty`, some nodes see nothing, not even themselves."""
    mask = torch.zeros(b, m, m, dtype=torch.bool)
    for s in range(b):
        mask[s, 0, 0] = True
        for i in range(1, m):
            p = int(torch.randint(max(0, i - 4), i, (1,), generator=g))
            mask[s, i] = mask[s, p]
            mask[s, i, i] = True
        if empty:
            mask[s, 1::3] = False
    return mask


def make(b, m, heads, groups, dim, slots, dtype, seed=0, sharp=1.0):
    g = torch.Generator().manual_seed(seed)
    q = (torch.randn(b, m, heads, dim, generator=g) * 1.5 * sharp).to(dtype)
    k = torch.randn(b, groups, slots, dim, generator=g).to(dtype)
    v = torch.randn(b, groups, slots, dim, generator=g).to(dtype)
    return g, q, k, v


def score_error(q, k, scale, dim):
    """A bound on any score's error: dim 2^-24 max|q| . |k| scale."""
    qm = q.double().abs().nan_to_num(0, 0, 0).flatten(0, -2).amax(0)
    km = k.double().abs().nan_to_num(0, 0, 0).flatten(0, -2).amax(0)
    most = float((qm * km).sum() * scale)
    return dim * 2.0 ** -24 * most + 2.0 ** -22 * most


def check_attention(q, k, v, pos, mask, scale, out, lse):
    dim, dtype = q.shape[-1], q.dtype
    b = q.shape[0]
    plist = [pos] * b if isinstance(pos, int) else [int(x) for x in pos]
    o, l = oracle.tree_attention(q, k, v, plist, mask, scale)
    n = max(plist) + q.shape[1]
    es = score_error(q, k, scale, dim)
    delta = 2.0 ** -16 + 2 * es + n * 2.0 ** -24 + 2.0 ** -20
    vmax = float(v.double().nan_to_num(0, 0, 0).abs().max())
    tol = torch.finfo(dtype).eps / 2 * o.abs() + 2 * delta * vmax + torch.finfo(dtype).smallest_normal * 2.0 ** -7
    got = out.double().cpu()
    assert torch.equal(got.isnan(), o.isnan())
    fin = ~o.isnan() & ~o.isinf()
    assert torch.equal(got[o.isinf()], o[o.isinf()])
    bad = ((got - o).abs() > tol) & fin
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {float(((got - o).abs() / tol)[fin].max()):.2f} x"
    none = l == -math.inf
    assert torch.equal(lse.cpu().double()[none], l[none])
    fin = ~none & ~l.isnan() & ~l.isinf()
    ltol = es + n * 2.0 ** -24 + 2.0 ** -21 * (l.abs() + 1)
    assert not (((lse.cpu().double() - l).abs() > ltol) & fin).any()


SHAPES = [  # b, m, heads, groups, dim, ctx: one token to some hundred rows, lengths at the seams of tiles and parts
    (1, 1, 40, 8, 64, 0), (1, 1, 40, 8, 64, 1), (1, 1, 40, 8, 64, 511), (1, 1, 40, 8, 64, 512), (1, 1, 7, 1, 64, 63),
    (1, 1, 12, 12, 128, 256), (1, 8, 40, 8, 64, 1024), (1, 8, 8, 2, 64, 0), (2, 13, 16, 2, 128, 300), (3, 5, 6, 3, 64, 64),
    (1, 33, 8, 2, 64, 100), (1, 32, 20, 4, 64, 31), (2, 70, 10, 2, 64, 129), (1, 130, 4, 1, 128, 65), (1, 6, 40, 8, 64, 2050),
    (1, 12, 5, 1, 64, 700), (1, 13, 5, 1, 128, 700),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_attention(dev, shape, tree, dtype):
    from flint_amd.attention import tree_attention
    b, m, heads, groups, dim, ctx = shape
    g, q, k, v = make(b, m, heads, groups, dim, ctx + m + 5, dtype, seed=m + ctx)
    # what lies behind the nodes is not read
    k[:, :, ctx + m:], v[:, :, ctx + m:] = math.nan, math.inf
    mask = tree_mask(g, b, m) if tree else None
    scale = dim ** -0.5
    out, lse = tree_attention(q.to(dev), k.to(dev), v.to(dev), ctx, None if mask is None else mask.to(dev), return_lse=True)
    k[:, :, ctx + m:], v[:, :, ctx + m:] = 0, 0
    check_attention(q, k, v, ctx, mask, scale, out, lse)


@pytest.mark.parametrize("m,heads,groups,dim", [(1, 10, 2, 64), (5, 10, 2, 64), (9, 8, 1, 128), (40, 8, 2, 64)])
def test_ragged_positions(dev, m, heads, groups, dim):
    """A length per sequence, from none to all slots; one outside gives NaN and touches no other."""
    from flint_amd.attention import tree_attention
    slots = 1500
    pos = [0, 1, 700, slots - m, 64, -1, slots - m + 1, 2 ** 31 - 1]
    g, q, k, v = make(len(pos), m, heads, groups, dim, slots, torch.bfloat16, seed=m)
    mask = tree_mask(g, len(pos), m)
    for pt in (torch.tensor(pos, dtype=torch.int32), torch.tensor(pos[:-1] + [2 ** 40], dtype=torch.int64)):
        out, lse = tree_attention(q.to(dev), k.to(dev), v.to(dev), pt.to(dev), mask.to(dev), 0.2, True)
        assert out[5:].isnan().all() and lse[5:].isnan().all()
        check_attention(q[:5], k[:5], v[:5], pos[:5], mask[:5], 0.2, out[:5], lse[:5])


@pytest.mark.parametrize("m,dim", [(4, 64), (9, 64), (9, 128), (40, 64)])
@pytest.mark.parametrize("pos", [0, 100])
def test_rows_that_see_nothing(dev, m, dim, pos):
    from flint_amd.attention import tree_attention
    g, q, k, v = make(2, m, 8, 2, dim, pos + m, torch.bfloat16, seed=pos)
    mask = tree_mask(g, 2, m, empty=True)
    out, lse = tree_attention(q.to(dev), k.to(dev), v.to(dev), pos, mask.to(dev), return_lse=True)
    if pos == 0:
        assert (out[:, 1] == 0).all() and (lse[:, 1] == -math.inf).all()
    check_attention(q, k, v, pos, mask, dim ** -0.5, out, lse)


@pytest.mark.parametrize("m,heads,groups,dim", [(6, 4, 2, 64), (16, 8, 2, 64), (16, 8, 2, 128), (40, 8, 2, 64), (40, 8, 1, 128)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_masked_nodes_poison_no_row(dev, m, heads, groups, dim, dtype):
    """Infinities and NaN in the K and V of nodes reach the nodes that see them and no other."""
    from flint_amd.attention import tree_attention
    pos = 70
    g, q, k, v = make(1, m, heads, groups, dim, pos + m, dtype, seed=3)
    mask = torch.eye(m, dtype=torch.bool)
    mask[:, 0] = True
    k[:, :, pos + 2], v[:, :, pos + 2] = math.nan, math.nan
    v[:, :, pos + 3, 5] = math.inf
    v[:, :, pos + 4, 7:9] = math.nan
    k[:, :, pos + 5] = -math.inf
    out, lse = tree_attention(q.to(dev), k.to(dev), v.to(dev), pos, mask.to(dev), return_lse=True)
    got = out.cpu()[0]
    assert got[2].isnan().all() and lse[0, 2].isnan().all()
    assert (got[3, :, 5] == math.inf).all() and got[4, :, 7:9].isnan().all() and got[4, :, 9:].isfinite().all()
    clean = [i for i in range(m) if i not in (2, 3, 4, 5)]
    assert got[clean].isfinite().all()
    k, v = k.nan_to_num(0, 0, 0), v.nan_to_num(0, 0, 0)
    o, _ = oracle.tree_attention(q, k, v, [pos], mask, dim ** -0.5)
    for i in clean:
        es = score_error(q, k, dim ** -0.5, dim)
        tol = torch.finfo(dtype).eps / 2 * o[0, i].abs() + 2 * (2.0 ** -16 + 2 * es + (pos + m) * 2.0 ** -24 + 2.0 ** -20) * float(v.abs().max())
        assert ((got[i].double() - o[0, i]).abs() <= tol).all()


def test_extreme_scores(dev):
    """Scores that pass the exponential's range either way: one key takes all."""
    from flint_amd.attention import tree_attention
    g, q, k, v = make(1, 3, 4, 2, 64, 600, torch.bfloat16, seed=1, sharp=60.0)
    out, lse = tree_attention(q.to(dev), k.to(dev), v.to(dev), 597, None, 4.0, True)
    # scores up to 10^4, whose fp32 error is up to 0.1: compare where one key leads by 20, so that no other counts, and
    # the leading weight's two 16-bit terms leave its value of v where it rounds to
    es = score_error(q, k, 4.0, 64)
    qd, kd = q.double(), k.double()
    for i in range(3):
        for h in range(4):
            s = (kd[0, h // 2, :598 + i] @ qd[0, i, h]) * 4.0
            top = s.topk(2).values
            if top[0] - top[1] > 20:
                assert torch.equal(out[0, i, h].cpu(), v[0, h // 2, int(s.argmax())])
            assert abs(float(lse[0, i, h]) - float(torch.logsumexp(s, 0))) <= es + 600 * 2.0 ** -24
    assert out.isfinite().all()


@pytest.mark.parametrize("m", [1, 7, 40])
def test_strides(dev, m):
    """Caches as [B, slots, key heads, dim] views, windows of larger caches, q of every order."""
    from flint_amd.attention import attention_weights, tree_attention
    g, q, k, v = make(2, m, 8, 2, 64, 400, torch.bfloat16, seed=9)
    mask = tree_mask(g, 2, m)
    want, wl = tree_attention(q.to(dev), k.to(dev), v.to(dev), 300, mask.to(dev), return_lse=True)
    ww = attention_weights(q.to(dev), k.to(dev), wl, 300, mask.to(dev))
    kt = k.transpose(1, 2).contiguous().to(dev).transpose(1, 2)
    big = torch.full((2, 3, 500, 64), math.nan, dtype=v.dtype, device=dev)
    big[:, 1:, 60:460] = v.to(dev)
    qt = q.permute(1, 2, 0, 3).contiguous().to(dev).permute(2, 0, 1, 3)
    odd = torch.empty(q.numel() + 1, dtype=q.dtype, device=dev)[1:].view(q.shape).copy_(q)
    for qq in (qt, odd):
        out, lse = tree_attention(qq, kt, big[:, 1:, 60:460], 300, mask.to(dev).to(torch.uint8), return_lse=True)
        assert torch.equal(out, want) and torch.equal(lse, wl)
        assert torch.equal(attention_weights(qq, kt, wl, 300, mask.to(dev)), ww)
    one, ol = tree_attention(q[1].to(dev), k[1].to(dev), v[1].to(dev), 300, mask[1].to(dev), return_lse=True)
    assert torch.equal(one, want[1]) and torch.equal(ol, wl[1])
    assert torch.equal(attention_weights(q[1].to(dev), k[1].to(dev), ol, 300, mask[1].to(dev)), ww[1])


def test_row_does_not_depend_on_repeats(dev):
    """Twenty calls, the same bits; on another stream too."""
    from flint_amd.attention import attention_weights, tree_attention
    g, q, k, v = make(1, 16, 40, 8, 64, 3000, torch.bfloat16, seed=5)
    q, k, v = q.to(dev), k.to(dev), v.to(dev)
    first, l0 = tree_attention(q, k, v, 2900, return_lse=True)
    w0 = attention_weights(q, k, l0, 2900)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    for i in range(20):
        with torch.cuda.stream(s if i % 2 else torch.cuda.current_stream()):
            out, lse = tree_attention(q, k, v, 2900, return_lse=True)
            w = attention_weights(q, k, lse, 2900)
        s.synchronize()
        torch.cuda.synchronize()
        assert torch.equal(out, first) and torch.equal(lse, l0) and torch.equal(w, w0)


WSHAPES = [(1, 1, 40, 8, 64, 0), (2, 1, 40, 8, 64, 130), (1, 1, 12, 12, 128, 64), (1, 6, 10, 2, 64, 63), (2, 7, 8, 1, 128, 200),
           (1, 33, 8, 2, 64, 100), (1, 100, 5, 1, 64, 0), (1, 64, 4, 2, 128, 190)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("shape", WSHAPES)
def test_weights(dev, shape, tree, dtype):
    from flint_amd.attention import attention_weights, tree_attention
    b, m, heads, groups, dim, ctx = shape
    slots = ctx + m + 70
    g, q, k, v = make(b, m, heads, groups, dim, slots, dtype, seed=m + ctx)
    k[:, :, ctx + m:] = math.nan
    mask = tree_mask(g, b, m, empty=True) if tree else None
    dm = None if mask is None else mask.to(dev)
    _, lse = tree_attention(q.to(dev), k.to(dev), v.to(dev), ctx, dm, return_lse=True)
    w = attention_weights(q.to(dev), k.to(dev), lse, ctx, dm)
    k[:, :, ctx + m:] = 0
    want = oracle.attention_weights(q, k, lse.cpu(), [ctx] * b, mask, dim ** -0.5)
    # each term e^(s - lse): the score's error and the exponent's argument's, then the sums over the rows
    rel = score_error(q, k, dim ** -0.5, dim) + 2.0 ** -21 * (float(lse[lse > -math.inf].abs().max()) + 1) + m * heads * 2.0 ** -24
    assert ((w.double().cpu() - want).abs() <= rel * want + 1e-30).all()
    assert (w[:, :, ctx + m:] == 0).all()
    base = torch.rand(w.shape, generator=g).to(dev)
    base[:, :, ctx + m:] = math.nan  # left as it is
    added = attention_weights(q.to(dev), k.to(dev), lse, ctx, dm, out=(acc := base.clone()))
    assert added is acc
    assert torch.equal(acc[:, :, :ctx + m], base[:, :, :ctx + m] + w[:, :, :ctx + m]) and acc[:, :, ctx + m:].isnan().all()


def test_weights_sum_to_the_rows(dev):
    """Every row hands out 1: over the keys of a head the weights sum to its rows."""
    from flint_amd.attention import attention_weights, tree_attention
    pos = torch.tensor([0, 17, 900, -1], dtype=torch.int32)
    g, q, k, v = make(4, 5, 16, 4, 64, 1000, torch.bfloat16, seed=2)
    _, lse = tree_attention(q.to(dev), k.to(dev), v.to(dev), pos.to(dev), return_lse=True)
    w = attention_weights(q.to(dev), k.to(dev), lse, pos.to(dev))
    assert ((w[:3].double().sum(-1) - 20.0).abs() <= 20 * (score_error(q, k, 0.125, 64) * 2 + 2.0 ** -18 + 1000 * 2.0 ** -24)).all()
    assert w[3].isnan().all()


def test_refusals(dev):
    from flint_amd.attention import attention_weights, tree_attention
    _, q, k, v = make(2, 3, 4, 2, 64, 20, torch.bfloat16)
    q, k, v = q.to(dev), k.to(dev), v.to(dev)
    lse = torch.zeros(2, 3, 4, device=dev)
    ok = dict(q=q, k_cache=k, v_cache=v, pos=5)
    eye = torch.eye(3, device=dev)
    for kw in (dict(q=q.float()), dict(q=q.cpu()), dict(k_cache=k.half()), dict(v_cache=v[:, :, :10]), dict(k_cache=k[:1]), dict(pos=-1),
               dict(pos=18), dict(pos=torch.tensor([1], device=dev)), dict(pos=torch.zeros(2, device=dev)), dict(pos=torch.zeros(2, dtype=torch.int32)),
               dict(mask=eye), dict(mask=eye.bool()[:2]), dict(mask=eye.bool().cpu()), dict(scale=0.0), dict(scale=-0.1), dict(scale=math.nan),
               dict(scale=math.inf), dict(q=q[..., :3, :]), dict(q=q[..., :32]), dict(q=q[:0], k_cache=k[:0], v_cache=v[:0]),
               dict(k_cache=k.transpose(2, 3).contiguous().transpose(2, 3)), dict(k_cache=torch.cat([k, k], -1)[..., 4:68])):
        with pytest.raises(ValueError):
            tree_attention(**{**ok, **kw})
    for kw in (dict(lse=lse.half()), dict(lse=lse[:1]), dict(out=torch.zeros(2, 2, 19, device=dev)), dict(out=torch.zeros(2, 2, 20)),
               dict(out=torch.zeros(2, 2, 40, device=dev)[..., ::2])):
        with pytest.raises(ValueError):
            attention_weights(**{**dict(q=q, k_cache=k, lse=lse, pos=5), **kw})


@pytest.mark.parametrize("b,m,ctx,dim", [(1, 1, 300, 64), (1, 8, 3000, 64), (3, 40, 700, 128), (2, 1, 9000, 64)])
def test_captured_and_replayed(dev, b, m, ctx, dim):
    """A captured call replays to the eager one's bits, on new inputs, with eager work in between; two graphs that were
    captured one after the other share nothing."""
    from flint_amd.attention import attention_weights, tree_attention
    slots = ctx + m
    ins = []
    for seed in range(3):
        g, q, k, v = make(b, m, 8, 2, dim, slots, torch.bfloat16, seed=seed)
        pos = torch.tensor([ctx - 5 * i * seed for i in range(b)], dtype=torch.int32)
        ins.append([x.to(dev) for x in (q, k, v, pos, tree_mask(g, b, m))])
    held = [x.clone() for x in ins[0]]

    def call(x):
        out, lse = tree_attention(x[0], x[1], x[2], x[3], x[4], return_lse=True)
        return out, lse, attention_weights(x[0], x[1], lse, x[3], x[4])
    want = [[y.clone() for y in call(x)] for x in ins]
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            got = call(held)
        graphs.append((gr, got))
    for i in (0, 1, 2, 1, 0, 2):
        for h, x in zip(held, ins[i]):
            h.copy_(x)
        for gr, got in graphs:
            gr.replay()
        call(ins[(i + 1) % 3])
        torch.cuda.synchronize()
        for gr, got in graphs:
            assert all(torch.equal(a, w) for a, w in zip(got, want[i]))


def test_two_streams_at_once(dev):
    """Calls that run at the same time have a workspace each."""
    from flint_amd.attention import tree_attention
    _, q, k, v = make(1, 9, 40, 8, 64, 20000, torch.bfloat16, seed=1)
    q, k, v = q.to(dev), k.to(dev), v.to(dev)
    want = [tree_attention(q, k, v, p) for p in (19000, 12345)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(15):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(tree_attention(q, k, v, (19000, 12345)[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i]) for i in range(2) for g in got[i])


@pytest.mark.parametrize("slots,b,groups", [(20000, 1, 1), (3000, 40, 8), (1 << 17, 1, 2)])
def test_single_tokens_of_many_lengths(dev, slots, b, groups):
    """One token a sequence behind every kind of length, parts of them empty for the shorter ones, against a float64
    product on the device."""
    from flint_amd.attention import tree_attention
    g = torch.Generator(device=dev).manual_seed(slots)
    heads = groups * 5
    q = torch.randn(b, 1, heads, 64, generator=g, device=dev).bfloat16()
    k, v = (torch.randn(b, groups, slots, 64, generator=g, device=dev).bfloat16() for _ in range(2))
    for lens in ([slots - 1] * b, [(slots - 1) * i // b for i in range(b)], [i % 3 for i in range(b)]):
        pos = torch.tensor(lens, dtype=torch.int32, device=dev)
        out, lse = tree_attention(q, k, v, pos, return_lse=True)
        n = max(lens) + 1
        seen = torch.arange(n, device=dev) <= pos[:, None]
        for j in range(groups):
            s = torch.matmul(q[:, 0, 5 * j:5 * j + 5].double(), k[:, j, :n].double().transpose(1, 2).contiguous()) * 0.125
            s = s.masked_fill(~seen[:, None], -math.inf)
            o = torch.matmul(torch.softmax(s, -1), v[:, j, :n].double())
            es = 64 * 2.0 ** -24 * 64 * 16 * 0.125 + 2.0 ** -20 * 16  # |q|, |k| below 5 in these draws: sum|q k| < 64 * 16
            tol = 2.0 ** -8 * o.abs() + 2 * (2.0 ** -16 + es + n * 2.0 ** -24) * 5.5
            assert ((out[:, 0, 5 * j:5 * j + 5].double() - o).abs() <= tol).all()
            assert ((lse[:, 0, 5 * j:5 * j + 5].double() - torch.logsumexp(s, -1)).abs() <= es + n * 2.0 ** -24 + 2.0 ** -18).all()


@pytest.mark.parametrize("m,rep,dim", [(40, 2, 64), (11, 3, 128), (21, 5, 64)])
def test_a_query_that_is_no_number_reaches_what_its_node_sees(dev, m, rep, dim):
    """Queries ordered by head: behind a head's last node lies the next head's first, which is NaN here."""
    from flint_amd.attention import attention_weights
    g, q, k, v = make(1, m, rep, 1, dim, 300, torch.bfloat16, seed=5)
    q[0, 0, 1] = math.nan
    pos = 55
    _, l = oracle.tree_attention(q, k, v, [pos], None, dim ** -0.5)
    want = oracle.attention_weights(q, k, l, [pos], None, dim ** -0.5)
    assert want.isnan().sum() == pos + 1
    qd = q.to(dev).transpose(1, 2).contiguous().transpose(1, 2)
    got = attention_weights(qd, k.to(dev), l.float().to(dev), pos).cpu()
    assert torch.equal(got.isnan(), want.isnan())


FAR = [  # b, m, heads, groups, dim, ctx: either kernel, one part of the keys and many
    (1, 1, 8, 2, 64, 64), (1, 1, 8, 2, 64, 1100), (1, 1, 8, 2, 64, 20000), (1, 1, 8, 2, 128, 30000), (1, 6, 8, 2, 64, 60000),
    (1, 40, 8, 2, 64, 5000), (1, 16, 8, 1, 128, 9000), (8, 300, 48, 48, 64, 1500),
]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("gap", [10.0, 15.0, 17.375, 20.0, 24.0])
@pytest.mark.parametrize("shape", FAR)
def test_weights_far_below_a_leading_key(dev, shape, gap, dtype):
    """Three leading keys whose values are 0, all others `gap` (or, of odd heads, half of that) below them: what these
    add up to, to the output's own precision.

    Scores are exact here (powers of two and multiples of 1/64). A weight's exponent and the factors that join parts have
    arguments below 64 in log2: 2^-19 each, three of them and the exponential's own error below 2^-16 of the weight. Its
    two terms leave 2^-17 of it in bf16; in fp16 2^-28 of the largest weight of its tile of up to 64 keys, which in the three
    tiles of a leading key is 2^-36 of that key's, elsewhere far below 2^-17 of the sum. fp32 sums in sequence: n / 8
    additions, at 2^-24 each, of the numerator and of the denominator."""
    from flint_amd.attention import tree_attention
    b, m, heads, groups, dim, ctx = shape
    rep, n = heads // groups, ctx + m
    g = torch.Generator(device=dev).manual_seed(ctx)
    q = torch.zeros(b, m, heads, dim, device=dev)
    q[..., 0] = 8.0
    if rep > 1:
        q[:, :, 1::2, 0] = 4.0
    k = torch.zeros(b, groups, n, dim, device=dev)
    k[..., 0] = torch.randint(-32, 33, (b, groups, n), generator=g, device=dev) / 64
    v = 32 * (0.5 + torch.rand(b, groups, n, dim, generator=g, device=dev))
    lead = [0, ctx // 2, ctx - 1]
    k[:, :, lead, 0] = gap
    v[:, :, lead] = 0
    q, k, v = q.to(dtype), k.to(dtype), v.to(dtype)
    assert (k[:, :, lead, 0] == gap).all()
    out, lse = tree_attention(q, k, v, ctx, None, 0.125, True)
    hidden = torch.arange(n, device=dev) > ctx + torch.arange(m, device=dev)[:, None]
    vmax = 48.0
    for s in range(b):
        for j in range(groups):
            sc = torch.matmul(q[s, :, j * rep:(j + 1) * rep].transpose(0, 1).double(), k[s, j].double().t().contiguous()) * 0.125
            sc = sc.masked_fill(hidden, -math.inf)
            o = torch.matmul(torch.softmax(sc, -1), v[s, j].double()).transpose(0, 1)
            rel = 2 * (2.0 ** -16 + 2.0 ** -17 + n / 8 * 2.0 ** -24)
            tol = torch.finfo(dtype).eps / 2 * o * (1 + rel) + rel * o + (3 * 64 * 2.0 ** -36 * vmax + 2.0 ** -25 if dtype == torch.float16 else 0.0)
            err = (out[s, :, j * rep:(j + 1) * rep].double() - o).abs()
            assert (err <= tol).all(), f"{float((err / tol).max()):.2f} x, {float((err / o).max()):.2e} of the value"
            l = torch.logsumexp(sc, -1).t()
            assert ((lse[s, :, j * rep:(j + 1) * rep].double() - l).abs() <= 2.0 ** -16 + n / 8 * 2.0 ** -24 + 2.0 ** -21 * l.abs()).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("order", ["rising", "falling", "back and forth"])
@pytest.mark.parametrize("m,heads,groups,dim,ctx", [(1, 4, 2, 64, 1400), (1, 4, 4, 64, 9000), (40, 4, 2, 64, 5000), (16, 8, 1, 128, 1000)])
def test_scores_that_rise_and_fall(dev, m, heads, groups, dim, ctx, order, dtype):
    """Levels of scores over 60, a hundred slots each, the keys of the highest level with values of 0: rel as
    above, and what the highest level's own tiles (two of 64 keys at 100 slots) leave, 2^-36 of its weight each."""
    from flint_amd.attention import tree_attention
    n = ctx + m
    g = torch.Generator(device=dev).manual_seed(ctx)
    level = torch.arange(n, device=dev) // 100
    steps = int(level[-1]) + 1
    height = torch.linspace(0, 1, steps, device=dev)
    if order == "falling":
        height = height.flip(0)
    elif order == "back and forth":
        height = torch.where(torch.arange(steps, device=dev) % 2 == 0, height, 1 - height)
    top = int(height.argmax())
    # from 0 to 44 below the highest level, that one 16 above the next
    score = ((height * 28).round() + 16 * (torch.arange(steps, device=dev) == top))[level]
    q = torch.zeros(1, m, heads, dim, device=dev)
    q[..., 0] = 8.0
    k = torch.zeros(1, groups, n, dim, device=dev)
    k[..., 0] = score
    v = 32 * (0.5 + torch.rand(1, groups, n, dim, generator=g, device=dev))
    v[:, :, level == top] = 0
    q, k, v = q.to(dtype), k.to(dtype), v.to(dtype)
    out, lse = tree_attention(q, k, v, ctx, None, 0.125, True)
    rep = heads // groups
    hidden = torch.arange(n, device=dev) > ctx + torch.arange(m, device=dev)[:, None]
    for j in range(groups):
        sc = torch.matmul(q[0, :, j * rep:(j + 1) * rep].transpose(0, 1).double(), k[0, j].double().t().contiguous()) * 0.125
        sc = sc.masked_fill(hidden, -math.inf)
        o = torch.matmul(torch.softmax(sc, -1), v[0, j].double()).transpose(0, 1)
        rel = 2 * (2.0 ** -16 + 2.0 ** -17 + n / 8 * 2.0 ** -24)
        # a row's sum is its highest weight or more, so what is left out of a weight is 2^-36 of the sum at most
        tol = torch.finfo(dtype).eps / 2 * o * (1 + rel) + rel * o + (3 * 64 * 2.0 ** -36 * 48 + 2.0 ** -25 if dtype == torch.float16 else 0.0)
        err = (out[0, :, j * rep:(j + 1) * rep].double() - o).abs()
        assert (err <= tol).all(), f"{float((err / tol).max()):.2f} x"
        assert ((lse[0, :, j * rep:(j + 1) * rep].double() - torch.logsumexp(sc, -1).t()).abs() <= 2.0 ** -14 + n / 8 * 2.0 ** -24).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,heads,groups,dim", [(1, 10, 2, 64), (6, 8, 2, 128), (40, 8, 2, 64), (150, 4, 1, 128)])
@pytest.mark.parametrize("ctx", [70, 1500, 2300, 3100, 5200, 50000])
def test_values_that_are_no_numbers(dev, ctx, m, heads, groups, dim, dtype):
    """An infinity or a NaN in the value of a slot that a node sees makes that dimension of it the same, however small its
    weight and however the keys are cut; infinities of both signs give NaN; the other dimensions keep their bits."""
    from flint_amd.attention import tree_attention
    n = ctx + m
    g, q, k, v = make(1, m, heads, groups, dim, n, dtype, seed=ctx + m)
    q, k, v = q.to(dev), k.to(dev), v.to(dev)
    q[..., 0] = 2.0
    k[:, :, 20, 0] = -60.0   # a weight of e^-15 and less
    k[:, :, 21, 0] = -2000.0  # e^-500: no fp32 number
    k[:, :, ctx // 2, 0] = 400.0  # takes all
    clean, lse = tree_attention(q, k, v, ctx, None, 0.125, True)
    bad = v.clone()
    bad[:, :, 0, 1] = math.inf
    bad[:, :, 20, 2] = -math.inf
    bad[:, :, 21, 3] = math.inf
    bad[:, :, ctx - 1, 4] = -math.inf
    bad[:, :, ctx // 2, 5] = math.inf
    bad[:, :, 5, 6], bad[:, :, ctx - 2, 6] = math.inf, -math.inf
    bad[:, :, 33, 7] = math.nan
    bad[:, :, ctx, 40] = -math.inf        # node 0
    bad[:, :, 9, 41], bad[:, :, ctx, 41] = -math.inf, math.inf
    bad[:, :, n - 1, 63] = math.inf       # the last node: seen by itself alone
    out, l2 = tree_attention(q, k, bad, ctx, None, 0.125, True)
    want = clean.clone()
    for d, x in ((1, math.inf), (2, -math.inf), (3, math.inf), (4, -math.inf), (5, math.inf), (6, math.nan), (7, math.nan), (40, -math.inf), (41, math.nan)):
        want[..., d] = x
    want[:, -1, :, 63] = math.inf
    assert torch.equal(l2, lse) and torch.equal(out.isnan(), want.isnan())
    assert torch.equal(out.nan_to_num(0.0, 7e4, -7e4), want.nan_to_num(0.0, 7e4, -7e4))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,heads,groups,dim", [(1, 5, 1, 64), (1, 10, 2, 128), (7, 6, 2, 64), (40, 4, 2, 64), (33, 3, 3, 128)])
def test_a_key_that_no_row_can_weigh(dev, m, heads, groups, dim, dtype):
    """A key whose scores are all -inf gathers 0, whatever stands behind the last row; a row whose lse is -inf adds nothing,
    not even to a key whose score is no number."""
    from flint_amd.attention import attention_weights, tree_attention
    pos = 100
    g, q, k, v = make(1, m, heads, groups, dim, pos + m + 3, dtype, seed=m)
    q[..., 3] = q[..., 3].abs() + 0.5
    k[:, :, 17, 3] = -math.inf
    k[:, :, pos, 3] = -math.inf
    _, lse = tree_attention(q.to(dev), k.to(dev), v.to(dev), pos, return_lse=True)
    got = attention_weights(q.to(dev), k.to(dev), lse, pos).cpu()
    want = oracle.attention_weights(q, k, lse.cpu(), [pos], None, dim ** -0.5)
    assert (want[:, :, [17, pos]] == 0).all() and (got[:, :, [17, pos]] == 0).all()
    rel = score_error(q, k.nan_to_num(0, 0, 0), dim ** -0.5, dim) + 2.0 ** -21 * (float(lse.abs().max()) + 1) + m * heads * 2.0 ** -24
    assert ((got.double() - want).abs() <= rel * want + 1e-30).all()
    k[:, :, 17, 3], k[:, :, 18, 3], k[:, :, 19, 5] = math.inf, math.nan, math.inf
    none = torch.full((1, m, heads), -math.inf, device=dev)
    assert (attention_weights(q.to(dev), k.to(dev), none, pos) == 0).all()


@pytest.mark.parametrize("dtype,big", [(torch.float16, 9.0e2), (torch.float16, 1.5e4), (torch.float16, 3.6e4), (torch.bfloat16, 6.0e4), (torch.bfloat16, 1.0e7), (torch.bfloat16, 1.0e16)])
@pytest.mark.parametrize("m,heads,groups,dim,ctx", [(1, 4, 2, 64, 300), (1, 4, 4, 64, 9000), (40, 4, 2, 64, 2000), (16, 8, 1, 128, 700)])
def test_scores_that_fp32_hardly_resolves(dev, m, heads, groups, dim, ctx, dtype, big):
    """Scores of 10^7 and far more, their differences exact multiples of a power of two: one key of a row leads all others
    by more than the score's own error, and its value is the row's (the others' weights are below 2^-60)."""
    from flint_amd.attention import tree_attention
    g = torch.Generator(device=dev).manual_seed(ctx)
    n = ctx + m
    q = torch.zeros(1, m, heads, dim, device=dev)
    q[..., :32] = big * (1 + torch.arange(m * heads, device=dev).view(1, m, heads, 1) % 5 / 8)
    k = torch.zeros(1, groups, n, dim, device=dev)
    level = torch.randint(1, 32, (1, groups, n), generator=g, device=dev) / 64
    for sign in (1.0, -1.0):
        k[..., :32] = (sign * big * (1 + level))[..., None]
        lead = torch.randint(0, ctx, (groups,), generator=g, device=dev)
        kk = k.clone()
        kk[0, torch.arange(groups), lead, :32] = big * (1.75 if sign > 0 else -0.875)
        v = torch.randn(1, groups, n, dim, generator=g, device=dev).to(dtype)
        qd, kd = q.to(dtype), kk.to(dtype)
        out, lse = tree_attention(qd, kd, v, ctx, None, 0.125, True)
        rep = heads // groups
        for j in range(groups):
            s = torch.matmul(qd[0, :, j * rep:(j + 1) * rep].double(), kd[0, j].double().t().contiguous()) * 0.125
            top = s.topk(2, -1).values
            # sums of 32 products: an error of 32 2^-24 of the score; the lead is 1/8 of it and more than 60 by far
            assert ((top[..., 0] - top[..., 1]) > 1e5).all()
            assert torch.equal(out[0, :, j * rep:(j + 1) * rep], v[0, j, lead[j]].expand(m, rep, dim))
            assert ((lse[0, :, j * rep:(j + 1) * rep].double() - top[..., 0]).abs() <= 2.0 ** -18 * top[..., 0].abs()).all()

"""Log probabilities, entropies, ranks and alternatives against the oracle's float64. Ranks and ids are exact. The
bounds of the others, with E = 2^-24 (half an fp32 step) and d the distances to the row's maximum:
- d is rounded once, d log2 e twice more: exp(d) is off by 3 E |d| + 2^-23 (the hardware's exp2, an ulp), relatively;
- s = sum exp(d): up to 96 values a thread, 9 steps across the workgroup, 32 chunks, each addition E: 140 E
  besides, so s is off by (3 U + 142 + ...) E <= (3 U + 150) E, with U = sum p |d|; log s by that and 2 E |log s|;
- a log probability adds E |d| and E |result|;
- u = sum exp(d) d the same with one factor d more: (3 Q + 150 U) E of its quotient by s, Q = sum p d^2."""
import math

import pytest
import torch

from flint_amd import _lib, generate, quantize
from flint_amd.model import Transformer
from flint_amd.synth import ModelArgs, synth_weights
from oracle import scoring

pytestmark = pytest.mark.gpu

E = 2.0 ** -24


def near(got, want, bound):
    if math.isnan(want):
        return math.isnan(got)
    if math.isinf(want):
        return got == want
    return abs(got - want) <= bound


def check(out, logits, tokens, top):
    """out of the GPU against the oracle's on the same logits (CPU, exact values)."""
    t = tokens if tokens is not None else torch.full((len(logits),), -1)
    for i, r in enumerate(scoring.logprobs(logits, t, top)):
        s_err = (3 * r["U"] + 150) * E
        log_err = s_err + 2 * E * abs(r["logsum"])
        if tokens is None:
            assert out.logprob is None and out.rank is None
        else:
            assert int(out.rank[i]) == r["rank"], i
            lp = r["logprob"]
            assert near(float(out.logprob[i]), lp, log_err + E * (2 * abs(lp) + abs(r["logsum"]))), i
        h_err = log_err + (3 * r["Q"] + 150 * r["U"]) * E + r["U"] * s_err + 2 * E * abs(r["entropy"])
        assert near(float(out.entropy[i]), r["entropy"], h_err), i
        if not top:
            assert out.top_ids is None and out.top_logprobs is None
            continue
        assert out.top_ids[i].tolist() == r["ids"].tolist(), i
        for got, want in zip(out.top_logprobs[i].tolist(), r["top"]):
            assert near(got, want, log_err + E * (2 * abs(want) + abs(r["logsum"]))), i


def host(out):
    return generate.TokenLogprobs(*(None if f is None else f.cpu() for f in out))


def rows_of(rows, vocab, seed, dtype):
    g = torch.Generator().manual_seed(seed)
    l = (torch.randn(rows, vocab, generator=g) * 3).to(torch.bfloat16).to(dtype)  # equal values are common
    return l, torch.randint(0, vocab, (rows,), generator=g, dtype=torch.int32)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab,top", [
    (1, 1, 1), (1, 1, 0), (3, 2, 2), (2, 7, 5), (5, 31, 31), (2, 63, 4), (4, 64, 8), (3, 65, 32), (2, 257, 20),
    (2, 511, 1), (3, 513, 5), (2, 1000, 32), (1, 2048, 20), (2, 4095, 5), (7, 4097, 20), (1, 8200, 32), (1, 32003, 20),
    (31, 32003, 8), (1, 49152, 20), (1, 49152, 0), (9, 49152, 32), (40, 49155, 5), (300, 5003, 5), (520, 16384, 3),
    (600, 33001, 20), (520, 49160, 5), (2, 160001, 20), (1, 1 << 20, 32), (3, (1 << 20) - 5, 7)])
def test_random_rows(dev, rows, vocab, top, dtype):
    logits, tokens = rows_of(rows, vocab, rows + vocab, dtype)
    out = host(generate.logprobs(logits.to(dev), tokens.to(dev), top))
    some = range(rows) if rows <= 40 else list(range(0, rows, rows // 13)) + [rows - 1]
    pick = lambda f: None if f is None else f[list(some)]  # noqa: E731
    check(generate.TokenLogprobs(*map(pick, out)), logits[list(some)], tokens[list(some)], top)


def hard_rows(vocab):
    """Rows where something can go wrong, and a token each."""
    g = torch.Generator().manual_seed(vocab)
    base = (torch.randn(vocab, generator=g) * 3).to(torch.bfloat16).float()
    low = torch.finfo(torch.bfloat16).min
    rows = []

    def add(r, t):
        rows.append((r, t))

    add(torch.zeros(vocab), vocab // 2)                                       # all equal
    add(torch.full((vocab,), -math.inf), vocab - 1)                           # nothing left
    one = torch.full((vocab,), -math.inf)
    one[vocab - 1] = 2.0
    add(one, vocab - 1)                                                       # one token left
    add(one, 0)                                                               # ... and a forbidden one asked for
    add(torch.where(torch.rand(vocab, generator=g) < 0.97, -math.inf, base), 1)
    lows = torch.where(torch.rand(vocab, generator=g) < 0.9, low, base)
    add(lows, 0)
    add(torch.full((vocab,), low), vocab // 3)                                # all of the lowest value
    huge = base.clone()
    huge[vocab // 2] = 3.3e38
    add(huge, vocab // 2)
    add(huge, 0)
    nan = base.clone()
    nan[vocab // 3] = math.nan
    nan[vocab - 1] = -math.nan
    add(nan, 0)
    add(nan, vocab - 1)
    add(torch.full((vocab,), math.nan), vocab - 1)
    inf = base.clone()
    inf[0] = math.inf
    inf[vocab // 2] = math.inf
    add(inf, vocab // 2)
    add(inf, 1)
    signs = torch.where(torch.rand(vocab, generator=g) < 0.5, 0.0, -0.0)
    add(signs, vocab - 1)                                                     # -0 equals 0
    add(torch.where(torch.rand(vocab, generator=g) < 0.5, 1.0, 0.0), vocab // 2)  # two values
    add(torch.arange(vocab).float().clamp(max=250.0), vocab - 1)              # rising
    add(-torch.arange(vocab).float().clamp(max=250.0), 0)                     # falling
    spike = torch.full((vocab,), -80.0)
    spike[vocab // 2] = 30.0
    add(spike, vocab // 2)                                                    # a certain token
    for bad in (-1, vocab, -2 ** 31, 2 ** 31 - 1):
        add(base, bad)                                                        # ids outside the vocabulary
    return torch.stack([r for r, _ in rows]).to(torch.bfloat16), torch.tensor([t for _, t in rows], dtype=torch.int32)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab,top", [(9, 9), (100, 20), (1003, 32), (5000, 8), (33333, 20), (49152, 5), (100003, 32)])
def test_rows_where_it_can_go_wrong(dev, vocab, top, dtype):
    logits, tokens = hard_rows(vocab)
    logits = logits.to(dtype)
    check(host(generate.logprobs(logits.to(dev), tokens.to(dev), top)), logits, tokens, top)
    if vocab in (1003, 33333):  # one at a time: rows are cut into other chunks
        for i in range(len(tokens)):
            check(host(generate.logprobs(logits[i].to(dev), tokens[i:i + 1].to(dev), top)), logits[i:i + 1],
                  tokens[i:i + 1], top)


def test_many_rows_of_equal_values(dev):
    """One chunk a row (more rows than workgroups) of few values: the candidates overflow."""
    g = torch.Generator().manual_seed(1)
    logits = torch.randint(0, 3, (700, 9001), generator=g).to(torch.bfloat16)
    tokens = torch.randint(0, 9001, (700,), generator=g, dtype=torch.int32)
    out = host(generate.logprobs(logits.to(dev), tokens.to(dev), 6))
    some = list(range(0, 700, 50))
    check(generate.TokenLogprobs(*(f[some] for f in out)), logits[some], tokens[some], 6)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_views_dtypes_and_shapes(dev, dtype):
    logits, tokens = rows_of(12, 1000, 3, dtype)
    want = host(generate.logprobs(logits.to(dev), tokens.to(dev), 5))
    check(want, logits, tokens, 5)

    def is_want(out):
        # other alignments take other loads, whose sums go in another order: the same within the bounds
        check(host(out), logits, tokens, 5)

    wide = torch.full((12, 1031), 99.0, dtype=dtype, device=dev)
    wide[:, :1000] = logits.to(dev)
    is_want(generate.logprobs(wide[:, :1000], tokens.to(dev), 5))              # rows apart, and not on 16 bytes
    shifted = torch.full((12, 1032), 99.0, dtype=dtype, device=dev)
    shifted[:, 1:1001] = logits.to(dev)
    is_want(generate.logprobs(shifted[:, 1:1001], tokens.to(dev), 5))
    is_want(generate.logprobs(logits.to(dev).t().contiguous().t(), tokens.to(dev), 5))
    is_want(generate.logprobs(logits.to(dev).view(3, 4, 1000), tokens.to(dev).view(3, 4), 5))
    is_want(generate.logprobs(logits.to(dev), tokens.to(dev).long(), 5))
    far = tokens.to(dev).long()
    far[3], far[4] = 2 ** 32 + 5, -2 ** 40                                      # outside, also cut to 32 bits
    out = generate.logprobs(logits.to(dev), far, 5)
    assert out.logprob[3].isnan() and out.logprob[4].isnan() and out.rank[3:5].tolist() == [-1, -1]
    one = logits[:1].expand(12, 1000)                                           # the same row again: stride 0
    check(host(generate.logprobs(logits[:1].to(dev).expand(12, 1000), tokens.to(dev), 5)), one, tokens, 5)
    check(host(generate.logprobs(logits.to(dev), None, 5)), logits, None, 5)
    check(host(generate.logprobs(logits.to(dev))), logits, None, 0)
    none = generate.logprobs(logits[:0].to(dev), tokens[:0].to(dev), 5)
    assert none.logprob.shape == (0,) and none.top_ids.shape == (0, 5)


def test_rows_beyond_32_bit_offsets(dev):
    """Two rows 2^32 + 8 values apart."""
    logits, tokens = rows_of(2, 3000, 5, torch.bfloat16)
    far = 2 ** 32 + 8
    buf = torch.empty(far + 3000, dtype=torch.bfloat16, device=dev)
    view = buf.as_strided((2, 3000), (far, 1))
    view.copy_(logits.to(dev))
    check(host(generate.logprobs(view, tokens.to(dev), 5)), logits, tokens, 5)


def test_refusals(dev):
    l, t = torch.zeros(4, 50, device=dev), torch.zeros(4, dtype=torch.int32, device=dev)
    for bad in (lambda: generate.logprobs(l.half(), t), lambda: generate.logprobs(l, t[:3]), lambda: generate.logprobs(l, t, 33),
                lambda: generate.logprobs(l[:, :3], t, 4), lambda: generate.logprobs(l, t, -1),
                lambda: generate.logprobs(l, t.cpu()), lambda: generate.logprobs(l, t.float()),
                lambda: generate.logprobs(l[:, :0], t), lambda: generate.logprobs(l.expand(3, 4, 50), t),
                lambda: generate.logprobs(torch.zeros(1, (1 << 20) + 1, device=dev)),
                lambda: generate.logprobs(torch.zeros((1 << 17) + 1, 2, device=dev))):
        with pytest.raises(ValueError):
            bad()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab", [(1, 4095), (1, 4096), (1, 4097), (2, 8191), (1, 8193), (3, 12296), (1, 131072),
                                        (1, 131073), (40, 65537), (1100, 4095), (1100, 4097), (1100, 8200)])
def test_where_steps_and_chunks_meet(dev, rows, vocab, dtype):
    """Few values, so that equal ones lie on both sides of every boundary; the tokens at the boundaries themselves."""
    g = torch.Generator().manual_seed(vocab)
    logits = torch.randint(0, 5, (rows, vocab), generator=g).to(dtype)
    logits[torch.rand(rows, vocab, generator=g) < 0.01] = -math.inf
    chunks = max(1, min(32, -(-vocab // 4096), 1024 // rows))
    per = -(-(-(-vocab // chunks)) // 8) * 8
    at = [0, vocab - 1, min(per, vocab) - 1, min(per, vocab - 1), min(4095, vocab - 1), min(4096, vocab - 1), vocab // 2]
    logits, some = logits.to(dev), sorted({0, rows - 1, rows // 2})
    for t in at:
        tokens = torch.full((rows,), t, dtype=torch.int32)
        out = host(generate.logprobs(logits, tokens.to(dev), 7))
        check(generate.TokenLogprobs(*(f[some] for f in out)), logits.cpu()[some], tokens[some], 7)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [4008, 5000, 20001])
def test_ranks_of_every_kind_of_token(dev, vocab, dtype):
    """The most likely token, the least likely, forbidden ones, NaN and its neighbours: everywhere in the row, in one row
    and in more rows than are cut into chunks."""
    g = torch.Generator().manual_seed(vocab)
    base = (torch.randn(vocab, generator=g) * 3).to(torch.bfloat16)
    rows, tokens = [], []
    for at in (0, 1, vocab // 2, 4007, vocab - 1):
        for value in (40.0, -40.0, -math.inf, math.nan, math.inf, float(base.max())):
            for other in (None, -math.inf, math.nan):
                r = base.clone()
                if other is not None:
                    r[torch.randint(0, vocab, (20,), generator=g)] = other
                    r[vocab - 1] = other
                r[at] = value
                rows.append(r)
                tokens.append(at)
    logits, tokens = torch.stack(rows).to(dtype), torch.tensor(tokens, dtype=torch.int32)
    check(host(generate.logprobs(logits.to(dev), tokens.to(dev), 3)), logits, tokens, 3)
    for i in range(0, len(rows), 7):
        check(host(generate.logprobs(logits[i].to(dev), tokens[i:i + 1].to(dev), 3)), logits[i:i + 1], tokens[i:i + 1], 3)
    many = torch.cat([logits] * 12)
    out = host(generate.logprobs(many.to(dev), tokens.repeat(12).to(dev), 3))
    check(generate.TokenLogprobs(*(f[-90:] for f in out)), logits, tokens, 3)


def test_results_can_be_saved(dev):
    import io
    lg, tok = rows_of(3, 100, 1, torch.float32)
    for tokens, top in ((tok.to(dev), 5), (tok.to(dev), 0), (None, 5), (None, 0)):
        out = generate.logprobs(lg.to(dev), tokens, top)
        buf = io.BytesIO()
        torch.save(list(out), buf)
        buf.seek(0)
        for a, b in zip(torch.load(buf, weights_only=True), out):
            assert (a is None and b is None) or torch.equal(a, b)


def test_two_streams_at_once(dev):
    lg, tok = rows_of(4, 49152, 1, torch.float32)
    logits, tokens = lg.to(dev), tok.to(dev)
    w = (torch.randn(9001, 256, generator=torch.Generator().manual_seed(2)) * 0.1).to(torch.bfloat16)
    head = quantize.DynamicInt8Linear.from_float(w.to(dev))
    feat = torch.randn(70, 256, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16).to(dev)
    calls = [lambda: generate.logprobs(logits, tokens, 5), lambda: generate.logprobs(logits[:1], tokens[:1], 20),
             lambda: generate.head_logprobs(feat, head.weight, head.scales, None, 8),
             lambda: generate.head_logprobs(feat[:3], head.weight, head.scales, tokens[:3], 8)]
    want = [host(f()) for f in calls]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in calls], []
    for _ in range(3):
        for s, f in zip(streams, calls):
            with torch.cuda.stream(s):
                got.append(f())
    torch.cuda.synchronize()
    for i, out in enumerate(got):
        for a, b in zip(host(out), want[i % len(calls)]):  # NaN: an id outside the smaller vocabulary
            assert (a is None and b is None) or torch.equal(a.nan_to_num(9.0), b.nan_to_num(9.0))


# ---- from features -----------------------------------------------------------------------------------

@pytest.mark.parametrize("m,n,k,top", [(1, 49152, 2560, 5), (8, 49152, 2560, 20), (1, 1000, 64, 3), (33, 1003, 1040, 32),
                                       (130, 5001, 256, 0), (700, 49152, 512, 5)])
def test_head(dev, m, n, k, top):
    g = torch.Generator().manual_seed(m + n)
    w = (torch.randn(n, k, generator=g) * 0.02).to(torch.bfloat16)
    x = torch.randn(m, k, generator=g).to(torch.bfloat16)
    tokens = torch.randint(0, n, (m,), generator=g, dtype=torch.int32)
    head = quantize.DynamicInt8Linear.from_float(w.to(dev))
    head.scales *= 4.0 / (0.02 * math.sqrt(k))
    out = host(generate.head_logprobs(x.to(dev), head.weight, head.scales, tokens.to(dev), top))
    logits = scoring.product(*scoring.quantize_rows(x), head.weight.cpu(), head.scales.cpu())
    some = list(range(m)) if m <= 40 else list(range(0, m, m // 13)) + [m - 1]
    pick = lambda f: None if f is None else f[some]  # noqa: E731
    check(generate.TokenLogprobs(*map(pick, out)), logits[some], tokens[some], top)
    # the same as the product and the log probabilities called one after the other
    y = quantize.linear_int8(x.to(dev), head.weight, head.scales, torch.float32)
    assert torch.equal(y.cpu()[some], logits[some])
    two = host(generate.logprobs(y, tokens.to(dev), top))
    assert torch.equal(two.rank, out.rank) and (top == 0 or torch.equal(two.top_ids, out.top_ids))


@pytest.mark.parametrize("top,given", [(6, True), (0, True), (3, False)])
def test_head_of_more_logits_than_one_block_holds(dev, top, given):
    """600000 logits a row, 111 rows of them in 256 MB: two whole blocks and a last one."""
    m, n, k = 250, 600000, 32
    g = torch.Generator().manual_seed(1)
    w = torch.randint(-128, 128, (n, k), generator=g).to(torch.int8)
    s = torch.rand(n, generator=g) * 1e-3
    x = torch.randn(m, k, generator=g).to(torch.bfloat16)
    tokens = torch.randint(0, n, (m,), generator=g, dtype=torch.int32)
    call = lambda a, b: host(generate.head_logprobs(x[a:b].to(dev), w.to(dev), s.to(dev),  # noqa: E731
                                                    tokens[a:b].to(dev) if given else None, top))
    out = call(0, m)
    some = [0, 110, 111, 221, 222, 249]
    logits = scoring.product(*scoring.quantize_rows(x[some]), w, s)
    pick = lambda f: None if f is None else f[some]  # noqa: E731
    check(generate.TokenLogprobs(*map(pick, out)), logits, tokens[some] if given else None, top)
    for a, b in zip(call(111, 222), out):
        assert a is None or a.dtype != torch.int32 or torch.equal(a, b[111:222])


def test_as_many_rows_as_there_may_be(dev):
    rows, vocab = 1 << 17, 100
    logits = torch.randn(rows, vocab, device=dev)
    tokens = torch.randint(0, vocab, (rows,), dtype=torch.int32, device=dev)
    out = host(generate.logprobs(logits, tokens, 4))
    some = [0, 1, 255, 256, 65536, rows - 1]
    check(generate.TokenLogprobs(*(f[some] for f in out)), logits[some].cpu(), tokens[some].cpu(), 4)


def test_head_refusals_and_shapes(dev):
    w, s = torch.zeros(40, 64, dtype=torch.int8, device=dev), torch.ones(40, device=dev)
    x, t = torch.zeros(6, 64, dtype=torch.bfloat16, device=dev), torch.zeros(6, dtype=torch.int32, device=dev)
    for bad in (lambda: generate.head_logprobs(x.float(), w, s, t), lambda: generate.head_logprobs(x[:, :48], w, s, t),
                lambda: generate.head_logprobs(x, w, s, t[:5]), lambda: generate.head_logprobs(x, w, s, t, 33),
                lambda: generate.head_logprobs(x, w.float(), s, t), lambda: generate.head_logprobs(x, w, s[:3], t)):
        with pytest.raises(ValueError):
            bad()
    out = generate.head_logprobs(x.view(2, 3, 64), w, s, t.view(2, 3).long(), 3)  # all logits 0
    assert out.rank.tolist() == [0] * 6 and out.top_ids.tolist() == [[0, 1, 2]] * 6
    assert generate.head_logprobs(x[:0], w, s, t[:0]).entropy.shape == (0,)
    x = x.clone()
    x[2, 5] = math.nan  # a broken row says so and leaves the others
    out = generate.head_logprobs(x, w, s, t, 3)
    assert out.logprob.isnan().tolist() == [False, False, True, False, False, False]


@pytest.mark.parametrize("rows,vocab", [(1, 49152), (5, 1000), (600, 9001)])
def test_captured_and_replayed(dev, rows, vocab):
    lg, tok = rows_of(rows, vocab, 1, torch.float32)
    logits, tokens = lg.to(dev), tok.to(dev)
    head = quantize.DynamicInt8Linear.from_float((torch.randn(vocab, 64) * 0.1).to(torch.bfloat16).to(dev))
    feat = torch.randn(rows, 64, device=dev).to(torch.bfloat16)
    generate.logprobs(logits, tokens, 5)
    torch.cuda.synchronize()
    g, h = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        a = generate.logprobs(logits, tokens, 5)
    with torch.cuda.graph(h):
        b = generate.head_logprobs(feat, head.weight, head.scales, tokens, 5)
    for seed in range(4):
        logits.copy_(rows_of(rows, vocab, seed + 10, torch.float32)[0])
        feat.copy_(torch.randn(rows, 64, generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16))
        g.replay()
        h.replay()
        g.replay()
        for got, want in zip(a, generate.logprobs(logits, tokens, 5)):
            assert torch.equal(got, want)
        for got, want in zip(b, generate.head_logprobs(feat, head.weight, head.scales, tokens, 5)):
            assert torch.equal(got, want)
        torch.cuda.synchronize()


# ---- as a model's user has them ------------------------------------------------------------------------

@pytest.fixture(scope="module")
def model(dev):
    args = ModelArgs.from_name("tiny")
    args.logits_scaling = 0.25  # logits that spread
    return Transformer.from_weights(args, synth_weights(args, seed=0), "cuda:0")


@pytest.mark.parametrize("n", [2, 3, 33, 34, 100])
def test_score_is_the_log_probabilities_of_the_models_logits(dev, model, n):
    tokens = torch.randint(0, 1024, (n,), generator=torch.Generator().manual_seed(n), dtype=torch.int32).to(dev)
    out = host(generate.score(model, tokens, top=4))
    logits = model.forward(tokens[:-1], 0)[0].float().cpu()  # one decode step per token
    given = torch.log_softmax(logits.double(), -1)[torch.arange(n - 1), tokens[1:].cpu().long()]
    assert out.logprob.shape == (n - 1,) and out.top_ids.shape == (n - 1, 4)
    # exactly those of the verify launches' own logits ...
    for s in range(0, n - 1, 32):
        _, lg, _ = model.verify(tokens[s:min(n - 1, s + 32)], s)
        lg = lg.cpu()
        e = s + lg.shape[0]
        check(generate.TokenLogprobs(*(f[s:e] for f in out)), lg, tokens[s + 1:e + 1].cpu(), 4)
        # ... and of the decode steps', up to what these two differ by: a log probability is a logit less the log of a
        # sum, and neither moves further than the row's furthest logit (2e-5: the fp32 sums, as in check)
        apart = (lg.double() - logits[s:e].double()).abs().amax(1)
        assert bool(((out.logprob[s:e].double() - given[s:e]).abs() <= 2 * apart + 2e-5).all())


@pytest.mark.parametrize("n", [2, 20, 150])
def test_score_through_the_8_bit_head(dev, model, n):
    tokens = torch.randint(0, 1024, (n,), generator=torch.Generator().manual_seed(n), dtype=torch.int32).to(dev)
    head = model.int8_head()
    out = host(generate.score(model, tokens, top=4, head=head))
    feat = model.prefill_features(tokens[:-1], 0)
    logits = scoring.product(*scoring.quantize_rows(feat.cpu()), head.weight.cpu(), head.scales.cpu())
    check(out, logits, tokens[1:].cpu(), 4)
    # the head's own error: a step of 1 / 127 of either row's maximum, K = 512 of them, against the bf16 head
    full = feat.cpu().double() @ model.packed.embed.cpu().double().T / model.config.logits_scaling
    x, w = feat.cpu().double(), model.packed.embed.cpu().double()
    sx, sw = x.abs().amax(1, keepdim=True) / 127, w.abs().amax(1, keepdim=True) / 127
    # |x w - x' w'| <= |x| sw / 2 + |w| sx / 2 + sx sw / 4, a sixty-fourth more for roundings
    bound = (x.abs().sum(1, keepdim=True) @ sw.T / 2 + sx @ w.abs().sum(1, keepdim=True).T / 2 + 512 * sx @ sw.T / 4)
    assert bool(((logits.double() - full).abs() <= bound * (1 + 1 / 64) / model.config.logits_scaling).all())


def test_prompt_features_are_the_models(dev, model):
    tokens = torch.randint(0, 1024, (70,), generator=torch.Generator().manual_seed(5), dtype=torch.int32).to(dev)
    model.setup_caches(1, 100)
    out = torch.empty(1, dtype=torch.int32, device=dev)
    feat = model.prefill_features(tokens, 0, out)
    plain = torch.empty(1, dtype=torch.int32, device=dev)
    k = model.k_cache.clone()
    model.prefill(tokens, 0, plain)
    assert torch.equal(k, model.k_cache) and int(out) == int(plain)
    assert torch.equal(model.prefill_features(tokens, 0), feat)
    _, _, ref = model.verify(tokens[:32], 0)
    d = (feat[:32].float() - ref.float()).norm() / ref.float().norm()
    assert float(d) < 0.02  # two layers, another order of sums


@pytest.mark.parametrize("sampled", [False, True])
def test_generate_with_log_probabilities(dev, model, sampled):
    prompt = torch.randint(0, 1024, (20,), generator=torch.Generator().manual_seed(1), dtype=torch.int32)
    kw = dict(temperature=0.9, top_k=50, seed=3) if sampled else {}
    plain = generate.generate(model, prompt, 8, **kw)
    seq, out = generate.generate(model, prompt, 8, logprobs=4, **kw)
    assert torch.equal(seq, plain)
    assert out.logprob.shape == (8,) and out.top_ids.shape == (8, 4)
    if not sampled:
        assert out.rank.tolist() == [0] * 8 and torch.equal(out.top_ids[:, 0], seq[20:])
        assert torch.equal(out.top_logprobs[:, 0], out.logprob)
    # the same tokens stepped through by hand
    model.setup_caches(1, 28)
    generate.prefill(model, prompt[:-1], 0)
    for i in range(8):
        logits = torch.empty(1024, dtype=torch.float32, device=dev)
        model.decode_step(seq[19 + i:20 + i], 19 + i, logits=logits)
        step = generate.logprobs(logits, seq[20 + i:21 + i], 4)
        for got, want in zip(out, step):
            assert torch.equal(got[i:i + 1], want)
    seq, out = generate.generate(model, prompt, 0, logprobs=2)
    assert len(seq) == 20 and out.logprob.shape == (0,) and out.top_ids.shape == (0, 2)
    with pytest.raises(ValueError):
        generate.generate(model, prompt, 2, logprobs=33)


def test_generate_refuses_log_probabilities_it_has_not(dev, model):
    prompt = torch.tensor([3, 5], dtype=torch.int32, device=dev)
    for n in (-1, 33):
        with pytest.raises(ValueError):
            generate.generate(model, prompt, 2, logprobs=n)
    seq, said = generate.generate(model, prompt, 0, logprobs=2)
    assert seq.tolist() == [3, 5] and said.logprob.shape == (0,) and said.top_ids.shape == (0, 2)


def test_features_of_a_prompt_of_several_passes(dev):
    """2100 tokens, three passes: the same as one call for each, and as the greedy prefill."""
    args = ModelArgs.from_name("tiny")
    args.block_size = 2304
    model = Transformer.from_weights(args, synth_weights(args, seed=0), "cuda:0")
    g = torch.Generator().manual_seed(9)
    tokens = torch.randint(0, model.config.vocab_size, (2100,), generator=g, dtype=torch.int32).to(dev)
    model.setup_caches(1, 2200)
    one, two = (torch.full((1,), -1, dtype=torch.int32, device=dev) for _ in range(2))
    feat = model.prefill_features(tokens, 0, one)
    parts = [model.prefill_features(tokens[:1024], 0), model.prefill_features(tokens[1024:2048], 1024),
             model.prefill_features(tokens[2048:], 2048)]
    assert torch.equal(feat, torch.cat(parts))
    model.prefill(tokens, 0, two)
    assert int(one) == int(two) >= 0
    said = generate.score(model, tokens, 2, model.int8_head())
    head = model.int8_head()
    want = generate.head_logprobs(feat[:-1], head.weight, head.scales, tokens[1:], 2)
    assert all(torch.equal(a, b) for a, b in zip(said, want))


@pytest.mark.parametrize("int8", [False, True])
def test_score_of_a_text_that_fills_the_positions(dev, int8):
    """128 positions, 129 tokens: the last one is only asked for."""
    args = ModelArgs.from_name("tiny")
    args.block_size = 128
    model = Transformer.from_weights(args, synth_weights(args, seed=0), "cuda:0")
    head = model.int8_head() if int8 else None
    tokens = torch.randint(0, args.vocab_size, (129,), generator=torch.Generator().manual_seed(2), dtype=torch.int32).to(dev)
    whole = host(generate.score(model, tokens, 3, head))
    model.check()
    part = host(generate.score(model, tokens[:128], 3, head))
    for a, b in zip(whole, part):
        assert a.shape[0] == 128 and torch.equal(a[:96], b[:96])
    if int8:
        logits = scoring.product(*scoring.quantize_rows(model.prefill_features(tokens[:128], 0).cpu()), head.weight.cpu(),
                                 head.scales.cpu())
    else:
        logits = model.verify(tokens[96:128], 96)[1].cpu()
    check(generate.TokenLogprobs(*(f[-len(logits):] for f in whole)), logits, tokens[-len(logits):].cpu(), 3)
    with pytest.raises(ValueError):
        generate.score(model, torch.cat([tokens, tokens[:1]]), 3, head)


@pytest.mark.parametrize("int8", [False, True])
def test_decoding_goes_on_from_a_scored_text(dev, model, int8):
    """The cache holds the rows of all tokens but the last, which is fed at its own position; the slots from there on are
    left as they were."""
    n = 50
    tokens = torch.randint(0, 1024, (n,), generator=torch.Generator().manual_seed(8), dtype=torch.int32).to(dev)
    model.setup_caches(1, 64)
    model.k_cache.fill_(7.0)
    generate.score(model, tokens, head=model.int8_head() if int8 else None)
    assert bool((model.k_cache[:, :, n - 1:] == 7.0).all()) and not bool((model.k_cache[:, :, :n - 1] == 7.0).all(3).any())
    after = model.decode_step(tokens[-1:], n - 1).clone()
    if int8:  # score's one pass over tokens[:-1], again
        model.prefill_features(tokens[:-1], 0)
    else:
        for s in range(0, n - 1, 32):
            model.verify(tokens[s:min(n - 1, s + 32)], s)
    assert torch.equal(model.decode_step(tokens[-1:], n - 1), after)


def test_score_refuses_before_it_runs(dev, model):
    tokens = torch.zeros(40, dtype=torch.int32, device=dev)
    model.setup_caches(1, 64)
    model.k_cache.fill_(7.0)
    for head in (None, model.int8_head()):
        for top in (-1, 33):
            with pytest.raises(ValueError):
                generate.score(model, tokens, top, head)
    assert bool((model.k_cache == 7.0).all())


def test_score_of_an_id_beyond_32_bits(dev):
    """Asked for last, it is outside the vocabulary; fed, the state says so."""
    model = Transformer.from_weights(ModelArgs.from_name("tiny"), synth_weights(ModelArgs.from_name("tiny"), seed=0), "cuda:0")
    tokens = torch.tensor([3, 4, 5, 2 ** 32 + 6], device=dev)
    for head in (None, model.int8_head()):
        out = generate.score(model, tokens, 2, head)
        model.check()
        assert out.rank.tolist()[2] == -1 and out.logprob.isnan().tolist() == [False, False, True]
    generate.score(model, tokens.flip(0), 2)
    with pytest.raises(_lib.FlError):
        model.check()
    model.reset_state()


def seams(rows, vocab, step=4096, most=32, workgroups=1024):
    """(values of a chunk, chunks) as the launcher cuts a row: chunks of as many whole steps as the largest needs, evenly
    filled in multiples of eight."""
    steps = -(-vocab // step)
    n = max(1, min(most, steps, workgroups // rows))
    n = -(-steps // -(-steps // n))
    per = -(-(-(-vocab // n)) // 8) * 8
    return per, -(-vocab // per)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab,chunks,chunk_steps", [
    (1, 131073, 17, 2), (1, 131072, 32, 1), (1, 400001, 25, 4), (40, 131073, 17, 2), (100, 49152, 6, 2), (128, 49152, 6, 2),
    (200, 49155, 5, 3), (300, 49155, 3, 5), (512, 20001, 2, 3), (1000, 20001, 1, 5)])
def test_tokens_and_ties_at_the_seams_of_chunks_of_several_steps(dev, rows, vocab, chunks, chunk_steps, dtype):
    """Equal values on both sides of every seam of chunks and of steps within them, the largest ones among them, and the
    tokens there."""
    per, n = seams(rows, vocab)
    assert n == chunks and -(-per // 4096) == chunk_steps
    g = torch.Generator().manual_seed(vocab + rows)
    logits = torch.randint(0, 5, (rows, vocab), generator=g).to(dtype)
    logits[torch.rand(rows, vocab, generator=g) < 0.01] = -math.inf
    starts = [c * per for c in range(1, n)]
    inner = [c * per + s * 4096 for c in range(n) for s in range(1, chunk_steps) if c * per + s * 4096 < min(vocab, (c + 1) * per)]
    ends = [min(vocab, (c + 1) * per) for c in range(n)]
    at = [p + d for p in starts + inner for d in (-1, 0)] + [ends[-1] - 1, 0]
    some = sorted({0, rows // 2, rows - 1})
    for r in some[:2]:  # the alternatives lie at the seams, in the order of their indices; the last row has them by chance
        logits[r, at] = 9.0
    logits = logits.to(dev)
    for t in sorted(set(at))[:: max(1, len(set(at)) // 14)] + [starts[0] if starts else 0, per - 1]:
        tokens = torch.full((rows,), t, dtype=torch.int32)
        out = host(generate.logprobs(logits, tokens.to(dev), 11))
        check(generate.TokenLogprobs(*(f[some] for f in out)), logits[some].cpu(), tokens[some], 11)
        assert out.top_ids[0].tolist() == sorted(set(at))[:11] or len(set(at)) < 11

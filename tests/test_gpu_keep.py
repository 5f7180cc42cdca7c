"""The cache operators as the engine runs them: prompts that gather weights, eviction and decoding from what stays,
trees wider than a verify launch, and sampled speculation over all of them."""
import pytest
import torch

from oracle import cache as oracle_cache
from tests.helpers import check_rows, fill_kv_random, log, make_pair, oracle_pair

pytestmark = pytest.mark.gpu


def tokens(args, n, seed):
    return torch.randint(0, args.vocab_size, (n,), generator=torch.Generator().manual_seed(seed), dtype=torch.int32)


@pytest.mark.parametrize("n,pos,window", [(17, 0, None), (40, 30, 7), (300, 100, None), (5, 3, 5), (1, 50, 1)])
def test_weights_of_a_prompt(dev, n, pos, window):
    """Layer 0's weights against 64 bits from the oracle's q and k: q and k are one linear of the same inputs, so single
    bf16 roundings apart (an ulp of one in a few hundred values: below 2^-8 of the score, e^s follows); every layer's
    rows hand out 1 each; a call adds to what is there, and the cache is a plain prompt's."""
    args, sd, eng, orc = make_pair("small", seed=3)
    eng.setup_caches(1, 512)
    orc.setup_caches(eng.max_seq_length)
    if pos:
        fill_kv_random(eng, orc, pos, seed=n)
    x = tokens(args, n, n + pos)
    w = eng.new_weights()
    nxt = torch.empty(1, dtype=torch.int32, device=dev)
    feat = torch.empty(n, args.dim, dtype=torch.bfloat16, device=dev)
    eng.prefill_weights(x.to(dev), pos, w, window, nxt, feat)
    eng.check()
    count = min(window or n, n)
    rep = args.n_head // args.n_local_heads
    assert ((w.double().sum(-1) - count * rep).abs() <= count * rep * 2.0 ** -12).all()
    assert (w[:, :, pos + n:] == 0).all()
    orc.trace = []
    orc.forward(x, pos)
    t = orc.trace[0]
    orc.trace = None
    q = t["q"].view(1, n, args.n_head, 64)[:, n - count:]
    k = orc.k_cache[0][None].clone()
    _, lse = oracle_cache.tree_attention(q, k, k, [pos + n - count], None, args.attn_scale)
    want = oracle_cache.attention_weights(q, k, lse, [pos + n - count], None, args.attn_scale)[0]
    e = float((w[0].double().cpu() - want).norm() / want.norm())
    log(f"weights of {n} tokens at {pos}: rel {e:.2e}")
    assert e <= 2.0 ** -7
    # the same call again adds the same
    before = w.clone()
    eng.prefill_weights(x.to(dev), pos, w, window)
    assert torch.equal(w, before + before)
    # K rows and features as a plain prompt's, up to fp32 order: layer 0's rows are the same linear
    k0 = eng.k_cache.clone()
    if n > 1:
        f2 = eng.prefill_features(x.to(dev), pos)
        assert torch.equal(eng.k_cache[0], k0[0])
        (alt, af), (ref, rf) = oracle_pair(orc, lambda: tuple(v.float() for v in orc.forward(x, pos)))
        d, f = float((feat.float() - f2.float()).norm() / f2.float().norm()), float((af - rf).norm() / rf.norm())
        log(f"features: two attentions {d:.2e} apart, the oracle's implementations {f:.2e}")
        assert d <= max(2 * f, 2.0 ** -8)


def test_window_is_the_rest(dev):
    """All weights = those of the first tokens + those of the window behind them, in two passes or one."""
    args, _, eng, _ = make_pair("small", seed=3)
    eng.setup_caches(1, 1400)
    x = tokens(args, 1300, 5).to(dev)  # two passes: 1024 and 276
    a, b, c = eng.new_weights(), eng.new_weights(), eng.new_weights()
    eng.prefill_weights(x, 0, a)
    eng.prefill_weights(x, 0, b, window=900)  # begins inside the first pass
    eng.prefill_weights(x[:400], 0, c)
    # the same rows; their K and V went through products of other shapes (1024 tokens against 400), a few roundings apart
    rel = float((a - b - c).norm() / a.norm())
    log(f"window: rel {rel:.2e}")
    assert rel <= 2.0 ** -8
    d = eng.new_weights()
    eng.prefill_weights(x, 0, d, window=10 ** 6)
    assert torch.equal(a, d)


@pytest.mark.parametrize("n,keep,recent,sink", [(60, 20, 8, 2), (200, 199, 0, 0), (333, 64, 64, 0)])
def test_decode_after_eviction(dev, n, keep, recent, sink):
    """What stays is what the definition keeps, and decode, verify, prompt and sampling go on from it at the old
    positions: the oracle on the same cut cache, its RoPE positions shifted."""
    args, sd, eng, orc = make_pair("small", seed=3)
    eng.setup_caches(1, 512)
    orc.setup_caches(eng.max_seq_length)
    x = tokens(args, n + 40, n)
    w = eng.new_weights()
    eng.prefill_weights(x[:n].to(dev), 0, w)
    k, v, wc = eng.k_cache.cpu(), eng.v_cache.cpu(), w.cpu()
    kept = eng.evict(w, n, keep, recent, sink)
    assert eng.shift == n - keep
    for l in range(args.n_layer):
        for g in range(args.n_local_heads):
            want = oracle_cache.kept_slots(wc[l, g].tolist(), n, keep, recent, sink)
            assert kept[l, g].tolist() == want
            assert torch.equal(eng.k_cache[l, g, :keep].cpu(), k[l, g, want]) and torch.equal(eng.v_cache[l, g, :keep].cpu(), v[l, g, want])
            assert torch.equal(w[l, g, :keep].cpu(), wc[l, g, want]) and (w[l, g, keep:] == 0).all()
    orc.k_cache.copy_(eng.k_cache.cpu())
    orc.v_cache.copy_(eng.v_cache.cpu())

    def orc_run(idx, slot):
        m = idx.numel()
        return oracle_pair(orc, lambda: (orc.forward(idx, slot, depth=torch.arange(m) + eng.shift)[0].float(),))
    # decode, then a verify of 3, a prompt of 30, at slots keep ..
    lg = torch.empty(args.vocab_size, dtype=torch.float32, device=dev)
    eng.decode_step(x[n:n + 1].to(dev), keep, logits=lg)
    (alt,), (ref,) = orc_run(x[n:n + 1], keep)
    check_rows(lg.cpu().view(1, -1), ref, alt, "small", f"decode after eviction {n} -> {keep}")
    _, vl, _ = eng.verify(x[n + 1:n + 4].to(dev), keep + 1)
    (alt,), (ref,) = orc_run(x[n + 1:n + 4], keep + 1)
    check_rows(vl.cpu(), ref, alt, "small", "verify after eviction")
    from flint_amd.generate import prefill
    prefill(eng, x[n + 4:n + 34], keep + 4)
    eng.decode_step(x[n + 34:n + 35].to(dev), keep + 34, logits=lg)
    (alt,), (ref,) = orc_run(x[n + 4:n + 35], keep + 4)
    check_rows(lg.cpu().view(1, -1), ref[-1:], alt[-1:], "small", "prompt after eviction")
    eng.check()
    # a second cut, then a fresh start
    eng.evict(w, keep + 35, 10, 0, 0)
    assert eng.shift == n - keep + keep + 35 - 10
    eng.setup_caches(1, 512)
    assert eng.shift == 0
    orc.setup_caches(eng.max_seq_length)
    eng.decode_step(x[:1].to(dev), 0, logits=lg)
    check_rows(lg.cpu().view(1, -1), orc.forward(x[:1], 0)[0].float(), orc.forward(x[:1], 0)[0].float(), "small", "fresh start")


def test_nothing_evicted_changes_nothing(dev):
    args, _, eng, _ = make_pair("small", seed=3)
    eng.setup_caches(1, 256)
    x = tokens(args, 50, 1).to(dev)
    w = eng.new_weights()
    eng.prefill_weights(x, 0, w)
    k, w0 = eng.k_cache.clone(), w.clone()
    eng.evict(w, 50, 50)
    eng.evict(w, 50, 80, 10, 10)
    assert eng.shift == 0 and torch.equal(eng.k_cache, k) and torch.equal(w, w0)


def test_positions_end_at_the_table(dev):
    from flint_amd import _lib
    args, _, eng, _ = make_pair("tiny", seed=3)  # 1024 positions
    eng.setup_caches(1, 1024)
    x = tokens(args, 1020, 1).to(dev)
    w = eng.new_weights()
    eng.prefill_weights(x, 0, w)
    eng.evict(w, 1020, 100, 10)
    for i in range(4):  # positions 1020 .. 1023 at slots 100 .. 103
        eng.decode_step(x[:1], 100 + i)
    with pytest.raises(_lib.FlError):
        eng.decode_step(x[:1], 104)
    with pytest.raises(_lib.FlError):
        eng.prefill_weights(x[:5], 100, w)
    eng.check()


def test_generate_keep(dev):
    """generate(keep=...) is prefill_weights and evict pass by pass, then decoding; keep of the prompt or more is none."""
    from flint_amd.generate import generate
    args, _, eng, _ = make_pair("small", seed=3)
    x = tokens(args, 1500, 9).to(dev)
    full = generate(eng, x[:200], 20)
    assert torch.equal(generate(eng, x[:200], 20, keep=199), full) and torch.equal(generate(eng, x[:200], 20, keep=1000), full)
    for kw in (dict(), dict(temperature=0.8, top_k=50, seed=3), dict(logprobs=2)):
        got = generate(eng, x, 12, keep=150, recent=40, sink=2, **kw)
        seq, said = got if "logprobs" in kw else (got, None)
        assert eng.shift == 1499 - 150
        eng.setup_caches(1, 150 + 1024 + 13)
        w = eng.new_weights()
        eng.prefill_weights(x[:1024], 0, w)
        eng.evict(w, 1024, 150, 40, 2)
        eng.prefill_weights(x[1024:1499], 150, w)
        eng.evict(w, 625, 150, 40, 2)
        tok = torch.empty(13, dtype=torch.int32, device=dev)
        tok[:1] = x[1499:]
        for i in range(12):
            if "temperature" in kw:
                eng.decode_sample(tok[i:i + 1], 150 + i, 0.8, 50, seed=3, offset=1499 + i, token_out=tok[i + 1:i + 2])
            else:
                eng.decode_step(tok[i:i + 1], 150 + i, token_out=tok[i + 1:i + 2])
        assert torch.equal(seq[:1500], x) and torch.equal(seq[1500:], tok[1:])
        assert said is None or said.logprob.shape == (12,)
    eng.check()
    for kw in (dict(keep=0), dict(keep=50, recent=50), dict(keep=100, recent=-1)):
        with pytest.raises(ValueError):
            generate(eng, x, 4, **kw)
    with pytest.raises(ValueError):
        generate(eng, tokens(args, 2048, 1), 4, keep=100)


def tree(m, seed):
    from flint_amd.spec import tree_depths, tree_mask
    g = torch.Generator().manual_seed(seed)
    parents = [-1] + [int(torch.randint(max(0, i - 6), i, (1,), generator=g)) for i in range(1, m)]
    return parents, torch.tensor(tree_depths(parents), dtype=torch.int32), torch.from_numpy(tree_mask(parents))


@pytest.mark.parametrize("m,pos", [(1, 20), (20, 0), (33, 100), (130, 37), (300, 10)])
def test_tree_features(dev, m, pos):
    """A tree in a prompt pass: the oracle's logits of its nodes, from the features."""
    args, sd, eng, orc = make_pair("small", seed=3)
    eng.setup_caches(1, 512)
    orc.setup_caches(eng.max_seq_length)
    if pos:
        fill_kv_random(eng, orc, pos, seed=m)
    x = tokens(args, m, m)
    _, depth, mask = tree(m, m)
    feat = eng.tree_features(x.to(dev), pos, depth.to(dev), mask.to(dev))
    eng.check()
    (alt, af), (ref, rf) = oracle_pair(orc, lambda: tuple(v.float() for v in orc.forward(x, pos, depth, mask)))
    lg = (torch.nn.functional.linear(feat.cpu(), orc.embed) / args.logits_scaling).float()
    check_rows(lg, ref, alt, "small", f"tree of {m} at {pos}")


def test_tree_refusals(dev):
    from flint_amd import _lib
    args, _, eng, _ = make_pair("tiny", seed=3)
    with pytest.raises(RuntimeError):
        eng.tree_features(torch.zeros(2, dtype=torch.int32, device=dev), 0, torch.zeros(2), torch.ones(2, 2))
    eng.setup_caches(1, 64)
    x = tokens(args, 40, 1).to(dev)
    _, depth, mask = tree(40, 1)
    for bad in (dict(depth=depth[:5]), dict(amask=mask[:5]), dict(tokens=x.long()), dict(tokens=x.cpu())):
        with pytest.raises(ValueError):
            eng.tree_features(**{**dict(tokens=x, pos=0, depth=depth, amask=mask), **bad})
    with pytest.raises(_lib.FlError):
        eng.tree_features(x, 30, depth, mask)
    w = eng.new_weights()
    for bad in (dict(weights=w[:1]), dict(weights=w.double()), dict(window=0), dict(token_out=torch.zeros(2, dtype=torch.int32, device=dev)),
                dict(feat=torch.zeros(40, args.dim, device=dev))):
        with pytest.raises(ValueError):
            eng.prefill_weights(**{**dict(tokens=x, pos=0, weights=w), **bad})
    with pytest.raises(ValueError):
        eng.evict(w, 100, 10)
    # a depth outside the RoPE table is recorded, as verify's
    depth = depth.clone()
    depth[3] = 5000
    eng.tree_features(x, 0, depth.to(dev), mask.to(dev))
    with pytest.raises(_lib.FlError):
        eng.check()
    eng.reset_state()


class Proposes:
    """A draft that draws every child from a distribution of its own, `branch` children per node, two levels."""

    def __init__(self, vocab, device, branch, seed=0, tell=True):
        g = torch.Generator(device=device).manual_seed(seed)
        self.q = torch.softmax(torch.randn(vocab, generator=g, device=device) * 2, 0)
        self.g, self.branch, self.tell, self.n = g, branch, tell, 0

    def chain(self, context, feats, k):
        self.n = min(k, 3)
        return torch.multinomial(self.q, self.n, replacement=True, generator=self.g).tolist() if self.n else []

    def tree(self, context, feats):
        b = self.branch
        parents = [-1] * b + [i // b for i in range(b * b)]
        self.n = len(parents)
        return torch.multinomial(self.q, self.n, replacement=True, generator=self.g).tolist(), parents

    def probs(self):
        return self.q.expand(self.n, -1) if self.tell else None


@pytest.mark.parametrize("mode,tell", [("chain", True), ("tree", True), ("chain", False)])
def test_sampled_speculation_is_the_samplers_distribution(dev, mode, tell):
    """The first two tokens of 600 runs against the sampler's own probabilities (top-k 3: nine pairs). A draft
    that tells its distribution draws tokens anew each run; one that does not proposes the same ones always. Five standard
    deviations of a count."""
    from flint_amd.generate import logits_to_probs, prefill
    from flint_amd.spec import SpecDecoder
    args, _, eng, _ = make_pair("tiny", seed=3)
    p0 = tokens(args, 6, 3).tolist()
    eng.setup_caches(1, 64)
    prefill(eng, torch.tensor(p0[:-1], dtype=torch.int32), 0)
    lg = torch.empty(args.vocab_size, dtype=torch.float32, device=dev)
    eng.decode_step(torch.tensor(p0[-1:], dtype=torch.int32, device=dev), len(p0) - 1, logits=lg)
    first = logits_to_probs(lg, 1.5, 3).cpu()
    want = {}
    for a in first.nonzero()[:, 0].tolist():
        eng.decode_step(torch.tensor([a], dtype=torch.int32, device=dev), len(p0), logits=lg)
        second = logits_to_probs(lg, 1.5, 3).cpu()
        for b in second.nonzero()[:, 0].tolist():
            want[a, b] = float(first[a] * second[b])
    draft = Proposes(args.vocab_size, dev, 2, tell=tell)
    draft.q = torch.zeros_like(draft.q)
    draft.q[[a for a, _ in want] + [b for _, b in want]] = 1.0  # so that some are accepted
    draft.q /= draft.q.sum()
    if not tell:
        fixed = [b for _, b in want][:3]
        draft.chain = lambda context, feats, k: fixed[:k]
    dec = SpecDecoder(eng, draft=draft, k=3)
    n, count, accepted = 600, dict.fromkeys(want, 0), 0
    for seed in range(n):
        out, stats = dec.generate(p0, 3, mode=mode, temperature=1.5, top_k=3, seed=seed)
        count[tuple(out[6:8])] += 1
        accepted += stats.tokens - stats.passes
    total = sum(want.values())  # bf16 probabilities: not quite 1
    for pair, p in want.items():
        p /= total
        # probabilities are bf16 and the verify kernel's logits a rounding off the decode kernel's: 2 % of p
        assert abs(count[pair] - n * p) <= 5 * (n * p * (1 - p)) ** 0.5 + 0.02 * n * p + 1, (pair, count, want)
    log(f"{mode}: {accepted} of {n} runs' tokens were accepted drafts")
    assert accepted > 0


def test_top_k_1_is_greedy(dev):
    """One candidate: the sampled loop emits the greedy loop's tokens (equal largest logits stay candidates: none here)."""
    from flint_amd.spec import LookupDraft, SpecDecoder
    args, _, eng, _ = make_pair("small", seed=3)
    p0 = (tokens(args, 12, 4).tolist() * 3)[:30]
    for mode in ("chain", "tree"):
        greedy, _ = SpecDecoder(eng, k=4).generate(p0, 24, mode=mode)
        sampled, _ = SpecDecoder(eng, k=4).generate(p0, 24, mode=mode, top_k=1, seed=7)
        again, _ = SpecDecoder(eng, k=4).generate(p0, 24, mode=mode, top_k=1, temperature=0.3, seed=8)
        same = next((i for i in range(len(greedy)) if greedy[i] != sampled[i]), len(greedy))
        log(f"{mode}: sampled and greedy agree for {same} of {len(greedy)}")
        assert sampled == again or same >= 30
        assert same >= 34
    assert LookupDraft().max_nodes == 32
    with pytest.raises(ValueError):
        SpecDecoder(eng).generate(p0, 4, top_k=0)


def test_wide_trees(dev):
    """Trees of more than 32 nodes through the prompt pass and the 8-bit head: repeatable, and as many tokens as asked for."""
    from flint_amd.spec import LookupDraft, SpecDecoder
    args, _, eng, _ = make_pair("small", seed=3)
    eng.setup_caches(1, 8)
    head = eng.int8_head()

    class Wide:
        def tree(self, context, feats):
            t = [(context[-1] * 7 + i * 13) % args.vocab_size for i in range(70)]
            return t, [-1] * 5 + [i // 5 for i in range(65)]
    for draft in (Wide(), LookupDraft(width=8, depth=10)):
        dec = SpecDecoder(eng, draft=draft, head=head)
        p0 = (tokens(args, 9, 4).tolist() * 4)[:33]
        for kw in (dict(), dict(temperature=0.9, seed=5)):
            a, sa = dec.generate(p0, 15, mode="tree", **kw)
            b, sb = dec.generate(p0, 15, mode="tree", **kw)
            assert a == b and len(a) >= 33 + 15 and a[:33] == p0
    eng.check()
    with pytest.raises(ValueError):
        SpecDecoder(eng, k=32)
    assert SpecDecoder(eng, k=100, head=head).k == 100


def test_workspace_covers_every_position(dev):
    """A prompt pass that gathers weights asks for a workspace before it knows how many keys are cached: enough for all."""
    from flint_amd import _lib
    args, _, eng, _ = make_pair("small", seed=3, block_size=16384)
    for slots in (64, 2048, 16384):
        eng.close()
        eng.max_seq_length = -1
        eng.setup_caches(1, slots)
        for m in (1, 2, 5, 12, 13, 40, 64, 200, 1024, 1025, 1100):
            if m > slots:
                continue
            plain, extra, need = (_lib.ctypes.c_int64() for _ in range(3))
            _lib.call("fl_prefill_workspace", eng._state, m, _lib.ctypes.byref(plain))
            _lib.call("fl_prefill_extra_workspace", eng._state, m, _lib.ctypes.byref(extra))
            room = extra.value - plain.value - min(m, 1024) * args.n_head * 4
            for t in {min(m, 1024), m % 1024 or min(m, 1024)}:
                d = _lib.AttnDesc(b=1, m=t, heads=args.n_head, groups=args.n_local_heads, dim=64, slots=slots, scale=0.125,
                                  q_m=args.n_head * 64, q_h=64, k_g=slots * 64, k_s=64, v_g=slots * 64, v_s=64)
                for pos in {0, 1, 500, 700, 1000, 1500, 2000, 4000, 8000, 11000, 12000, 12300, 14000, slots - t}:
                    if pos <= slots - t:
                        d.pos0 = pos
                        _lib.call("fl_tree_attention_workspace", _lib.ctypes.byref(d), 1, _lib.ctypes.byref(need))
                        assert need.value <= room, (slots, m, t, pos)


@pytest.mark.parametrize("pos", [3000, 11000, 15000])
def test_short_prompt_far_into_the_cache(dev, pos):
    """A few tokens behind many: the weights sum to the rows and the features are a plain prompt's."""
    args, _, eng, _ = make_pair("small", seed=3, block_size=16384)
    eng.setup_caches(1, 16384)
    g = torch.Generator(device=dev).manual_seed(pos)
    for c in (eng.k_cache, eng.v_cache):
        c[:, :, :pos].copy_(torch.randn(c[:, :, :pos].shape, generator=g, device=dev) * 0.5)
    x = tokens(args, 12, 3).to(dev)
    w = eng.new_weights()
    feat = torch.empty(12, args.dim, dtype=torch.bfloat16, device=dev)
    eng.prefill_weights(x, pos, w, feat=feat)
    rep = args.n_head // args.n_local_heads
    assert ((w.double().sum(-1) - 12 * rep).abs() <= 12 * rep * 2.0 ** -10).all()
    plain = eng.prefill_features(x, pos)
    assert float((feat.float() - plain.float()).norm() / plain.float().norm()) <= 2.0 ** -6
    eng.check()


def test_noise_counts_positions(dev):
    """decode_sample's default counter is the token's position, also where eviction has made slots and positions differ:
    the same slot again, at another position, has other noise."""
    args, _, eng, _ = make_pair("small", seed=3)
    eng.setup_caches(1, 256)
    x = tokens(args, 100, 1).to(dev)
    w = eng.new_weights()
    eng.prefill_weights(x, 0, w)
    out = torch.empty(2, dtype=torch.int32, device=dev)
    lg = torch.empty(args.vocab_size, dtype=torch.float32, device=dev)

    def both(slot, position, seed):
        eng.decode_sample(x[:1], slot, 50.0, None, seed=seed, token_out=out[:1], logits=lg)  # nearly flat: noise decides
        eng.decode_sample(x[:1], slot, 50.0, None, seed=seed, offset=position, token_out=out[1:])
        return out.tolist()
    for seed in range(8):
        a, b = both(100, 100, seed)
        assert a == b
    eng.evict(w, 100, 30, 4, 2)
    slots = 0
    from flint_amd.generate import decode_one_token
    for seed in range(8):
        a, b = both(30, 100, seed)
        assert a == b == int(decode_one_token(eng, x[:1], 30, temperature=50.0, seed=seed)[0])
        eng.decode_sample(x[:1], 30, 50.0, None, seed=seed, offset=30, token_out=out[:1])
        slots += int(out[0]) == a
    assert slots < 8
    eng.check()


def test_more_slots_than_positions_are_refused_whole(dev):
    """An eviction whose slots would lie behind the RoPE table is refused before a row moves."""
    args, _, eng, _ = make_pair("tiny", seed=3)  # 1024 positions
    eng.setup_caches(1, 1024)
    x = tokens(args, 1020, 1).to(dev)
    w = eng.new_weights()
    eng.prefill_weights(x, 0, w)
    eng.evict(w, 1020, 100, 10)
    assert eng.shift == 920
    k, v, w0 = eng.k_cache.clone(), eng.v_cache.clone(), w.clone()
    for n in (105, 1024):
        with pytest.raises(ValueError):
            eng.evict(w, n, 50, 10)
        assert eng.shift == 920 and torch.equal(eng.k_cache, k) and torch.equal(eng.v_cache, v) and torch.equal(w, w0)
    eng.evict(w, 104, 50, 10)
    assert eng.shift == 974


def leads(eng, text, tok):
    """How far the largest logit behind `text` lies before that of `tok` (0: it is a largest one)."""
    from flint_amd.generate import prefill
    lg = torch.empty(eng.config.vocab_size, dtype=torch.float32, device=eng.device)
    prefill(eng, torch.tensor(text[:-1], dtype=torch.int32), 0)
    eng.decode_step(torch.tensor(text[-1:], dtype=torch.int32, device=eng.device), len(text) - 1, logits=lg)
    return float(lg.max() - lg[tok])


@pytest.mark.parametrize("mode", ["chain", "tree"])
def test_top_k_1_at_any_temperature(dev, mode):
    """One candidate: whatever the temperature and the seed, each run is the greedy loop's up to a place where two logits
    are equal, or an ulp of bf16 apart (the decode kernel's logits against the verify kernel's)."""
    from flint_amd.spec import SpecDecoder
    args, _, eng, _ = make_pair("small", seed=3)
    p0 = (tokens(args, 12, 4).tolist() * 3)[:30]
    greedy, _ = SpecDecoder(eng, k=4).generate(p0, 24, mode=mode)
    runs = [greedy] + [SpecDecoder(eng, k=4).generate(p0, 24, mode=mode, top_k=1, temperature=t, seed=s)[0] for t, s in ((1.0, 7), (0.3, 8), (2.0, 9))]
    assert len(greedy) >= 54
    for run in runs[1:]:
        at = next((i for i in range(54) if greedy[i] != run[i]), None)
        log(f"{mode}: agree for {'all' if at is None else at}")
        if at is not None:
            gap = [leads(eng, greedy[:at], t) for t in (greedy[at], run[at])]
            assert max(gap) <= 2.0 ** -7 * 8, gap  # logits below 8 here: two roundings to bf16


class Interleaved:
    """Proposes the text's own continuation, every node of it behind one that is no part of the text."""

    def __init__(self, text, vocab, depth):
        self.text, self.vocab, self.depth, self.at = text, vocab, depth, []

    def tree(self, context, feats):
        n = len(context)
        self.at.append(n)
        if list(context) != self.text[:n]:
            return [], []
        toks, pars, last = [], [], -1
        for t in self.text[n:n + self.depth]:
            toks += [(t + 1) % self.vocab, t]
            pars += [last, last]
            last = len(toks) - 1
        return toks, pars


class Junk:
    def __init__(self, vocab):
        self.vocab = vocab

    def tree(self, context, feats):
        return [(context[-1] + 1 + i) % self.vocab for i in range(40)], [-1] * 40


def test_wide_trees_of_the_right_tokens(dev):
    """A path of some forty nodes that are no prefix of the tree: the tokens are those that the 8-bit head puts first
    behind the emitted text, and the cache rows those of that text."""
    from flint_amd.quantize import linear_int8
    from flint_amd.spec import SpecDecoder
    args, _, eng, _ = make_pair("small", seed=3)
    eng.setup_caches(1, 8)
    head = eng.int8_head()
    p0 = tokens(args, 20, 6).tolist()
    text, slow = SpecDecoder(eng, draft=Junk(args.vocab_size), head=head).generate(p0, 60, mode="tree")
    text = text[:80]
    draft = Interleaved(text, args.vocab_size, 45)
    out, fast = SpecDecoder(eng, draft=draft, head=head).generate(p0, 60, mode="tree")
    got = out[:80]
    log(f"{slow.passes} and {fast.passes} passes; agree for {next((i for i in range(80) if got[i] != text[i]), 80)} of 80")
    assert max(b - a for a, b in zip(draft.at, draft.at[1:])) > 33  # a path that is moved in two pieces
    n = 79
    k = eng.k_cache[:, :, :n].clone()
    feat = eng.prefill_features(torch.tensor(got[:n], dtype=torch.int32, device=dev), 0)
    lg = linear_int8(feat, head.weight, head.scales, torch.float32)
    top = lg.max(dim=1).values
    said = lg[torch.arange(19, n), torch.tensor(got[20:], device=dev)]
    # the same rows through products of other shapes: features some bf16 roundings apart
    size = float(lg.abs().max())
    assert (top[19:] - said <= 2.0 ** -5 * size).all(), (top[19:] - said).max()
    assert (lg[19:].argmax(1).tolist() == got[20:]) or int((top[19:] - said > 0).sum()) <= 6
    ref = eng.k_cache[:, :, :n].float()
    rel = ((k.float() - ref).square().sum((0, 1, 3)) / ref.square().sum((0, 1, 3))).sqrt()  # of each slot
    log(f"rows of the cache: worst slot {float(rel.max()):.2e} off")
    assert (rel[20:n] <= 2.0 ** -4).all()
    eng.check()

"""Verification of drafted tokens against the target's probabilities: equal to the definition, token for token."""
import math

import numpy as np
import pytest
import torch

from oracle import cache as oracle

pytestmark = pytest.mark.gpu


def make(b, m, v, seed, tree=True, draft=True, dtype=torch.float32, close=0.5):
    """(p, q, tokens, parents, accept_u, sample_u) on the CPU: a draft that is near the target."""
    g = torch.Generator().manual_seed(seed)
    l = torch.randn(b, m, v, generator=g) * 2
    p = torch.softmax(l, -1).to(dtype)
    q = torch.softmax(l[:, :m - 1] + close * torch.randn(b, m - 1, v, generator=g), -1).to(dtype) if m > 1 else torch.zeros(b, 0, v, dtype=dtype)
    parents = torch.full((b, m), -1, dtype=torch.int32)
    tokens = torch.zeros(b, m, dtype=torch.int32)
    for s in range(b):
        for i in range(1, m):
            parents[s, i] = int(torch.randint(max(0, i - 4), i, (1,), generator=g)) if tree else i - 1
            tokens[s, i] = int(torch.multinomial(q[s, parents[s, i]].float(), 1, generator=g))
    return (p, q if draft else None, tokens, parents if tree else None, torch.rand(b, m, generator=g), torch.rand(b, generator=g))


def check(args, dev):
    from flint_amd.spec import accept_sampled
    p, q, tokens, parents, ua, us = args
    on = lambda t: None if t is None else t.to(dev)  # noqa: E731
    got = accept_sampled(on(p), on(tokens), on(ua), on(us), on(parents), on(q))
    for s in range(p.shape[0]):
        path, token = oracle.accept(p[s].double().tolist(), None if q is None else q[s].double().tolist(), tokens[s].tolist(),
                                    None if parents is None else parents[s].tolist(), ua[s].tolist(), float(us[s]))
        assert got.path[s].tolist() == path + [-1] * (p.shape[1] - len(path))
        assert int(got.count[s]) == len(path) and int(got.token[s]) == token
    return got


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("draft", [True, False])
@pytest.mark.parametrize("tree", [True, False])
@pytest.mark.parametrize("b,m,v", [(1, 1, 1), (1, 2, 5), (3, 5, 100), (16, 9, 1003), (2, 32, 4096), (40, 6, 64), (5, 3, 17000), (1, 70, 300), (2, 4, 65537)])
def test_accept(dev, b, m, v, tree, draft, dtype):
    check(make(b, m, v, seed=m * v + b, tree=tree, draft=draft, dtype=dtype), dev)


def test_border_numbers(dev):
    """u of 0 and of just under 1; tokens of probability 0; rows that are all on one token; p equal to q."""
    for u in (0.0, 1.0 - 2.0 ** -24):
        for draft in (True, False):
            p, q, tokens, parents, ua, us = make(8, 6, 50, 3, draft=draft)
            p[0, 0] = 0
            p[0, 0, 7] = 1.0
            p[1, :, 3:] = 0
            p[2, 0, int(tokens[2, 1])] = 0
            if draft:
                q[3] = p[3, :-1]
                q[4, 0, int(tokens[4, 1])] = 0
            tokens[5, 1:] = 7  # the same token again and again
            ua[:], us[:] = u, u
            check((p, q, tokens, parents, ua, us), dev)


def test_rows_without_a_distribution(dev):
    p, q, tokens, parents, ua, us = make(6, 4, 40, 5)
    p[0] = 0
    p[1] = math.nan
    p[2, :, 4] = math.inf
    p[3, :, ::2] = -1.0
    p[4, :, ::3] = math.nan
    q[5] = 1.0
    got = check((p, q, tokens, parents, ua, us), dev)
    assert got.token[:3].tolist() == [-1, -1, -1] and int(got.token[4]) >= 0


def test_padding_and_strange_trees(dev):
    """Padded nodes, tokens outside the vocabulary, parents that are no earlier node, 64-bit ids."""
    p, q, tokens, parents, ua, us = make(6, 8, 30, 7)
    ua[:] = 0.0
    parents[0, 3:] = -1
    tokens[1, 1:3] = torch.tensor([30, -5], dtype=torch.int32)
    parents[2, 4], parents[2, 5] = 4, 7
    parents[3, 0] = 5
    parents[4, 1:] = -1
    check((p, q, tokens, parents, ua, us), dev)
    tokens, parents = tokens.long(), parents.long()
    tokens[5, 1], parents[5, 2] = 2 ** 32, -2 ** 40
    from flint_amd.spec import accept_sampled
    got = accept_sampled(p.to(dev), tokens.to(dev), ua.to(dev), us.to(dev), parents.to(dev), q.to(dev))
    path, token = oracle.accept(p[5].double().tolist(), q[5].double().tolist(), tokens[5].tolist(), parents[5].tolist(), ua[5].tolist(), float(us[5]))
    assert got.path[5].tolist()[:len(path)] == path and int(got.token[5]) == token


@pytest.mark.parametrize("draft", [True, False])
def test_distribution(dev, draft):
    """The first token that comes out, drafted or drawn, is distributed as the target's row: 200000 trees of three
    children; a count of n p differs from its mean by five standard deviations once in 10^6."""
    from flint_amd.spec import accept_sampled
    n, v, m = 200000, 12, 4
    g = torch.Generator(device=dev).manual_seed(1)
    p0 = torch.softmax(torch.randn(v, generator=g, device=dev) * 1.5, 0)
    q0 = torch.softmax(torch.randn(v, generator=g, device=dev) * 1.5, 0)
    p, q = p0.expand(1, m, v), q0.expand(1, m - 1, v)
    parents = torch.tensor([-1, 0, 0, 0], dtype=torch.int32, device=dev)
    counts = torch.zeros(v, device=dev, dtype=torch.long)
    done = 0
    while done < n:
        b = 50000
        tok = torch.zeros(b, m, dtype=torch.int32, device=dev)
        tok[:, 1:] = torch.multinomial(q0.expand(b, v), m - 1, replacement=True, generator=g).int() if draft else \
            q0.topk(m - 1).indices.int()
        got = accept_sampled(p.expand(b, m, v).contiguous(), tok, torch.rand(b, m, generator=g, device=dev),
                             torch.rand(b, generator=g, device=dev), parents.expand(b, m).contiguous(),
                             q.expand(b, m - 1, v).contiguous() if draft else None)
        first = torch.where(got.count > 1, tok.gather(1, got.path[:, 1:2].clamp(min=0).long())[:, 0], got.token)
        counts += torch.bincount(first.long(), minlength=v)
        done += b
    mean = p0.double() * done
    assert ((counts - mean).abs() <= 5 * (mean * (1 - p0.double())).sqrt() + 1).all(), (counts.tolist(), mean.tolist())


def test_one_tree_without_a_batch(dev):
    from flint_amd.spec import accept_sampled
    p, q, tokens, parents, ua, us = (x.to(dev) for x in make(1, 6, 90, 11))
    a = accept_sampled(p, tokens, ua, us, parents, q)
    b = accept_sampled(p[0], tokens[0], ua[0], us, parents[0], q[0])
    assert b.path.shape == (6,) and torch.equal(b.path, a.path[0]) and torch.equal(b.count, a.count) and torch.equal(b.token, a.token)
    assert accept_sampled(p[:0], tokens[:0], ua[:0], us[:0]).path.shape == (0, 6)
    t = p.transpose(1, 2).contiguous().transpose(1, 2)  # strided rows
    assert torch.equal(accept_sampled(t, tokens, ua, us, parents, q).path, a.path)
    assert np.array_equal(accept_sampled(p, tokens, ua, us, parents, q).token.cpu().numpy(), a.token.cpu().numpy())


def test_refusals(dev):
    from flint_amd.spec import accept_sampled
    p, q, tokens, parents, ua, us = (x.to(dev) for x in make(2, 4, 20, 1))
    ok = dict(probs=p, tokens=tokens, accept_u=ua, sample_u=us, parents=parents, draft_probs=q)
    for kw in (dict(probs=p.half()), dict(probs=p[..., None]), dict(tokens=tokens.float()), dict(tokens=tokens[:, :3]), dict(tokens=tokens.cpu()),
               dict(parents=parents[:1]), dict(accept_u=ua.double()), dict(accept_u=ua[:1]), dict(sample_u=us[:1]), dict(sample_u=us.cpu()),
               dict(draft_probs=q.bfloat16()), dict(draft_probs=p), dict(probs=torch.zeros(1, 1025, 4, device=dev)), dict(probs=p[..., :0])):
        with pytest.raises(ValueError):
            accept_sampled(**{**ok, **kw})


def test_captured_and_replayed(dev):
    from flint_amd.spec import accept_sampled
    ins = [[x.to(dev) for x in make(5, 9, 700, seed)] for seed in range(3)]
    held = [x.clone() for x in ins[0]]

    def call(x):
        return accept_sampled(x[0], x[2], x[4], x[5], x[3], x[1])
    want = [[y.clone() for y in call(x)] for x in ins]
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        got = call(held)
    for i in (0, 1, 2, 0, 2):
        for h, x in zip(held, ins[i]):
            h.copy_(x)
        gr.replay()
        call(ins[(i + 1) % 3])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want[i]))


@pytest.mark.parametrize("v", [15, 16, 17, 1023, 1024, 1025, 16384, 16385, 262145])
@pytest.mark.parametrize("where", ["first", "last", "seam"])
def test_weight_in_one_place(dev, v, where):
    """All of a row's weight in one or two indices, at the seams of the waves' pieces: the last token is one of them."""
    from flint_amd.spec import accept_sampled
    seg = -(-(-(-v // 16)) // 64) * 64
    at = {"first": 0, "last": v - 1, "seam": min(v - 1, seg)}[where]
    other = max(0, at - 1)
    p = torch.zeros(3, 1, v, device=dev)
    p[:, 0, at] = 0.5
    p[1, 0, other] += 0.25
    us = torch.tensor([0.999, 0.0, 0.999], device=dev)
    got = accept_sampled(p, torch.zeros(3, 1, dtype=torch.int32, device=dev), torch.zeros(3, 1, device=dev), us)
    assert got.token.tolist() == [at, other, at] and got.count.tolist() == [1, 1, 1]


def test_rows_of_leaves_are_not_looked_at(dev):
    """A draft row that no child was drawn from may hold anything; so may one whose first child is accepted."""
    from flint_amd.spec import accept_sampled
    p, q, tokens, parents, ua, us = make(6, 8, 3000, 21)
    inner = torch.zeros(6, 7, dtype=torch.bool)
    for s in range(6):
        inner[s, parents[s, 1:].long()] = True
    want = accept_sampled(*(x.to(dev) for x in (p, tokens, ua, us, parents, q)))
    for junk in (float("nan"), float("inf"), -1.0):
        got = accept_sampled(*(x.to(dev) for x in (p, tokens, ua, us, parents, torch.where(inner[..., None], q, junk))))
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("draft", [True, False])
def test_many_children_of_one_node(dev, draft):
    """A root with 1023 children, unlikely ones and many of them twice, nearly all rejected."""
    m, v = 1024, 1500
    p, q, _, _, ua, us = make(3, m, v, 31, draft=draft)
    g = torch.Generator().manual_seed(32)
    low = p[:, 0].argsort(dim=1)[:, :1000].int()
    tokens = low.gather(1, torch.randint(0, 1000, (3, m), generator=g))
    parents = torch.zeros(3, m, dtype=torch.int32)
    parents[:, 0] = -1
    ua = 1.0 - 0.01 * ua
    ua[1, 1000] = ua[2, 70] = 0.0
    check((p, q, tokens, parents, ua, us), dev)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("v", [70, 3000, 49152])
def test_what_little_is_left(dev, v, dtype):
    """Rejected tokens that hold nearly all of a row: Z is the sum of what is left, not a difference of large numbers."""
    m = 8
    g = torch.Generator().manual_seed(v)
    p = (torch.rand(6, 1, v, generator=g) + 0.5).repeat(1, m, 1) * 2.0 ** -70
    p[:, :, 5] = 0.5
    p[1:, :, 9] = 2.0 ** -30
    p[2, :, 7] = 2.0 ** -50
    p[3, :, 5] = 3.0e38
    p[4, :, 5] = math.inf
    p = p.to(dtype)
    tokens = torch.tensor([[0, 5, 9, 7, 5, 11, 12, 13]] * 6, dtype=torch.int32)
    parents = torch.tensor([[-1] + [0] * 7] * 6, dtype=torch.int32)
    ua = torch.full((6, m), 1.0 - 2.0 ** -24)
    ua[:, 5:] = torch.rand(6, 3, generator=g)
    ua[5, 5:] = 1e-5
    us = torch.rand(6, generator=g)
    got = check((p, None, tokens, parents, ua, us), dev)
    assert int(got.count[0]) == 1 and int(got.token[0]) not in (5, 9, 7)

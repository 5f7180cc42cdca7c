"""Speculation and long texts over a key / value cache, measured: attention of a tree of drafted tokens
(one token alone included) over the cache, the attention weight that each cached key gathers, eviction
of the keys that gathered least, and verification of drafted tokens against the target's probabilities
from given random numbers.

run() has each operator twice: in plain torch, and (where `own` is true) as the call that a program makes
of flint_amd. Sizes are the flint-3b model's (40 query heads over 8 key heads of 64, 40 layers, vocabulary
49152), and ragged ones around them.

Definitions. Node m of a sequence sits in cache slot pos + m; it attends to the slots [0, pos) and to pos + j
where mask[m, j] (None: a chain, j <= m). o = sum_k p_k v_k, p = softmax over those keys of scale q.k, lse = log
sum exp of the same; a row that sees nothing gives 0 and -inf. The weight of a key is the sum of its p over
the nodes and the query heads of its group. Eviction keeps, of the slots [0, n), the first `sink`, the last
`recent` and of the others those of the largest weight, `keep` in all, ties to the lower slot, moved together
in order. Verification walks from the root: the children of a node are tried in order, child t accepted where
u q(t) Z < w(t); at first w = p, the target's row of the node, and Z = 1; a rejection takes Z q off w (where no
draft probabilities are given, q is all at t), not below 0, and Z becomes the sum of w. The last node's token is
the first index where the running sum of w passes sample_u times its sum (p's, should w hold nothing).
"""
import math

import torch

own = False  # run() makes the framework's calls in place of the plain form

DEV = "cuda"
HEADS, GROUPS, DIM, LAYERS, VOCAB = 40, 8, 64, 40, 49152  # of flint-3b


def _attn(name, b, m, ctx, heads=HEADS, groups=GROUPS, dim=DIM, dtype="bfloat16", tree=False, ragged=False,
          kind="attention"):
    return dict(name=name, kind=kind, b=b, m=m, ctx=ctx, heads=heads, groups=groups, dim=dim, dtype=dtype, tree=tree,
                ragged=ragged)


def listed():
    return [
        # one token behind a short chat: the shortest call of a decode step
        _attn("attention-1-512", 1, 1, 512),
        # the 8-node tree of a speculative pass
        _attn("attention-8-1024", 1, 8, 1024, tree=True),
        # trees of 13 nodes for 16 sequences of any length, heads of another model's layout
        _attn("attention-16x13-odd", 16, 13, 8011, heads=32, groups=4, dim=128, dtype="float16", tree=True, ragged=True),
        # one token far into a very long document
        _attn("attention-1-131072", 1, 1, 131072),
        # a pass of 1024 prompt tokens behind earlier ones
        _attn("attention-1024-4096", 1, 1024, 4096),
        # one decode step of 24 sequences: what their caches' keys gather
        _attn("weights-24x1-odd", 24, 1, 2777, ragged=True, kind="weights"),
        # a pass of 512 prompt tokens behind 8192: what every key gathered from it
        _attn("weights-512-8192", 1, 512, 8192, kind="weights"),
        # one layer of a short chat cut to half
        dict(name="evict-1-1100", kind="evict", layers=1, groups=GROUPS, dim=DIM, n=1100, keep=512, recent=64, sink=4),
        # all layers of a long document cut to a quarter
        dict(name="evict-40-8192", kind="evict", layers=LAYERS, groups=GROUPS, dim=DIM, n=8192, keep=2048, recent=256,
             sink=4),
        # a chain of four drafted tokens with the draft's probabilities
        dict(name="verify-chain-4", kind="verify", b=1, m=5, vocab=VOCAB, tree=False, draft=True, dtype="float32"),
        # the widest tree of a draft that proposes without probabilities
        dict(name="verify-tree-32", kind="verify", b=1, m=32, vocab=VOCAB, tree=True, draft=False, dtype="float32"),
        # trees of nine for a full batch, each child drawn from the draft's row
        dict(name="verify-48x9-odd", kind="verify", b=48, m=9, vocab=32003, tree=True, draft=True, dtype="float32"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attention", "attention", "attention", "weights", "evict", "verify", "verify"])
    if kind in ("attention", "weights"):
        b = rng.choice([1, 1, _log_int(rng, 2, 32)])
        m = rng.choice([1, _log_int(rng, 2, 32), _log_int(rng, 33, 1024)])
        ctx = _log_int(rng, 1, 131072)
        groups, rep = rng.choice([(8, 5), (8, 5), (8, 4), (4, 8), (2, 4), (12, 1), (1, 7)])
        dim = rng.choice([64, 64, 128])
        while b * m * (ctx + m) * groups * rep * dim > 1024 * 4608 * HEADS * DIM:  # the largest product
            m = (m + 1) // 2 if m > 16 else m
            ctx, b = (ctx + 1) // 2, (b + 1) // 2
        while b * (ctx + m) * groups * dim > 131072 * GROUPS * DIM:  # the largest cache
            ctx, b = (ctx + 1) // 2, (b + 1) // 2
        return dict(kind=kind, b=b, m=m, ctx=ctx, heads=groups * rep, groups=groups, dim=dim,
                    dtype=rng.choice(["bfloat16", "bfloat16", "float16"]), tree=m > 1 and rng.random() < 0.5,
                    ragged=b > 1)
    if kind == "evict":
        layers, groups, dim = rng.choice([1, LAYERS, rng.randint(1, 12)]), rng.choice([2, 4, 8]), rng.choice([64, 128])
        n = _log_int(rng, 20, 131072)
        while layers * groups * n * dim > LAYERS * GROUPS * 8192 * DIM:
            n //= 2
        keep = max(1, int(n * rng.uniform(0.05, 0.95)))
        sink = min(keep, rng.choice([0, 0, 4]))
        return dict(kind="evict", layers=layers, groups=groups, dim=dim, n=n, keep=keep, sink=sink,
                    recent=int((keep - sink) * rng.choice([0.0, 0.1, rng.random()])))
    b, m, vocab = rng.choice([1, 1, _log_int(rng, 2, 64)]), rng.randint(2, 32), _log_int(rng, 1000, 160000)
    while b * m * vocab > 48 * 9 * 32003:
        b, m = (b + 1) // 2, max(2, m - 1)
    return dict(kind="verify", b=b, m=m, vocab=vocab, tree=rng.random() < 0.6, draft=rng.random() < 0.6,
                dtype=rng.choice(["float32", "float32", "bfloat16"]))


# ---- inputs, from the seed alone ------------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _positions(case):
    """Cached keys of each sequence: ctx, or any length up to it."""
    b, ctx = case["b"], case["ctx"]
    return [ctx * (2 * i + 1) // (2 * b) for i in range(b)] if case["ragged"] else [ctx] * b


def _parents(g, b, m, tree):
    """int32 [b, m], -1 at the root; a tree's nodes hang below one of the five before them."""
    i = torch.arange(m, device=DEV)
    if not tree:
        return (i - 1).int().expand(b, m).contiguous()
    back = 1 + (torch.rand(b, m, generator=g, device=DEV) * i.clamp(max=5)).int()
    return torch.where(i > 0, i - back, -1).int()


def _ancestors(parents):
    """uint8 [b, m, m]: 1 where column j is row i or above it."""
    b, m = parents.shape
    mask = torch.zeros(b, m, m, dtype=torch.uint8, device=DEV)
    rows = torch.arange(b, device=DEV)
    mask[:, 0, 0] = 1
    for i in range(1, m):
        mask[:, i] = mask[rows, parents[:, i].long()]
        mask[:, i, i] = 1
    return mask


def prepare(case, seed):
    g = _gen(seed)
    st = dict(case=case)
    if case["kind"] in ("attention", "weights"):
        b, m, d, dt = case["b"], case["m"], case["dim"], getattr(torch, case["dtype"])
        pos = _positions(case)
        order = torch.randperm(b, generator=g, device=DEV).tolist()
        pos = [pos[i] for i in order]
        slots = -(-(max(pos) + m) // 8) * 8 + 8  # caches come in eights; some of it is free
        st["q"] = (torch.randn(b, m, case["heads"], d, generator=g, device=DEV) * 1.5).to(dt)
        # keys of a few dimensions of large mean, as rotated keys have; values plain
        k = torch.randn(b, case["groups"], slots, d, generator=g, device=DEV)
        k += 2.0 * torch.randn(case["groups"], 1, d, generator=g, device=DEV) * (torch.arange(d, device=DEV) % 16 == 0)
        st["k"] = k.to(dt)
        st["v"] = torch.randn(b, case["groups"], slots, d, generator=g, device=DEV).to(dt)
        st["scale"] = d ** -0.5
        st["pos"] = torch.tensor(pos, dtype=torch.int32, device=DEV) if b > 1 else pos[0]
        st["mask"] = _ancestors(_parents(g, b, m, True)) if case["tree"] else None
        if case["kind"] == "weights":
            st["lse"] = _attention(st)[1]
        return st
    if case["kind"] == "evict":
        lead, n, d = (case["layers"], case["groups"]), case["n"], case["dim"]
        slots = n + n // 8 // 8 * 8
        st["k"] = torch.randn(*lead, slots, d, generator=g, device=DEV).to(torch.bfloat16)
        st["v"] = torch.randn(*lead, slots, d, generator=g, device=DEV).to(torch.bfloat16)
        # a few keys gather most; some none at all, so that equal weights are common
        w = torch.exp(3.0 * torch.randn(*lead, slots, generator=g, device=DEV) - 4.0)
        st["w"] = torch.where(torch.rand(*lead, slots, generator=g, device=DEV) < 0.2, 0.0, w)
        # where the kept rows go: a smaller cache
        new = -(-case["keep"] // 8) * 8
        st["out"] = (torch.zeros(*lead, new, d, dtype=torch.bfloat16, device=DEV),
                     torch.zeros(*lead, new, d, dtype=torch.bfloat16, device=DEV),
                     torch.zeros(*lead, new, device=DEV))
        return st
    b, m, v = case["b"], case["m"], case["vocab"]
    logits = torch.randn(b, m, v, generator=g, device=DEV)
    logits += 6.0 * torch.rand(b, m, v, generator=g, device=DEV) ** 40  # some tokens stand out
    p = torch.softmax(3.0 * logits, dim=-1)
    st["p"] = torch.where(p < p.amax(dim=-1, keepdim=True) * 1e-6, 0.0, p).to(getattr(torch, case["dtype"]))
    st["parents"] = _parents(g, b, m, case["tree"]) if case["tree"] else None
    par = _parents(g, b, m, False) if st["parents"] is None else st["parents"]
    logits += 0.35 * torch.randn(b, m, v, generator=g, device=DEV)  # the draft's mind
    q = torch.softmax(3.0 * logits[:, :m - 1], dim=-1)
    rows = torch.arange(b, device=DEV)
    if case["draft"]:
        tok = torch.multinomial(q.view(-1, v), m, replacement=True, generator=g).view(b, m - 1, m)
        st["q"] = q.to(getattr(torch, case["dtype"]))
    else:  # the draft's best few, in order
        tok, st["q"] = q.topk(min(m, v), dim=-1).indices, None
    tokens, used = torch.zeros(b, m, dtype=torch.long, device=DEV), torch.zeros(b, m, dtype=torch.long, device=DEV)
    for i in range(1, m):
        at = par[:, i].long()
        tokens[:, i] = tok[rows, at, used[rows, at]]
        used[rows, at] += 1
    st["tokens"] = tokens.int()
    st["accept_u"] = torch.rand(b, m, generator=g, device=DEV)
    st["sample_u"] = torch.rand(b, generator=g, device=DEV)
    return st


# ---- one pass ---------------------------------------------------------------------------------------

def _seen(st, slots):
    """bool [b, 1, m, slots]: what each node attends to."""
    b, m = st["q"].shape[:2]
    pos = torch.as_tensor(st["pos"], device=DEV).reshape(-1, 1, 1).expand(b, 1, 1)
    j = torch.arange(slots, device=DEV) - pos  # [b, 1, slots]: node of a slot
    if st["mask"] is None:
        return (j <= torch.arange(m, device=DEV)[:, None])[:, None]
    inside = ((j >= 0) & (j < m)).expand(b, m, slots)
    tree = st["mask"].bool().gather(2, j.clamp(0, m - 1).expand(b, m, slots))
    return torch.where(inside, tree, j < 0)[:, None]


def _scores(st, ftype=torch.float32):
    """[b, groups, heads of a group, m, slots]: scale q.k, -inf where a node does not attend."""
    b, m, heads, d = st["q"].shape
    groups = st["k"].shape[1]
    slots = int(max(_positions(st["case"]))) + m
    q = st["q"].to(ftype).view(b, m, groups, heads // groups, d).permute(0, 2, 3, 1, 4).reshape(b, groups, -1, d)
    s = (q @ st["k"][:, :, :slots].to(ftype).transpose(2, 3).contiguous()) * st["scale"]
    s = s.view(b, groups, heads // groups, m, slots)
    return s.masked_fill_(~_seen(st, slots)[:, None], -math.inf)


def _attention(st, ftype=torch.float32):
    """(o [b, m, heads, d], lse [b, m, heads]), in ftype."""
    s = _scores(st, ftype)
    b, groups, rep, m, slots = s.shape
    top = s.amax(dim=-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = s.sub_(top).exp_()
    total = p.sum(dim=-1, keepdim=True)
    o = p.view(b, groups, rep * m, slots) @ st["v"][:, :, :slots].to(ftype)
    o = o.view(b, groups, rep, m, -1) / torch.where(total == 0, 1.0, total)
    lse = (total.log() + top)[..., 0]
    return (o.permute(0, 3, 1, 2, 4).reshape(b, m, groups * rep, -1),
            lse.permute(0, 3, 1, 2).reshape(b, m, groups * rep))


def _weights(st, ftype=torch.float32):
    s = _scores(st, ftype)
    b, groups, rep, m, slots = s.shape
    lse = st["lse"].to(ftype).view(b, m, groups, rep).permute(0, 2, 3, 1)[..., None]
    w = torch.zeros(b, groups, st["k"].shape[2], dtype=ftype, device=DEV)
    w[:, :, :slots] = s.sub_(lse).exp_().nan_to_num_(nan=0.0).sum(dim=(2, 3))
    return w


def _kept(case, w):
    """Slots that stay, int64 [..., keep], rising."""
    n, keep, recent, sink = case["n"], case["keep"], case["recent"], case["sink"]
    w = w[..., :n].clone()
    w[..., :sink] = math.inf
    w[..., n - recent:] = math.inf
    return w.sort(dim=-1, descending=True, stable=True).indices[..., :keep].sort(dim=-1).values


def _verify(p, q, tokens, parents, accept_u, sample_u):
    """64 bits throughout: a token next to a border must not fall on its other side. The nodes of a tree come
    parents first, so one walk over them in order is the walk down the tree."""
    b, m, v = p.shape
    rows = torch.arange(b, device=p.device)
    cur = torch.zeros(b, dtype=torch.long, device=p.device)
    z = torch.ones(b, dtype=torch.float64, device=p.device)
    w = p[:, 0].double()
    path = torch.full((b, m), -1, dtype=torch.int32, device=p.device)
    path[:, 0] = 0
    count = torch.ones(b, dtype=torch.long, device=p.device)
    for i in range(1, m):
        t = tokens[:, i].long()
        tried = (parents[:, i] == cur) if parents is not None else cur == i - 1
        qrow = None if q is None else q[rows, cur.clamp(max=m - 2)].double()
        qt = 1.0 if q is None else qrow[rows, t]
        yes = tried & (accept_u[:, i].double() * qt * z < w[rows, t])
        no = tried & ~yes
        if q is None:
            less = w.clone()
            less[rows, t] = 0.0
        else:
            less = (w - z[:, None] * qrow).clamp(min=0.0)
        w = torch.where(no[:, None], less, torch.where(yes[:, None], p[:, i].double(), w))
        z = torch.where(no, w.sum(dim=1), torch.where(yes, 1.0, z))
        path.scatter_(1, torch.where(yes, count, m - 1)[:, None],
                      torch.where(yes, i, path.gather(1, torch.where(yes, count, m - 1)[:, None])[:, 0])[:, None].int())
        cur, count = torch.where(yes, i, cur), count + yes
    w = torch.where(w.sum(dim=1, keepdim=True) > 0, w, p[rows, cur].double())
    run_ = w.cumsum(dim=1)
    token = (run_ <= sample_u.double()[:, None] * run_[:, -1:]).sum(dim=1).clamp(max=v - 1)
    return path, count.int(), token.int()


def run(st):
    case = st["case"]
    kind = case["kind"]
    if own:
        from flint_amd import attention, spec
        if kind == "attention":
            return attention.tree_attention(st["q"], st["k"], st["v"], st["pos"], st["mask"], st["scale"],
                                            return_lse=True)
        if kind == "weights":
            return attention.attention_weights(st["q"], st["k"], st["lse"], st["pos"], st["mask"], st["scale"])
        if kind == "evict":
            kept = attention.evict(st["k"], st["v"], st["w"], case["n"], case["keep"], recent=case["recent"],
                                   sink=case["sink"], out=st["out"])
            return (kept, *st["out"])
        return tuple(spec.accept_sampled(st["p"], st["tokens"], st["accept_u"], st["sample_u"], st["parents"], st["q"]))
    if kind == "attention":
        o, lse = _attention(st)
        return o.to(st["q"].dtype), lse
    if kind == "weights":
        return _weights(st)
    if kind == "evict":
        kept = _kept(case, st["w"])
        k, v, w = st["out"]
        rows = kept[..., None].expand(*kept.shape, case["dim"])
        k[..., :case["keep"], :] = st["k"].gather(2, rows)
        v[..., :case["keep"], :] = st["v"].gather(2, rows)
        w[..., :case["keep"]] = st["w"].gather(2, kept)
        return kept.int(), k, v, w
    return _verify(st["p"], st["q"], st["tokens"], st["parents"], st["accept_u"], st["sample_u"])


# ---- what a pass cannot do without ---------------------------------------------------------------------

def work(case):
    if case["kind"] in ("attention", "weights"):
        b, m, heads, groups, d = (case[x] for x in ("b", "m", "heads", "groups", "dim"))
        keys = sum(_positions(case)) + b * m
        seen = sum(p * m for p in _positions(case)) + b * (m if case["tree"] else m * (m + 1) // 2)
        rows = b * m * heads
        mask = b * m * m if case["tree"] else 0
        if case["kind"] == "attention":  # K and V once, q in, o and lse out
            return {"bytes": keys * groups * d * 4 + rows * (4 * d + 4) + mask, "flops": 4 * seen * heads * d}
        return {"bytes": keys * groups * (2 * d + 4) + rows * (2 * d + 4) + mask, "flops": 2 * seen * heads * d}
    if case["kind"] == "evict":
        lead = case["layers"] * case["groups"]
        # all weights once, the kept rows of K and V in and out, their weights and slots out
        return {"bytes": lead * (4 * case["n"] + case["keep"] * (8 * case["dim"] + 8)), "flops": lead * case["n"]}
    size = 4 if case["dtype"] == "float32" else 2
    # of each sequence the row that the last token is drawn from, with the draft's, and the numbers of every node
    return {"bytes": case["b"] * (case["vocab"] * size * (2 if case["draft"] else 1) + case["m"] * (16 + 2 * size)),
            "flops": case["b"] * case["vocab"] * 4}


# ---- the same in 64 bits, from the definitions -----------------------------------------------------------

def _softmax_rows(case, st):
    """For each sequence and group: (keys seen bool [m, n], scores fp64 [heads of a group, m, n]), n its own keys."""
    b, m, heads, d = st["q"].shape
    groups = st["k"].shape[1]
    pos = st["pos"].tolist() if b > 1 else [st["pos"]]
    for i in range(b):
        n = pos[i] + m
        seen = torch.ones(m, n, dtype=torch.bool, device=DEV)
        new = torch.ones(m, m, device=DEV).tril() if st["mask"] is None else st["mask"][i]
        seen[:, pos[i]:] = new != 0
        for j in range(groups):
            q = st["q"][i, :, j * (heads // groups):(j + 1) * (heads // groups)].double().transpose(0, 1)
            yield i, j, n, seen, torch.matmul(q, st["k"][i, j, :n].double().t().contiguous()) * st["scale"]


def exact(case, seed):
    """Whole numbers have no value here: the verified tokens and the kept slots."""
    if case["kind"] == "verify":
        return None
    st = prepare(case, seed)
    if case["kind"] == "evict":
        k, v, w = (x.double() for x in st["out"])
        slot = torch.arange(case["n"], device=DEV)
        safe = (slot < case["sink"]) | (slot >= case["n"] - case["recent"])
        free = case["keep"] - case["sink"] - case["recent"]
        for l in range(case["layers"]):
            for g in range(case["groups"]):
                score = st["w"][l, g, :case["n"]].double().cpu().numpy()
                order = (-score).argsort(kind="stable")
                order = torch.from_numpy(order).to(DEV)
                stays = safe.clone()
                stays[order[~safe[order]][:free]] = True
                at = stays.nonzero()[:, 0]
                k[l, g, :len(at)], v[l, g, :len(at)] = st["k"][l, g, at].double(), st["v"][l, g, at].double()
                w[l, g, :len(at)] = st["w"][l, g, at].double()
        return None, k, v, w
    b, m, heads, d = st["q"].shape
    rep = heads // st["k"].shape[1]
    if case["kind"] == "weights":
        total = torch.zeros(st["k"].shape[:3], dtype=torch.float64, device=DEV)
        for i, j, n, seen, s in _softmax_rows(case, st):
            lse = st["lse"][i, :, j * rep:(j + 1) * rep].double().t()[..., None]
            total[i, j, :n] = torch.where(seen, torch.exp(s - lse), 0.0).sum(dim=1).sum(dim=0)
        return total
    o = torch.zeros(b, m, heads, d, dtype=torch.float64, device=DEV)
    lse = torch.full((b, m, heads), -math.inf, dtype=torch.float64, device=DEV)
    for i, j, n, seen, s in _softmax_rows(case, st):
        log_total = torch.logsumexp(torch.where(seen, s, -math.inf), dim=-1)
        p = torch.where(seen, torch.exp(s - log_total[..., None]), 0.0)
        h = slice(j * rep, (j + 1) * rep)
        o[i, :, h] = torch.matmul(p, st["v"][i, j, :n].double()).transpose(0, 1)
        lse[i, :, h] = log_total.t()
    return o, lse

"""Scoring tokens through 8-bit linears, measured: the matrix product of 8-bit integers with a scale
for each token and channel, the linear that quantises its input rows on the way, log probabilities
of given tokens with entropy, rank and top alternatives, and both joined at the vocabulary head
(features in, log probabilities out).

run() has each operator twice: in plain torch, and (where `own` is true) as the call that a program
makes of flint_amd. Sizes are the flint-3b model's (hidden 2560, feed-forward 8192, vocabulary
49152), and ragged ones around them.

Definitions. A row r of bf16 values is held in 8 bits as scale s = fp32(max|r| / 127) and whole
numbers q = r / s rounded to the nearest, ties to even (s = 0: q = 0; a row with a NaN or an infinity:
s = NaN, q = 0). A product is y[m, n] = (sum_k xq[m, k] wq[n, k]) (xs[m] ws[n]), the sum exact, fp32
behind it, bf16 at the end (fp32 for logits). Of logits l: logprob = l[t] - log sum exp l, entropy =
-sum p log p, rank = how many indices come before t when sorted by value (NaN first, ties to the lower
index), the first `top` of that order and their log probabilities.
"""
import math

import torch

own = False  # run() makes the framework's calls in place of the plain form

DEV = "cuda"
# (N, K) of the linears of one flint-3b layer: QKV, attention output, gate + up, down
SHAPES = {"qkv": (3584, 2560), "o": (2560, 2560), "gate_up": (16384, 2560), "down": (2560, 8192)}
VOCAB, DIM = 49152, 2560


def listed():
    return [
        # one token through the attention output projection: the shortest call of a decode step
        dict(name="linear-1-o", kind="linear", m=1, n=2560, k=2560),
        # a few drafted tokens through a layer of other sizes than the 3B model's
        dict(name="linear-7-odd", kind="linear", m=7, n=5003, k=1408),
        # the widest speculative tree through gate + up
        dict(name="linear-32-gate-up", kind="linear", m=32, n=16384, k=2560),
        # a chat turn's prompt, of a length that fits no tile, into a ragged output size
        dict(name="linear-333-odd", kind="linear", m=333, n=2570, k=2560),
        # a long prompt through gate + up
        dict(name="linear-2048-gate-up", kind="linear", m=2048, n=16384, k=2560),
        # rows quantised once for several linears: a short prompt through the down projection
        dict(name="product-64-down", kind="product", m=64, n=2560, k=8192),
        # ... and a pass of 1024 prompt tokens through QKV
        dict(name="product-1024-qkv", kind="product", m=1024, n=3584, k=2560),
        # the log probability of the token just decoded, with 20 alternatives
        dict(name="logprobs-1", kind="logprobs", rows=1, vocab=VOCAB, top=20, dtype="float32", masked=False),
        # the rows of a verified tree under a grammar that forbids most tokens, in some rows all of them
        dict(name="logprobs-31-masked", kind="logprobs", rows=31, vocab=32003, top=8, dtype="bfloat16", masked=True),
        # a prompt of 1024 tokens scored from its logits
        dict(name="logprobs-1024", kind="logprobs", rows=1024, vocab=VOCAB, top=5, dtype="float32", masked=False),
        # eight verified tokens scored from their features through the 8-bit vocabulary head
        dict(name="head-8", kind="head", m=8, n=VOCAB, k=DIM, top=5),
        # a prompt of 1024 tokens scored from its features
        dict(name="head-1024", kind="head", m=1024, n=VOCAB, k=DIM, top=5),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["linear", "linear", "product", "logprobs", "logprobs", "head"])
    if kind == "logprobs":
        rows, vocab = rng.choice([1, _log_int(rng, 2, 40), _log_int(rng, 41, 1500)]), _log_int(rng, 1000, 160000)
        while rows * vocab > 1024 * VOCAB:
            rows = (rows + 1) // 2
        return dict(kind="logprobs", rows=rows, vocab=vocab, top=rng.choice([0, 1, 5, 20, rng.randint(2, 32)]),
                    dtype=rng.choice(["float32", "bfloat16"]), masked=rng.random() < 0.3)
    m = rng.choice([1, _log_int(rng, 2, 32), _log_int(rng, 33, 2048)])
    n, k = _log_int(rng, 500, 16384), 16 * _log_int(rng, 16, 512)
    if kind == "head":
        m, n, k = min(m, 1024), _log_int(rng, 1000, VOCAB), 16 * _log_int(rng, 16, DIM // 16)
        return dict(kind="head", m=m, n=n, k=k, top=rng.choice([0, 1, 5, rng.randint(2, 32)]))
    if m > 1 and rng.random() < 0.5:  # a layer of the 3B model
        n, k = rng.choice(sorted(SHAPES.values()))
    while m * n * k > 2048 * 16384 * 2560:
        m //= 2
    return dict(kind=kind, m=m, n=n, k=k)


# ---- inputs, from the seed alone ------------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _quantized(x):
    """(whole numbers int8, scales fp32) of the rows of x; the quotients in 64 bits: x / s next to a
    half must not be rounded onto it."""
    amax = x.float().abs().amax(dim=1)
    s = torch.where(amax.isfinite(), amax / 127, math.nan)
    q = (x.double() / s.double()[:, None]).round()
    return q.nan_to_num(nan=0.0).clamp(-127, 127).to(torch.int8), s


def _weight(g, n, k):
    return _quantized((torch.randn(n, k, generator=g, device=DEV) * 0.02).to(torch.bfloat16))


def _rows(g, m, k):
    """Activations as the linears of a transformer meet them: near normal, a few channels far larger."""
    x = torch.randn(m, k, generator=g, device=DEV)
    x[:, torch.randint(0, k, (max(1, k // 512),), generator=g, device=DEV)] *= 12.0
    return x.to(torch.bfloat16)


def _tokens(g, m, n):
    return torch.randint(0, n, (m,), generator=g, device=DEV, dtype=torch.int32)


def prepare(case, seed):
    g = _gen(seed)
    if case["kind"] == "logprobs":
        rows, vocab = case["rows"], case["vocab"]
        # bf16 values, as the decode and verify kernels write them: equal logits are common
        l = (torch.randn(rows, vocab, generator=g, device=DEV) * 2.5).to(torch.bfloat16)
        t = _tokens(g, rows, vocab)
        if case["masked"]:
            mask = torch.rand(rows, vocab, generator=g, device=DEV) < 0.9
            l.masked_fill_(mask.scatter_(1, t.long()[:, None], False), -math.inf)  # the token given was allowed
            l[1::7].clamp_(min=torch.finfo(l.dtype).min)  # masks of the type's lowest value
            l[5::9] = -math.inf                           # nothing left
        return dict(case=case, logits=l.to(getattr(torch, case["dtype"])), tokens=t)
    wq, ws = _weight(g, case["n"], case["k"])
    st = dict(case=case, wq=wq, ws=ws)
    x = _rows(g, case["m"], case["k"])
    if case["kind"] == "product":
        st["xq"], st["xs"] = _quantized(x)
    elif case["kind"] == "linear":
        st["x"] = x
    else:  # features such that logits spread by about 4, as a trained head's do
        st["ws"] = ws * (4.0 / (0.02 * math.sqrt(case["k"])))
        st["x"], st["tokens"] = x, _tokens(g, case["m"], case["n"])
    return st


# ---- one pass ---------------------------------------------------------------------------------------

def _product(xq, xs, wq, ws):
    """fp32 [M, N]; the sums in 64 bits: they are exact, and pass 2^24."""
    acc = xq.double() @ wq.double().T
    return acc.float() * (xs[:, None] * ws[None, :])


def _order(l):
    """int64 keys, all different, in the order of the values (NaN above all), equal ones by falling index."""
    b = (l.float() + 0.0).masked_fill(l.isnan(), math.nan).view(torch.int32).long()
    return (torch.where(b < 0, -2 ** 31 - b, b) << 32) - torch.arange(l.shape[1], device=l.device)


def _logprobs(l, tokens, top):
    t, n = tokens.long()[:, None], l.shape[1]
    key = _order(l)
    rank = (key > key.gather(1, t)).sum(dim=1).int()
    l = l.float()
    d = l - l.amax(dim=1, keepdim=True)
    e = d.exp()
    s = e.sum(dim=1)
    logsum = s.log()
    logprob = d.gather(1, t)[:, 0] - logsum
    # a value whose probability is nothing adds nothing
    entropy = logsum - torch.where(e == 0, 0.0, d * e).sum(dim=1) / s
    if not top:
        return logprob, entropy, rank, None, None
    best = key.topk(top, dim=1).values  # sorted; the index is in the low 32 bits, falling
    ids = (-best) & 0xFFFFFFFF
    return logprob, entropy, rank, ids.int(), d.gather(1, ids) - logsum[:, None]


def run(st):
    case = st["case"]
    kind = case["kind"]
    if own:
        from flint_amd import generate, quantize
        if kind == "linear":
            return quantize.linear_int8(st["x"], st["wq"], st["ws"])
        if kind == "product":
            return quantize.gemm_int8(st["xq"], st["xs"], st["wq"], st["ws"])
        if kind == "logprobs":
            return generate.logprobs(st["logits"], st["tokens"], top=case["top"])
        return generate.head_logprobs(st["x"], st["wq"], st["ws"], st["tokens"], top=case["top"])
    if kind == "product":
        return _product(st["xq"], st["xs"], st["wq"], st["ws"]).to(torch.bfloat16)
    if kind == "logprobs":
        return _logprobs(st["logits"], st["tokens"], case["top"])
    y = _product(*_quantized(st["x"]), st["wq"], st["ws"])
    return y.to(torch.bfloat16) if kind == "linear" else _logprobs(y, st["tokens"], case["top"])


# ---- what a pass cannot do without ---------------------------------------------------------------------

def work(case):
    out = lambda rows: rows * (4 + 12 + 8 * case["top"])  # noqa: E731  token in; three numbers and the alternatives out
    if case["kind"] == "logprobs":
        rows, vocab = case["rows"], case["vocab"]
        # per value: a maximum, a difference, an exponential, two sums and a product, a comparison for the rank
        return {"bytes": rows * vocab * (4 if case["dtype"] == "float32" else 2) + out(rows), "flops": 7 * rows * vocab}
    m, n, k = case["m"], case["n"], case["k"]
    if case["kind"] == "head":
        return {"bytes": n * (k + 4) + 2 * m * k + out(m), "flops": 2 * m * n * k + 7 * m * n}
    return {"bytes": n * (k + 4) + (2 * m * k if case["kind"] == "linear" else m * (k + 4)) + 2 * m * n,
            "flops": 2 * m * n * k}


# ---- the same in 64 bits, from the definitions -----------------------------------------------------------

def _held(x):
    """The float64 values that 8 bits hold of the rows of x (scales are fp32 numbers)."""
    s = (x.double().abs().amax(dim=1, keepdim=True) / 127).float().double()
    return torch.where(s > 0, torch.round(x.double() / s) * s, 0.0)


def exact(case, seed):
    """Whole numbers have no value here; ids would need the order of values that differ in their last bits."""
    st = prepare(case, seed)
    kind = case["kind"]
    if kind == "logprobs":
        l = st["logits"].double()
    else:
        x = st["xq"].double() * st["xs"].double()[:, None] if kind == "product" else _held(st["x"])
        l = x @ (st["wq"].double() * st["ws"].double()[:, None]).T
        if kind != "head":
            return l
    lse = torch.logsumexp(l, dim=1, keepdim=True)
    p = torch.exp(l - lse)
    logp = l - torch.where(lse == -math.inf, math.nan, lse)
    entropy = -torch.special.xlogy(p, p).sum(dim=1)
    entropy = torch.where(logp.isnan().any(dim=1), math.nan, entropy)
    given = logp[torch.arange(len(l), device=l.device), st["tokens"].long()]
    best = logp.sort(dim=1, descending=True).values[:, :case["top"]] if case["top"] else None
    return given, entropy, None, None, best

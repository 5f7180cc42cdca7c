"""Plain 64-bit forms of the cache operators: attention of a tree's nodes over a cache, the weight that
each key gathers, eviction, and verification of drafted tokens. Written from the definitions, one sequence and one
head at a time; what a row does not see is never multiplied in."""
import math

import torch


def seen_keys(pos, m, mask, i):
    """Slots that node i of a sequence sees, in order."""
    nodes = range(i + 1) if mask is None else [j for j in range(m) if mask[i][j]]
    return list(range(pos)) + [pos + j for j in nodes]


def tree_attention(q, k, v, pos, mask, scale):
    """(o [B, M, heads, dim], lse [B, M, heads]) in float64. pos: a list; mask: None, [M, M] or [B, M, M] bool."""
    b, m, heads, d = q.shape
    rep = heads // k.shape[1]
    q, k, v = q.double(), k.double(), v.double()
    o = torch.zeros(b, m, heads, d, dtype=torch.float64, device=q.device)
    lse = torch.full((b, m, heads), -math.inf, dtype=torch.float64, device=q.device)
    for s in range(b):
        tree = None if mask is None else (mask if mask.dim() == 2 else mask[s]).tolist()
        for i in range(m):
            keys = seen_keys(pos[s], m, tree, i)
            if not keys:
                continue
            at = torch.tensor(keys, device=q.device)
            kk, vv = k[s][:, at], v[s][:, at]                               # [groups, n, d]
            sc = (kk[:, None] * q[s, i].view(-1, rep, 1, d)).sum(-1) * scale  # [groups, rep, n]
            lse[s, i] = torch.logsumexp(sc, dim=-1).view(-1)
            p = torch.exp(sc - lse[s, i].view(-1, rep, 1))
            o[s, i] = (p[..., None] * vv[:, None]).sum(2).view(heads, d)
    return o, lse


def attention_weights(q, k, lse, pos, mask, scale):
    """float64 [B, groups, slots]."""
    b, m, heads, d = q.shape
    groups = k.shape[1]
    w = torch.zeros(k.shape[:3], dtype=torch.float64, device=q.device)
    for s in range(b):
        tree = None if mask is None else (mask if mask.dim() == 2 else mask[s]).tolist()
        for i in range(m):
            keys = seen_keys(pos[s], m, tree, i)
            if not keys:
                continue
            at = torch.tensor(keys, device=q.device)
            sc = (k[s].double()[:, at][:, None] * q[s, i].double().view(groups, -1, 1, d)).sum(-1) * scale
            l = lse[s, i].double().view(groups, -1, 1)
            w[s][:, at] += torch.where(l == -math.inf, 0.0, torch.exp(sc - l)).sum(1)
    return w


def kept_slots(w, n, keep, recent, sink):
    """Slots of one head that stay, rising; w a list of floats."""
    keep = min(keep, n)
    if keep == n:
        return list(range(n))
    always = [i for i in range(n) if i < sink or i >= n - recent]
    others = [i for i in range(n) if sink <= i < n - recent]
    others.sort(key=lambda i: (not math.isnan(w[i]), -w[i] if not math.isnan(w[i]) else 0.0, i))
    return sorted(always + others[:keep - len(always)])


def accept(p, q, tokens, parents, accept_u, sample_u):
    """One tree: (path, token). p [M][V], q [M - 1][V] or None (numpy float64 arrays or lists), in Python floats."""
    m, v = len(p), len(p[0])
    cur, path, w, z = 0, [0], [x if x > 0 else 0.0 for x in p[0]], 1.0
    start = list(w)
    for i in range(1, m):
        par = i - 1 if parents is None else parents[i]
        t = tokens[i]
        if par != cur or not 0 <= t < v:
            continue
        qt = 1.0 if q is None else q[cur][t]
        if accept_u[i] * qt * z < w[t]:
            cur = i
            path.append(i)
            w, z = [x if x > 0 else 0.0 for x in p[i]], 1.0
            start = list(w)
            continue
        if q is None:
            w[t] = 0.0
        else:
            w = [a - z * b if a - z * b > 0 else 0.0 for a, b in zip(w, q[cur])]
        z = math.fsum(w)
    if not math.fsum(w) > 0:
        w = start
    total = math.fsum(w)
    if not 0 < total < math.inf:
        return path, -1
    run, token = 0.0, -1
    for i, x in enumerate(w):
        run += x
        if x > 0:
            token = i
            if run > sample_u * total:
                break
    return path, token

"""Plain CPU forms of the 8-bit integer linear and of log probabilities, in 64 bits.

quantize_rows and product define every bit; logprobs is the definition in float64, with the order of
indices (value, larger first; NaN above all; equal values by rising index) exact.
"""
import numpy as np
import torch


def quantize_rows(x):
    """(q int8 [M, K], s float32 [M]) of bf16 rows: s = fp32(max|row| * fp32(1 / 127)), q = row / s to the nearest,
    ties to even. The scale is the product: for maxima of the bf16 significands 143, 144, 175, 207, 208 and 239 it is
    an ulp below fp32(max|row| / 127), and half the maximum becomes 64, not 63. A row with a NaN or an infinity: s NaN, q 0."""
    xf = x.float().numpy()
    amax = np.abs(xf).max(axis=1)
    s = np.where(np.isfinite(amax), amax * (np.float32(1) / np.float32(127)), np.float32("nan")).astype(np.float32)
    with np.errstate(invalid="ignore", divide="ignore"):
        # a quotient of 8 by 24 bits that is not a half is at least 2^-25 of it away: float64 decides
        q = np.rint(xf.astype(np.float64) / s.astype(np.float64)[:, None])
    q = np.clip(np.nan_to_num(q, nan=0.0, posinf=0.0, neginf=0.0), -127, 127)
    q[~(s > 0)] = 0
    return torch.from_numpy(q.astype(np.int8)), torch.from_numpy(s)


def product(xq, xs, wq, ws):
    """fp32 [M, N]: the exact sum, rounded to fp32, times fp32(xs ws)."""
    acc = xq.double() @ wq.double().T  # whole numbers below 2^53: exact
    return acc.float() * (xs[:, None] * ws[None, :])


def order(row):
    """Indices of a row (numpy floats) in their order: NaN first, then larger values, equal ones by index."""
    r = row.astype(np.float64) + 0.0
    nan = np.isnan(r)
    return np.lexsort((np.arange(len(r)), -np.where(nan, 0.0, r), ~nan))


def logprobs(logits, tokens, top):
    """Per row: dict(logprob, entropy, rank, ids, top) in float64, and what their error bounds need: the sums U =
    sum p |d|, Q = sum p d^2 of the distances d to the maximum."""
    out = []
    for row, t in zip(logits.double().numpy(), tokens.tolist()):
        v = len(row)
        o = order(row)
        place = np.empty(v, dtype=np.int64)
        place[o] = np.arange(v)
        m = row.max() if not np.isnan(row).any() else np.nan
        inside = 0 <= t < v
        r = dict(rank=int(place[t]) if inside else -1, ids=o[:top], U=0.0, Q=0.0)
        if not np.isfinite(m):
            r.update(logprob=np.nan, entropy=np.nan, top=np.full(top, np.nan), logsum=np.nan)
        else:
            d = row - m
            e = np.exp(d)
            s = e.sum()
            p = e / s
            on = e > 0
            r.update(logprob=d[t] - np.log(s) if inside else np.nan, entropy=float(np.log(s) - (p[on] * d[on]).sum()),
                     top=d[o[:top]] - np.log(s), logsum=np.log(s), U=float((p[on] * -d[on]).sum()),
                     Q=float((p[on] * d[on] ** 2).sum()))
        out.append(r)
    return out

"""Speculative decoding, greedy or sampled, over fl_verify: the chain loop (reference spec_mega.py:89-117) and
the tree loop with KV compaction (reference spec_tree.py:85-133).

Each pass feeds the pending token (the root, not yet in the cache) plus a draft to one verify
launch at cache slots pos..pos+M-1, takes the target's greedy token per node (fl_verify's
on-device argmax), accepts the longest draft prefix (chain) or root-to-leaf path (tree) that the
target agrees with, and for a tree moves the accepted nodes' K/V rows into contiguous slots with
fl_kv_move. The emitted tokens equal sequential greedy decoding of the same model (reference
result.md:111-113), up to argmax ties that the verify and decode kernels break differently.

The draft is pluggable. The reference's EAGLE head (train/draft_model.py) is trained weights
and not part of this package; a draft here is any object with

    chain(context, feats, k) -> list[int]             up to k proposed tokens after context
    tree(context, feats)     -> (tokens, parents)      nodes below the root, parents[i] in
                                                        [-1, i) (-1 = the root), parents first

where context is every token so far (prompt, emitted tokens, and last the pending root) and feats
is a bf16 [n, dim] device view of the final-norm features of the verified tokens (the input an
EAGLE head consumes, reference spec_mega.py:112). LookupDraft (prompt-lookup n-gram matching)
needs no weights.

With a temperature or top_k the loop samples (accept_sampled): the emitted tokens are distributed as
the sampler's own (generate.sample), whatever the draft proposes. A draft that drew its tokens from
distributions of its own also has

    probs() -> fp32 device [nodes - 1, vocab] or None   of the proposal just made: row i the
                                                        distribution that the children of node i were
                                                        drawn from, each on its own (node 0 = the root;
                                                        a chain's node i + 1 is its i-th token)
"""
import os
import time
from collections import namedtuple

import numpy as np
import torch

from . import _lib
from .generate import _ids, logits_to_probs, prefill
from .quantize import linear_int8

# accept_sampled as one call of the torch extension, as quantize's linears
_accept_fast = None
if "FLINT_AMD_LIB" not in os.environ:
    try:
        from ._torch_ops import accept_fast as _accept_fast
    except ImportError:
        pass


WIDE_NODES = 1024  # of a tree in a prompt pass (Transformer.tree_features)


def tree_depths(parents):
    """Depth of each node of a tree in verify order (node 0 = root, parents[0] = -1, every other
    parent an earlier node); raises ValueError on any other parent array. Reference
    spec_tree.py:98-100 builds the same depth list from the draft."""
    depth = []
    for i, p in enumerate(parents):
        p = int(p)
        if i == 0:
            if p != -1:
                raise ValueError("node 0 is the root and has parent -1")
            depth.append(0)
            continue
        if not 0 <= p < i:
            raise ValueError(f"node {i}: parent {p} is not an earlier node")
        depth.append(depth[p] + 1)
    return depth


def tree_mask(parents):
    """Ancestor-or-self mask uint8 [M, M]: mask[i][j] = 1 when j is i or one of its ancestors
    (reference spec_tree.py:101-104). A chain's mask is lower-triangular."""
    tree_depths(parents)
    m = len(parents)
    mask = np.zeros((m, m), dtype=np.uint8)
    for i in range(m):
        j = i
        while j != -1:
            mask[i, j] = 1
            j = int(parents[j])
    return mask


def accept_chain(targets, draft):
    """Number of leading draft tokens the target agrees with: draft[j] is accepted while
    targets[j] (the target's greedy token after cand[0..j]) equals it (reference
    spec_mega.py:106-110)."""
    acc = 0
    for t, d in zip(targets, draft):
        if int(t) != int(d):
            break
        acc += 1
    return acc


def accept_tree(cand, parents, targets):
    """Longest root-to-leaf path the target agrees with: from the root, step to the first child
    (in node order) whose token is the target's greedy token at the current node (reference
    spec_tree.py:109-118). Returns the node indices of the path, root first."""
    children = [[] for _ in cand]
    for i in range(1, len(cand)):
        children[int(parents[i])].append(i)
    path = [0]
    cur = 0
    while True:
        want = int(targets[cur])
        nxt = next((c for c in children[cur] if int(cand[c]) == want), None)
        if nxt is None:
            return path
        path.append(nxt)
        cur = nxt


# What accept_sampled returns, for B trees of M nodes: path int32 [B, M], the accepted nodes, 0 first, then -1; count
# int32 [B] of them; token int32 [B], the one behind the path.
Accepted = namedtuple("Accepted", "path count token")


def accept_sampled(probs, tokens, accept_u, sample_u, parents=None, draft_probs=None):
    """Speculative sampling on the GPU (fl_accept): which path of each drafted tree the target's distribution accepts,
    and the token behind it, drawn so that path and token are distributed as the target's own samples. From given
    random numbers in [0, 1), so the same call gives the same tokens.

    probs: fp32 or bf16 device [B, M, V] (or [M, V]), row i the target's distribution after node i (as
    generate.logits_to_probs gives it). tokens: int [B, M], of the nodes (node 0 is the root, its own is not looked
    at). accept_u: fp32 [B, M], sample_u: fp32 [B]. parents: int [B, M], -1 at the root, parents before children
    (None: a chain); a node without an earlier node as its parent (-1: padding) is no part of the tree. draft_probs:
    of probs' type, [B, M - 1, V], row i the distribution from which the children of node i were drawn, independently
    of each other; None: they were proposed without one (top candidates, a lookup).

    Children are tried in order: child t is accepted where accept_u q(t) Z < w(t), with w = probs' row and Z = 1 at
    first; a rejection takes Z q off w (all of t without draft_probs), not below 0, and Z becomes the sum of w. The last
    node's token is the first index at which the running sum of w passes sample_u times its sum (-1 where that is not
    a positive number). Returns Accepted (without B: of one tree, count and token of one element)."""
    if _accept_fast is not None and probs.is_cuda:
        r = _accept_fast(probs, tokens, accept_u, sample_u, parents, draft_probs,
                         torch._C._cuda_getCurrentRawStream(probs.get_device()))
        if r is not None:
            return Accepted(*r)
    one = probs.dim() == 2
    if one:
        probs = probs[None]
        draft_probs = None if draft_probs is None else draft_probs[None]
    if not probs.is_cuda or probs.dim() != 3 or probs.dtype not in (torch.float32, torch.bfloat16):
        raise ValueError("probs must be an fp32 or bf16 CUDA (HIP) tensor [B, M, V]")
    b, m, v = probs.shape
    dev = probs.device
    if not 1 <= m <= 1024 or not 1 <= v <= 1 << 20 or b > 65536:
        raise ValueError("1..1024 nodes, a vocabulary of 1..2^20 and at most 65536 trees")
    if draft_probs is not None and (draft_probs.dtype != probs.dtype or draft_probs.device != dev
                                    or draft_probs.shape != (b, m - 1, v)):
        raise ValueError(f"draft_probs must be [{b}, {m - 1}, {v}] of probs' type and device")
    for t, name in ((tokens, "tokens"), (parents, "parents")):
        if t is not None and (t.device != dev or t.dtype not in (torch.int32, torch.int64) or t.numel() != b * m):
            raise ValueError(f"{name} must be {b * m} int32 or int64 on probs' device")
    for t, name, n in ((accept_u, "accept_u", b * m), (sample_u, "sample_u", b)):
        if t.device != dev or t.dtype != torch.float32 or t.numel() != n:
            raise ValueError(f"{name} must be {n} fp32 numbers on probs' device")
    path = torch.empty(b, m, dtype=torch.int32, device=dev)
    count, token = torch.empty(b, dtype=torch.int32, device=dev), torch.empty(b, dtype=torch.int32, device=dev)
    if b:
        # in names, so that no copy's memory is given to the next before the launch
        probs, tokens, accept_u, sample_u = (x.detach().contiguous() for x in (probs, _ids(tokens), accept_u, sample_u))
        parents = None if parents is None else _ids(parents).contiguous()
        draft_probs = None if draft_probs is None else draft_probs.detach().contiguous()
        with torch.cuda.device(dev):
            _lib.call("fl_accept", _lib.ptr(probs), _lib.ptr(draft_probs), int(probs.dtype == torch.bfloat16),
                      _lib.ptr(tokens), _lib.ptr(parents), _lib.ptr(accept_u), _lib.ptr(sample_u), _lib.ptr(path),
                      _lib.ptr(count), _lib.ptr(token), b, m, v, _lib.stream_ptr())
    return Accepted(path[0] if one else path, count, token)


def compaction_moves(path, pos):
    """(src, dst) cache slots that bring the accepted path's rows to slots pos..pos+L: node
    path[s] was written at slot pos+path[s] and belongs at pos+s (its RoPE already used position
    pos+s, its depth). Rows already in place are left out (reference spec_tree.py:125-128)."""
    src, dst = [], []
    for s in range(1, len(path)):
        if path[s] != s:
            src.append(pos + int(path[s]))
            dst.append(pos + s)
    return src, dst


class LookupDraft:
    """Prompt-lookup draft: find earlier occurrences of the context's last n tokens (n from
    max_ngram down to min_ngram, the most recent occurrence first) and propose what followed
    them. tree() merges up to `width` distinct continuations into a trie of at most
    max_nodes - 1 nodes below the root: up to 1024 nodes in all, of which a SpecDecoder without a
    head takes 32."""

    def __init__(self, max_ngram=3, min_ngram=1, width=2, depth=4, max_nodes=_lib.MAX_VERIFY):
        if not 1 <= min_ngram <= max_ngram:
            raise ValueError("need 1 <= min_ngram <= max_ngram")
        self.max_ngram, self.min_ngram = int(max_ngram), int(min_ngram)
        self.width, self.depth = int(width), int(depth)
        self.max_nodes = min(int(max_nodes), WIDE_NODES)

    def reset(self):
        """Forget the indexed context (SpecDecoder.generate calls this at the start of a run)."""
        self._ctx, self._pos = [], {}

    def _index(self, ctx):
        """Positions of every n-gram (min_ngram <= n <= max_ngram) of ctx, oldest first, kept
        across calls and extended when ctx extends the indexed context (the loop's case: the
        whole indexed context must be a prefix of ctx, compared element by element)."""
        old = getattr(self, "_ctx", [])
        n0 = len(old)
        if not (n0 and len(ctx) >= n0 and ctx[:n0] == old):
            n0, self._pos = 0, {}
        for n in range(self.min_ngram, self.max_ngram + 1):
            for i in range(max(0, n0 - n + 1), len(ctx) - n + 1):
                self._pos.setdefault(tuple(ctx[i:i + n]), []).append(i)
        self._ctx = list(ctx)
        return self._pos

    def _continuations(self, context, k, limit):
        ctx = context if isinstance(context, list) else [int(t) for t in context]
        n_ctx = len(ctx)
        pos = self._index(ctx)
        found, seen = [], set()
        for n in range(min(self.max_ngram, n_ctx - 1), self.min_ngram - 1, -1):
            for start in reversed(pos.get(tuple(ctx[n_ctx - n:]), ())):
                if start >= n_ctx - n:          # the suffix itself
                    continue
                cont = tuple(ctx[start + n:start + n + k])
                if cont and cont not in seen:
                    seen.add(cont)
                    found.append(list(cont))
                    if len(found) >= limit:
                        return found
        return found

    def chain(self, context, feats, k):
        conts = self._continuations(context, k, 1)
        return conts[0] if conts else []

    def tree(self, context, feats):
        tokens, parents = [], []
        kids = {}                                    # (parent, token) -> node; -1 = root
        for cont in self._continuations(context, self.depth, self.width):
            par = -1
            for t in cont:
                node = kids.get((par, t))
                if node is None:
                    if len(tokens) >= self.max_nodes - 1:
                        break
                    tokens.append(t)
                    parents.append(par)
                    node = kids[(par, t)] = len(tokens) - 1
                par = node
        return tokens, parents


class SpecStats:
    def __init__(self):
        self.passes = 0
        self.tokens = 0
        self.nodes = 0
        self.seconds = 0.0

    @property
    def tokens_per_pass(self):
        return self.tokens / self.passes if self.passes else 0.0

    def __repr__(self):
        return (f"SpecStats(passes={self.passes}, tokens={self.tokens}, nodes={self.nodes}, "
                f"tokens_per_pass={self.tokens_per_pass:.2f}, seconds={self.seconds:.4f})")


class SpecDecoder:
    """Speculative decoding of one sequence on a flint_amd Transformer, greedy or sampled.

    generate(prompt, max_new, mode="chain" | "tree") sets up the model's caches (like
    generate.generate), prefills the prompt, and returns (prompt + new tokens as a host int list,
    SpecStats). Generation stops after max_new tokens or at the first eos token (which is kept).
    """

    def __init__(self, model, draft=None, k=4, head=None):
        """head: a quantize.DynamicInt8Linear (Transformer.int8_head) through which a pass of more than 32 nodes gets its
        logits (Transformer.tree_features; up to 1024 nodes then); such a pass gives the tokens of the model with that head."""
        self.model = model
        self.draft = draft if draft is not None else LookupDraft()
        self.k = int(k)
        self.head = head
        nv = self._nodes = _lib.MAX_VERIFY if head is None else WIDE_NODES
        if not 0 <= self.k < nv:
            raise ValueError(f"k must be in [0, {nv - 1}]")
        dev = model.device
        # tokens | depth | parents | amask staged in one pinned buffer, one copy per pass
        self._host = torch.zeros(3 * nv + nv * nv // 4, dtype=torch.int32, pin_memory=dev.type == "cuda")
        self._dev = torch.zeros_like(self._host, device=dev)
        self._tout = torch.empty(nv, dtype=torch.int32, device=dev)
        self._feat = torch.empty(nv, model.config.dim, dtype=torch.bfloat16, device=dev)

    def _verify(self, cand, parents, pos, logits=False):
        """Stage a pass's nodes on the device and run them; (greedy tokens as a device tensor, logits or None, feat)."""
        m = len(cand)
        nv = self._nodes
        vocab = self.model.config.vocab_size
        if any(not 0 <= t < vocab for t in cand):
            raise ValueError(f"draft token outside [0, {vocab})")
        h = self._host.numpy()
        h[:m] = cand
        h[nv:nv + m] = tree_depths(parents)
        h[2 * nv:2 * nv + m] = parents
        h[3 * nv:].view(np.uint8)[:m * m] = tree_mask(parents).reshape(-1)
        used = 3 * nv + (m * m + 3) // 4
        self._dev[:used].copy_(self._host[:used], non_blocking=True)
        lg = torch.empty(m, vocab, dtype=torch.float32, device=self.model.device) if logits and m <= _lib.MAX_VERIFY else False
        if m == 1:
            # a lone root is one decode step (same cache slot, RoPE position, argmax and final-norm
            # feature as a verify of M = 1), and the decode kernel is the faster of the two
            self.model.decode_step(self._dev[:1], pos, token_out=self._tout[:1], feat=self._feat[0],
                                   logits=lg[0] if logits else None)
            return self._tout[:1], lg, self._feat[:1]
        depth = self._dev[nv:nv + m]
        amask = self._dev[3 * nv:].view(torch.uint8)[:m * m].view(m, m)
        if m > _lib.MAX_VERIFY:
            feat = self.model.tree_features(self._dev[:m], pos, depth, amask)
            lg = linear_int8(feat, self.head.weight, self.head.scales, torch.float32)
            return lg.argmax(dim=1).int(), lg, feat
        tout, lg, feat = self.model.verify(self._dev[:m], pos, depth=depth, amask=amask, logits=lg, feat=self._feat[:m],
                                           tokens_out=self._tout[:m])
        return tout[:m], lg, feat

    def _greedy(self, cand, parents, pos):
        """One pass: (accepted path, next token, features of all nodes)."""
        tout, _, feat = self._verify(cand, parents, pos)
        tgt = tout.tolist()
        path = accept_tree(cand, parents, tgt)
        return path, tgt[path[-1]], feat

    def _sampled(self, cand, parents, pos, temperature, top_k, gen, draft_probs):
        """The same, sampled."""
        m, nv, dev = len(cand), self._nodes, self.model.device
        _, logits, feat = self._verify(cand, parents, pos, logits=True)
        probs = logits_to_probs(logits, temperature, top_k)
        u = torch.rand(m + 1, generator=gen, device=dev)
        got = accept_sampled(probs, self._dev[:m], u[:m], u[m:], parents=self._dev[2 * nv:2 * nv + m], draft_probs=draft_probs)
        out = torch.cat([got.count, got.token, got.path]).tolist()
        if out[1] < 0:
            raise RuntimeError("a row of logits without a distribution")
        return out[2:2 + out[0]], out[1], feat

    @torch.no_grad()
    def generate(self, prompt, max_new, mode="chain", eos=None, temperature=None, top_k=None, seed=0):
        """Greedy, or sampled where temperature or top_k is given (as generate.sample, from torch's generator seeded with
        `seed`: a run repeats itself, and differs from generate.generate's Philox noise)."""
        if mode not in ("chain", "tree"):
            raise ValueError("mode is 'chain' or 'tree'")
        if top_k is not None and int(top_k) < 1:
            raise ValueError("top_k must be >= 1")
        sampled = temperature is not None or top_k is not None
        if hasattr(self.draft, "reset"):
            self.draft.reset()
        ids = [int(t) for t in (prompt.reshape(-1).tolist() if torch.is_tensor(prompt) else prompt)]
        if not ids:
            raise ValueError("empty prompt")
        model, nv = self.model, self._nodes
        T = len(ids)
        max_seq = T + int(max_new) + nv
        if self.head is not None:  # room for the widest tree, as far as there are positions
            max_seq = max(T + int(max_new) + _lib.MAX_VERIFY, min(max_seq, model.packed.rope.shape[0] // 8 * 8))
        model.setup_caches(1, max_seq)
        feats = torch.empty(max_seq, model.config.dim, dtype=torch.bfloat16, device=model.device)
        stats = SpecStats()
        out = list(ids)
        if max_new <= 0:
            return out, stats
        if T > 1:
            prefill(model, torch.tensor(ids[:-1], dtype=torch.int32), 0)
        pos = T - 1
        # reference spec_mega.py:92-93: the last prompt token through the verify kernel
        gen = torch.Generator(device=model.device).manual_seed(int(seed)) if sampled else None
        temp = 1.0 if temperature is None else float(temperature)

        def step(cand, parents, pos, draft_probs=None):
            if sampled:
                return self._sampled(cand, parents, pos, temp, top_k, gen, draft_probs)
            return self._greedy(cand, parents, pos)

        _, nxt, vfeat = step([ids[-1]], [-1], pos)
        feats[0:1].copy_(vfeat[:1])
        n_feat, pos = 1, pos + 1
        new = 0
        t0 = time.perf_counter()
        while True:
            out.append(nxt)
            new += 1
            if new >= max_new or nxt == eos:
                break
            room = min(nv, max_seq - pos)
            context = out
            if mode == "chain":
                d = [int(t) for t in self.draft.chain(context, feats[:n_feat], min(self.k, room - 1))]
                d = d[:room - 1]
                cand = [nxt] + d
                parents = list(range(-1, len(d)))
            else:
                toks, pars = self.draft.tree(context, feats[:n_feat])
                toks, pars = [int(t) for t in toks][:room - 1], [int(p) for p in pars][:room - 1]
                cand = [nxt] + toks
                parents = [-1] + [p + 1 for p in pars]          # draft parents -> verify node indices
            q = None
            if sampled and len(cand) > 1 and hasattr(self.draft, "probs"):
                q = self.draft.probs()
                q = None if q is None else q[:len(cand) - 1]  # a proposal cut to the room that is left
            path, after, vfeat = step(cand, parents, pos, q)
            if mode == "tree":
                src, dst = compaction_moves(path, pos)
                for i in range(0, len(src), _lib.MAX_VERIFY):  # rising: a later move's source is no earlier one's destination
                    model.kv_move(src[i:i + _lib.MAX_VERIFY], dst[i:i + _lib.MAX_VERIFY])
            if path[-1] == len(path) - 1:                      # a prefix of the nodes
                feats[n_feat:n_feat + len(path)].copy_(vfeat[:len(path)])
            else:
                idx = torch.tensor(path, device=model.device)
                feats[n_feat:n_feat + len(path)].copy_(vfeat.index_select(0, idx))
            n_feat += len(path)
            stats.passes += 1
            stats.nodes += len(cand)
            stop = False
            for node in path[1:]:
                out.append(int(cand[node]))
                new += 1
                if new >= max_new or cand[node] == eos:
                    stop = True
                    break
            if stop:
                break
            pos += len(path)
            nxt = after
        if model.device.type == "cuda":
            torch.cuda.synchronize()
        stats.seconds = time.perf_counter() - t0
        stats.tokens = new
        return out, stats

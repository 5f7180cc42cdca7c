"""Attention over a K/V cache as a call of its own (fl_tree_attention), the weight that every cached key gathers
(fl_attention_weights), and eviction of the keys that gathered least (fl_evict).

The attention is that of the verify launch (reference kernels/verify_mega.cu:106-244, spec_tree.py:46-51): node m of a
sequence sits in cache slot pos + m and attends to [0, pos) and to pos + j where mask[m, j]. Caches are
[..., key heads, slots, dim], as Transformer's k_cache and v_cache; other orders come as transposed views.
"""
import math
import os

import torch

from . import _lib
from .quantize import workspace

# each operator in one call of the torch extension, for the arguments it takes as they are, as quantize's linears
_tree_attention_fast = _attention_weights_fast = _evict_fast = None
if "FLINT_AMD_LIB" not in os.environ:
    try:
        from ._torch_ops import attention_weights_fast as _attention_weights_fast
        from ._torch_ops import evict_fast as _evict_fast
        from ._torch_ops import tree_attention_fast as _tree_attention_fast
    except ImportError:
        pass


def _check(cond, text):
    if not cond:
        raise ValueError(text)


def _strides16(t, name):
    """t's strides, for the kernels' 16-byte loads."""
    _check(t.stride(-1) == 1 and all(s % 8 == 0 for s, n in zip(t.stride()[:-1], t.shape) if n > 1)
           and t.data_ptr() % 16 == 0,
           f"{name}: the last dimension must be contiguous, the other strides and the start on 16 bytes")
    return [s if n > 1 else 0 for s, n in zip(t.stride()[:-1], t.shape)]


def _describe(q, k, v, pos, mask, scale):
    """(desc, q, pos, mask) of checked arguments; q, pos and mask as the kernels take them, to be held until the launch."""
    for t, name in ((q, "q"), (k, "k_cache"), (v, "v_cache")):
        _check(t is None or t.is_cuda and t.dtype in (torch.bfloat16, torch.float16) and t.dtype == q.dtype
               and t.device == q.device, f"{name} must be a bf16 or fp16 CUDA (HIP) tensor of q's type and device")
        _check(t is None or t.dim() == 4, f"{name}: four dimensions (three for one sequence)")
    b, m, heads, dim = q.shape
    groups, slots = k.shape[1], k.shape[2]
    _check(k.shape[0] == b and k.shape[3] == dim and (v is None or v.shape == k.shape),
           "k_cache and v_cache must be [B, key heads, slots, dim] of q's [B, nodes, heads, dim]")
    _check(dim in (64, 128), "heads of 64 or 128 dimensions")
    _check(b >= 1 and m >= 1 and groups >= 1 and heads >= 1 and heads % groups == 0,
           "one sequence, node and head at least, and as many query heads for each key head")
    _check(m <= slots <= 1 << 30, "at least as many slots as nodes, at most 2^30")
    _check(b <= 65536 and m <= 32768 and heads <= 4096 and m * (heads // groups) <= 1 << 24,
           "at most 65536 sequences, 32768 nodes, 4096 heads and 2^24 rows of a key head")
    scale = dim ** -0.5 if scale is None else float(scale)
    _check(0.0 < scale < 3e38, "scale must be positive and finite")
    # queries are small: those that the kernels cannot load as they lie are copied, caches are not
    if q.stride(-1) != 1 or any(s % 8 for s, n in zip(q.stride()[:-1], q.shape) if n > 1) or q.data_ptr() % 16:
        q = q.clone(memory_format=torch.contiguous_format)
    d = _lib.AttnDesc(b=b, m=m, heads=heads, groups=groups, dim=dim, slots=slots, fp16=int(q.dtype == torch.float16),
                      scale=scale)
    d.q_b, d.q_m, d.q_h = _strides16(q, "q")
    _check((m - 1) * d.q_m + (heads - 1) * d.q_h + dim <= 1 << 30, "q: a sequence's queries within 2^30 values")
    d.k_b, d.k_g, d.k_s = _strides16(k, "k_cache")
    _check(d.k_s <= 1 << 23, "k_cache: slots at most 2^23 values apart")
    if v is not None:
        d.v_b, d.v_g, d.v_s = _strides16(v, "v_cache")
        _check(d.v_s <= 1 << 23, "v_cache: slots at most 2^23 values apart")
    if torch.is_tensor(pos) and pos.is_cuda:
        _check(pos.dtype in (torch.int32, torch.int64) and pos.numel() == b and pos.device == q.device,
               "pos: an int, or one int32 or int64 for each sequence on q's device")
        # a 64-bit position outside the cache stays outside it
        pos = (pos.clamp(-1, 2 ** 31 - 1) if pos.dtype == torch.int64 else pos).reshape(b).to(torch.int32).contiguous()
    else:
        _check(not torch.is_tensor(pos) or pos.numel() == 1, "pos: an int, or a device tensor")
        d.pos0, pos = int(pos), None
        _check(0 <= d.pos0 <= slots - m, f"pos must be 0 .. {slots - m}")
    if mask is not None:
        _check(mask.is_cuda and mask.device == q.device and mask.dtype in (torch.bool, torch.uint8),
               "mask must be bool or uint8, on q's device")
        _check(mask.shape in ((m, m), (b, m, m)), f"mask must be [{m}, {m}] or [{b}, {m}, {m}]")
        mask = mask.contiguous().view(torch.uint8)
        d.mask_b = m * m if mask.dim() == 3 and b > 1 else 0
    return d, q, pos, mask


def tree_attention(q, k_cache, v_cache, pos, mask=None, scale=None, return_lse=False):
    """Attention of the nodes of drafted trees (or chains, prompts, single tokens) over K/V caches, on the GPU.

    q bf16 or fp16 device [B, M, heads, dim], k_cache and v_cache [B, key heads, slots, dim] (without B: one sequence),
    dim 64 or 128; the nodes' own K and V are in the caches already. Strided caches are read as they lie, given a
    contiguous last dimension and the rest on 16 bytes. pos: cached keys before node 0, an int or a device int per
    sequence (one outside 0 .. slots - M gives NaN). mask bool or uint8 [M, M] or [B, M, M]: node i sees node j (None: a
    chain, j <= i). scale: of the scores, positive (None: dim ** -0.5). Returns the output in q's shape and type and, with
    return_lse, the log sum exp of the scaled scores (fp32 [B, M, heads]). A node that sees nothing gives 0 and -inf; an
    infinity or a NaN in the value of a slot that it sees makes that dimension the same, however small its weight
    (infinities of both signs: NaN). Calls of 2^32 threads or more (one token each of 65536 sequences of 128 key heads)
    raise FlError. No gradient."""
    if _tree_attention_fast is not None and q.is_cuda:
        at, p0 = (None, pos) if type(pos) is int else (pos, 0)
        if at is None or type(at) is torch.Tensor:
            r = _tree_attention_fast(q, k_cache, v_cache, at, p0, mask, q.shape[-1] ** -0.5 if scale is None else float(scale),
                                     return_lse, torch._C._cuda_getCurrentRawStream(q.get_device()))
            if r is not None:
                return r if return_lse else r[0]
    one = q.dim() == 3
    if one:
        q, k_cache, v_cache = q[None], k_cache[None], v_cache[None]
    q, k_cache, v_cache = q.detach(), k_cache.detach(), v_cache.detach()
    d, q, pos, mask = _describe(q, k_cache, v_cache, pos, mask, scale)
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    lse = torch.empty(q.shape[:3], dtype=torch.float32, device=q.device) if return_lse else None
    with torch.cuda.device(q.device):
        ref = _lib.ctypes.byref(d)
        work = workspace("fl_tree_attention_workspace", ref, int(pos is None), device=q.device)
        _lib.call("fl_tree_attention", ref, _lib.ptr(q), _lib.ptr(k_cache), _lib.ptr(v_cache), _lib.ptr(pos),
                  _lib.ptr(mask), _lib.ptr(out), _lib.ptr(lse), _lib.ptr(work), _lib.stream_ptr())
    if one:
        out, lse = out[0], None if lse is None else lse[0]
    return (out, lse) if return_lse else out


def attention_weights(q, k_cache, lse, pos, mask=None, scale=None, out=None):
    """The attention weight that each slot of a cache gathers from the nodes: fp32 [B, key heads, slots], the sum over
    the nodes and the query heads of a key head of softmax's probability; 0 in slots that no node sees. Arguments as
    tree_attention's, lse as it returns it. out: a contiguous tensor of that shape to add to (slots from pos + M on are
    left as they are); it is returned. Sums have a fixed order."""
    if _attention_weights_fast is not None and out is None and q.is_cuda:
        at, p0 = (None, pos) if type(pos) is int else (pos, 0)
        if at is None or type(at) is torch.Tensor:
            r = _attention_weights_fast(q, k_cache, lse, at, p0, mask, q.shape[-1] ** -0.5 if scale is None else float(scale),
                                        torch._C._cuda_getCurrentRawStream(q.get_device()))
            if r is not None:
                return r
    one = q.dim() == 3
    if one:
        q, k_cache, lse = q[None], k_cache[None], lse[None]
    q, k_cache = q.detach(), k_cache.detach()
    d, q, pos, mask = _describe(q, k_cache, None, pos, mask, scale)
    _check(lse.is_cuda and lse.device == q.device and lse.dtype == torch.float32 and lse.shape == q.shape[:3],
           "lse must be fp32 [B, M, heads] on q's device")
    lse = lse.detach().contiguous()
    add = out is not None
    if add:
        want = k_cache.shape[1:3] if one else k_cache.shape[:3]
        _check(out.is_cuda and out.device == q.device and out.dtype == torch.float32 and out.shape == want
               and out.is_contiguous(), f"out must be a contiguous fp32 tensor of {tuple(want)} on q's device")
    else:
        out = torch.empty(k_cache.shape[1:3] if one else k_cache.shape[:3], dtype=torch.float32, device=q.device)
    with torch.cuda.device(q.device):
        _lib.call("fl_attention_weights", _lib.ctypes.byref(d), _lib.ptr(q), _lib.ptr(k_cache), _lib.ptr(lse),
                  _lib.ptr(pos), _lib.ptr(mask), _lib.ptr(out), int(add), _lib.stream_ptr())
    return out


def _rows(t, lead, name):
    """fl_rows of t [*lead, slots, dim], its leading dimensions as an outer and an inner one: ((outer, inner), rows)."""
    _check(t.is_cuda and t.element_size() * t.shape[-1] % 16 == 0 and t.stride(-1) == 1 and t.data_ptr() % 16 == 0
           and t.dim() == len(lead) + 2 and tuple(t.shape[:-2]) == tuple(lead),
           f"{name}: a CUDA (HIP) tensor [..., slots, dim] of the same leading dimensions, its rows whole 16 bytes")
    es = t.element_size()
    dims = [(n, s) for n, s in zip(t.shape[:-2], t.stride()[:-2]) if n > 1]
    merged = []
    for n, s in dims:  # dimensions that lie behind each other are one
        if merged and merged[-1][1] == n * s:
            merged[-1] = (merged[-1][0] * n, s)
        else:
            merged.append((n, s))
    return merged, [s * es for _, s in merged], t.stride(-2) * es if t.shape[-2] > 1 else t.shape[-1] * es


def evict(k_cache, v_cache, weights, n, keep, recent=0, sink=0, out=None):
    """Cuts each head's cache to the `keep` slots that matter: of the slots [0, n) the first `sink`, the last `recent`
    and of the others those of the largest weight (equal ones: the lower slot; a NaN counts as the largest). Their rows
    move, in order, to the slots 0 .. keep - 1.

    k_cache, v_cache: device [..., slots, dim] of any type (rows of whole 16 bytes, at most 4096), strided in the
    leading dimensions and between slots; weights: contiguous fp32 [..., slots]. In place (out None) the weights move
    with the rows, those of keep .. n - 1 become 0, and the rows there stay what they were. out = (k, v) or (k, v, weights) of
    [..., keep or more, ...] takes them instead and leaves the caches alone; it must not overlap them. What is written
    must not overlap itself or each other either; K and V may lie between each other's rows. Returns the kept slots, int32
    [..., keep], rising. keep >= n keeps all."""
    if _evict_fast is not None and k_cache.is_cuda and (out is None or len(out) in (2, 3)):
        ko, vo, wo = (None, None, None) if out is None else out if len(out) == 3 else (*out, None)
        kept = _evict_fast(k_cache, v_cache, weights, n, keep, recent, sink, ko, vo, wo,
                           torch._C._cuda_getCurrentRawStream(k_cache.get_device()))
        if kept is not None:
            return kept
    lead = k_cache.shape[:-2]
    _check(k_cache.dim() >= 2 and v_cache.shape == k_cache.shape and v_cache.dtype == k_cache.dtype
           and v_cache.device == k_cache.device, "k_cache and v_cache must be of one shape, type and device")
    dev, slots = k_cache.device, k_cache.shape[-2]
    _check(slots <= 1 << 30, "at most 2^30 slots")
    _check(weights.is_cuda and weights.device == dev and weights.dtype == torch.float32
           and weights.shape == k_cache.shape[:-1] and weights.is_contiguous(),
           "weights must be contiguous fp32 [..., slots] on the caches' device")
    n, recent, sink = int(n), int(recent), int(sink)
    _check(0 <= n <= slots, f"n must be 0 .. {slots}")
    keep = min(int(keep), n)
    _check(n == 0 or keep >= 1, "keep must be 1 or more")
    _check(recent >= 0 and sink >= 0, "recent and sink must not be negative")
    if keep < n:
        _check(recent + sink <= keep, "recent and sink together must not exceed keep")
    else:  # nothing leaves
        recent = sink = 0
    heads = math.prod(lead)
    _check(heads <= 65535, "at most 65535 heads")
    row_bytes = k_cache.shape[-1] * k_cache.element_size()
    _check(row_bytes <= 4096, "rows of at most 4096 bytes")
    tensors = [(k_cache, "k_cache"), (v_cache, "v_cache")]
    if out is not None:
        _check(len(out) in (2, 3), "out must be (k, v) or (k, v, weights)")
        for t, name in ((out[0], "out k"), (out[1], "out v")):
            _check(t.dtype == k_cache.dtype and t.device == dev and t.dim() == k_cache.dim() and t.shape[-1] == k_cache.shape[-1]
                   and t.shape[-2] >= keep and t.shape[-2] == out[0].shape[-2],
                   f"{name} must be [..., {keep} or more, {k_cache.shape[-1]}] of the caches' type and device")
            tensors.append((t, name))
        if len(out) == 3 and out[2] is not None:
            _check(out[2].is_cuda and out[2].device == dev and out[2].dtype == torch.float32 and out[2].is_contiguous()
                   and out[2].shape == out[0].shape[:-1], "out weights must be contiguous fp32 of out k's slots")
        for t in [x for x in out if x is not None]:
            for src in (k_cache, v_cache, weights):
                _check(not _overlap(t, src), "out must not overlap the caches or the weights")
    # what is written: no row twice, and none by two workgroups that do not wait for each other
    written, name = ((k_cache, v_cache, weights), "caches") if out is None else ((*out, None)[:3], "out")
    for t in written[:2]:
        _check(t.numel() == 0 or _apart(t), f"{name}: rows that heads or slots share cannot be written")
        _check(written[2] is None or not _overlap(t, written[2]), f"{name}: K and V must not overlap the weights")
    _check(not _rows_meet(*written[:2]), f"{name}: K and V must not be the same memory")
    kept = torch.empty(*lead, keep, dtype=torch.int32, device=dev)
    if heads == 0 or n == 0:
        return kept
    described = [_rows(t, lead, name) for t, name in tensors]
    # one split of the heads into outer and inner that fits every tensor
    shapes = [[m[0] for m in merged] for merged, _, _ in described]
    widest = max(shapes, key=len)
    _check(len(widest) <= 2, "leading dimensions of more than two different strides")
    inner = widest[1] if len(widest) == 2 else 1
    rows = []
    for (t, name), (merged, strides, row) in zip(tensors, described):
        if len(merged) == 2:
            _check([m[0] for m in merged] == widest, f"{name}: its leading dimensions split otherwise than the others'")
            o, i = strides
        elif len(merged) == 1:
            o, i = strides[0] * inner, strides[0] if inner > 1 else 0
        else:
            o = i = 0
        _check(o % 16 == 0 and i % 16 == 0 and row % 16 == 0, f"{name}: strides must be whole 16 bytes")
        rows.append(_lib.Rows(t.data_ptr(), o, i, row))
    ref = [_lib.ctypes.byref(r) for r in rows] + [None] * (4 - len(rows))
    w_out = out[2] if out is not None and len(out) == 3 else None
    with torch.cuda.device(dev):
        _lib.call("fl_evict", ref[0], ref[1], _lib.ptr(weights), heads // inner, inner, slots, row_bytes, n, keep, recent,
                  sink, _lib.ptr(kept), ref[2], ref[3], _lib.ptr(w_out), 0 if out is None else out[0].shape[-2],
                  _lib.stream_ptr())
    return kept


def _apart(t):
    """Whether t's elements are all at addresses of their own, dimension within dimension (so that no row is another's)."""
    extent = 1
    for s, n in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n > 1):
        if s < extent:
            return False
        extent += (n - 1) * s
    return True


def _rows_meet(a, b):
    """Whether K and V share memory; both _apart. Two views of other strides whose spans meet count as sharing; views of the
    same strides may lie between each other, as K and V of a slot next to each other do."""
    if not _overlap(a, b):
        return False
    dims = sorted(((s, n) for s, n in zip(a.stride(), a.shape) if n > 1), reverse=True)
    if dims != sorted(((s, n) for s, n in zip(b.stride(), b.shape) if n > 1), reverse=True):
        return True
    d, odd = divmod(b.data_ptr() - a.data_ptr(), a.element_size())

    def meet(d, i):  # two elements d apart in a's dimensions from i on: of the outer one, the multiple below d or above it
        if i == len(dims):
            return d == 0
        s, n = dims[i]
        return any(abs(k) < n and meet(d - k * s, i + 1) for k in (d // s, d // s + 1))
    return odd != 0 or meet(d, 0)


def _overlap(a, b):
    """Whether the memory that two tensors span meets."""
    def span(t):
        end = t.data_ptr() + (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * t.element_size()
        return (t.data_ptr(), end) if t.numel() else (0, 0)
    (a0, a1), (b0, b1) = span(a), span(b)
    return a0 < b1 and b0 < a1

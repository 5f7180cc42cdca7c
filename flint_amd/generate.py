"""Greedy generation loop over the HIP decode kernel.

Mirrors reference engine/generate.py:57-81,137-206 (prefill / decode_one_token / decode_n_tokens /
generate) for greedy sampling and chat.py:71-96 (logits_at / pick / respond). Tokens stay on
the device between steps: step i reads the token step i-1 wrote, so the loop issues launches
back-to-back with no host synchronisation (gpt-fast's decode loop has none either). The prompt
runs as GEMM passes over up to 1024 tokens (fl_prefill), a short one through the verify kernel.
"""
import os
from collections import namedtuple

import torch

# the whole of logprobs / head_logprobs as one call of the torch extension, as quantize's linears
_logprobs_fast = _head_logprobs_fast = None
if "FLINT_AMD_LIB" not in os.environ:
    try:
        from ._torch_ops import head_logprobs_fast as _head_logprobs_fast
        from ._torch_ops import logprobs_fast as _logprobs_fast
    except ImportError:
        pass

# prompts of more tokens than this run as fl_prefill passes: up to 16 tokens are one token pass of the verify
# launch (flint-3b, 40 layers: 16 tokens 1.8 ms against 2.6 in a pass, 24 tokens 2.8 against 2.6)
PREFILL_MIN = 16


def prefill(model, x, input_pos, chunk=32):
    """Feed prompt tokens x (int32 device [T]) at positions input_pos[0]..; returns the greedy next
    token (int32 device [1]) after the last one (reference engine/generate.py:57-60, which runs
    the prompt through one forward). With the default chunk, more than PREFILL_MIN tokens go through
    fl_prefill, up to 1024 per pass. Fewer, or a smaller chunk, go through the verify kernel
    `chunk` (<= 32) tokens per launch with a causal mask: each launch reads every weight once for
    the whole chunk and appends the chunk's K/V rows."""
    from . import _lib
    x = x.reshape(-1).to(device=model.device, dtype=torch.int32)
    p0 = int(input_pos.reshape(-1)[0]) if torch.is_tensor(input_pos) else int(input_pos)
    chunk = max(1, min(int(chunk), _lib.MAX_VERIFY))
    n = x.numel()
    out = torch.empty(1, dtype=torch.int32, device=model.device)
    if n == 0:
        return out
    if chunk == _lib.MAX_VERIFY and n > PREFILL_MIN and hasattr(model, "prefill"):
        try:
            return model.prefill(x, p0, out)
        except torch.OutOfMemoryError:
            pass  # no room for its workspace: the verify launches need none
    cache = getattr(model, "_prefill_masks", None)
    if cache is None:
        cache = model._prefill_masks = {}
    for s in range(0, n, chunk):
        m = min(chunk, n - s)
        if m not in cache:
            cache[m] = (torch.arange(m, dtype=torch.int32, device=model.device),
                        torch.tril(torch.ones(m, m, dtype=torch.uint8, device=model.device)),
                        torch.empty(m, model.config.vocab_size, dtype=torch.float32, device=model.device),
                        torch.empty(m, model.config.dim, dtype=torch.bfloat16, device=model.device),
                        torch.empty(m, dtype=torch.int32, device=model.device))
        depth, amask, logits, feat, toks = cache[m]
        model.verify(x[s:s + m], p0 + s, depth=depth, amask=amask, logits=logits, feat=feat,
                     tokens_out=toks)
    out.copy_(toks[m - 1:m])
    return out


def sample(logits, temperature=1.0, top_k=None, seed=0, offset=0, noise=None, probs=False):
    """Sample one token per logit row on the GPU (reference engine/generate.py:36-55:
    logits_to_probs + multinomial_sample_one_no_sync). logits: fp32 device [V] or [rows, V]
    (bf16 values, as the decode and verify kernels write them). The exponential noise comes from
    Philox4x32-10 keyed by `seed` at counter (index, row, offset), or from `noise` (same shape as
    logits). Returns (tokens int32 device [rows], probs fp32 [rows, V] or None)."""
    from . import _lib
    lg = logits.float().contiguous()
    rows, vocab = (1, lg.numel()) if lg.dim() == 1 else (lg.shape[0], lg.shape[-1])
    if top_k is not None and int(top_k) < 1:
        raise ValueError("top_k must be >= 1")
    out = torch.empty(rows, dtype=torch.int32, device=lg.device)
    pr = torch.empty(rows, vocab, dtype=torch.float32, device=lg.device) if probs else None
    nz = None if noise is None else noise.float().contiguous()
    if nz is not None and nz.numel() != lg.numel():
        raise ValueError("noise must have the logits' shape")
    _lib.call("fl_sample", _lib.ptr(lg), rows, vocab, float(temperature), int(top_k or 0),
              int(seed) & (2 ** 64 - 1), int(offset) & (2 ** 64 - 1), _lib.ptr(nz), _lib.ptr(out),
              _lib.ptr(pr), _lib.stream_ptr())
    return out, pr


def logits_to_probs(logits, temperature=1.0, top_k=None):
    """Reference generate.py:41-49 on the GPU: probs fp32 device (bf16 values), logits' shape."""
    _, pr = sample(logits, temperature, top_k, probs=True)
    return pr.view(logits.shape)


# What logprobs and head_logprobs return, for R rows of logits: logprob fp32 [R] and rank int32 [R] of the tokens
# given (None without tokens), entropy fp32 [R], top_ids int32 and top_logprobs fp32 [R, top] (None for top = 0).
TokenLogprobs = namedtuple("TokenLogprobs", "logprob entropy rank top_ids top_logprobs")

TOP_MAX = 32  # alternatives at most


def _logprob_outputs(rows, tokens, top, dev):
    f32, i32 = dict(dtype=torch.float32, device=dev), dict(dtype=torch.int32, device=dev)
    return TokenLogprobs(torch.empty(rows, **f32) if tokens is not None else None, torch.empty(rows, **f32),
                         torch.empty(rows, **i32) if tokens is not None else None,
                         torch.empty(rows, top, **i32) if top else None, torch.empty(rows, top, **f32) if top else None)


def _check_logprob_args(rows, vocab, tokens, top, dev):
    """tokens as the kernels take them: int32 [rows] or None."""
    if not 0 <= top <= min(TOP_MAX, vocab):
        raise ValueError(f"top must be 0..{min(TOP_MAX, vocab)}")
    if rows > 1 << 17 or not 1 <= vocab <= 1 << 20:
        raise ValueError("at most 2^17 rows and a vocabulary of 1..2^20")
    if tokens is None:
        return None
    if tokens.device != dev or tokens.dtype not in (torch.int32, torch.int64):
        raise ValueError("tokens must be int32 or int64, on the logits' device")
    if tokens.numel() != rows:
        raise ValueError(f"tokens: {tokens.numel()} ids for {rows} rows")
    return _ids(tokens).contiguous()


def _ids(tokens):
    """tokens as int32 [n]; 64-bit ids outside the vocabulary stay outside it."""
    tokens = tokens.reshape(-1)
    return (tokens.clamp(-1, 2 ** 31 - 1) if tokens.dtype == torch.int64 else tokens).to(torch.int32)


def logprobs(logits, tokens=None, top=0):
    """Log probabilities of rows of logits (fp32 or bf16 device [V] or [..., V], strided rows too) on the GPU, in one
    pass over them (fl_logprobs): of tokens (int, one per row; an id outside the vocabulary, as a padded row has,
    gives NaN and rank -1) the log probability and the rank (0: the most likely; equal logits rank by
    index), of every row the entropy in nats and the `top` (up to 32) most likely ids with their log probabilities. A
    logit of -inf (a masked token) has probability 0; a row with nothing but -inf, or with a NaN or a +inf, gives NaN.
    Alternatives take several times as long (of many rows up to sixty times) where masks of the type's lowest value
    leave a handful of tokens, or masks of -inf one range of ids that does not begin at the row's start.
    Returns TokenLogprobs over the flattened rows; they carry no gradient."""
    top = int(top)
    if _logprobs_fast is not None and logits.is_cuda:
        r = _logprobs_fast(logits, tokens, top, torch._C._cuda_getCurrentRawStream(logits.get_device()))
        if r is not None:
            return TokenLogprobs(*r)
    from . import _lib  # here: the two lines take 1.5 us
    from .quantize import workspace
    if not logits.is_cuda or logits.dtype not in (torch.float32, torch.bfloat16):
        raise ValueError("logits must be an fp32 or bf16 CUDA (HIP) tensor")
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError("logits must be [..., V]")
    vocab = logits.shape[-1]
    lg = logits.detach()
    lg = lg.reshape(-1, vocab) if lg.dim() != 2 else lg
    rows = lg.shape[0]
    if rows and (lg.stride(1) != 1 or (rows > 1 and lg.stride(0) < vocab)):
        lg = lg.contiguous()
    tokens = _check_logprob_args(rows, vocab, tokens, top, lg.device)
    out = _logprob_outputs(rows, tokens, top, lg.device)
    if rows:
        with torch.cuda.device(lg.device):
            work = workspace("fl_logprobs_workspace", rows, vocab, top, device=lg.device)
            _lib.call("fl_logprobs", _lib.ptr(lg), int(lg.dtype == torch.bfloat16), lg.stride(0), rows, vocab,
                      _lib.ptr(tokens), top, *map(_lib.ptr, out), _lib.ptr(work), _lib.stream_ptr())
    return out


def head_logprobs(feat, weight, scales, tokens=None, top=0):
    """logprobs of the logits that an 8-bit vocabulary head (weight int8 [V, K], scales fp32 [V], as of
    quantize.DynamicInt8Linear) gives for features (bf16 device [..., K], as of verify, prefill or decode), without
    all of those logits in memory (fl_head_logprobs). The logits are fp32 and exact integer sums behind two scales, so
    a row's ranks and ids do not depend on the batch it is scored in."""
    top = int(top)
    if _head_logprobs_fast is not None and feat.is_cuda:
        r = _head_logprobs_fast(feat, weight, scales, tokens, top,
                                torch._C._cuda_getCurrentRawStream(feat.get_device()))
        if r is not None:
            return TokenLogprobs(*r)
    from . import _lib
    from .quantize import _check_weight, aligned16, workspace
    _check_weight(weight, scales)
    n, k = weight.shape
    if not feat.is_cuda or feat.dtype != torch.bfloat16:
        raise ValueError("feat must be a torch.bfloat16 CUDA (HIP) tensor")
    if feat.dim() < 1 or feat.shape[-1] != k or feat.device != weight.device:
        raise ValueError(f"feat must be [..., {k}], on the weight's device")
    x = aligned16(feat.detach().reshape(-1, k).contiguous())
    rows = x.shape[0]
    tokens = _check_logprob_args(rows, n, tokens, top, x.device)
    out = _logprob_outputs(rows, tokens, top, x.device)
    if rows:
        wa = aligned16(weight)
        with torch.cuda.device(x.device):
            work = workspace("fl_head_logprobs_workspace", rows, n, k, top, device=x.device)
            _lib.call("fl_head_logprobs", _lib.ptr(x), _lib.ptr(wa), _lib.ptr(scales), _lib.ptr(tokens),
                      top, *map(_lib.ptr, out), _lib.ptr(work), rows, n, k, _lib.stream_ptr())
    return out


@torch.no_grad()
def score(model, tokens, top=0, head=None):
    """How likely a text is to the model: TokenLogprobs of tokens[1:] (int device [T], T from 2 to block_size + 1),
    row i of the distribution after tokens[:i + 1] at tokens[i + 1]. The K/V rows of tokens[:-1] are in the cache
    afterwards: to go on, feed tokens[-1] at position T - 1.

    head None: the model's own bf16 LM head, through the verify kernel's logits, 32 tokens at a time. head a
    quantize.DynamicInt8Linear (Transformer.int8_head): one pass over the prompt and its features through the
    8-bit head."""
    from . import _lib
    x = _ids(tokens.to(model.device))
    n = x.numel() - 1
    if n < 1:
        raise ValueError("score needs two tokens or more")
    if head is None:  # refusals before the model has run
        _check_logprob_args(1, model.config.vocab_size, None, int(top), model.device)
    else:
        _check_logprob_args(n, head.weight.shape[0], None, int(top), model.device)
    # the last token takes no position here; room for it, to decode on from it, where there is one (caches come in eights)
    model.setup_caches(1, n + 1 if n + 1 <= model.packed.rope.shape[0] // 8 * 8 else n)
    if head is not None:
        return head_logprobs(model.prefill_features(x[:n], 0), head.weight, head.scales, x[1:], top)
    parts = []
    for s in range(0, n, _lib.MAX_VERIFY):
        e = min(n, s + _lib.MAX_VERIFY)
        _, logits, _ = model.verify(x[s:e], s, feat=False)
        parts.append(logprobs(logits, x[s + 1:e + 1], top))
    return TokenLogprobs(*(None if f[0] is None else torch.cat(f) for f in zip(*parts)))


def decode_one_token(model, x, input_pos, logits=None, temperature=None, top_k=None, seed=0):
    """(next_token int32 device [1], logits) for one token at input_pos: greedy, or sampled when
    temperature or top_k is given (reference generate.py:62-66, sample at :52-55), with the
    position as the noise counter."""
    pos = int(input_pos.reshape(-1)[0]) if torch.is_tensor(input_pos) else int(input_pos)
    if logits is None:
        logits = torch.empty(model.config.vocab_size, dtype=torch.float32, device=model.device)
    out = torch.empty(1, dtype=torch.int32, device=model.device)
    tok = x.reshape(-1)[:1].to(torch.int32)
    if temperature is not None or top_k is not None:  # sampled in the decode launch itself
        t = 1.0 if temperature is None else temperature
        model.decode_sample(tok, pos, t, top_k, seed=seed, offset=pos, token_out=out, logits=logits)
    else:
        model.decode_step(tok, pos, token_out=out, logits=logits)
    return out, logits


def decode_n_tokens(model, cur_token, input_pos, num_new_tokens, out=None):
    """Greedy-decode num_new_tokens tokens after cur_token (int32 device [1]) at input_pos.
    Returns int32 device [num_new_tokens]; no host synchronisation inside the loop."""
    pos = int(input_pos.reshape(-1)[0]) if torch.is_tensor(input_pos) else int(input_pos)
    buf = torch.empty(num_new_tokens + 1, dtype=torch.int32, device=model.device)
    buf[:1] = cur_token.reshape(-1)[:1]
    for i in range(num_new_tokens):
        model.decode_step(buf[i:i + 1], pos + i, token_out=buf[i + 1:i + 2])
    if out is not None:
        out.copy_(buf[1:])
        return out
    return buf[1:]


@torch.no_grad()
def generate(model, prompt, max_new_tokens, temperature=None, top_k=None, seed=0, logprobs=None):
    """Generate: returns int32 device [T + max_new_tokens] = prompt + new tokens. Greedy (the
    argmax fused into the decode kernel) unless temperature or top_k is given; then each step
    samples in the decode launch itself (fl_decode_sample) with the step's position as the noise
    counter. Tokens stay on the device either way (no host synchronisation in the loop).
    logprobs = n (0..32): (tokens, TokenLogprobs of the new ones with n alternatives each) of the
    model's own distribution, before temperature and top_k."""
    if logprobs is not None:
        _check_logprob_args(1, model.config.vocab_size, None, int(logprobs), model.device)
    prompt = prompt.reshape(-1).to(device=model.device, dtype=torch.int32)
    T = prompt.numel()
    model.setup_caches(1, T + max_new_tokens)
    seq = torch.empty(T + max_new_tokens, dtype=torch.int32, device=model.device)
    seq[:T] = prompt
    if T > 1:
        prefill(model, prompt[:-1], 0)
    sampled = temperature is not None or top_k is not None
    t = 1.0 if temperature is None else temperature
    said, logits = [], None
    if logprobs is not None:
        logits = torch.empty(model.config.vocab_size, dtype=torch.float32, device=model.device)
    # the last prompt token produces the first new token
    for i in range(max_new_tokens):
        p = T - 1 + i
        out = seq[p + 1:p + 2]
        if sampled:
            model.decode_sample(seq[p:p + 1], p, t, top_k, seed=seed, offset=p, token_out=out, logits=logits)
        else:
            model.decode_step(seq[p:p + 1], p, token_out=out, logits=logits)
        if logits is not None:
            said.append(_logprobs(logits, out, logprobs))
    if logits is None:
        return seq
    if not said:
        return seq, _logprob_outputs(0, seq[:0], int(logprobs), seq.device)
    return seq, TokenLogprobs(*(None if f[0] is None else torch.cat(f) for f in zip(*said)))


_logprobs = logprobs  # generate's argument of that name hides it there

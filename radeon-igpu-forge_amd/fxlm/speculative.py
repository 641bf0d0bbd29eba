"""fxlm.speculative: drafted decoding, besides its attention (fxlm.attention.tree_attention).

A draft model proposes a tree of tokens behind each sequence; the target model runs the whole tree
in one pass (GPT.tree_step), ``sampling_probs`` turns its logits into the probabilities that
GPT.generate would sample from, ``verify_draft`` accepts a path of the tree so that the accepted
tokens and the one after them are distributed as the target's own samples, and ``compact_cache``
moves the path's keys and values together in every layer's cache.  The reference has no drafting
(its ml/fxlm/sample.py:62-73 samples one token a pass).  All of it is inference: what these functions
return has no gradient, whatever their inputs require.

A tree is two (B, N) tensors: tokens, and parents (a node's parent lies below it).  Node 0 is the
root, the sequence's last token, whose key is not in the cache yet; a node with a parent of -1 is
padding.
"""
import torch

from fxgpu.abi import host


def _taken(r, name):
    """r, what the host module returned, which is None for what none of the checks names"""
    if r is None:
        raise ValueError(f"{name}: tensors of a layout or size that it does not take")
    return r


def sampling_probs(logits, temperature=1.0, top_k=0):
    """logits (..., V) fp32 or bf16 -> probabilities (..., V) fp32: softmax(logits / temperature)
    over each row's top_k largest logits and the equals of the last of them (over all for
    top_k <= 0), as GPT.generate samples.  A row of -inf gives zeros; NaN or +inf gives NaN.  Without
    a gradient (inference)."""
    if not 1e-30 <= float(temperature) <= 1e30:
        raise ValueError(f"temperature {temperature} must lie in [1e-30, 1e30]")
    r = host.sampling_probs(logits, float(temperature), int(top_k))
    if r is None:
        if logits.dtype not in (torch.float32, torch.bfloat16):
            raise TypeError(f"logits must be float32 or bfloat16, got {logits.dtype}")
        if not logits.is_cuda:
            raise TypeError("logits must be a cuda tensor")
        if logits.dim() < 1 or logits.shape[-1] < 1:
            raise ValueError(f"logits must be (..., V), got {tuple(logits.shape)}")
        x = logits.contiguous()   # a slice of positions, or rows at an odd address
        r = host.sampling_probs(x if x.data_ptr() % 16 == 0 else x.clone(), float(temperature), int(top_k))
    return _taken(r, "sampling_probs")


def verify_draft(probs, tokens, parents, uniform, draft_probs=None):
    """Accept a path of each sequence's tree against the target's probabilities.

    probs (B, N, V) fp32: row i is the target's distribution after node i.  tokens (B, N) int64,
    parents (B, N) int32 cuda: the tree.  uniform (B, N) fp32: independent numbers of [0, 1), one
    a node (the root's draws the last token).  draft_probs (B, N, V) fp32: row i is the
    distribution that node i's children were drawn from, independently (the row of a node without
    children may hold anything); None: proposals without one (looked up, or the likeliest), each
    certain of its token.  N <= 64, V <= 1,048,576.

    From the root, the children of the node that is reached are asked in their order.  One with
    token x is accepted with probability min(1, p(x) / q(x)); a refusal leaves
    norm(max(p - q, 0)) as the target's distribution for the next (without draft_probs: p without
    x).  Where none is accepted the last token is drawn from what is left: the first whose running
    sum passes uniform[b, 0] times the whole (from the row itself where nothing is left; -1 where
    that has no mass).  Sums are in 64 bits.  Nodes whose token is no id below V are never asked.

    Returns tokens (B, N) int64 (the accepted ones and the last, then -1), path (B, N) int32 (the
    accepted nodes, 0 first, then -1) and counts (B,) int32, the length of both.
    """
    r = host.verify_draft(probs, tokens, parents, uniform, draft_probs)
    if r is None:
        if probs.dim() != 3:
            raise ValueError(f"probs must be (B, N, V), got {tuple(probs.shape)}")
        B, N, V = probs.shape
        if N < 1 or N > 64 or V < 1:
            raise ValueError(f"probs {tuple(probs.shape)}: a tree has 1 to 64 nodes")
        for nm, t, want, shape in (("probs", probs, torch.float32, (B, N, V)), ("tokens", tokens, torch.int64, (B, N)),
                                   ("parents", parents, torch.int32, (B, N)), ("uniform", uniform, torch.float32, (B, N)),
                                   ("draft_probs", draft_probs, torch.float32, (B, N, V))):
            if t is None:
                continue
            if t.dtype != want:
                raise TypeError(f"{nm} must be {want}, got {t.dtype}")
            if not t.is_cuda:
                raise TypeError(f"{nm} must be a cuda tensor")
            if tuple(t.shape) != shape:
                raise ValueError(f"{nm} must be {shape}, got {tuple(t.shape)}")
        p, q = (None if t is None else t.contiguous() if t.data_ptr() % 16 == 0 else t.clone(memory_format=torch.contiguous_format)
                for t in (probs, draft_probs))
        r = host.verify_draft(p, tokens.contiguous(), parents.contiguous(), uniform.contiguous(), q)
    return _taken(r, "verify_draft")


def compact_cache(cache, ctx, path, counts):
    """Move each sequence's accepted rows together: in every tensor of cache, a list of (k, v)
    pairs (B, Tmax, Hkv, Dh) bf16 (GPT.init_cache's), row ctx[b] + path[b, d] to row ctx[b] + d
    for d < counts[b].  ctx, counts (B,) and path (B, N) int32 cuda, a path ascending
    (verify_draft's); entries outside the cache are passed over.  A tensor that is in the list more
    than once (layers that share one) is compacted once.  In place; returns ctx + counts, the new
    lengths, which count the entries that are passed over.  Rows past them keep what they held."""
    r = host.compact_cache(cache, ctx, path, counts)
    if r is None:
        flat = [t for kv in cache for t in kv]
        if not flat:
            raise ValueError("cache holds no tensors")
        s = flat[0].shape
        for t in flat:
            if any(st == 0 and n > 1 for st, n in zip(t.stride(), t.shape)):
                raise ValueError("an expanded cache cannot be compacted")
            if t.dtype != torch.bfloat16 or not t.is_cuda:
                raise TypeError("caches must be bfloat16 cuda tensors")
            if t.dim() != 4 or t.shape != s or min(s) < 1 or s[3] % 8 or s[0] > 65535:
                raise ValueError(f"caches must share one shape (B, Tmax, Hkv, Dh), Dh a multiple of 8: {tuple(t.shape)}")
            if t.stride(-1) != 1 or any(x % 8 for x in t.stride()[:-1]) or t.data_ptr() % 16:
                raise ValueError("caches: last dim must be contiguous, other strides multiples of 8 "
                                 "elements and the base 16-byte aligned")
        for nm, t in (("ctx", ctx), ("path", path), ("counts", counts)):
            if t.dtype != torch.int32 or not t.is_cuda:
                raise TypeError(f"{nm} must be an int32 cuda tensor")
        if tuple(ctx.shape) != (s[0],) or tuple(counts.shape) != (s[0],) or path.dim() != 2 or path.shape[0] != s[0] or path.shape[1] < 1:
            raise ValueError(f"ctx and counts ({s[0]},), path ({s[0]}, N): {tuple(ctx.shape)} {tuple(counts.shape)} {tuple(path.shape)}")
        r = host.compact_cache(cache, ctx.contiguous(), path.contiguous(), counts.contiguous())
    return _taken(r, "compact_cache")

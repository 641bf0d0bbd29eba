"""Drafted decoding in 64 bits: attention of a tree of tokens over a cache, the probabilities that
are sampled from, the verification of drafted tokens, and the cache's compaction.  Plain loops over
the definitions; the reference has no counterpart (its ml/fxlm/sample.py:62-73 samples a token a
pass)."""
import math

import numpy as np
import torch


def ancestors(parents):
    """(N,) int64 bit sets of a tree given by its parents (-1: the root's, and padding's): a node's
    own bit and its ancestors'; 0 for padding."""
    bits = []
    for i, p in enumerate(parents):
        bits.append(1 if i == 0 else 0 if p < 0 else bits[p] | 1 << i)
    return torch.tensor([b - (1 << 64) if b >> 63 else b for b in bits], dtype=torch.int64)


def tree_attention(q, k, v, ctx, tree, first=0, scale=None, k_new=None, v_new=None):
    """(o, lse, size, k, v): o (B,N,H,Dh) and lse (B,N,H) float64; size the sum of p |v| / sum p, what
    roundings of p are relative to; k, v the caches after the call."""
    B, N, H, D = q.shape
    T, Hkv = k.shape[1:3]
    scale = 1 / math.sqrt(D) if scale is None else scale
    k, v = k.clone(), v.clone()
    o = torch.zeros(B, N, H, D, dtype=torch.float64)
    size = torch.zeros_like(o)
    lse = torch.full((B, N, H), -math.inf, dtype=torch.float64)
    for b in range(B):
        c = min(max(int(ctx[b]), 0), T)
        bits = [int(x) & (2 ** 64 - 1) for x in tree[b]]
        real = [bits[i] >> (first + i) & 1 for i in range(N)]
        if k_new is not None:
            for i in range(N):
                if real[i] and c + first + i < T:
                    k[b, c + first + i], v[b, c + first + i] = k_new[b, i], v_new[b, i]
        for i in range(N):
            if not real[i]:
                continue
            rows = list(range(c)) + [c + j for j in range(first + N) if bits[i] >> j & 1 and c + j < T
                                     and (j < first or real[j - first])]
            if not rows:
                continue
            for h in range(H):
                kk, vv = k[b, rows, h * Hkv // H].double(), v[b, rows, h * Hkv // H].double()
                s = scale * (kk @ q[b, i, h].double())
                m = s.max()
                p = torch.exp(s - m)
                o[b, i, h] = (p @ vv) / p.sum()
                size[b, i, h] = (p @ vv.abs()) / p.sum()
                lse[b, i, h] = m + p.sum().log()
    return o, lse, size, k, v


def sampling_probs(logits, temperature=1.0, top_k=0):
    x = logits.double()
    if 0 < top_k < x.shape[-1]:
        kth = x.sort(-1, descending=True).values[..., top_k - 1:top_k]
        x = torch.where(x >= kth, x, -math.inf)
    return torch.softmax(x / temperature, -1)


def verify_draft(probs, tokens, parents, uniform, draft_probs=None):
    B, N, V = probs.shape
    out, path = torch.full((B, N), -1, dtype=torch.int64), torch.full((B, N), -1, dtype=torch.int32)
    counts = torch.zeros(B, dtype=torch.int32)
    for b in range(B):
        cur, n = 0, 0
        path[b, 0] = 0
        while True:
            row = probs[b, cur].double().numpy()
            left, total, took = np.maximum(row, 0.0), 1.0, None   # what rejections leave, and its sum
            for i in range(cur + 1, N):
                x = int(tokens[b, i])
                if int(parents[b, i]) != cur or not 0 <= x < V:
                    continue
                if draft_probs is None:
                    q = np.zeros(V)
                    q[x] = 1.0
                else:
                    q = draft_probs[b, cur].double().numpy()
                if float(uniform[b, i]) * total * q[x] < left[x]:
                    took = i
                    break
                if draft_probs is None:
                    total -= left[x]
                    left = left.copy()
                    left[x] = 0.0
                else:   # left holds total times the normalised target
                    left = np.maximum(left - total * q, 0.0)
                    total = left.sum()
            if took is None:
                break
            out[b, n], path[b, n + 1], cur, n = tokens[b, took], took, took, n + 1
        if not left.sum() > 0:
            left = np.maximum(row, 0.0)
        cdf = np.cumsum(left)
        if cdf[-1] > 0:
            out[b, n] = min(int(np.searchsorted(cdf, float(uniform[b, 0]) * cdf[-1], side="right")), int(np.nonzero(left > 0)[0][-1]))
        counts[b] = n + 1
    return out, path, counts


def compact_cache(cache, ctx, path, counts):
    """The caches afterwards and the new lengths."""
    after = []
    for t in (t for kv in cache for t in kv):
        t2 = t.clone()
        for b in range(t.shape[0]):
            for d in range(int(counts[b])):
                t2[b, int(ctx[b]) + d] = t[b, int(ctx[b]) + int(path[b, d])]
        after.append(t2)
    return after, ctx + counts

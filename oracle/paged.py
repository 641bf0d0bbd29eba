"""A paged KV cache and a beam search's selection in 64 bits: attention of one token over a row's
pages, the tables' upkeep, and the best continuations of beams.  Plain loops over the definitions; the
reference has no counterpart (its ml/fxlm/sample.py:62-73 samples a token a pass)."""
import math

import torch


def _clamped(n, most):
    return min(max(int(n), 0), most)


def paged_attention(q, k, v, table, lens, scale=None, k_new=None, v_new=None):
    """(o, lse, size, k, v): o (R,H,Dh) and lse (R,H) float64; size the sum of p |v| / sum p, what roundings of p are
    relative to; k, v the pools after the call."""
    R, H, D = q.shape
    N, P, Hkv = k.shape[:3]
    scale = 1 / math.sqrt(D) if scale is None else scale
    k, v = k.clone(), v.clone()
    o = torch.zeros(R, H, D, dtype=torch.float64)
    size = torch.zeros_like(o)
    lse = torch.full((R, H), -math.inf, dtype=torch.float64)
    for r in range(R):
        n = _clamped(lens[r], table.shape[1] * P)
        places = [(int(table[r, j // P]), j % P) for j in range(n)]
        if n and k_new is not None and 0 <= places[-1][0] < N:
            k[places[-1]], v[places[-1]] = k_new[r], v_new[r]
        places = [p for p in places if 0 <= p[0] < N]
        if not places:
            continue
        page, at = (torch.tensor(x) for x in zip(*places))
        for h in range(H):
            kk, vv = k[page, at, h * Hkv // H].double(), v[page, at, h * Hkv // H].double()
            s = scale * (kk @ q[r, h].double())
            p = torch.exp(s - s.max())
            o[r, h] = (p @ vv) / p.sum()
            size[r, h] = (p @ vv.abs()) / p.sum()
            lse[r, h] = s.max() + torch.log(p.sum())
    return o, lse, size, k, v


def extend_pages(table, lens, add, uses, page, most=1, cache=None):
    """(slots, lens, table, uses, cache) after the call."""
    table, uses = table.clone(), uses.clone()
    cache = None if cache is None else [tuple(t.clone() for t in kv) for kv in cache]
    R, M = table.shape
    N = uses.numel()
    slots, out = torch.full((R, most), -1, dtype=torch.int64), lens.clone()
    rows = []
    for r in range(R):
        n, a = _clamped(lens[r], M * page), _clamped(add[r], most)
        if a == 0 or n + a > M * page:
            continue
        held = int(table[r, n // page]) if n % page else None
        if held is not None and (not 0 <= held < N or (cache is None and uses[held] > 1)):
            continue
        rows.append((r, n, a, held))
    writers = {}
    for r, n, _, held in rows:
        if held is not None and uses[held] > 1:
            writers.setdefault(held, []).append((-(n % page), r))
    free = torch.nonzero(uses == 0)[:, 0].tolist()
    # (the longest writes behind every other holder's tokens, so one that is refused its copy loses none)
    copied = {r for p, rs in writers.items() for _, r in (rs if len(rs) < uses[p] else sorted(rs)[1:])}
    wanted = 0
    for r, n, a, held in rows:
        cols = ([n // page] if r in copied else []) + list(range(-(-n // page), -(-(n + a) // page)))
        wanted += len(cols)
        if cols and wanted > len(free):
            continue
        for i, c in enumerate(cols):
            p = free[wanted - len(cols) + i]
            if r in copied and i == 0:
                uses[held] -= 1
                for kv in cache or ():
                    for t in kv:
                        t[p, :n % page] = t[held, :n % page]
            table[r, c] = p
            uses[p] = 1
        out[r] = n + a
        for i in range(a):
            slots[r, i] = int(table[r, (n + i) // page]) * page + (n + i) % page
    return slots, out, table, uses, cache


def store_pages(k, v, slots, k_pages, v_pages):
    """The pools after the call."""
    k_pages, v_pages = k_pages.clone(), v_pages.clone()
    N, P = k_pages.shape[:2]
    for r in range(slots.shape[0]):
        for t in range(slots.shape[1]):
            s = int(slots[r, t])
            if 0 <= s < N * P:
                k_pages[s // P, s % P], v_pages[s // P, s % P] = k[r, t], v[r, t]
    return k_pages, v_pages


def reorder_pages(table, lens, parents, uses, page):
    """(lens, table, uses) after the call."""
    was, table, uses, out = table, table.clone(), uses.clone(), torch.zeros_like(lens)
    R, M = table.shape
    n = [_clamped(x, M * page) for x in lens]
    for r in range(R):
        for p in was[r, :-(-n[r] // page)].tolist():
            if 0 <= p < uses.numel():
                uses[p] -= 1
        par = int(parents[r])
        if 0 <= par < R:
            c = -(-n[par] // page)
            table[r, :c] = was[par, :c]
            out[r] = n[par]
            for p in was[par, :c].tolist():
                if 0 <= p < uses.numel():
                    uses[p] += 1
    return out, table, uses


def beam_select(logits, scores, done=None, fill=0, weight=None):
    """(scores float64, parents, tokens, ranks): as the operator, with the ranks (B, K + 1) that they were ordered by, that of the
    best one left out behind them."""
    B, K, V = logits.shape
    out = torch.full((B, K), -math.inf, dtype=torch.float64)
    ranks = torch.full((B, K + 1), -math.inf, dtype=torch.float64)
    rows = torch.full((B, K), -1, dtype=torch.int32)
    toks = torch.full((B, K), fill, dtype=torch.int64)
    for b in range(B):
        cand = []   # (not NaN, -rank, beam, -logit, token, score)
        for k in range(K):
            s, w = float(scores[b, k]), 1.0 if weight is None else float(weight[b, k])
            if s == -math.inf:
                continue
            if not 0 < w < math.inf:
                s = math.nan
            if s != s or (done is not None and bool(done[b, k])):
                cand.append((s == s, -w * s if s == s else 0.0, k, 0.0, fill, s))
                continue
            x = logits[b, k].double()
            lp = torch.log_softmax(x, -1)
            if bool(x.isnan().any()) or bool((x == math.inf).any()):
                cand.append((False, 0.0, k, 0.0, fill, math.nan))
                continue
            for v in torch.argsort(x, descending=True, stable=True)[:K].tolist():
                if x[v] != -math.inf and s + float(lp[v]) != -math.inf:
                    cand.append((True, -w * (s + float(lp[v])), k, -float(x[v]), v, s + float(lp[v])))
        for i, (num, rank, k, _, v, s) in enumerate(sorted(cand)[:K]):
            out[b, i], rows[b, i], toks[b, i], ranks[b, i] = s, b * K + k, v, -rank if num else math.nan
        if len(cand) > K:
            ranks[b, K] = -sorted(cand)[K][1]
    return out, rows, toks, ranks

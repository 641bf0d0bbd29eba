"""A paged KV cache and beam selection on the GPU against the 64-bit oracle (oracle/paged.py).

Tolerances.  Attention: an output is rounded once (2^-8 of it, bf16's half step); p enters its product in
two bf16 parts, which leave at most 2^-16 of it (a rounding of 2^-8 of what a rounding of 2^-8 leaves);
scores, exponentials and sums are fp32: a score's error is at most (D + 8) 2^-24 of the sum of |q k| scale,
which moves every p by that much relatively, and 2^-18 covers the exponentials and the sums of up to 64
partial ones.  Beam selection: a logit's distance d from the maximum is rounded twice (the difference, and
its product with log2 e, itself rounded: 3 2^-24 |d|), each exponential is 2^-23 off and a chunk's sum in
fp32 goes through at most 64 roundings, so log sum exp is off by at most 3 2^-24 sum p |d| + 66 2^-23; the
score is rounded once.  Tables, slots, uses and moved rows are exact."""
import math
import random

import pytest
import torch

from oracle import paged as op

pytestmark = pytest.mark.gpu


def _ints(x, dev=None):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def _same(x, y):
    return torch.equal(x.cpu().view(torch.int16), y.cpu().view(torch.int16))


# ---- attention -----------------------------------------------------------------------------


def _case(R, H, Hkv, D, P, M, lens, seed=0, heads=False, share=False):
    """Rows of lens keys over a pool with four pages more than they need; behind a row's pages anything."""
    g = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g).bfloat16()   # noqa: E731
    need = [min(max(-(-n // P), 0), M) for n in lens]
    ids = torch.randperm(sum(need) + 4, generator=g).int()
    table = torch.randint(-9, 2 ** 31 - 1, (R, M), generator=g).int()
    at = 0
    for r in range(R):
        table[r, :need[r]] = ids[at:at + need[r]]
        at += need[r]
        if share and r % 2 and need[r - 1] > 1:   # the row before's pages but its last
            c = min(need[r - 1] - 1, max(need[r] - 1, 0))
            table[r, :c] = table[r - 1, :c]
    N = sum(need) + 4
    pool = (lambda: rn(N, Hkv, P, D).transpose(1, 2)) if heads else (lambda: rn(N, P, Hkv, D))
    return {"q": rn(R, H, D), "k": pool(), "v": pool(), "table": table, "lens": _ints(lens), "kn": rn(R, Hkv, D), "vn": rn(R, Hkv, D)}


def _to(dev, c):
    # (a transposed pool keeps its layout)
    return {n: t.to(dev) for n, t in c.items()}


def _check(dev, c, new, d=None):
    from fxlm import paged_attention
    kn, vn = (c["kn"], c["vn"]) if new else (None, None)
    ro, rl, size, rk, rv = op.paged_attention(c["q"], c["k"], c["v"], c["table"], c["lens"], k_new=kn, v_new=vn)
    d = _to(dev, c) if d is None else d
    o, l = paged_attention(d["q"], d["k"], d["v"], d["table"], d["lens"], return_lse=True, k_new=d["kn"] if new else None,   # noqa: E741
                           v_new=d["vn"] if new else None)
    D = c["q"].shape[-1]
    mag = float(c["q"].double().norm(dim=-1).max() * rk.double().norm(dim=-1).nan_to_num(0, 0, 0).max()) / math.sqrt(D)
    score = (D + 8) * 2.0 ** -24 * mag
    assert torch.isfinite(o).all()
    err, tol = (o.double().cpu() - ro).abs(), 2.0 ** -8 * ro.abs() + (2 * score + 2.0 ** -16 + 2.0 ** -18) * size
    assert (err <= tol).all(), float((err - tol).max())
    none = rl == -math.inf
    lc = l.double().cpu()
    assert torch.equal(lc == -math.inf, none) and not o.cpu()[none].any()
    assert ((lc - rl).abs() <= score + 2.0 ** -18 + 2.0 ** -22 * rl.abs())[~none].all()
    assert _same(d["k"], rk) and _same(d["v"], rv)
    return d, o, l


# a row of nothing, of one key, ends inside a half tile, at its end, at a tile's and a page's end; 1 to 40 heads a key head
# (one tile of 16, two, and two groups); tables that are split over workgroups (more than 1,536 keys) and not
@pytest.mark.parametrize("new", [True, False])
@pytest.mark.parametrize("R,H,Hkv,D,P,M,lens", [
    (1, 1, 1, 64, 16, 1, [1]),
    (1, 1, 1, 128, 16, 1, [0]),
    (6, 2, 2, 64, 16, 5, [0, 15, 16, 17, 33, 80]),
    (4, 6, 3, 128, 32, 9, [31, 32, 287, 288]),
    (3, 12, 4, 64, 64, 8, [511, 64, 1]),
    (3, 16, 1, 128, 16, 40, [640, 3, 300]),
    (3, 17, 1, 64, 128, 4, [130, 0, 512]),
    (2, 40, 1, 128, 32, 20, [601, 77]),
    (2, 40, 1, 64, 32, 20, [601, 77]),
    (1, 2, 2, 64, 16, 200, [3190]),                       # split from here on
    (3, 4, 4, 128, 16, 130, [2080, 0, 1]),
    (2, 33, 1, 128, 64, 40, [2500, 2560]),
    (70, 2, 1, 64, 16, 110, [(37 * i) % 1750 for i in range(70)]),   # more rows than lanes
    (3, 8, 2, 128, 1024, 4, [4096, 1025, 1000]),
    (5, 20, 2, 128, 256, 9, [2304, 5, 700, 0, 2049]),
    (2, 8, 8, 128, 16, 1000, [16000, 40]),                # the entries past a wave's 64
])
def test_paged_attention(dev, R, H, Hkv, D, P, M, lens, new):
    for heads in (False, True):
        _check(dev, _case(R, H, Hkv, D, P, M, lens, seed=R + H + P, heads=heads), new)


def test_paged_attention_rows_share_pages(dev):
    for M, n in ((20, 300), (130, 2000)):
        _check(dev, _case(6, 4, 2, 64, 16, M, [n, n, n - 40, n + 17, 16, 40], seed=n, share=True), False)


# long tables over a small pool, their rows sharing pages
@pytest.mark.parametrize("R,H,Hkv,P,M,lens", [
    (32, 12, 12, 64, 50, [(419 * i) % 1000 for i in range(31)] + [3200]),
    (32, 12, 12, 64, 50, [i % 3 for i in range(32)]),            # fewer steps than workgroups
    (170, 2, 2, 32, 100, [(97 * i) % 300 for i in range(169)] + [3200]),
    (170, 33, 1, 32, 100, [(97 * i) % 300 for i in range(169)] + [3200]),
])
def test_paged_attention_of_many_rows_of_a_small_pool(dev, R, H, Hkv, P, M, lens):
    for new in (False, True):
        _check(dev, _case(R, H, Hkv, 64, P, M, lens, seed=R + H, share=not new), new)


def test_paged_attention_lengths_outside_the_table(dev):
    # a negative length is none, one past the table is the table's
    for M in (3, 120):
        _check(dev, _case(4, 4, 2, 64, 16, M, [-5, 16 * M + 1, 2 ** 31 - 1, 16 * M], seed=M), True)


@pytest.mark.parametrize("M,lens", [(12, [190, 77, 20]), (150, [2400, 1000, 170])])
def test_paged_attention_entries_that_are_no_pages(dev, M, lens):
    # inside a row: the keys of such entries are nobody's, the new key's among them
    c = _case(3, 6, 2, 128, 16, M, lens, seed=M)
    N = c["k"].shape[0]
    c["table"][0, 3], c["table"][0, 4], c["table"][1, 0] = -1, N, 2 ** 31 - 1
    c["table"][2, (lens[2] - 1) // 16] = -2 ** 31
    for new in (True, False):
        _check(dev, c, new)
    c["table"][1] = -1       # a row of nothing else
    _check(dev, c, True)


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_paged_attention_stale_rows_may_hold_anything(dev, bad):
    for M, lens in ((12, [190, 77, 0, 16]), (150, [2399, 1000, 0, 16])):
        c = _case(4, 6, 2, 64, 16, M, lens, seed=M)
        keep = torch.zeros(c["k"].shape[:2], dtype=torch.bool)
        for r, n in enumerate(lens):
            for j in range(n - 1):     # the last key comes from the call
                keep[c["table"][r, j // 16], j % 16] = True
        for t in ("k", "v"):
            c[t][~keep] = bad
        rk, rv = c["k"].clone(), c["v"].clone()
        from fxlm import paged_attention
        d = _to(dev, c)
        o = paged_attention(d["q"], d["k"], d["v"], d["table"], d["lens"], k_new=d["kn"], v_new=d["vn"])
        for r, n in enumerate(lens):
            if n:
                rk[c["table"][r, (n - 1) // 16], (n - 1) % 16], rv[c["table"][r, (n - 1) // 16], (n - 1) % 16] = c["kn"][r], c["vn"][r]
        assert _same(d["k"], rk) and _same(d["v"], rv)
        z = {n: t.clone() for n, t in c.items()}
        for t in ("k", "v"):
            z[t][~keep] = 0
        assert torch.equal(o, _check(dev, z, True)[1])


def test_paged_attention_strided_views(dev):
    # q, k_new and v_new out of one projection; pools as views with room between heads, pages and rows; a table's first columns
    from fxlm import paged_attention
    R, H, Hkv, D, P, M = 3, 6, 2, 64, 32, 60
    g = torch.Generator(device=dev).manual_seed(5)
    qkv = torch.randn(R, H + 2 * Hkv, D, device=dev, generator=g).bfloat16()
    q, kn, vn = qkv.split([H, Hkv, Hkv], dim=1)
    both = torch.randn(P, 2, 190, Hkv + 1, D + 8, device=dev, generator=g).bfloat16()
    k, v = (both[:, i, :, :Hkv, :D].transpose(0, 1) for i in range(2))
    kept = both.clone()
    wide = torch.randperm(190, device=dev, generator=g)[:180].int().view(R, M)
    table = torch.cat([wide, torch.full((R, 7), 10 ** 9, device=dev, dtype=torch.int32)], 1)[:, :M]
    lens = _ints([1900, 333, 64], dev)
    o, l = paged_attention(q, k, v, table, lens, return_lse=True, k_new=kn, v_new=vn)   # noqa: E741
    for r, n in enumerate(lens.tolist()):
        page = int(wide[r, (n - 1) // P])
        kept[(n - 1) % P, 0, page, :Hkv, :D], kept[(n - 1) % P, 1, page, :Hkv, :D] = kn[r], vn[r]
    assert torch.equal(both, kept)        # the new rows, and nothing between them
    o2, l2 = paged_attention(q.contiguous(), k.contiguous(), v.contiguous(), wide.t().contiguous().t(), lens.repeat_interleave(2)[::2], return_lse=True)
    assert torch.equal(o, o2) and torch.equal(l, l2)


def test_paged_attention_scales(dev):
    from fxlm import paged_attention
    c = _case(2, 2, 1, 64, 16, 9, [100, 144], seed=8)
    d = _to(dev, c)
    for scale in (0.02, 1.0):
        ro, _, size, _, _ = op.paged_attention(c["q"], c["k"], c["v"], c["table"], c["lens"], scale=scale)
        o = paged_attention(d["q"], d["k"], d["v"], d["table"], d["lens"], scale=scale)
        score = 72 * 2.0 ** -24 * scale * float(c["q"].double().norm(dim=-1).max() * c["k"].double().norm(dim=-1).max())
        assert ((o.double().cpu() - ro).abs() <= 2.0 ** -8 * ro.abs() + (2 * score + 2.0 ** -16 + 2.0 ** -18) * size).all()
    for scale in (0.0, -1.0, math.inf, math.nan):
        with pytest.raises(ValueError):
            paged_attention(d["q"], d["k"], d["v"], d["table"], d["lens"], scale=scale)


def test_paged_attention_in_a_pool_past_32_bits(dev):
    # a page's first element past 2^32; both at a pool's far end
    from fxlm import paged_attention
    P, Hkv, D = 64, 4, 128
    N = (2 ** 32 + 2 ** 24) // (P * Hkv * D)
    c = _case(2, 8, Hkv, D, P, 40, [2500, 70], seed=3)
    n = c["k"].shape[0]
    pools = [torch.empty(N, P, Hkv, D, device=dev, dtype=torch.bfloat16) for _ in range(2)]
    for p, t in zip(pools, ("k", "v")):
        p[N - n:] = c[t].to(dev)
    ro, _ = paged_attention(*(c[t].to(dev) for t in ("q", "k", "v", "table", "lens")), k_new=c["kn"].to(dev), v_new=c["vn"].to(dev), return_lse=True)
    o, _ = paged_attention(c["q"].to(dev), *pools, (c["table"] + (N - n)).to(dev), c["lens"].to(dev), k_new=c["kn"].to(dev), v_new=c["vn"].to(dev),
                           return_lse=True)
    assert torch.equal(o, ro)
    page = int(c["table"][0, 2499 // P])
    assert _same(pools[0][N - n + page, 2499 % P], c["kn"][0]) and _same(pools[1][N - n + page, 2499 % P], c["vn"][0])


# pools that are loaded past the caches: each of the kernel's forms, with the bits of the same rows in a small pool
@pytest.mark.parametrize("R,H,Hkv,D,P,M,lens", [
    (900, 4, 4, 64, 16, 20, [(53 * i) % 321 for i in range(900)]),      # not split
    (500, 20, 1, 128, 64, 20, [(531 * i) % 1281 for i in range(500)]),
    (6, 8, 4, 64, 256, 200, [3000, 0, 1, 2048, 255, 1700]),             # split: four heads a workgroup, two, one
    (6, 8, 4, 128, 128, 200, [3000, 0, 1, 2048, 255, 1700]),
    (6, 6, 6, 64, 256, 200, [3000, 0, 1, 2048, 255, 1700]),
    (6, 40, 2, 128, 256, 200, [3000, 0, 1, 2048, 255, 1700]),
    (6, 5, 5, 64, 256, 200, [3000, 0, 1, 2048, 255, 1700]),
    (6, 32, 1, 64, 1024, 200, [3000, 0, 1, 2048, 255, 1700]),
])
@pytest.mark.parametrize("heads", [False, True])
def test_paged_attention_in_large_pools(dev, R, H, Hkv, D, P, M, lens, heads):
    from fxlm import paged_attention
    c = _case(R, H, Hkv, D, P, M, lens, seed=D + P, heads=heads)
    n = c["k"].shape[0]
    N = max(n, (2 ** 28 + 2 ** 22) // (P * Hkv * D * 4))
    assert min(R * M, N) * P * Hkv * D * 4 >= 2 ** 28 > min(R * M, n) * P * Hkv * D * 4
    d = _to(dev, c)
    kn, vn = d["kn"], d["vn"]
    big = []
    for t in ("k", "v"):
        x = torch.full((N, Hkv, P, D) if heads else (N, P, Hkv, D), math.nan, device=dev, dtype=torch.bfloat16)
        x = x.transpose(1, 2) if heads else x
        x[N - n:] = d[t]
        big.append(x)
    o, l = paged_attention(d["q"], *big, d["table"] + (N - n), d["lens"], return_lse=True, k_new=kn, v_new=vn)   # noqa: E741
    _, ro, rl = _check(dev, c, True) if R < 100 else (None, *paged_attention(*(d[t] for t in ("q", "k", "v", "table", "lens")), return_lse=True, k_new=kn, v_new=vn))
    assert torch.equal(o, ro) and torch.equal(l, rl)


def test_paged_attention_on_another_stream_and_in_graphs(dev):
    # two captured calls with workspaces of their own, replayed in turn between eager calls, lengths changed in between
    from fxlm import paged_attention
    cs = [_to(dev, _case(3, 4, 2, 64, 16, 130, [2000, 17, 900], seed=s)) for s in range(2)]
    run = lambda c: paged_attention(c["q"], c["k"], c["v"], c["table"], c["lens"], return_lse=True)   # noqa: E731
    ref = [run(c) for c in cs]
    side = torch.cuda.Stream(device=dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        o, l = run(cs[0])   # noqa: E741
    side.synchronize()
    assert torch.equal(o, ref[0][0]) and torch.equal(l, ref[0][1])
    graphs = []
    for c in cs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = run(c)
        graphs.append((g, out))
    for lens in ([2000, 17, 900], [5, 0, 2080], [1, 1500, 33]):
        for c in cs:
            c["lens"].copy_(_ints(lens))
        for g, _ in graphs:
            g.replay()
        for c, (_, out) in zip(cs, graphs):
            for a, b in zip(run(c), out):
                assert torch.equal(a, b)


def test_paged_attention_and_selection_on_two_streams_at_once(dev):
    from fxlm import beam_select, paged_attention
    cs = [_to(dev, _case(4, 4, 2, 64, 16, 130, [2000, 17, 900, 1300], seed=s)) for s in range(2)]
    g = torch.Generator(device=dev).manual_seed(1)
    xs = [(torch.randn(6, 4, 30011, device=dev, generator=g), torch.randn(6, 4, device=dev, generator=g)) for _ in range(2)]
    run = lambda i: (*paged_attention(*(cs[i][n] for n in ("q", "k", "v", "table", "lens")), return_lse=True), *beam_select(*xs[i]))   # noqa: E731
    want = [run(i) for i in range(2)]
    streams = [torch.cuda.Stream(device=dev) for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(8):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(run(i))
    torch.cuda.synchronize()
    for i in range(2):
        for out in got[i]:
            for a, b in zip(out, want[i]):
                assert torch.equal(a, b)


# ---- tables --------------------------------------------------------------------------------


def _tables(g, R, M, P, N, most, full=0.6):
    """A pool in use: rows of any length, some with the pages of others, entries behind a row's pages of any kind."""
    r = random.Random(int(torch.randint(0, 2 ** 31, (1,), generator=g)))
    table = torch.randint(-3, N + 3, (R, M), generator=g).int()
    lens, ids = [], torch.randperm(N, generator=g).tolist()
    left = int(N * full)
    for i in range(R):
        n = r.choice([0, r.randint(0, M * P), r.randint(0, min(M * P, 3 * P)), P * r.randint(0, M)])
        if i and r.random() < 0.4:    # a beam of the row before: all of its pages, or but the last
            n = lens[i - 1] if r.random() < 0.7 else max(0, (lens[i - 1] - 1) // P * P)
            table[i, :-(-n // P)] = table[i - 1, :-(-n // P)]
        else:
            n = min(n, left * P)
            c = -(-n // P)
            for j in range(c):
                table[i, j] = ids.pop()
            left -= c
        lens.append(n)
    uses = torch.zeros(N, dtype=torch.int32)
    for i, n in enumerate(lens):
        for p in table[i, :-(-n // P)].tolist():
            uses[p] += 1
    add = _ints([r.choice([0, 1, 1, 1, most, r.randint(0, most)]) for _ in range(R)])
    return table, _ints(lens), add, uses


def _check_extend(dev, table, lens, add, uses, P, most, cache=None, d=None):
    from fxlm import extend_pages
    want = op.extend_pages(table, lens, add, uses, P, most, cache)
    d = {"table": table.to(dev), "uses": uses.to(dev)} if d is None else d
    dc = None if cache is None else [tuple(t.to(dev) for t in kv) for kv in cache]
    slots, n = extend_pages(d["table"], lens.to(dev), add.to(dev), d["uses"], P, most, dc)
    for a, b in zip((slots, n, d["table"], d["uses"]), want):
        assert torch.equal(a.cpu(), b)
    if cache is not None:
        for kv, rkv in zip(dc, want[4]):
            for a, b in zip(kv, rkv):
                assert _same(a, b)
    return want


# few rows and many, pages for all and too few of them, slots in the same launch and in one of their own, pools that are no
# multiple of what a thread looks through, wide tables
@pytest.mark.parametrize("R,M,P,N,most", [
    (1, 1, 16, 1, 1), (1, 3, 16, 5, 20), (5, 6, 16, 40, 1), (9, 4, 64, 30, 3), (40, 12, 16, 700, 1), (64, 40, 32, 3000, 200), (300, 9, 16, 1500, 1),
    (300, 9, 16, 1100, 40), (2500, 5, 16, 20001, 5), (8192, 2, 128, 33000, 1), (3, 300, 16, 70000, 4800),
])
def test_extend_pages(dev, R, M, P, N, most):
    g = torch.Generator().manual_seed(R + M)
    for full in (0.3, 0.98):
        t = _tables(g, R, M, P, N, most, full)
        _check_extend(dev, *t, P, most)
        _check_extend(dev, *t, P, most, [(torch.randn(N, P, 1, 8, generator=g).bfloat16(),) * 2] if N * P < 10 ** 6 else None)


def test_extend_pages_of_a_pool_in_which_the_free_ones_are_far(dev):
    # the search goes through several turns of the workgroup, at an odd address
    g = torch.Generator().manual_seed(1)
    N = 100003
    uses = torch.ones(N + 1, dtype=torch.int32)
    uses[60001:60004] = 0
    uses[99999:] = 0
    buf = uses.to(dev)
    for first in (0, 1):
        u = uses[first:N + first].clone()
        table, lens, add = torch.randint(0, N, (7, 4), generator=g).int(), _ints([16, 0, 32, 5, 0, 0, 1]), _ints([1, 1, 1, 1, 17, 40, 1])
        d = {"table": table.to(dev), "uses": buf.clone()[first:N + first]}
        _check_extend(dev, table, lens, add, u, 16, 40, d=d)


@pytest.mark.parametrize("R,N", [(7, 2 ** 18 - 1), (7, 2 ** 18), (300, 300001), (1500, 2 ** 20 + 70003)])
def test_extend_pages_of_large_pools(dev, R, N):
    # pools whose free pages are counted first: at the far end, here and there (more turns than a wave looks up at once), too few, none
    g = torch.Generator().manual_seed(R)
    buf = torch.ones(N + 3, dtype=torch.int32, device=dev)
    table, lens = torch.randint(0, N, (R, 4), generator=g).int(), torch.randint(0, 33, (R,), generator=g).int()
    add = torch.randint(0, 20, (R,), generator=g).int()
    for free, first in ((torch.arange(N - 4000, N), 0), (torch.randperm(N, generator=g)[:5000], 1), (torch.tensor([5, N // 2, N - 1]), 2), (torch.tensor([], dtype=torch.int64), 3)):
        u = torch.ones(N, dtype=torch.int32)
        u[free] = 0
        u[table[:, 0].long()] = 1
        u[table[:, 1].long()] = 1
        buf[first:N + first] = u.to(dev)
        _check_extend(dev, table, lens, add, u, 16, 20, d={"table": table.to(dev), "uses": buf[first:N + first].clone() if first == 0 else buf[first:N + first]})
        buf.fill_(1)


def test_extend_pages_at_the_edges_of_its_arguments(dev):
    # lengths below zero and past the table, additions below zero and past `most`, an open page that is none, a table of too few
    # pages; strided views
    N, P, M = 50, 16, 4
    table = torch.full((9, M + 3), -1, dtype=torch.int32)
    table[:, 0] = torch.arange(9) * 5
    table[5, 0], table[6, 0] = -1, N
    lens, add = _ints([-4, 70, 64, 10, 10, 10, 10, 16, 0]), _ints([3, 1, 1, -2, 99, 1, 1, 48, 65])
    uses = torch.zeros(N, dtype=torch.int32)
    uses[torch.arange(0, 45, 5)] = 1
    from fxlm import extend_pages
    for most in (1, 7, 65):
        want = op.extend_pages(table[:, :M], lens, add, uses, P, most)
        dt, du = table.to(dev), uses.to(dev)
        slots, n = extend_pages(dt[:, :M], lens.to(dev), add.to(dev).repeat_interleave(2)[::2], du, P, most)
        for a, b in zip((slots, n, dt[:, :M], du), want):
            assert torch.equal(a.cpu(), b)
        assert torch.equal(dt[:, M:].cpu(), table[:, M:])


def test_extend_pages_copies_in_every_layer(dev):
    # 33 layers, more tensors than one launch takes; pools of two layouts; rows behind the copied ones stay
    from fxlm import extend_pages
    g = torch.Generator().manual_seed(6)
    N, P, H, D, L = 24, 16, 3, 64, 33
    table = _ints([[1, 2, -1], [1, 2, -1], [1, 2, -1], [4, 5, -1], [4, 5, -1], [7, -1, -1]])
    lens, add = _ints([21, 21, 21, 31, 31, 16]), _ints([1, 1, 1, 1, 0, 1])
    uses = torch.zeros(N, dtype=torch.int32)
    uses[[1, 2, 4, 5, 7]] = _ints([3, 3, 2, 2, 1])
    cache = [tuple(torch.randn(N, H, P, D, generator=g).bfloat16().transpose(1, 2) if i % 2 else torch.randn(N, P, H, D, generator=g).bfloat16()
                   for _ in range(2)) for i in range(L)]
    want = _check_extend(dev, table, lens, add, uses, P, 1, cache)
    assert want[1].tolist() == [22, 22, 22, 32, 31, 17] and want[3][[2, 5]].tolist() == [1, 1]
    with pytest.raises(ValueError):
        extend_pages(table.to(dev), lens.to(dev), add.to(dev), uses.to(dev), P, 1, [])
    with pytest.raises(ValueError):
        extend_pages(table.to(dev), lens.to(dev), add.to(dev), uses[:20].to(dev), P, 1, [tuple(t.to(dev) for t in cache[0])])


@pytest.mark.parametrize("R,M,P,N", [(1, 1, 16, 4), (6, 5, 16, 40), (40, 64, 16, 3000), (333, 130, 64, 60000), (1500, 7, 16, 12000), (8192, 3, 16, 30000)])
def test_reorder_pages(dev, R, M, P, N):
    from fxlm import reorder_pages
    g = torch.Generator().manual_seed(R)
    for kind in range(4):
        table, lens, _, uses = _tables(g, R, M, P, N, 1)
        par = {0: torch.randint(-2, R + 2, (R,), generator=g), 1: torch.randperm(R, generator=g), 2: torch.arange(R) // 4 * 4, 3: torch.full((R,), -1)}[kind].int()
        want = op.reorder_pages(table, lens, par, uses, P)
        wide = torch.cat([table, torch.full((R, 2), 77, dtype=torch.int32)], 1).to(dev)
        du = uses.to(dev)
        n = reorder_pages(wide[:, :M], lens.to(dev), par.to(dev), du, P)
        for a, b in zip((n, wide[:, :M], du), want):
            assert torch.equal(a.cpu(), b)
        assert bool((wide[:, M:] == 77).all())


def test_reorder_pages_lengths_outside_the_table_and_entries_that_are_no_pages(dev):
    from fxlm import reorder_pages
    table = _ints([[3, -1, 99], [4, 5, 6], [7, 8, 2 ** 31 - 1]])
    lens, par, uses = _ints([48, 100, -3]), _ints([1, 0, 0]), _ints([1] * 9)
    want = op.reorder_pages(table, lens, par, uses, 16)
    dt, du = table.to(dev), uses.to(dev)
    n = reorder_pages(dt, lens.to(dev), par.to(dev), du, 16)
    for a, b in zip((n, dt, du), want):
        assert torch.equal(a.cpu(), b)


@pytest.mark.parametrize("R,T,H,D,P,heads", [(1, 1, 1, 8, 16, False), (2, 37, 3, 64, 16, True), (3, 300, 2, 128, 64, False), (1, 5, 40, 72, 16, True)])
def test_store_pages(dev, R, T, H, D, P, heads):
    from fxlm import store_pages
    g = torch.Generator().manual_seed(T)
    N = -(-R * T // P) + 2
    pool = lambda: torch.randn(N, H, P, D, generator=g).bfloat16().transpose(1, 2) if heads else torch.randn(N, P, H, D, generator=g).bfloat16()   # noqa: E731
    kp, vp = pool(), pool()
    qkv = torch.randn(R, T, 3 * H, D, generator=g).bfloat16()
    slots = torch.randperm(N * P, generator=g)[:R * T].view(R, T)
    slots[torch.rand(R, T, generator=g) < 0.3] = -1
    slots[0, 0] = N * P        # outside
    if T > 2:
        slots[0, 1:3] = torch.tensor([-2 ** 63, 2 ** 63 - 1])
    want = op.store_pages(qkv[:, :, H:2 * H], qkv[:, :, 2 * H:], slots, kp, vp)
    dk, dv, dq = kp.to(dev), vp.to(dev), qkv.to(dev)
    store_pages(dq[:, :, H:2 * H], dq[:, :, 2 * H:], slots.t().contiguous().to(dev).t(), dk, dv)
    assert _same(dk, want[0]) and _same(dv, want[1])


def test_a_cache_in_use(dev):
    """Rows come, grow, fork, move and end; every step's attention is that of plain caches, and the pages' uses add up."""
    from fxlm import PagedCache, paged_attention, store_pages
    R, H, Hkv, D, P = 10, 4, 2, 64, 16
    g = torch.Generator().manual_seed(11)
    r = random.Random(11)
    c = PagedCache(R, 12, P, 12, 1, Hkv, D, dev)
    (kp, vp), = c.kv
    plain = [[] for _ in range(R)]     # (k, v) rows
    rn = lambda *s: torch.randn(*s, generator=g).bfloat16()   # noqa: E731
    refused = 0
    for step in range(40):
        if step % 3 == 0:    # prompts into the empty rows
            add = [r.randint(1, 40) if not p and r.random() < 0.7 else 0 for p in plain]
            k, v = rn(R, 40, Hkv, D), rn(R, 40, Hkv, D)
            slots = c.extend(_ints(add, dev), 40)
            store_pages(k.to(dev), v.to(dev), slots, kp, vp)
            for i, n in enumerate(add):
                if n and int(slots[i, 0]) >= 0:
                    plain[i] = [(k[i, t], v[i, t]) for t in range(n)]
                refused += n > 0 and int(slots[i, 0]) < 0
        kn, vn, q = rn(R, Hkv, D), rn(R, Hkv, D), rn(R, H, D)
        ok = c.extend((c.lens > 0).int())[:, 0] >= 0
        lens = torch.where(ok, c.lens, 0)
        o = paged_attention(q.to(dev), kp, vp, c.table, lens, k_new=kn.to(dev), v_new=vn.to(dev)).cpu()
        for i in range(R):
            if not bool(ok[i]):
                refused += len(plain[i]) > 0
                assert not o[i].any()
                continue
            plain[i] = plain[i] + [(kn[i], vn[i])]
            kk, vv = (torch.stack(x)[None] for x in zip(*plain[i]))
            n = len(plain[i])
            table = torch.arange(-(-n // 16), dtype=torch.int32)[None]
            pad = lambda t: torch.cat([t, torch.zeros(1, -n % 16, Hkv, D).bfloat16()], 1).view(-1, 16, Hkv, D)   # noqa: E731
            ro, _, size, _, _ = op.paged_attention(q[i:i + 1], pad(kk), pad(vv), table, _ints([n]))
            assert ((o[i].double() - ro[0]).abs() <= 2.0 ** -8 * ro[0].abs() + 2.0 ** -13 * size[0]).all()
        par = [r.choice([i, i, i, r.randrange(R), -1]) if r.random() < 0.5 else i for i in range(R)]
        c.reorder(_ints(par, dev))
        plain = [list(plain[p]) if p >= 0 else [] for p in par]
        assert c.lens.tolist() == [len(p) for p in plain]
        held = torch.zeros(12, dtype=torch.int32)
        for i, p in enumerate(plain):
            for x in c.table[i, :-(-len(p) // P)].tolist():
                held[x] += 1
        assert torch.equal(c.uses.cpu(), held)
    assert refused > 0     # the pool was too small now and then
    c.end()
    assert not c.uses.any() and not c.lens.any()


def test_tables_in_a_graph(dev):
    # reordering, pages, stores and attention captured once and replayed between eager work, against the same calls one by one
    from fxlm import extend_pages, paged_attention, reorder_pages, store_pages
    g = torch.Generator().manual_seed(4)
    R, M, P, N, H, D = 12, 9, 16, 200, 2, 64
    table, lens, _, uses = _tables(g, R, M, P, N, 1, 0.3)
    pools = [torch.randn(N, P, H, D, generator=g).bfloat16().to(dev) for _ in range(2)]
    a = {"table": table.to(dev), "lens": lens.to(dev), "uses": uses.to(dev), "k": pools[0].clone(), "v": pools[1].clone(),
         "par": torch.zeros(R, dtype=torch.int32, device=dev), "add": torch.zeros(R, dtype=torch.int32, device=dev), "x": torch.zeros(3, R, 3, H, D, device=dev).bfloat16()}
    b = {n: t.clone() for n, t in a.items()}

    def step(s):
        n = reorder_pages(s["table"], s["lens"], s["par"], s["uses"], P)
        slots, n = extend_pages(s["table"], n, s["add"], s["uses"], P, 3, [(s["k"], s["v"])])
        s["lens"].copy_(n)
        store_pages(s["x"][0], s["x"][1], slots, s["k"], s["v"])
        return paged_attention(s["x"][2][:, 0], s["k"], s["v"], s["table"], n)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(a)
    for i in range(6):
        for n, t in (("par", torch.randint(-1, R, (R,), generator=g).int()), ("add", torch.randint(0, 4, (R,), generator=g).int()),
                     ("x", torch.randn(3, R, 3, H, D, generator=g).bfloat16())):
            a[n].copy_(t)
            b[n].copy_(t)
        graph.replay()
        want = step(b)
        torch.cuda.synchronize()
        for n in a:
            assert torch.equal(a[n].view(torch.int16) if a[n].dtype == torch.bfloat16 else a[n], b[n].view(torch.int16) if b[n].dtype == torch.bfloat16 else b[n]), (i, n)
        assert torch.equal(out, want)


# ---- beams ---------------------------------------------------------------------------------


def _check_beams(dev, x, scores, done=None, fill=0, weight=None, exact=False):
    """Scores against the oracle's; parents and tokens too, where no other continuation ranks within both sides' errors."""
    from fxlm import beam_select
    B, K, V = x.shape
    ro, rr, rt, rank = op.beam_select(x, scores, done, fill, weight)
    to = lambda t: None if t is None else t.to(dev)   # noqa: E731
    out, rows, toks = (t.cpu() for t in beam_select(x.to(dev), to(scores), to(done), fill, to(weight)))
    xd = x.double()
    d = (xd.amax(-1, keepdim=True) - xd).nan_to_num(0, 0, 0)
    p = torch.softmax(xd.nan_to_num(0, 0), -1)
    lse = (3 * 2.0 ** -24 * (p * d).sum(-1) + 66 * 2.0 ** -23).amax(-1)[:, None]       # (B, 1)
    fin = torch.isfinite(ro)
    assert torch.equal(torch.isnan(out), torch.isnan(ro)) and torch.equal(out[torch.isinf(ro)].double(), ro[torch.isinf(ro)])
    assert ((out.double() - ro).abs() <= lse + 2.0 ** -24 * ro.abs())[fin].all()
    w = 1.0 if weight is None else float(weight.max())
    # (a beam's own continuations have the order of its logits)
    gap = (rank[:, :-1, None] - rank[:, None]).abs().nan_to_num(math.inf, math.inf, math.inf)       # (B, K, K + 1)
    gap[..., :-1][rr[:, :, None] == rr[:, None]] = math.inf
    clear = (gap.amin(-1) > 2 * w * lse) | exact
    assert torch.equal(rows[clear], rr[clear]) and torch.equal(toks[clear], rt[clear])
    assert int(clear.sum()) >= 0.5 * B * K
    return out, rows, toks


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("B,K,V", [(1, 1, 1), (2, 3, 2), (1, 4, 50304), (3, 5, 1000), (2, 8, 8191), (2, 8, 8193), (2, 2, 8200), (1, 32, 40001), (7, 6, 257),
                                   (1, 3, 131071), (40, 16, 300)])
def test_beam_select(dev, B, K, V, bf16):
    g = torch.Generator().manual_seed(V + K)
    x = torch.randn(B, K, V, generator=g) * 3
    x = x.bfloat16() if bf16 else x
    s = -torch.rand(B, K, generator=g).cumsum(-1) * 2
    done = torch.rand(B, K, generator=g) < 0.3
    _check_beams(dev, x, s)
    _check_beams(dev, x, s, done, V - 1, torch.rand(B, K, generator=g) + 0.2)
    s[0, 0] = -math.inf
    _check_beams(dev, x, s, done, 5)


def test_beam_select_largest_vocabulary(dev):
    from fxlm import beam_select
    g = torch.Generator().manual_seed(1)
    _check_beams(dev, torch.randn(1, 2, 1048576, generator=g), torch.tensor([[0.0, -0.5]]))
    for shape in ((1, 2, 1048577), (1, 33, 5)):
        with pytest.raises(ValueError):
            beam_select(torch.zeros(shape, device=dev), torch.zeros(shape[:2], device=dev))


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("V", [40, 9000, 50304])
def test_beam_select_equals_and_masks(dev, V, bf16):
    inf, t = math.inf, torch.bfloat16 if bf16 else torch.float32
    K = 6
    low = torch.finfo(t).min
    rows = torch.zeros(12, K, V)
    rows[0] = 1.5                                  # all equal: the lowest tokens of the lowest beam
    rows[1], rows[1, :, 30:33] = -inf, 2.0         # three tokens left
    rows[2], rows[2, :, [7, V - 1]] = low, 1.0     # masks of the lowest value
    rows[3] = torch.arange(V) / V                  # ascending: bf16 rounds to equals
    rows[4] = -torch.arange(V) / V
    rows[5], rows[5, 0, 9] = -inf, 0.0             # one token in all
    rows[6] = -inf                                 # none
    rows[7, 2, V // 2] = math.nan
    rows[8, 1, 3], rows[8, 4, 5] = inf, math.nan
    rows[9, :, 1::2] = -0.0                        # both zeros are equal
    rows[10], rows[10, :, V - 3:] = -3e38, -2e38   # sums past the type's range
    rows[11] = (torch.arange(V) % 7 == 3).float()  # many equals at the top
    x = rows.to(t)
    s = torch.zeros(12, K)
    _check_beams(dev, x, s, exact=True)
    s[:, 1:] = -inf                                # a search's first step
    _check_beams(dev, x, s, exact=True)
    s[3, 0], s[4, 2] = math.nan, math.nan
    done = torch.zeros(12, K, dtype=torch.bool)
    done[0, 0] = done[3, 0] = done[5, 1] = True
    _check_beams(dev, x, s, done, 2, exact=True)


def test_beam_select_adversarial_order(dev):
    # the largest logits all in few threads' places, more of them than a list holds
    g = torch.Generator().manual_seed(2)
    V, K = 8192, 32
    x = torch.randn(1, K, V, generator=g)
    for e in (4, 8):
        i = torch.arange(V)
        x[0, :, (i // e) % 64 < 31] += 50.0
    _check_beams(dev, x, torch.zeros(1, K) - torch.arange(K) * 0.01)


def test_beam_select_of_many_sequences(dev):
    g = torch.Generator().manual_seed(8)
    x = torch.randn(3000, 8, 50, generator=g) * 2
    _check_beams(dev, x, -torch.rand(3000, 8, generator=g).cumsum(-1), torch.rand(3000, 8, generator=g) < 0.2)


def test_beam_select_views_and_streams(dev):
    from fxlm import beam_select
    g = torch.Generator(device=dev).manual_seed(3)
    big = torch.randn(4, 5, 3, 1001, device=dev, generator=g)
    s = torch.randn(5, 4, device=dev, generator=g)
    x = big[:, :, 1].transpose(0, 1)           # (5, 4, 1001), strided
    want = beam_select(x.contiguous(), s)
    side = torch.cuda.Stream(device=dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        got = beam_select(x, s.t().contiguous().t())
    side.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    odd = torch.empty(1 + 5 * 4 * 1001, device=dev)[1:].view(5, 4, 1001).copy_(x)    # an odd address
    for a, b in zip(beam_select(odd, s), want):
        assert torch.equal(a, b)


# ---- the model -----------------------------------------------------------------------------


def _model(dev, vocab=64, layers=2, seq=160, d=128, heads=2, tie=True, seed=0):
    from fxlm import GPT, GPTConfig
    torch.manual_seed(seed)
    m = GPT(GPTConfig(vocab_size=vocab, seq_len=seq, n_layer=layers, n_head=heads, d_model=d, tie_embeddings=tie)).to(dev).bfloat16()
    with torch.no_grad():
        m.pos_emb.normal_(std=0.1)
        m.tok_emb.weight.mul_(8.0)     # logits apart from each other
    return m


# the model's logits by its paths: bf16 activations, each rounded (2^-8 of it) in products of unlike kernels, a few layers deep
LOGITS = 0.06


@pytest.mark.parametrize("R", [3, 70])
def test_paged_steps_are_the_models_forward(dev, R):
    # rows of unlike lengths, padding that is no id; few rows and more than the few-row products take
    m = _model(dev)
    g = torch.Generator().manual_seed(R)
    T, n = 40, 6
    idx = torch.randint(0, 64, (R, T + n), generator=g)
    lens = torch.randint(1, T + 1, (R,), generator=g).int()
    prompt = idx[:, :T].clone()
    prompt[torch.arange(T)[None] >= lens[:, None]] = 10 ** 12
    cache = m.paged_cache(R + 1, R * 4, 16)
    rows = torch.randperm(R + 1, generator=g)[:R].to(dev)
    lg = [m.paged_prefill(prompt.to(dev), lens.to(dev), cache, rows)]
    tok = torch.zeros(R + 1, dtype=torch.int64, device=dev)
    seqs = [idx[r, :lens[r]].tolist() for r in range(R)]
    for i in range(n):
        for r in range(R):
            seqs[r].append(int(idx[r, T + i]))
        tok[rows] = idx[:, T + i].to(dev)
        full = m.paged_step(tok, cache)
        assert full[[r for r in range(R + 1) if r not in rows.tolist()]].isnan().all()
        lg.append(full[rows])
    lg = torch.stack(lg, 1).cpu()
    for r in range(min(R, 12)):
        with torch.no_grad():
            ref = m(torch.tensor([seqs[r]], device=dev))[0, lens[r] - 1:].float().cpu()
        assert ((lg[r] - ref).abs() <= LOGITS * ref.abs().max()).all(), float((lg[r] - ref).abs().max() / ref.abs().max())


@pytest.mark.parametrize("kw", [{"tie_embeddings": False}, {"linear_impl": "torch", "norm_impl": "torch", "mlp_impl": "torch"}])
def test_paged_steps_of_other_models(dev, kw):
    # a head of its own, torch's own layers; a hook on the embedding, which is then called
    from fxlm import GPT, GPTConfig
    torch.manual_seed(2)
    m = GPT(GPTConfig(**{**dict(vocab_size=64, seq_len=80, n_layer=2, n_head=2, d_model=128), **kw})).to(dev).bfloat16()
    idx, lens = torch.randint(0, 64, (3, 20), device=dev), _ints([20, 3, 11], dev)
    tok = torch.tensor([5, 63, 0], device=dev)
    seen = []
    outs = []
    for hook in (False, True):
        if hook:
            m.tok_emb.register_forward_hook(lambda mod, args, out: seen.append(out.shape))
        cache = m.paged_cache(3, 8, 16)
        m.paged_prefill(idx, lens, cache)
        seen.clear()
        outs.append(m.paged_step(tok, cache))
        assert len(seen) == hook
    assert torch.equal(*outs)
    for r, n in enumerate(lens.tolist()):
        with torch.no_grad():
            ref = m(torch.cat([idx[r, :n], tok[r:r + 1]])[None])[0, -1].float()
        assert ((outs[0][r] - ref).abs() <= LOGITS * ref.abs().max()).all()
    out, scores = m.beam_search(idx, 6, beams=3, lens=lens)
    assert out.shape == (3, 3, 6) and torch.isfinite(scores).all()


def test_paged_step_rows_that_cannot_go_on(dev):
    # no pages, no position, no id: NaN, and the other rows as they were
    m = _model(dev, seq=48)
    idx = torch.randint(0, 64, (3, 48), device=dev)
    cache = m.paged_cache(4, 7, 16)
    lg = m.paged_prefill(idx, _ints([48, 16, 40], dev), cache)
    assert torch.isfinite(lg).all() and cache.uses.sum() == 7
    tok = torch.tensor([1, 1, 2, 3], device=dev)
    out = m.paged_step(tok, cache)
    assert out[[0, 1, 3]].isnan().all() and torch.isfinite(out[2]).all() and cache.lens.tolist() == [48, 16, 41, 0]
    ref = m(torch.cat([idx[2:, :40], tok[2:3, None]], 1))[0, -1].float()
    assert ((out[2] - ref).abs() <= LOGITS * ref.abs().max()).all()
    tok[2] = 64
    assert m.paged_step(tok, cache).isnan().all()
    lg2 = m.paged_prefill(idx, _ints([48, 0, 33], dev), cache, torch.tensor([2, 3, 1], device=dev))
    # row 0 keeps its three pages; of the four that are free row 1 takes three, and row 2, which comes after it, gets none
    assert torch.isfinite(lg2[2]).all() and lg2[[0, 1]].isnan().all() and cache.lens.tolist() == [48, 33, 0, 0]


def test_paged_step_of_some_rows(dev):
    m = _model(dev)
    idx, lens = torch.randint(0, 64, (4, 20), device=dev), _ints([20, 5, 16, 11], dev)
    a, b = m.paged_cache(4, 12, 16), m.paged_cache(4, 12, 16)
    for c in (a, b):
        m.paged_prefill(idx, lens, c)
    tok = torch.tensor([1, 2, 3, 4], device=dev)
    on = torch.tensor([True, False, True, False], device=dev)
    want, got = m.paged_step(tok, a), m.paged_step(tok, b, on)
    assert torch.equal(got[on], want[on]) and got[~on].isnan().all() and b.lens.tolist() == [21, 5, 17, 11]
    # the others go on from where they were
    got = m.paged_step(tok, b, ~on)
    assert torch.equal(got[~on], want[~on]) and got[on].isnan().all() and b.lens.tolist() == a.lens.tolist()
    assert not m.paged_step(tok, b, torch.zeros_like(on)).isfinite().any() and b.lens.tolist() == a.lens.tolist()


def test_generate_with_lengths(dev):
    m = _model(dev)
    idx, lens = torch.randint(0, 64, (5, 30), device=dev), _ints([30, 1, 17, 16, 9], dev)
    outs = []
    for graph in (True, False):
        outs.append(m.generate(idx, 12, temperature=1e-3, top_k=1, graph=graph, lens=lens))
    assert torch.equal(*outs)
    # each the likeliest of the whole model's logits, up to what the paths differ by
    for r, n in enumerate(lens.tolist()):
        seq = torch.cat([idx[r, :n], outs[0][r]])[None]
        with torch.no_grad():
            lg = m(seq)[0, n - 1:-1].float()
        assert (lg.gather(1, outs[0][r][:, None])[:, 0] >= lg.amax(-1) - 2 * LOGITS * lg.abs().amax()).all()


def _score(m, prompt, out, eos=None):
    with torch.no_grad():
        lp = torch.log_softmax(m(torch.cat([prompt, out])[None])[0, len(prompt) - 1:-1].double(), -1).gather(1, out[:, None])[:, 0]
    if eos is not None and bool((out == eos).any()):
        lp = lp[:int((out == eos).int().argmax()) + 1]
    return float(lp.sum()), len(lp)


@pytest.mark.parametrize("B,K,T,n,page", [(1, 4, 20, 10, 16), (3, 5, 37, 30, 16), (2, 32, 16, 5, 32), (17, 4, 9, 4, 16)])
def test_beam_search_scores(dev, B, K, T, n, page):
    # scores are those of the whole model over the beams' tokens; best first, no two alike; the same with and without a graph
    m = _model(dev)
    g = torch.Generator().manual_seed(T)
    idx, lens = torch.randint(0, 64, (B, T), generator=g).to(dev), torch.randint(1, T + 1, (B,), generator=g).int().to(dev)
    for ln in (None, lens):
        out, scores = m.beam_search(idx, n, beams=K, lens=ln, page=page)
        out2, scores2 = m.beam_search(idx, n, beams=K, lens=ln, page=page, graph=False)
        assert torch.equal(out, out2) and torch.equal(scores, scores2)
        assert out.shape == (B, K, n) and (scores[:, 1:] <= scores[:, :-1]).all()
        for b in range(B):
            assert len({tuple(x) for x in out[b].tolist()}) == K
            for k in range(0, K, max(1, K // 4)):
                ref, _ = _score(m, idx[b, :T if ln is None else int(ln[b])], out[b, k])
                assert abs(float(scores[b, k]) - ref) <= 0.02 * n + 0.02 * abs(ref)


def test_beam_search_with_an_end(dev):
    m = _model(dev, vocab=16)
    idx = torch.randint(0, 16, (4, 12), device=dev)
    for penalty in (0.0, 1.0):
        out, scores = m.beam_search(idx, 14, beams=6, eos=3, length_penalty=penalty)
        ended = 0
        for b in range(4):
            ranks = []
            for k in range(6):
                ref, n = _score(m, idx[b], out[b, k], 3)
                assert abs(float(scores[b, k]) - ref) <= 0.02 * 14 + 0.02 * abs(ref)
                ended += n < 14
                assert n == 14 or (out[b, k, n - 1:] == 3).all()
                ranks.append(float(scores[b, k]) / n ** penalty)
            assert all(x >= y - 1e-5 * abs(y) for x, y in zip(ranks, ranks[1:]))
        assert ended > 0


def test_beam_search_finds_the_best_where_it_tries_all(dev):
    # 8 tokens, 32 beams: two steps are exhaustive, and so is the third's choice of 32 among all that the best 32 go on by
    m = _model(dev, vocab=8, seed=3)
    prompt = torch.randint(0, 8, (1, 7), device=dev)
    out, scores = m.beam_search(prompt, 2, beams=32)
    every = torch.cartesian_prod(torch.arange(8), torch.arange(8)).to(dev)
    ref = torch.tensor([_score(m, prompt[0], t)[0] for t in every]).sort(descending=True)
    assert ((scores[0].cpu().double() - ref.values[:32]).abs() <= 0.02 * 2 + 0.02 * ref.values[:32].abs()).all()
    # fewer continuations than beams
    out, scores = m.beam_search(prompt, 1, beams=12)
    assert torch.isfinite(scores[0, :8]).all() and (scores[0, 8:] == -math.inf).all() and sorted(out[0, :8, 0].tolist()) == list(range(8))


def test_beam_search_refuses_a_model_that_is_not_finite(dev):
    m = _model(dev)
    with torch.no_grad():
        m.lnf_w[3] = math.nan
    with pytest.raises(RuntimeError):
        m.beam_search(torch.randint(0, 64, (2, 9), device=dev), 5)


def test_refusals_on_the_gpu(dev):
    from fxlm import beam_select, extend_pages, paged_attention, reorder_pages, store_pages
    bf = lambda *s: torch.zeros(*s, device=dev).bfloat16()   # noqa: E731
    q, k, t, n = bf(2, 4, 64), bf(5, 16, 2, 64), torch.zeros(2, 3, dtype=torch.int32, device=dev), _ints([1, 1], dev)
    odd = bf(5 * 16 * 2 * 64 + 1)[1:].view(5, 16, 2, 64)
    for err, args in [(TypeError, (q, k, k, t.long(), n)), (TypeError, (q, k, k, t[:1], n)), (TypeError, (q, k, k, t, n.long())), (TypeError, (q, k, k, t, n[:1])),
                      (ValueError, (q, odd, k, t, n)), (ValueError, (q, k[:0], k[:0], t, n)), (ValueError, (q[:, :, :32], k, k, t, n)),
                      (TypeError, (q, k.cpu(), k, t, n))]:
        with pytest.raises(err):
            paged_attention(*args)
    far = torch.empty(16 * 2 ** 23, device=dev, dtype=torch.bfloat16).as_strided((1, 16, 1, 64), (8, 2 ** 23, 64, 1))
    with pytest.raises(ValueError):     # a page's rows too far apart
        paged_attention(q[:, :2], far, far, t, n)
    u = torch.zeros(5, dtype=torch.int32, device=dev)
    for err, args, kw in [(TypeError, (t, n, n, u.cpu(), 16), {}), (TypeError, (t, n[:1], n, u, 16), {}), (ValueError, (t, n, n, u, 16), {"most": 0}),
                          (ValueError, (t.expand(2, -1)[:1].expand(2, -1), n, n, u, 16), {}), (TypeError, (t, n, n, u.repeat_interleave(2)[::2], 16), {}),
                          (ValueError, (t, n, n, u, 16), {"cache": [(k, k[:4])]}), (ValueError, (t, n, n, u, 32), {"cache": [(k, k)]}),
                          (ValueError, (t, n, n, u, 16), {"cache": [(k, odd)]}), (ValueError, (torch.zeros(8193, 1, dtype=torch.int32, device=dev), n, n, u, 16), {})]:
        with pytest.raises(err):
            extend_pages(*args, **kw)
        if not kw:
            with pytest.raises(err):
                reorder_pages(*args)
    for err, args in [(TypeError, (bf(2, 3, 2, 64), bf(2, 3, 2, 64), n[:, None].expand(2, 3), k, k)),
                      (ValueError, (bf(2, 3, 1, 64), bf(2, 3, 1, 64), torch.zeros(2, 3, dtype=torch.int64, device=dev), k, k)),
                      (ValueError, (bf(2, 3, 2, 64), bf(2, 3, 2, 64), torch.zeros(2, 3, dtype=torch.int64, device=dev), k[:1].expand(5, -1, -1, -1), k))]:
        with pytest.raises(err):
            store_pages(*args)
    x, s = torch.zeros(2, 3, 7, device=dev), torch.zeros(2, 3, device=dev)
    for err, args, kw in [(TypeError, (x, s.double()), {}), (ValueError, (x, s[:1]), {}), (TypeError, (x, s), {"done": s}), (TypeError, (x, s), {"weight": s.cpu()}),
                          (TypeError, (x.half(), s), {})]:
        with pytest.raises(err):
            beam_select(*args, **kw)

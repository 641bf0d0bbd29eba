"""Drafted decoding on the GPU against the 64-bit oracle (oracle/drafting.py).

Tolerances.  Tree attention: an output is rounded once (2^-8 of it, bf16's half step) and each p
is rounded to bf16 before its product (2^-8 of the sum of p |v|); scores, exponentials and sums are
fp32: a score's error is at most (D + 8) 2^-24 of the sum of |q k| scale, which moves every p by that
much relatively, and 2^-18 covers the exponentials and the sums of up to 64 partial ones.
Probabilities (fp32): a difference from the maximum is rounded once and multiplied by 1 / T, so p is
2^-24 (l - m) / T off besides the exponential's and the sum's few steps (128 of 2^-24).
Tokens, paths and moved rows are exact."""
import math

import pytest
import torch

from oracle import drafting as od

pytestmark = pytest.mark.gpu


def _parents(g, N, branch, count):
    p = [-1]
    for i in range(1, N):
        p.append(max(0, (i - 1) // branch - int(torch.randint(0, 2, (1,), generator=g))) if i < count else -1)
    return p


def _tree_case(B, N, H, Hkv, D, T, ctx, first=0, branch=2, seed=0, ragged=False):
    g = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g).bfloat16()   # noqa: E731
    tree = torch.stack([od.ancestors(_parents(g, first + N, branch, first + N - (b % N if ragged else 0)))[first:] for b in range(B)])
    return {"q": rn(B, N, H, D), "k": rn(B, T, Hkv, D), "v": rn(B, T, Hkv, D), "ctx": torch.tensor(ctx, dtype=torch.int32),
            "tree": tree, "first": first, "kn": rn(B, N, Hkv, D), "vn": rn(B, N, Hkv, D)}


def _check_tree(dev, c, new=True, o_nan_ok=False):
    from fxlm import tree_attention
    kn, vn = (c["kn"], c["vn"]) if new else (None, None)
    ro, rl, size, rk, rv = od.tree_attention(c["q"], c["k"], c["v"], c["ctx"], c["tree"], c["first"], k_new=kn, v_new=vn)
    d = {n: t.to(dev) if torch.is_tensor(t) else t for n, t in c.items()}
    o, l = tree_attention(d["q"], d["k"], d["v"], d["ctx"], d["tree"], first=c["first"], return_lse=True,   # noqa: E741
                          k_new=d["kn"] if new else None, v_new=d["vn"] if new else None)
    D = c["q"].shape[-1]
    # the largest sum of |q k| scale that any score can have
    mag = float(c["q"].double().norm(dim=-1).max() * max(rk.double().norm(dim=-1).nan_to_num(0, 0, 0).max(), 0.0)) / math.sqrt(D)
    score = (D + 8) * 2.0 ** -24 * mag
    fin = torch.isfinite(ro)
    tol = 2.0 ** -8 * (ro.abs() + size) + (2 * score + 2.0 ** -18) * size
    oc = o.double().cpu()
    assert torch.equal(torch.isfinite(oc), fin)
    assert ((oc - ro).abs() <= tol)[fin].all(), float(((oc - ro).abs() - tol)[fin].max())
    assert torch.equal(oc.isnan(), ro.isnan()) and torch.equal(oc[oc.isinf()], ro[ro.isinf()])
    lc = l.double().cpu()
    fl = torch.isfinite(rl)
    assert torch.equal(lc[~fl].nan_to_num(7.0, 9.0, -9.0), rl[~fl].nan_to_num(7.0, 9.0, -9.0))
    assert ((lc - rl).abs() <= score + 2.0 ** -18 + 2.0 ** -22 * rl.abs())[fl].all()
    same = lambda x, y: torch.equal(x.view(torch.int16), y.view(torch.int16))   # noqa: E731
    assert same(d["k"].cpu(), rk) and same(d["v"].cpu(), rv)
    return d, o, l


# rows of a key head: up to 32, 64, 128, 256 and past 256; caches that are split (long, few heads) and not;
# contexts of nothing, of one key, ending inside a tile and at its end
@pytest.mark.parametrize("new", [True, False])
@pytest.mark.parametrize("B,N,H,Hkv,D,T,ctx,first", [
    (1, 1, 1, 1, 64, 1, [0], 0),
    (1, 1, 1, 1, 128, 70, [64], 0),
    (2, 8, 3, 3, 64, 300, [217, 0], 0),
    (3, 16, 4, 2, 64, 1200, [1000, 31, 32], 0),
    (2, 16, 4, 2, 64, 2500, [2400, 1], 0),            # split
    (1, 5, 2, 1, 128, 5000, [4900], 0),               # split, one key head
    (3, 1, 2, 2, 64, 3000, [2990, 5, 0], 7),          # one token behind seven
    (2, 33, 4, 4, 128, 700, [600, 64], 0),            # 33 rows
    (2, 64, 2, 1, 64, 4200, [4100, 63], 0),           # 128 rows, split, 64 nodes
    (1, 57, 6, 2, 128, 2300, [2200], 3),              # 171 rows, split
    (1, 64, 5, 1, 64, 2100, [1999], 0),               # 320 rows: two groups, split
    (2, 64, 8, 1, 128, 500, [77, 400], 0),            # 512 rows: two groups
    (70, 2, 1, 1, 64, 1700, [(37 * i) % 1600 for i in range(70)], 0),   # more sequences than lanes
    (16, 17, 32, 8, 64, 4200, [40 + 9 * i for i in range(11)] + [4100, 0, 1100, 31, 7], 0),   # many key heads, split for the long one
])
def test_tree_attention(dev, B, N, H, Hkv, D, T, ctx, first, new):
    for branch, ragged in ((1, False), (3, first == 0)):
        _check_tree(dev, _tree_case(B, N, H, Hkv, D, T, ctx, first, branch, seed=B * N + D, ragged=ragged), new)


@pytest.mark.parametrize("B,N,H,Hkv,D,T,ctx", [(1, 1, 4, 4, 64, 500, [400]), (1, 8, 4, 4, 64, 300, [217]), (3, 16, 4, 2, 128, 500, [401, 0, 33]),
                                               (2, 1, 64, 2, 64, 2500, [2400, 700]), (1, 32, 1, 1, 64, 2100, [700])])
def test_tree_attention_of_few_rows_rounds_its_output_alone(dev, B, N, H, Hkv, D, T, ctx):
    # up to 32 rows a key head, as in the decode attention: one rounding to bf16, the output's (2^-8 of it); p reaches its
    # product to 2^-16, besides what the scores, exponentials and sums are off by (above)
    from fxlm import tree_attention
    c = _tree_case(B, N, H, Hkv, D, T, ctx, branch=2, seed=N + T)
    ro, _, size, rk, _ = od.tree_attention(c["q"], c["k"], c["v"], c["ctx"], c["tree"], k_new=c["kn"], v_new=c["vn"])
    o = tree_attention(*(c[n].to(dev) for n in ("q", "k", "v", "ctx", "tree")), k_new=c["kn"].to(dev), v_new=c["vn"].to(dev))
    score = (D + 8) * 2.0 ** -24 * float(c["q"].double().norm(dim=-1).max() * rk.double().norm(dim=-1).max()) / math.sqrt(D)
    tol = 2.0 ** -8 * ro.abs() + (2 * score + 2.0 ** -16 + 2.0 ** -18) * size
    err = (o.double().cpu() - ro).abs()
    assert (err <= tol).all(), float((err - tol).max())


def test_tree_attention_at_the_end_of_the_cache(dev):
    # nodes whose rows lie past the cache are nobody's key and not written; a context past it is the cache's
    for T, ctx, first in ((70, [66, 70], 0), (70, [64, 69], 3), (70, [71, 500], 0), (70, [-3, 5], 0)):
        for new in (True, False):
            _check_tree(dev, _tree_case(2, 9, 2, 1, 64, T, ctx, first, 2, seed=T + ctx[0]), new)


def test_tree_attention_strided_views(dev):
    # q, k_new and v_new out of one projection; caches with room between heads and sequences; a shared tree
    from fxlm import tree_attention
    B, N, H, Hkv, D, T = 2, 12, 6, 2, 64, 1500
    g = torch.Generator(device=dev).manual_seed(5)
    qkv = torch.randn(B, N, H + 2 * Hkv, D, device=dev, generator=g).bfloat16()
    both = torch.randn(T, 2, B, Hkv + 1, D + 8, device=dev, generator=g).bfloat16()
    k, v = (both[:, i, :, :Hkv, :D].transpose(0, 1) for i in range(2))
    kept = both.clone()
    q, kn, vn = qkv.split([H, Hkv, Hkv], dim=2)
    ctx = torch.tensor([1400, 333], dtype=torch.int32, device=dev)
    tree = od.ancestors([-1] + [i // 2 for i in range(N - 1)]).to(dev)
    o, l = tree_attention(q, k, v, ctx, tree, return_lse=True, k_new=kn, v_new=vn)   # noqa: E741
    o2, l2 = tree_attention(q.contiguous(), k.contiguous(), v.contiguous(), ctx.repeat_interleave(2)[::2],
                            tree.expand(B, -1).contiguous(), return_lse=True)
    assert torch.equal(o, o2) and torch.equal(l, l2)
    for b in range(B):
        kept[int(ctx[b]):int(ctx[b]) + N, 0, b, :Hkv, :D] = kn[b]
        kept[int(ctx[b]):int(ctx[b]) + N, 1, b, :Hkv, :D] = vn[b]
    assert torch.equal(both, kept)        # the rows of the tree, and nothing between them


@pytest.mark.parametrize("T", [300, 3000])   # one unit a sequence, and split
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_tree_attention_values_that_are_not_finite(dev, bad, T):
    # stale rows behind the tree and padding's rows may hold anything; a node's own row reaches the queries
    # that see it alone
    c = _tree_case(2, 10, 2, 2, 64, T, [T - 100, 40], 0, 2, seed=9)
    c["tree"][0, 7] = 0
    for t in ("k", "v"):
        c[t][0, T - 100 + 10:] = bad
        c[t][1, 50:] = bad
        c[t][0, T - 93] = bad       # the padding's
    c["kn"][0, 7] = bad
    c["vn"][0, 7] = bad
    _check_tree(dev, c)
    c["vn"][0, 3, :, 5] = bad       # single elements of a value; every element of another
    c["vn"][1, 2] = bad
    _, o, _ = _check_tree(dev, c)
    seen = [(int(c["tree"][0, i]) >> 3) & 1 for i in range(10)]
    assert any(seen) and not all(seen)
    assert [bool((~torch.isfinite(o[0, i])).any()) for i in range(10)] == [bool(s) for s in seen]
    c["kn"][1, 4, 0] = math.nan     # and of a key
    c["k"][1, 44, 0] = math.nan
    from fxlm import tree_attention
    d = {n: t.to(dev) if torch.is_tensor(t) else t for n, t in c.items()}
    o = tree_attention(d["q"], d["k"], d["v"], d["ctx"], d["tree"], k_new=d["kn"], v_new=d["vn"])
    for i in range(10):
        if (int(c["tree"][1, i]) >> 4) & 1:
            assert o[1, i, 0].isnan().all()
        elif not (int(c["tree"][1, i]) >> 2) & 1:
            assert torch.isfinite(o[1, i]).all()


def test_tree_attention_agrees_with_decode_attention(dev):
    # one node, its key in place: the decode step's softmax over lens = ctx + 1 keys
    from fxlm import tree_attention
    from fxlm.attention import decode_attention
    g = torch.Generator(device=dev).manual_seed(2)
    B, H, D, T = 3, 4, 64, 2000
    q = torch.randn(B, H, D, device=dev, generator=g).bfloat16()
    k, v = (torch.randn(B, T, H, D, device=dev, generator=g).bfloat16() for _ in range(2))
    ctx = torch.tensor([1999, 0, 700], dtype=torch.int32, device=dev)
    a, la = decode_attention(q, k, v, ctx + 1, return_lse=True)
    o, l = tree_attention(q[:, None], k, v, ctx, torch.ones(B, 1, dtype=torch.int64, device=dev), return_lse=True)   # noqa: E741
    assert ((a.double() - o[:, 0].double()).abs() <= 2.0 ** -7 * a.double().abs() + 2.0 ** -8).all()
    assert ((la - l[:, 0]).abs() <= 1e-4).all()


def test_tree_attention_of_far_rows(dev):
    # rows behind element 2^31 of a cache: 2 sequences of 1,100,000 rows of 8 heads of 128
    from fxlm import tree_attention
    B, T, H, D, N = 2, 1100000, 8, 128, 4
    k = torch.zeros(B, T, H, D, device=dev, dtype=torch.bfloat16)
    v = torch.zeros_like(k)
    g = torch.Generator(device=dev).manual_seed(4)
    at = T - 100
    k[1, at:], v[1, at:] = (torch.randn(T - at, H, D, device=dev, generator=g).bfloat16() for _ in range(2))
    k[1, :at, :, 0] = -60.0          # scores far below the tail's
    q = torch.randn(B, N, H, D, device=dev, generator=g).bfloat16()
    q[..., 0] = 40.0
    kn, vn = (torch.randn(B, N, H, D, device=dev, generator=g).bfloat16() for _ in range(2))
    tree = od.ancestors([-1, 0, 0, 2]).expand(B, -1)
    ctx = torch.tensor([3, T - 9], dtype=torch.int32, device=dev)
    o = tree_attention(q, k, v, ctx, tree.to(dev), k_new=kn, v_new=vn)
    assert torch.equal(k[1, T - 9:T - 5], kn[1]) and torch.equal(v[1, T - 9:T - 5], vn[1])
    ro, _, size, _, _ = od.tree_attention(q[1:].cpu(), k[1:, at:].cpu(), v[1:, at:].cpu(), [T - 9 - at], tree[1:], k_new=kn[1:].cpu(), v_new=vn[1:].cpu())
    assert ((o[1:].double().cpu() - ro).abs() <= 2.0 ** -8 * (ro.abs() + size) + 1e-3 * size).all()


# ---- probabilities ---------------------------------------------------------------------------


def _check_probs(dev, x, T, k):
    from fxlm import sampling_probs
    p = sampling_probs(x.to(dev), T, k)
    ref = od.sampling_probs(x, T, k)
    assert p.dtype == torch.float32 and p.shape == x.shape
    pc = p.double().cpu()
    m = x.double().amax(-1, keepdim=True)
    far = ((m - x.double()) / T).nan_to_num(0, 0, 0).clamp_max(200)
    assert torch.equal(pc > 0, ref > 1.2e-38) or ((pc > 0) != (ref > 1.2e-38)).logical_and(ref > 3e-38).sum() == 0
    err = (pc - ref).abs() - (2.0 ** -24 * (128 + 2 * far) * ref + 1.2e-38)
    assert (err <= 0).all(), float(err.max())
    return p


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape,k", [((1,), 0), ((3, 1), 5), ((2, 7), 3), ((5, 255), 0), ((2, 3, 1000), 50), ((4, 4097), 4096), ((3, 50304), 50),
                                     ((2, 50304), 1), ((2, 50303), 0), ((3, 131071), 200), ((2, 131071), 20000), ((1, 300001), 50)])
def test_sampling_probs(dev, shape, k, dtype):
    g = torch.Generator().manual_seed(len(shape) + k)
    x = (torch.randn(*shape, generator=g) * 3).to(dtype)
    for T in (0.7, 1.0):
        _check_probs(dev, x, T, k)


def test_sampling_probs_orders_and_ties(dev):
    V = 9000
    up = torch.arange(V).float() / 500
    x = torch.stack([up, up.flip(0), torch.zeros(V), torch.cat([torch.full((V - 70,), -1.0), torch.full((70,), 2.0)]),
                     torch.where(torch.arange(V) % 2 == 0, 0.0, -0.0), up.roll(V // 2)])
    for k in (1, 49, 50, 64, 70, 71, 1024, 1025, 8999):
        p = _check_probs(dev, x, 0.9, k)
        assert (p[2] > 0).all() and (p[4] > 0).all()                     # equals of the last kept stay: both zeros alike
        assert int((p[3] > 0).sum()) == (70 if k <= 70 else V)
        assert int((p[0] > 0).sum()) == k
    # a row that one thread's stride holds the largest of
    y = torch.randn(V, generator=torch.Generator().manual_seed(1))
    y[::1024] += 30
    y[4::4096] += 30
    _check_probs(dev, y[None], 1.0, 50)


def test_sampling_probs_masked_and_not_finite(dev):
    from fxlm import sampling_probs
    x = torch.randn(6, 5001, generator=torch.Generator().manual_seed(7))
    x[0, 100:] = -math.inf
    x[1, :] = -math.inf
    x[2, 77] = math.nan
    x[3, 5000] = math.inf
    x[4, 1:] = torch.finfo(torch.float32).min     # masks of the type's lowest value
    x[5, :] = torch.finfo(torch.float32).min
    for k in (0, 50, 200):
        p = sampling_probs(x.to(dev), 0.5, k).cpu()
        assert torch.equal(p[0] > 0, od.sampling_probs(x[:1], 0.5, k)[0] > 0) and abs(float(p[0].sum()) - 1) < 1e-5
        assert not p[1].any() and p[2].isnan().all() and p[3].isnan().all()
        assert float(p[4, 0]) == 1.0 and not p[4, 1:].any()
        assert ((p[5] - 1 / 5001).abs() <= 2.0 ** -20 / 5001).all()
    # temperatures at the ends: the largest alone, and all that are not masked alike
    p = sampling_probs(x[:1].to(dev), 1e-30).cpu()
    assert float(p[0, x[0].argmax()]) == 1.0 and int((p > 0).sum()) == 1
    p = sampling_probs(x[:1].to(dev), 1e30).cpu()
    assert ((p[0, :100] - 0.01).abs() <= 2.0 ** -20 / 100).all() and not p[0, 100:].any()
    # a slice of positions, rows at an odd address
    y = torch.randn(3, 5, 1003, generator=torch.Generator().manual_seed(8)).to(dev)
    assert torch.equal(sampling_probs(y[:, -1], 0.8, 20), sampling_probs(y[:, -1].clone(), 0.8, 20))
    flat = y.flatten()[1:1 + 4 * 1001].view(4, 1001)
    assert torch.equal(sampling_probs(flat, 0.8, 20), sampling_probs(flat.clone(), 0.8, 20))
    assert sampling_probs(y[:0]).shape == (0, 5, 1003)


@pytest.mark.parametrize("T", [9.999999414548473e29, 9.999999414548476e29, 9.7e29, 8.3e29, 1e29])
def test_sampling_probs_masked_at_the_largest_temperatures(dev, T):
    # log2(e) / T in two floats: of the first two what the first float leaves is no float at all
    from fxlm import sampling_probs
    x = torch.randn(2, 5001, generator=torch.Generator().manual_seed(9))
    x[:, 100:] = -math.inf
    x[1, 7] = -1e30
    for k in (0, 200):
        p = sampling_probs(x.to(dev), T, k).double().cpu()
        ref = od.sampling_probs(x, T, k)
        # exact differences, one rounding each of the product, the power and the quotient, and the sum's 100 terms
        assert ((p - ref).abs() <= 2.0 ** -24 * 128 * ref).all() and not p[:, 100:].any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V,k,left", [(256, 50, None), (257, 200, None), (512, 384, None), (1000, 300, None), (2000, 300, None), (5001, 50, 40),
                                      (5001, 50, 50), (5001, 50, 51), (5001, 384, 1030), (50304, 50, 1), (50304, 200, 199), (131071, 50, 49)])
def test_sampling_probs_of_few_logits(dev, V, k, left, dtype):
    # fewer threads than top_k hold logits: a short row, or one that a mask leaves few of (the rest -inf, or the lowest value)
    g = torch.Generator().manual_seed(V + k)
    x = (torch.randn(4, V, generator=g) * 3).to(dtype)
    if left:
        out = torch.ones(4, V, dtype=torch.bool).scatter_(1, torch.rand(4, V, generator=g).topk(left, -1).indices, False)
        x[:3][out[:3]] = -math.inf
        x[3][out[3]] = torch.finfo(dtype).min
    _check_probs(dev, x, 0.8, k)


def test_sampling_probs_of_a_masked_row_takes_no_counted_passes(dev):
    # 40 logits of 50,304 with top-k 50 took 8 times what 60 did: each -inf was listed, the list ran over, and 32 passes over
    # the row found the bound.  Four times would be that again
    from fxlm import sampling_probs
    x = torch.randn(50304, generator=torch.Generator().manual_seed(2))

    def least(left):
        y = x.clone()
        y[torch.randperm(50304, generator=torch.Generator().manual_seed(left))[left:]] = -math.inf
        y = y[None].to(dev)
        took = []
        for i in range(8):
            a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            a.record()
            for _ in range(100):
                sampling_probs(y, 0.8, 50)
            b.record()
            torch.cuda.synchronize()
            took.append(a.elapsed_time(b))
        return min(took)

    assert least(40) < 4 * least(60)


@pytest.mark.parametrize("V,dtype", [(20003, torch.float32), (50304, torch.float32), (65536, torch.bfloat16), (131071, torch.bfloat16)])
def test_sampling_probs_of_many_long_rows(dev, V, dtype):
    # more rows than the GPU runs at once, rows without probabilities among them: each as it is alone
    from fxlm import sampling_probs
    n = torch.cuda.get_device_properties(dev).multi_processor_count
    x = (torch.randn(2 * n + 3, V, device=dev, generator=torch.Generator(device=dev).manual_seed(V)) * 2).to(dtype)
    x[1] = -math.inf
    x[n - 1, 5] = math.nan
    x[n] = -math.inf
    x[n + 2, V - 1] = math.inf
    x[2 * n + 1, :V - 1] = -math.inf
    x[3] = 0.5                          # equals: more than the list holds
    for k in (0, 50):
        p = sampling_probs(x, 0.8, k)
        assert not p[1].any() and not p[n].any() and p[n - 1].isnan().all() and p[n + 2].isnan().all()
        for rows in torch.arange(2 * n + 3).split(64):
            rows = torch.tensor([i for i in rows.tolist() if i not in (1, n - 1, n, n + 2)], device=dev)
            y, pc = x[rows].double(), p[rows].double()
            ref = od.sampling_probs(y, 0.8, k)
            far = ((y.amax(-1, keepdim=True) - y) / 0.8).nan_to_num(0, 0, 0).clamp_max(200)
            assert ((pc > 0) != (ref > 1.2e-38)).logical_and(ref > 3e-38).sum() == 0
            assert ((pc - ref).abs() <= 2.0 ** -24 * (128 + 2 * far) * ref + 1.2e-38).all()   # as above
        assert torch.equal(sampling_probs(x, 0.8, k).nan_to_num(2), p.nan_to_num(2))


@pytest.mark.parametrize("V,dtype", [(70001, torch.float32), (140003, torch.bfloat16)])
def test_sampling_probs_of_many_rows_past_the_registers(dev, V, dtype):
    # rows of which a workgroup holds a part and reads the rest again, several a workgroup
    from fxlm import sampling_probs
    n = torch.cuda.get_device_properties(dev).multi_processor_count + 40
    x = (torch.randn(n, V, device=dev, generator=torch.Generator(device=dev).manual_seed(V)) * 2).to(dtype)
    x[2, V - 40000:] = -math.inf
    x[n - 1, V - 1] = 40
    for k in (0, 50):
        p = sampling_probs(x, 0.8, k)
        rows = [0, 1, 2, 39, 40, 41, n - 41, n - 40, n - 2, n - 1]
        y, pc = x[rows].double().cpu(), p[rows].double().cpu()
        ref = od.sampling_probs(y, 0.8, k)
        far = ((y.amax(-1, keepdim=True) - y) / 0.8).nan_to_num(0, 0, 0).clamp_max(200)
        assert ((pc > 0) != (ref > 1.2e-38)).logical_and(ref > 3e-38).sum() == 0
        assert ((pc - ref).abs() <= 2.0 ** -24 * (128 + 2 * far) * ref + 1.2e-38).all()   # as above
        assert torch.equal(sampling_probs(x, 0.8, k), p)


def test_sampling_probs_of_more_rows_than_a_launch_has(dev):
    from fxlm import sampling_probs
    n = 2 ** 22 + 13                 # workgroups of 1,024 threads: past 2^32 work items
    x = torch.randn(16, 5, generator=torch.Generator().manual_seed(3))
    for dtype in (torch.float32, torch.bfloat16):
        r = x.to(dtype).to(dev)
        want = sampling_probs(r, 0.7, 3)
        got = sampling_probs(r.repeat(n // 16 + 1, 1)[:n].contiguous(), 0.7, 3)
        assert torch.equal(got[:n // 16 * 16].view(-1, 16, 5), want.expand(n // 16, 16, 5)) and torch.equal(got[n // 16 * 16:], want[:n % 16])


def test_batches_past_a_launch_are_refused(dev):
    from fxlm import tree_attention, verify_draft
    n = 2 ** 22
    one = torch.ones(n, 1, 1, device=dev)
    zero = torch.zeros(n, 1, dtype=torch.int64, device=dev)
    with pytest.raises(ValueError, match="grid too large"):
        verify_draft(one, zero, zero.int() - 1, one[..., 0] * 0)
    B = 2 ** 17                      # 64 key heads each: 2^23 workgroups of 512 threads
    q = torch.zeros(1, 1, 64, 64, dtype=torch.bfloat16, device=dev).expand(B, -1, -1, -1)
    kv = torch.zeros(1, 1, 64, 64, dtype=torch.bfloat16, device=dev).expand(B, -1, -1, -1)
    with pytest.raises(ValueError, match="grid too large"):
        tree_attention(q, kv, kv, torch.zeros(B, dtype=torch.int32, device=dev), torch.ones(1, dtype=torch.int64, device=dev))


# ---- verification ----------------------------------------------------------------------------


def _draft_case(B, N, V, branch, seed, ragged, drafted, k=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(B, N, V, generator=g) * 2
    p = od.sampling_probs(x, 0.8, k).float()
    q = od.sampling_probs(x * 0.9 + 0.7 * torch.randn(B, N, V, generator=g), 0.8, k).float()
    par = torch.tensor([_parents(g, N, branch, N - (b % N if ragged else 0)) for b in range(B)], dtype=torch.int32)
    tok = torch.zeros(B, N, dtype=torch.int64)
    for b in range(B):
        for i in range(N):
            tok[b, i] = torch.multinomial(q[b, max(int(par[b, i]), 0)], 1, generator=g)
    return p, tok, par, torch.rand(B, N, generator=g), q if drafted else None


def _check_verify(dev, p, tok, par, u, q):
    from fxlm import verify_draft
    got = verify_draft(*(t.to(dev) for t in (p, tok, par, u)), draft_probs=None if q is None else q.to(dev))
    ref = od.verify_draft(p, tok, par, u, q)
    for a, r, name in zip(got, ref, ("tokens", "path", "counts")):
        assert torch.equal(a.cpu(), r), name
    return got


@pytest.mark.parametrize("drafted", [True, False])
@pytest.mark.parametrize("B,N,V,branch,k", [(1, 1, 1, 1, 0), (3, 2, 2, 1, 0), (5, 6, 257, 1, 0), (40, 8, 100, 2, 0), (30, 16, 1000, 3, 20),
                                            (9, 64, 513, 4, 0), (12, 7, 50304, 6, 0), (3, 5, 131071, 4, 50), (200, 4, 33, 3, 0)])
def test_verify_draft(dev, B, N, V, branch, k, drafted):
    for seed in range(3):
        _check_verify(dev, *_draft_case(B, N, V, branch, 100 * seed + N, seed == 1, drafted, k))


def test_verify_draft_of_the_largest_vocabulary(dev):
    # 2^20 ids, the most that it takes; one more is refused
    for drafted in (True, False):
        _check_verify(dev, *_draft_case(2, 4, 2 ** 20, 2, 7, False, drafted, 0))
    from fxlm import verify_draft
    i = torch.zeros(1, 2, dtype=torch.int64, device=dev)
    with pytest.raises(ValueError):
        verify_draft(torch.zeros(1, 2, 2 ** 20 + 1, device=dev), i, i.int() - 1, torch.zeros(1, 2, device=dev))


def test_verify_draft_edges(dev):
    # ids outside the vocabulary, parents that are none, numbers at the ends, rows without mass, duplicates
    p, tok, par, u, q = _draft_case(16, 12, 300, 3, 5, False, True)
    tok[0, 1:4], tok[1, 1], par[2, 3], par[3, 5], par[4, 1] = 300, -7, 3, 9, -5
    u[5], u[6], u[7, 0] = 0.0, 1.0 - 2.0 ** -24, 1.0 - 2.0 ** -24
    p[8], p[9, 0, 5:] = 0.0, 0.0
    tok[10, 1:] = tok[10, 1]
    q[11] = p[11]                    # the draft is the target: every first child is accepted
    q[12], p[13, :, ::2] = 0.0, 0.0
    for d in (q, None):
        out, path, n = _check_verify(dev, p, tok, par, u, d)
        assert int(out[8, 0]) == -1 and int(n[8]) == 1
        assert int((out[9, 0] < 5)) or int(n[9]) > 1
    # NaN is no mass: refused, and a row of it gives -1
    p[:], u[:] = math.nan, 0.5
    from fxlm import verify_draft
    out, path, n = verify_draft(*(t.to(dev) for t in (p, tok, par, u)), draft_probs=q.to(dev))
    assert (n == 1).all() and (out == -1).all() and (path[:, 0] == 0).all() and (path[:, 1:] == -1).all()


@pytest.mark.parametrize("V", [5, 700, 20001])
def test_verify_draft_rows_that_nothing_was_drawn_from(dev, V):
    # a leaf's draft row is nobody's distribution: whatever it holds, the last token comes from the target's row
    p, tok, par, u, q = _draft_case(24, 9, V, 2, 3, False, True)
    q = (q + 3 * p) / 4              # near the target: walks that reach the leaves
    leaf = torch.ones(24, 9, dtype=torch.bool)
    leaf.scatter_(1, par.clamp_min(0).long(), False)
    for bad in (math.nan, math.inf, -math.inf, 1e38):
        q[leaf] = bad
        _, path, n = _check_verify(dev, p, tok, par, u, q)
        end = path.cpu().gather(1, n.cpu().long()[:, None] - 1)[:, 0].long()
        assert bool(leaf[torch.arange(24), end].any())


def test_verified_tokens_are_distributed_as_the_target(dev):
    # 200,000 sequences, 5 standard deviations: the first token, and the second after each first
    from fxlm import verify_draft
    g = torch.Generator(device=dev).manual_seed(11)
    B, N, V = 200000, 6, 6
    p = torch.softmax(torch.randn(N, V, device=dev, generator=g), -1)
    q = torch.softmax(torch.randn(N, V, device=dev, generator=g), -1)
    # children of the root 1 and 2, of 1: 3 and 4, of 2: 5; a node's distribution hangs on its token: here each has its own
    par = torch.tensor([-1, 0, 0, 1, 1, 2], dtype=torch.int32, device=dev).expand(B, N).contiguous()
    tok = torch.stack([torch.multinomial(q[max(i, 0)], B, replacement=True, generator=g) for i in (-1, 0, 0, 1, 1, 2)], 1)
    # a distribution by token, so that the law of (first, second) is a product: rows of p and q by the parent's token
    P = torch.softmax(torch.randn(V, V, device=dev, generator=g), -1)
    pr = p[None].expand(B, N, V).clone()
    pr[:, 1:] = P[tok[:, 1:]]
    qr = q[None].expand(B, N, V).contiguous()
    out, path, n = verify_draft(pr, tok, par, torch.rand(B, N, device=dev, generator=g), draft_probs=qr)
    f = torch.bincount(out[:, 0], minlength=V).double() / B
    p0 = p[0].double()
    assert ((f - p0).abs() <= 5 * (p0 * (1 - p0) / B).sqrt()).all()
    two = n >= 2
    for x in range(V):
        s = out[two & (out[:, 0] == x), 1]
        if len(s) > 1000:
            f, px = torch.bincount(s, minlength=V).double() / len(s), P[x].double()
            assert ((f - px).abs() <= 5 * (px * (1 - px) / len(s)).sqrt()).all()


# ---- compaction ------------------------------------------------------------------------------


@pytest.mark.parametrize("L,B,N,H,D,T", [(1, 1, 1, 1, 64, 2), (3, 4, 9, 2, 64, 50), (2, 3, 64, 12, 64, 200), (40, 2, 5, 1, 128, 20), (33, 1100, 3, 1, 8, 6)])
def test_compact_cache(dev, L, B, N, H, D, T):
    from fxlm import compact_cache
    g = torch.Generator().manual_seed(L + N)
    cache = [tuple(torch.randint(-30000, 30000, (B, T, H, D), generator=g, dtype=torch.int16).view(torch.bfloat16) for _ in range(2)) for _ in range(L)]
    counts = torch.tensor([1 + (5 * b) % N for b in range(B)], dtype=torch.int32)
    ctx = torch.tensor([(7 * b) % (T - N + 1) for b in range(B)], dtype=torch.int32)
    path = torch.full((B, N), -1, dtype=torch.int32)
    for b in range(B):
        path[b, :counts[b]] = torch.cat([torch.zeros(1), 1 + torch.randperm(N - 1, generator=g)[:counts[b] - 1].sort().values]).int()
    ref, rctx = od.compact_cache(cache, ctx, path, counts)
    mine = [(k.to(dev), v.transpose(1, 2).contiguous().to(dev).transpose(1, 2)) for k, v in cache]     # two layouts
    got = compact_cache(mine, ctx.to(dev), path.to(dev), counts.to(dev))
    assert torch.equal(got.cpu(), rctx)
    for t, r in zip((t for kv in mine for t in kv), ref):
        assert torch.equal(t.cpu().view(torch.int16), r.contiguous().view(torch.int16))


def test_compact_cache_passes_over_what_is_outside(dev):
    from fxlm import compact_cache
    k = torch.arange(2 * 12 * 8).view(2, 12, 1, 8).bfloat16().to(dev)
    v = k + 1
    k0 = k.clone()
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)   # noqa: E731
    got = compact_cache([(k, v)], i32(10, -4), i32([0, 5, 900], [0, 2, 3]), i32(3, 3))      # past the cache; a negative context
    assert torch.equal(k, k0) and got.tolist() == [13, -1]
    got = compact_cache([(k, v)], i32(2, 2), i32([-1, -1, -1], [0, 3, 3]), i32(-5, 9))      # counts outside: none, all
    k0[1, 3], k0[1, 4] = k0[1, 5].clone(), k0[1, 5].clone()
    assert torch.equal(k, k0) and torch.equal(v, k0 + 1) and got.tolist() == [2, 5]


def test_compact_cache_moves_a_shared_tensor_once(dev):
    from fxlm import compact_cache
    k, v = (torch.randn(2, 20, 1, 64, device=dev).bfloat16() for _ in range(2))
    ctx, path, n = (torch.tensor(x, dtype=torch.int32, device=dev) for x in ([3, 4], [[0, 2, 3, 7], [0, 1, 4, 5]], [4, 4]))
    ref, _ = od.compact_cache([(k.cpu(), v.cpu())], ctx.cpu(), path.cpu(), n.cpu())
    compact_cache([(k, v), (k, v), (v, k)], ctx, path, n)
    assert torch.equal(k.cpu(), ref[0]) and torch.equal(v.cpu(), ref[1])


# ---- together --------------------------------------------------------------------------------


def test_operators_in_a_row_on_another_stream_and_in_a_graph(dev):
    # attention over the drafted tree, probabilities, verification, compaction: eager on the current stream,
    # on another one, and captured twice and replayed with new inputs
    from fxlm import compact_cache, sampling_probs, tree_attention, verify_draft
    B, N, H, D, T, V = 3, 9, 4, 64, 4000, 700
    g = torch.Generator().manual_seed(21)
    head = (torch.randn(V, H * D, generator=g) * 0.3).to(dev)

    def inputs(seed):
        g = torch.Generator().manual_seed(seed)
        rn = lambda *s: torch.randn(*s, generator=g).bfloat16().to(dev)   # noqa: E731
        par = [_parents(g, N, 2, N) for _ in range(B)]
        return {"q": rn(B, N, H, D), "kn": rn(B, N, H, D), "vn": rn(B, N, H, D), "k": rn(B, T, H, D), "v": rn(B, T, H, D),
                "ctx": torch.tensor([3000, 40 + seed, 1111], dtype=torch.int32, device=dev), "tree": torch.stack([od.ancestors(p) for p in par]).to(dev),
                "par": torch.tensor(par, dtype=torch.int32, device=dev), "tok": torch.randint(0, V, (B, N), generator=g).to(dev),
                "u": torch.rand(B, N, generator=g).to(dev) * 0.02}

    def step(s):
        o = tree_attention(s["q"], s["k"], s["v"], s["ctx"], s["tree"], k_new=s["kn"], v_new=s["vn"])
        p = sampling_probs(torch.mm(o.view(B * N, -1).float(), head.t()).view(B, N, V), 0.9, 40)
        out, path, n = verify_draft(p, s["tok"], s["par"], s["u"])
        ctx = compact_cache([(s["k"], s["v"])], s["ctx"], path, n)
        return o, p, out, path, n, ctx

    want = {}
    for seed in (1, 2, 3):
        s = inputs(seed)
        want[seed] = [t.clone() for t in step(s)] + [s["k"].clone(), s["v"].clone()]
        for b in range(B):   # what verification saw, by the oracle
            r = od.verify_draft(want[seed][1].cpu(), s["tok"].cpu(), s["par"].cpu(), s["u"].cpu())
            assert all(torch.equal(a.cpu(), x) for a, x in zip(want[seed][2:5], r))
    side = torch.cuda.Stream()
    s = inputs(1)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = list(step(s))
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got + [s["k"], s["v"]], want[1]))
    graphs = []
    for _ in range(2):
        s = inputs(1)
        with torch.cuda.stream(side):
            step(s)
        torch.cuda.current_stream().wait_stream(side)
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            got = step(s)
        graphs.append((gr, s, got))
    for seed in (2, 1, 3, 3):
        for gr, s, got in graphs:
            for n, t in inputs(seed).items():
                s[n].copy_(t)
        for gr, s, got in graphs:       # two graphs, one behind the other
            gr.replay()
        torch.cuda.synchronize()
        for gr, s, got in graphs:
            for a, b in zip(list(got) + [s["k"], s["v"]], want[seed]):
                assert torch.equal(a, b), seed
        x = inputs(seed)                # eager work between the replays
        assert all(torch.equal(a, b) for a, b in zip(step(x), want[seed]))


# ---- the model's steps -----------------------------------------------------------------------


def _model(dev, seed=0, seq_len=160, n_layer=2, **kw):
    from fxlm.model import GPT, GPTConfig
    torch.manual_seed(seed)
    m = GPT(GPTConfig(vocab_size=256, seq_len=seq_len, n_layer=n_layer, n_head=2, d_model=128, **kw)).to(dev).bfloat16().eval()
    for blk in m.blocks:
        torch.nn.init.normal_(blk.proj.weight, std=0.05)
        torch.nn.init.normal_(blk.fc2.weight, std=0.05)
    return m


@pytest.mark.parametrize("B,kw", [(2, {}), (9, {}), (2, dict(norm_impl="torch", mlp_impl="torch", linear_impl="torch"))])
def test_tree_step_logits_are_the_full_forwards(dev, B, kw):
    # every node of a tree against a full forward over its own prefix (9 x 8 rows: past the few-row kernels);
    # the bound of the cached step's test
    m = _model(dev, **kw)
    g = torch.Generator(device=dev).manual_seed(3)
    T, parents = 37, [-1, 0, 0, 1, 1, 2, 4, 6]
    N, depth = len(parents), [0, 1, 1, 2, 2, 2, 3, 4]
    idx = torch.randint(0, 256, (B, T), device=dev, generator=g)
    tok = torch.randint(0, 256, (B, N), device=dev, generator=g)
    cache = m._new_cache(B, T + N)
    m.prefill(idx, cache)
    ctx = torch.full((B,), T, dtype=torch.int32, device=dev)
    bits, dep = od.ancestors(parents).to(dev), torch.tensor(depth, device=dev)
    lg = m.tree_step(tok, dep, cache, ctx, bits)
    again = m._new_cache(B, T + N)
    m.prefill(idx, again)
    parts = [m.tree_step(tok[:, a:b], dep[a:b], again, ctx, bits[a:b], first=a) for a, b in ((0, 1), (1, 3), (3, 6), (6, 8))]
    with torch.no_grad():
        for i in range(N):
            chain = []
            j = i
            while j >= 0:
                chain.append(j)
                j = parents[j]
            ref = m(torch.cat([idx, tok[:, chain[::-1]]], 1))[:, -1].float()
            scale = max(1.0, float(ref.abs().max()))
            assert float((lg[:, i] - ref).abs().max()) <= 3e-2 * scale
            assert float((torch.cat(parts, 1)[:, i] - ref).abs().max()) <= 3e-2 * scale


def test_tree_step_of_padding_with_tokens_that_are_no_ids(dev):
    # what verify_draft returns behind the last token is -1: nodes that are padding, and no node sees them
    m = _model(dev)
    idx = torch.randint(0, 256, (2, 11), device=dev, generator=torch.Generator(device=dev).manual_seed(4))
    ctx = torch.full((2,), 11, dtype=torch.int32, device=dev)
    dep = torch.tensor([0, 1, 2, 2, 1], dtype=torch.int32, device=dev)
    bits = od.ancestors([-1, 0, 1, -1, -1]).to(dev)
    res = []
    for t3, t4 in ((7, 9), (-1, 256), (2 ** 62, -2 ** 62)):
        cache = m._new_cache(2, 20)
        m.prefill(idx, cache)
        tok = torch.tensor([[1, 2, 3, t3, t4]] * 2, device=dev)
        res.append((m.tree_step(tok, dep, cache, ctx, bits)[:, :3], [t[:, :14].clone() for kv in cache for t in kv]))
    for lg, rows in res[1:]:
        assert torch.equal(lg, res[0][0]) and all(torch.equal(a, b) for a, b in zip(rows, res[0][1]))


@pytest.mark.parametrize("first,hook", [(0, False), (1, False), (0, True)])
def test_tree_step_of_nodes_that_cannot_be(dev, first, hook):
    # no id, no position of the model, no row of the cache: NaN for the node and those that see it, and for no other; with a
    # hook on the embedding, which is called then, too
    m = _model(dev, seq_len=40)
    called = []
    if hook:
        m.tok_emb.register_forward_hook(lambda *a: called.append(1))
    parents, dep = [-1, 0, 0, 1, 2, 4], torch.tensor([0, 1, 1, 2, 2, 3], dtype=torch.int32, device=dev)
    bits = od.ancestors(parents).to(dev)
    idx = torch.randint(0, 256, (3, 37), device=dev, generator=torch.Generator(device=dev).manual_seed(4))

    def step(ctx, tok, rows, depth=dep, bits=bits):
        cache = m._new_cache(3, rows)
        m.prefill(idx[:, :max(ctx)], cache)
        ctx = torch.tensor(ctx, dtype=torch.int32, device=dev)
        tok = torch.tensor(tok, device=dev)
        if first:
            m.tree_step(tok[:, :1], depth[..., :1], cache, ctx, bits[:1])
        return m.tree_step(tok[:, first:], depth[..., first:], cache, ctx, bits[first:], first=first)

    good = [[1, 2, 3, 4, 5, 6]] * 3
    ref = step([30] * 3, good, 48)
    assert torch.isfinite(ref).all() and bool(called) == hook
    assert torch.equal(step([30] * 3, good, 48, depth=dep.long().expand(3, -1)), ref)
    for bad in (256, -1, 2 ** 40):
        lg = step([30] * 3, [good[0], [1, 2, bad, 4, 5, 6], good[0]], 48)
        want = torch.zeros(3, 6, dtype=torch.bool, device=dev)
        want[1, [2, 4, 5]] = True
        assert torch.equal(lg.isnan().all(-1), want[:, first:]) and torch.equal(lg.isnan().any(-1), want[:, first:])
        assert torch.equal(lg[~want[:, first:]], ref[~want[:, first:]])
    # depth 3 of the second sequence is position 40 of 40
    lg = step([36, 37, 36], good, 48)
    assert lg.isnan().all(-1).tolist() == [[False] * (6 - first), [False] * (5 - first) + [True], [False] * (6 - first)]
    # and of a cache of 35 rows node 5 has none, of 33 rows nodes 3 to 5 have none
    for rows, gone in ((35, [5]), (33, [3, 4, 5])):
        lg = step([30] * 3, good, rows)
        assert lg.isnan().all(-1).tolist() == [[i in gone for i in range(first, 6)]] * 3
    # padding's may lie behind the cache
    lg = step([30] * 3, good, 48, bits=od.ancestors([-1, 0, 0, -1, -1, -1]).to(dev))
    assert torch.equal(step([30] * 3, good, 33, bits=od.ancestors([-1, 0, 0, -1, -1, -1]).to(dev)), lg) and torch.isfinite(lg).all()


@pytest.mark.parametrize("proposals,branches", [("sampled", (2, 2, 1)), ("likeliest", (3, 1)), ("sampled", (1, 1, 1, 1))])
def test_speculate_greedy_is_the_models_own(dev, proposals, branches):
    # top_k = 1: whatever the draft proposes, each token is the model's own choice within the rounding of its logits
    m, d = _model(dev, n_layer=3), _model(dev, seed=5, n_layer=1)
    g = torch.Generator(device=dev).manual_seed(6)
    idx = torch.randint(0, 256, (3, 20), device=dev, generator=g)
    for draft in (d, m):
        out = m.speculate(idx, 33, draft, branches=branches, temperature=1.0, top_k=1, generator=g, proposals=proposals)
        assert out.shape == (3, 33) and out.dtype == torch.int64
        x = torch.cat([idx, out], 1)
        with torch.no_grad():
            lg = m(x[:, :-1])[:, 19:].float()
        gap = lg.max(-1).values - lg.gather(2, out[:, :, None])[:, :, 0]
        assert bool((gap <= 3e-2 * lg.abs().amax(-1).clamp_min(1.0)).all())


def test_speculate_samples_as_generate_does(dev):
    # the second token's law over 6,000 sequences of one prompt, against the model's own probabilities given
    # the first: 5 standard deviations
    m, d = _model(dev, n_layer=1, seq_len=16), _model(dev, seed=5, n_layer=1, seq_len=16)
    g = torch.Generator(device=dev).manual_seed(8)
    B = 6000
    idx = torch.randint(0, 256, (1, 5), device=dev, generator=g).expand(B, -1).contiguous()
    out = m.speculate(idx, 3, d, branches=(2, 1), temperature=0.9, top_k=4, generator=g)
    assert out.shape == (B, 3) and int(out.min()) >= 0
    first, count = out[:, 0].unique(return_counts=True)
    x = first[count.argmax()]
    rows = out[out[:, 0] == x]
    with torch.no_grad():
        p = od.sampling_probs(m(torch.cat([idx[:1], x.view(1, 1)], 1))[0, -1].float().cpu(), 0.9, 4)
    f = torch.bincount(rows[:, 1].cpu(), minlength=256).double() / len(rows)
    # the logits of a batched bf16 pass differ by roundings: 2 % of a probability besides
    assert ((f - p).abs() <= 5 * (p * (1 - p) / len(rows)).sqrt() + 0.02 * p).all()
    assert set(f.nonzero()[:, 0].tolist()) <= set((p > 0).nonzero()[:, 0].tolist())


@pytest.mark.parametrize("proposals,branches", [("sampled", (2, 1)), ("sampled", (1, 3)), ("likeliest", (2, 2))])
def test_speculate_samples_every_token_as_generate_does(dev, proposals, branches):
    # each token's law given the most frequent tokens before it, over 20,000 sequences of one prompt: the second hangs on the
    # root's draft row, the third on the rows of inner nodes, the later ones on caches compacted in rounds before
    m, d = _model(dev, n_layer=1, seq_len=16), _model(dev, seed=5, n_layer=1, seq_len=16)
    g = torch.Generator(device=dev).manual_seed(18)
    B, n = 20000, 6
    idx = torch.randint(0, 256, (1, 5), device=dev, generator=g).expand(B, -1).contiguous()
    out = m.speculate(idx, n, d, branches=branches, temperature=0.7, top_k=3, generator=g, proposals=proposals)
    assert out.shape == (B, n) and int(out.min()) >= 0
    rows, x = out, idx[:1]
    for i in range(n):
        with torch.no_grad():
            p = od.sampling_probs(m(x)[0, -1].float().cpu(), 0.7, 3)
        f = torch.bincount(rows[:, i].cpu(), minlength=256).double() / len(rows)
        # as above: 5 standard deviations, and 2 % for the roundings of the logits
        assert ((f - p).abs() <= 5 * (p * (1 - p) / len(rows)).sqrt() + 0.02 * p).all(), i
        best = f.argmax().to(dev)
        rows, x = rows[rows[:, i] == best], torch.cat([x, best.view(1, 1)], 1)
    assert len(rows) >= 20


def test_speculate_without_finite_logits(dev):
    m, d = _model(dev, seq_len=40), _model(dev, seed=2, seq_len=40, n_layer=1)
    idx = torch.randint(0, 256, (2, 30), device=dev)
    with torch.no_grad():
        d.lnf_w[3] = math.nan
    with pytest.raises(RuntimeError, match="not finite"):
        m.speculate(idx, 4, d)
    with pytest.raises(RuntimeError, match="not finite"):
        d.speculate(idx, 4, m)


@pytest.mark.parametrize("proposals", ["sampled", "likeliest"])
def test_speculate_reads_the_device_once_a_round(dev, proposals, monkeypatch):
    import warnings

    import fxlm.model as M
    m, d = _model(dev, seq_len=40), _model(dev, seed=2, seq_len=40, n_layer=1)
    idx = torch.randint(0, 256, (2, 5), device=dev)
    rounds = []
    verify = M.verify_draft
    monkeypatch.setattr(M, "verify_draft", lambda *a, **kw: rounds.append(1) or verify(*a, **kw))

    def reads(n):   # (waits for the GPU, rounds) of a call
        rounds.clear()
        with warnings.catch_warnings(record=True) as w:
            warnings.simplefilter("always")
            torch.cuda.set_sync_debug_mode("warn")
            try:
                m.speculate(idx, n, d, proposals=proposals, generator=torch.Generator(device=dev).manual_seed(3))
            finally:
                torch.cuda.set_sync_debug_mode("default")
        return sum("synchroniz" in str(x.message) for x in w), len(rounds)

    reads(3)
    (a, ra), (b, rb) = reads(2), reads(30)
    assert a > 0 and rb > ra and b - a == rb - ra


def test_operators_on_two_streams_at_once(dev):
    # each call has a workspace of its own: two streams' calls, none waiting for the other, against the same calls in turn
    from fxlm import sampling_probs, tree_attention, verify_draft
    cases = [{n: t.to(dev) if torch.is_tensor(t) else t for n, t in _tree_case(2, 16, 4, 2, 64, 9000, [8900, 70 + s], seed=s).items()} for s in range(2)]
    drafts = [[t.to(dev) for t in _draft_case(6, 9, 3000, 2, s, False, True)] for s in range(2)]

    def calls(i):
        c, (p, tok, par, u, q) = cases[i], drafts[i]
        r = [tree_attention(c["q"], c["k"], c["v"], c["ctx"], c["tree"], return_lse=True, k_new=c["kn"], v_new=c["vn"]) for _ in range(8)][-1]
        return list(r) + [sampling_probs(p * 50, 0.7, 40)] + list(verify_draft(p, tok, par, u, draft_probs=q))

    want = [calls(0), calls(1)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [None, None]
    for _ in range(3):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i] = calls(i)
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_speculate_ends_and_refuses(dev):
    m, d = _model(dev, seq_len=40), _model(dev, seed=2, seq_len=40, n_layer=1)
    idx = torch.randint(0, 256, (2, 30), device=dev)
    g = torch.Generator(device=dev).manual_seed(1)
    for n in (0, 1, 2, 10):          # 10: to the last position
        out = m.speculate(idx, n, d, generator=g)
        assert out.shape == (2, n) and (n == 0 or 0 <= int(out.min()) <= int(out.max()) < 256)
    for kw in ({"max_new": 11}, {"branches": (4, 4, 3)}, {"branches": (0,)}, {"proposals": "best"}):
        with pytest.raises(ValueError):
            m.speculate(idx, **{"max_new": 4, "draft": d, **kw})
    with pytest.raises(ValueError):
        m.tree_step(idx[:, 0], torch.zeros(1, dtype=torch.int32, device=dev), m._new_cache(2, 40), torch.zeros(2, dtype=torch.int32, device=dev),
                    torch.ones(1, dtype=torch.int64, device=dev))

"""A paged KV cache and beam selection on the CPU: the 64-bit oracle against what defines it, and what
the wrappers refuse before anything is launched."""
import itertools
import math

import pytest
import torch

from oracle import attention as oatt
from oracle import paged as op


def _i(*x):
    return torch.tensor(x, dtype=torch.int32)


def test_paged_attention_is_the_last_row_of_causal_attention():
    torch.manual_seed(2)
    T, H, D, P = 37, 2, 64, 16
    q, k, v = (torch.randn(1, T, H, D).bfloat16() for _ in range(3))
    ref, lse = oatt.attn_fwd(q, k, v, True)
    table = _i(4, 1, 3)[None]
    kp, vp = torch.zeros(6, P, H, D).bfloat16(), torch.zeros(6, P, H, D).bfloat16()
    for j in range(T):
        kp[table[0, j // P], j % P], vp[table[0, j // P], j % P] = k[0, j], v[0, j]
    o, l, _, k2, v2 = op.paged_attention(q[:, -1], kp, vp, table, _i(T))   # noqa: E741
    assert torch.allclose(o, ref[:, -1], atol=1e-12) and torch.allclose(l, lse[:, :, -1], atol=1e-12)
    kp[3, 4], vp[3, 4] = 9, 9        # the last key's place
    o2, _, _, k3, v3 = op.paged_attention(q[:, -1], kp, vp, table, _i(T), k_new=k[:, -1], v_new=v[:, -1])
    assert torch.equal(o, o2) and torch.equal(k2, k3) and torch.equal(v2, v3)


def test_tables_of_a_small_pool():
    # three rows of pages of 16: 20 tokens, 16, none; pages 2, 0 and 5 are held
    table, lens = _i(2, 0, -1, 5, -1, -1, -1, -1, -1).view(3, 3), _i(20, 16, 0)
    uses = _i(1, 0, 1, 0, 0, 1, 0)
    slots, n, t, u, _ = op.extend_pages(table, lens, _i(1, 1, 17), uses, 16, most=17)
    assert n.tolist() == [21, 17, 17] and u.tolist() == [1, 1, 1, 1, 1, 1, 0]
    assert t.tolist() == [[2, 0, -1], [5, 1, -1], [3, 4, -1]]
    assert slots[0, :2].tolist() == [4, -1] and slots[1, 0] == 16 and slots[2].tolist() == [48 + i for i in range(16)] + [64]
    # row 0 goes on twice, row 1 ends
    n2, t2, u2 = op.reorder_pages(t, n, _i(0, -1, 0), u, 16)
    assert n2.tolist() == [21, 0, 21] and t2[2, :2].tolist() == [2, 0] and u2.tolist() == [2, 0, 2, 0, 0, 0, 0]
    # both write: the lower one keeps the open page, the other has its rows
    cache = [(torch.arange(7 * 16.).view(7, 16, 1, 1), torch.arange(7 * 16.).view(7, 16, 1, 1) + 1)]
    slots, n3, t3, u3, c3 = op.extend_pages(t2, n2, _i(1, 1, 1), u2, 16, cache=cache)
    # (row 1, without tokens, begins anew)
    assert n3.tolist() == [22, 1, 22] and t3[:, :2].tolist() == [[2, 0], [1, 1], [2, 3]] and u3.tolist() == [1, 1, 2, 1, 0, 0, 0]
    assert c3[0][0][3, :5].flatten().tolist() == [0, 1, 2, 3, 4] and slots[2, 0] == 48 + 5
    # one of them writes: it gets its own; without the pools it gets nothing
    assert op.extend_pages(t2, n2, _i(1, 0, 0), u2, 16, cache=cache)[2][0].tolist() == [2, 1, -1]
    assert op.extend_pages(t2, n2, _i(1, 0, 0), u2, 16)[1].tolist() == [21, 0, 21]


@pytest.mark.parametrize("weight", [None, 0.5])
def test_beam_selection_is_the_best_of_all(weight):
    torch.manual_seed(4)
    B, K, V = 3, 4, 6
    x, s = torch.randn(B, K, V) * 2, -torch.rand(B, K) * 3
    w = None if weight is None else torch.rand(B, K) + weight
    out, rows, toks, _ = op.beam_select(x, s, weight=w)
    lp = torch.log_softmax(x.double(), -1) + s.double()[..., None]
    rank = lp if w is None else lp * w.double()[..., None]
    for b in range(B):
        best = sorted(itertools.product(range(K), range(V)), key=lambda kv: -float(rank[b][kv]))[:K]
        assert [(int(r) - b * K, int(t)) for r, t in zip(rows[b], toks[b])] == best
        assert torch.allclose(out[b], torch.stack([lp[b][kv] for kv in best]))


def test_beam_selection_at_its_edges():
    inf = math.inf
    x = torch.tensor([[[1., 1., 0.], [5., 5., 5.], [-inf, -inf, 2.], [0., math.nan, 0.]]])
    # a beam that does not exist, equal logits, masked tokens
    out, rows, toks, _ = op.beam_select(x[:, :3], torch.tensor([[0., -inf, 0.]]), fill=2)
    assert rows.tolist() == [[2, 0, 0]] and toks.tolist() == [[2, 0, 1]] and out[0, 0] == 0
    # NaN first; a done beam goes on by the fill token; too few continuations
    out, rows, toks, _ = op.beam_select(x, torch.tensor([[-inf, -1., -inf, 0.]]), done=torch.tensor([[False, True, False, False]]), fill=1)
    assert rows.tolist() == [[3, 1, -1, -1]] and toks.tolist() == [[1, 1, 1, 1]] and out[0, 0].isnan() and out[0, 1:].tolist() == [-1, -inf, -inf]


def test_wrappers_refuse():
    from fxlm import beam_select, extend_pages, paged_attention, reorder_pages, store_pages
    bf = lambda *s: torch.zeros(*s).bfloat16()   # noqa: E731
    q, k, t, n = bf(2, 4, 64), bf(5, 16, 2, 64), torch.zeros(2, 3, dtype=torch.int32), _i(1, 1)
    for err, args, kw in [
            (TypeError, (q, k, k, t, n), {}),                              # off the GPU
            (TypeError, (q.float(), k, k, t, n), {}),
            (ValueError, (q[0], k, k, t, n), {}),
            (ValueError, (q, k, k[:, :8], t, n), {}),
            (ValueError, (q, k[:, :8], k[:, :8], t, n), {}),               # pages of 8
            (ValueError, (q, bf(5, 48, 2, 64), bf(5, 48, 2, 64), t, n), {}),
            (ValueError, (q[:, :3], k, k, t, n), {}),                      # 3 heads on 2
            (ValueError, (bf(2, 4, 96), bf(5, 16, 2, 96), bf(5, 16, 2, 96), t, n), {}),
            (ValueError, (q, k, k, t, n), {"k_new": bf(2, 2, 64)}),
            (ValueError, (q, k, k, t, n), {"k_new": bf(2, 4, 64), "v_new": bf(2, 4, 64)}),
            (ValueError, (q, bf(1, 16, 2, 64).expand(5, -1, -1, -1), k, t, n), {"k_new": bf(2, 2, 64), "v_new": bf(2, 2, 64)}),
    ]:
        with pytest.raises(err):
            paged_attention(*args, **kw)
    for err, args, kw in [
            (TypeError, (t, n, n, _i(0, 0), 16), {}),
            (TypeError, (t.long(), n, n, _i(0, 0), 16), {}),
            (ValueError, (t, n, n, _i(0, 0), 24), {}),
    ]:
        with pytest.raises(err):
            extend_pages(*args, **kw)
        with pytest.raises(err):
            reorder_pages(*args, **kw)
    with pytest.raises(TypeError):
        store_pages(bf(2, 3, 2, 64), bf(2, 3, 2, 64), torch.zeros(2, 3, dtype=torch.int64), k, k)
    with pytest.raises(ValueError):
        store_pages(bf(2, 3, 2, 64), bf(2, 4, 2, 64), torch.zeros(2, 3, dtype=torch.int64), k, k)
    x, s = torch.zeros(2, 3, 7), torch.zeros(2, 3)
    for err, args in [(TypeError, (x, s)), (TypeError, (x.half(), s)), (ValueError, (x[0], s)), (ValueError, (torch.zeros(1, 33, 7), torch.zeros(1, 33)))]:
        with pytest.raises(err):
            beam_select(*args)


def test_paged_cache_refuses():
    from fxlm import PagedCache
    for rows, pages, page, width in ((0, 4, 16, 4), (1, 0, 16, 4), (1, 4, 20, 4), (9000, 4, 16, 4), (1, 4, 16, 0)):
        with pytest.raises(ValueError):
            PagedCache(rows, pages, page, width, 1, 1, 64, "cpu")


def test_beam_search_refuses():
    from fxlm import GPT, GPTConfig
    m = GPT(GPTConfig(vocab_size=8, seq_len=32, n_layer=1, n_head=1, d_model=64))
    idx = torch.zeros(1, 20, dtype=torch.int64)
    for kw in ({"max_new": 13}, {"max_new": 4, "beams": 33}, {"max_new": 4, "beams": 0}, {"max_new": 4, "lens": _i(0)}, {"max_new": 4, "lens": _i(21)}):
        with pytest.raises(ValueError):
            m.beam_search(idx, **kw)
    with pytest.raises(ValueError):
        m.generate(idx, 13, lens=_i(20))
    with pytest.raises(ValueError):
        m.generate(idx, 3, lens=_i(0))


def test_beam_search_refuses_pages_and_penalties():
    from fxlm import GPT, GPTConfig
    m = GPT(GPTConfig(vocab_size=8, seq_len=32, n_layer=1, n_head=1, d_model=64))
    idx = torch.zeros(1, 20, dtype=torch.int64)
    for kw in ({"page": 0}, {"page": 24}, {"length_penalty": math.nan}, {"length_penalty": math.inf}, {"length_penalty": -100.0}):
        with pytest.raises(ValueError):
            m.beam_search(idx, 4, **kw)
    with pytest.raises(ValueError):
        m.paged_cache(2, 4, 0)


def test_beam_selection_without_a_rank():
    # a weight that is no positive finite number gives its beam no rank: NaN, and first
    inf = math.inf
    x, s = torch.tensor([[[0., 1.], [3., 2.], [1., 0.], [0., 0.]]]), torch.tensor([[-1., -2., -3., -inf]])
    for bad in (0.0, -1.0, inf, -inf, math.nan):
        out, rows, toks, _ = op.beam_select(x, s, fill=1, weight=torch.tensor([[1., bad, 1., bad]]))
        assert out[0, 0].isnan() and rows[0, 0] == 1 and toks[0, 0] == 1 and not (rows[0, 1:] == 1).any() and torch.isfinite(out[0, 1:]).all()

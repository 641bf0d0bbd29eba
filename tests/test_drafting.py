"""Drafted decoding on the CPU: the 64-bit oracle against what defines it, and what the wrappers
refuse before anything is launched."""
import math

import pytest
import torch

from oracle import attention as oatt
from oracle import drafting as od


def test_a_chain_is_causal_attention():
    torch.manual_seed(1)
    B, T, H, D, c = 2, 11, 2, 64, 6
    q, k, v = (torch.randn(B, T, H, D).bfloat16() for _ in range(3))
    ref, lse = oatt.attn_fwd(q, k, v, True)
    tree = od.ancestors([-1, 0, 1, 2, 3]).expand(B, -1)
    for kn, vn in ((None, None), (k[:, c:].clone(), v[:, c:].clone())):
        kc, vc = k.clone(), v.clone()
        if kn is not None:
            kc[:, c:] = 0
            vc[:, c:] = 0
        o, l2, _, k2, v2 = od.tree_attention(q[:, c:], kc, vc, torch.full((B,), c), tree, k_new=kn, v_new=vn)
        assert torch.allclose(o, ref[:, c:], atol=1e-12) and torch.allclose(l2, lse[:, :, c:].transpose(1, 2), atol=1e-12)
        assert torch.equal(k2, k) and torch.equal(v2, v)


def test_ancestors_reach_the_sign_bit():
    bits = od.ancestors(list(range(-1, 63)))
    assert bits[63].item() == -1 and bits[62].item() == 2 ** 63 - 1
    assert od.ancestors([-1, 0, -1, 1]).tolist() == [1, 3, 0, 11]


@pytest.mark.parametrize("drafted", [True, False])
def test_verified_tokens_are_distributed_as_the_target(drafted):
    # the first token's law, by the law of large numbers over sequences: three children of the root
    # drawn from q (or the same three proposals), 30,000 sequences, 5 standard deviations
    g = torch.Generator().manual_seed(3)
    B, N, V = 30000, 4, 5
    p = torch.tensor([.1, .35, .05, .3, .2])
    q = torch.tensor([.3, .1, .2, .2, .2])
    if drafted:
        tok = torch.multinomial(q, B * N, replacement=True, generator=g).view(B, N)
    else:
        tok = torch.tensor([0, 3, 1, 4]).expand(B, N).contiguous()
    par = torch.tensor([-1, 0, 0, 0], dtype=torch.int32).expand(B, N).contiguous()
    out, path, n = od.verify_draft(p.expand(B, N, V), tok, par, torch.rand(B, N, generator=g), q.expand(B, N, V) if drafted else None)
    freq = torch.bincount(out[:, 0], minlength=V).double() / B
    assert ((freq - p).abs() <= 5 * (p * (1 - p) / B).sqrt()).all()
    assert set(n.tolist()) <= {1, 2}


def test_wrappers_refuse():
    from fxlm import compact_cache, sampling_probs, tree_attention, verify_draft
    bf = lambda *s: torch.zeros(*s).bfloat16()   # noqa: E731
    q, k, c, t = bf(2, 3, 4, 64), bf(2, 16, 2, 64), torch.zeros(2, dtype=torch.int32), torch.ones(2, 3, dtype=torch.int64)
    for err, args, kw in [
            (TypeError, (q, k, k, c, t), {}),                              # off the GPU
            (TypeError, (q.float(), k, k, c, t), {}),
            (ValueError, (q[0], k, k, c, t), {}),
            (ValueError, (q, k, k[:, :8], c, t), {}),
            (ValueError, (bf(2, 3, 5, 64), k, k, c, t), {}),               # 5 query heads, 2 key heads
            (ValueError, (bf(2, 3, 4, 96), bf(2, 16, 2, 96), bf(2, 16, 2, 96), c, t), {}),
            (ValueError, (q, k, k, c, t), {"first": 62}),
            (ValueError, (q, k, k, c, t), {"first": -1}),
            (ValueError, (bf(2, 65, 4, 64), k, k, c, torch.ones(2, 65, dtype=torch.int64)), {}),
            (ValueError, (bf(2, 0, 4, 64), k, k, c, t[:, :0]), {}),
            (ValueError, (q, k, k, c, t), {"k_new": bf(2, 3, 2, 64)}),     # without v_new
            (ValueError, (q, k, k, c, t), {"k_new": bf(2, 3, 4, 64), "v_new": bf(2, 3, 4, 64)}),
            (ValueError, (q, k[:1].expand(2, -1, -1, -1), k, c, t), {"k_new": bf(2, 3, 2, 64), "v_new": bf(2, 3, 2, 64)})]:
        with pytest.raises(err):
            tree_attention(*args, **kw)
            pytest.fail(f"not refused: {kw} {[tuple(a.shape) for a in args]}")
    x = torch.zeros(2, 10)
    for err, args, kw in [(TypeError, (x,), {}), (TypeError, (x.half(),), {}), (ValueError, (x,), {"temperature": 0.0}),
                          (ValueError, (x,), {"temperature": math.inf}), (ValueError, (x,), {"temperature": math.nan}),
                          (ValueError, (x,), {"temperature": 1e-31}), (ValueError, (x,), {"temperature": 1e31})]:
        with pytest.raises(err):
            sampling_probs(*args, **kw)
    p, tok, par, u = torch.zeros(2, 3, 10), torch.zeros(2, 3, dtype=torch.int64), torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, 3)
    for err, args, kw in [
            (TypeError, (p, tok, par, u), {}), (TypeError, (p.double(), tok, par, u), {}), (TypeError, (p, tok.int(), par, u), {}),
            (TypeError, (p, tok, par.long(), u), {}), (ValueError, (p[0], tok, par, u), {}),
            (ValueError, (torch.zeros(2, 65, 4), tok, par, u), {})]:
        with pytest.raises(err):
            verify_draft(*args, **kw)
    cache, path = [(k, k.clone())], torch.zeros(2, 3, dtype=torch.int32)
    for err, args in [(TypeError, (cache, c, path, c)), (ValueError, ([], c, path, c)), (TypeError, ([(k.float(), k)], c, path, c)),
                      (ValueError, ([(k[:1].expand(2, -1, -1, -1), k)], c, path, c))]:
        with pytest.raises(err):
            compact_cache(*args)


def test_host_module_returns_nothing_off_the_gpu():
    # host.cpp's own checks return nothing for tensors that are not the GPU's: nothing is launched
    from fxgpu.abi import host
    q, k = torch.zeros(1, 2, 2, 64).bfloat16(), torch.zeros(1, 8, 2, 64).bfloat16()
    c, t = torch.zeros(1, dtype=torch.int32), torch.ones(1, 2, dtype=torch.int64)
    assert host.tree_attention(q, k, k, c, t, 0, 0.125, True, None, None) is None
    assert host.sampling_probs(torch.zeros(2, 8), 1.0, 0) is None
    assert host.verify_draft(torch.zeros(1, 2, 8), t, t.int(), torch.zeros(1, 2), None) is None
    assert host.compact_cache([(k, k)], c, t.int(), c) is None
    assert host.compact_cache([], c, t.int(), c) is None

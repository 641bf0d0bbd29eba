"""Beams with the same logits and the same scores rank alike, wherever their rows begin in memory: a vocabulary that is no
whole number of 16-byte vectors has them begin at every offset of one.  Nothing here has a tolerance."""
import pytest
import torch

pytestmark = pytest.mark.gpu


# one chunk a row and many, short chunks and long ones (more rows than CUs take in short ones)
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("B,K,V", [(3, 8, 257), (5, 7, 1001), (2, 8, 8191), (1, 5, 50257), (40, 8, 50257), (2, 32, 30011), (33, 8, 131071), (2, 3, 131069), (1, 2, 1048575)])
def test_beams_alike(dev, B, K, V, bf16):
    from fxlm import beam_select
    g = torch.Generator(device=dev).manual_seed(V + K)
    for spread in (0.3, 4.0):
        row = torch.randn(V, device=dev, generator=g) * spread
        row[V // 2] = row.max() + 0.5       # one best token
        x = (row.bfloat16() if bf16 else row).expand(B, K, V).contiguous()
        s = torch.full((B, K), -1.25, device=dev)
        scores, parents, tokens = beam_select(x, s)
        assert (scores == scores[0, 0]).all()
        assert torch.equal(parents.long().cpu(), torch.arange(B * K).view(B, K)) and (tokens == V // 2).all()
        # the same row at each place of a batch of others
        y = torch.randn(B, K, V, device=dev, generator=g).to(x.dtype)
        y[:, K - 1] = x[:, K - 1]
        lone = torch.full((B, K), -torch.inf, device=dev)
        lone[:, K - 1] = -1.25
        assert (beam_select(y, lone)[0][:, 0] == scores[0, 0]).all()


@pytest.mark.parametrize("V", [1001, 50257])
def test_pairs_of_beams_alike(dev, V):
    # beams 0 and 2, 1 and 3 alike: their continuations take turns, the lower beam first
    from fxlm import beam_select
    g = torch.Generator(device=dev).manual_seed(V)
    x = torch.randn(60, 2, V, device=dev, generator=g).repeat(1, 2, 1)
    s = torch.randn(60, 2, device=dev, generator=g).repeat(1, 2)
    scores, parents, tokens = beam_select(x, s)
    k = parents.long() % 4
    assert (k[:, 0::2] < 2).all() and torch.equal(k[:, 1::2], k[:, 0::2] + 2)
    assert torch.equal(tokens[:, 0::2], tokens[:, 1::2]) and torch.equal(scores[:, 0::2], scores[:, 1::2])

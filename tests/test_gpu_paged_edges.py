"""Calls of a paged cache's functions at the ends of what they take, on the GPU, against the 64-bit oracle."""
import pytest
import torch

from oracle import paged as op

pytestmark = pytest.mark.gpu


def _ints(x, dev=None):
    return torch.tensor(x, dtype=torch.int32, device=dev)


# slots in the same launch as the tables, and in one of their own; lengths past the table by what is added, by less and by more
@pytest.mark.parametrize("R,most", [(4, 2), (4, 65), (4, 3000), (700, 2), (700, 40), (5000, 7)])
def test_extend_pages_lengths_past_the_table(dev, R, most):
    from fxlm import extend_pages
    P, M = 16, 4
    lens = _ints([64 + (r * 7 + most) % (most + 2) if r % 3 else 64 + min(most, 1 + r % 7) for r in range(R)])
    add = torch.where(torch.arange(R) % 3 == 0, lens - 64, _ints([r * 5 % (most + 2) for r in range(R)])).int()
    lens[1], add[1] = 40, 3                  # one that fits
    lens[R - 1], add[R - 1] = 65, 1          # the last row: nothing is behind it
    assert int(((lens - 64 == add.clamp(0, most)) & (add > 0)).sum()) >= 2
    table = torch.arange(R * M, dtype=torch.int32).view(R, M)
    uses = torch.cat([torch.ones(R * M, dtype=torch.int32), torch.zeros(9, dtype=torch.int32)])
    want = op.extend_pages(table, lens, add, uses, P, most)
    dt, du = table.to(dev), uses.to(dev)
    got = extend_pages(dt, lens.to(dev), add.to(dev), du, P, most)
    for a, b in zip((*got, dt, du), want):
        assert torch.equal(a.cpu(), b)
    assert (got[0].cpu()[lens > 64] == -1).all() and int((got[0] >= 0).sum()) == min(3, most)


def test_extend_pages_of_as_many_tokens_as_there_can_be(dev):
    # 2^31 - 1 slots of a row, 16 GiB: the last ones' numbers are just below the type's end
    from fxlm import extend_pages
    most = 2 ** 31 - 1
    table, uses = torch.full((1, 4), -1, dtype=torch.int32, device=dev), torch.zeros(6, dtype=torch.int32, device=dev)
    slots, n = extend_pages(table, _ints([0], dev), _ints([40], dev), uses, 16, most)
    assert slots.shape == (1, most) and n.tolist() == [40] and slots[0, :40].tolist() == list(range(40))
    assert int(slots[0, 40:].amax()) == -1 and int(slots[0, 40:].amin()) == -1
    assert table.tolist() == [[0, 1, 2, -1]] and uses.tolist() == [1, 1, 1, 0, 0, 0]


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("K,V", [(4, 2), (4, 9001), (32, 300)])
def test_beam_select_of_weights_that_are_none(dev, K, V, bf16):
    from fxlm import beam_select
    g = torch.Generator().manual_seed(V)
    x, s = torch.randn(6, K, V, generator=g), -torch.rand(6, K, generator=g)
    x = x.bfloat16() if bf16 else x
    s[:, 3], done, w = -torch.inf, torch.zeros(6, K, dtype=torch.bool), torch.ones(6, K)
    done[:, 2] = True
    for b, bad in enumerate((0.0, -1.0, torch.inf, -torch.inf, torch.nan)):     # (the last sequence's weights are good)
        w[b, 1] = w[b, 2] = w[b, 3] = bad       # of a beam that goes on, one that is done and one that does not exist
    ro, rr, rt, _ = op.beam_select(x, s, done, 1, w)
    out, rows, toks = (t.cpu() for t in beam_select(x.to(dev), s.to(dev), done.to(dev), 1, w.to(dev)))
    assert torch.equal(out.isnan(), ro.isnan()) and int(out.isnan().sum()) == 10 and out[:5, :2].isnan().all()
    assert torch.equal(rows[:5, :2], rr[:5, :2]) and (toks[:5, :2] == 1).all()
    # log sum exp: 66 2^-23 of exponentials and sums, 3 2^-24 of the mean distance from the maximum (below 9); the score's own rounding
    num = ~ro.isnan()
    assert ((out.double() - ro).abs()[num] <= 2.0 ** -23 * 80 + 2.0 ** -24 * ro.abs()[num]).all()


def test_extend_pages_without_copies_needs_nothing_for_each_page(dev):
    # many rows over a large pool of their own pages
    from fxlm import extend_pages
    R, N = 300, 1 << 24
    table, uses = torch.full((R, 2), -1, dtype=torch.int32, device=dev), torch.zeros(N, dtype=torch.int32, device=dev)
    lens, add = torch.zeros(R, dtype=torch.int32, device=dev), torch.ones(R, dtype=torch.int32, device=dev)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats(dev)
    held = torch.cuda.memory_allocated(dev)
    slots, n = extend_pages(table, lens, add, uses, 16)
    assert torch.cuda.max_memory_allocated(dev) - held < N
    assert slots[:, 0].tolist() == list(range(0, 16 * R, 16)) and (n == 1).all() and int(uses.sum()) == R


@pytest.mark.parametrize("eos", [None, 5])
def test_beams_that_do_not_exist_have_no_prompts_tokens(dev, eos):
    # 4 tokens: 16 continuations by two for 32 beams
    from fxlm import GPT, GPTConfig
    torch.manual_seed(4)
    m = GPT(GPTConfig(vocab_size=4, seq_len=32, n_layer=1, n_head=1, d_model=64)).to(dev).bfloat16()
    with torch.no_grad():
        m.tok_emb.weight.mul_(8.0)
    out, scores = m.beam_search(torch.randint(0, 4, (3, 9), device=dev), 2, beams=32, eos=eos)
    assert torch.isfinite(scores[:, :16]).all() and (scores[:, 16:] == -torch.inf).all()
    assert (out[:, 16:] == (eos or 0)).all()
    for b in range(3):
        assert len({tuple(t) for t in out[b, :16].tolist()}) == 16


def test_paged_attention_of_more_steps_than_are_counted(dev):
    # 2^31 keys of 512 heads are 2^26 steps of 128 groups of heads: past 32 bits, where 256 heads are just below
    from fxlm import paged_attention
    table, lens = torch.zeros(1, 2 ** 21 - 1, dtype=torch.int32, device=dev), _ints([3], dev)
    for H in (256, 512):
        q, k = torch.ones(1, H, 64, device=dev).bfloat16(), torch.ones(1, 1024, H, 64, device=dev).bfloat16()
        if H == 256:
            assert (paged_attention(q, k, k, table, lens) == 1).all()
        else:
            with pytest.raises(ValueError):
                paged_attention(q, k, k, table, lens)


@pytest.mark.parametrize("R,H,Hkv,D,P,M", [(64, 32, 8, 128, 16, 512), (35, 20, 2, 128, 32, 300), (16, 12, 12, 64, 16, 64)])
def test_paged_attention_repeats(dev, R, H, Hkv, D, P, M):
    # ragged rows whose pieces are cut and joined, the new keys written by the first call and again by each: the same bits every time
    from fxlm import paged_attention
    g = torch.Generator(device=dev).manual_seed(R)
    lens = torch.randint(0, M * P // 2 + 1, (R,), device=dev, generator=g).int()
    N = R * M // 2 + 1
    table = torch.randperm(N, device=dev, generator=g)[:R * (M // 2)].int().view(R, M // 2)
    table = torch.cat([table, torch.full((R, M - M // 2), -1, device=dev, dtype=torch.int32)], 1)
    q, k, v, kn, vn = (torch.randn(s, device=dev, generator=g).bfloat16() for s in ((R, H, D), (N, P, Hkv, D), (N, P, Hkv, D), (R, Hkv, D), (R, Hkv, D)))
    want = None
    for _ in range(20):
        got = paged_attention(q, k, v, table, lens, return_lse=True, k_new=kn, v_new=vn)
        want = want or got
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])

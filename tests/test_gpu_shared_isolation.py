"""Attention over a shared prefix: what a query does not see does not reach it, where a CTA takes the items of many sequences one after the other."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def filled(fmt, batch, tokens, heads, dim, prefix, own, page=64, seed=0):
    """A cache of one layer, every sequence with `own` tokens; prefix and own tables."""
    from pi05_megakernel_b200.cache import KvCache
    g = torch.Generator(device="cuda").manual_seed(seed)
    pp, op = -(-prefix // page), -(-own // page)
    c = KvCache(pp + batch * op, 1, page, heads, dim, fmt)
    order = torch.randperm(c.pages, generator=g, device="cuda").int()
    ptab, tab = order[:pp].contiguous(), order[pp:].view(batch, op).contiguous()
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda").to(torch.bfloat16)
    if prefix:
        c.write(rnd(1, 1, prefix, heads, dim), rnd(1, 1, prefix, heads, dim), ptab[None])
    c.write(rnd(batch, 1, own, heads, dim), rnd(batch, 1, own, heads, dim), tab)
    c.status()
    return c, ptab, tab, torch.full((batch,), own, dtype=torch.int32, device="cuda"), rnd


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("own", [64, 128, 192, 250, 256, 512])
def test_a_value_that_is_not_a_number_stays_in_its_sequence(own, bad):
    """64 sequences x 8 KV heads over at most 148 CTAs: each takes several items, whose last tiles only some queries see.  A value that is not a number in one
    head of one sequence makes the queries NaN that see it; every other output is the clean run's, bit for bit."""
    from pi05_megakernel_b200.shared import SharedPrefixAttention
    batch, tokens, heads, dim = 64, 4, 8, 128
    c, ptab, tab, lengths, rnd = filled("bf16", batch, tokens, heads, dim, 1024, own)
    q = rnd(batch, tokens, 32, dim)
    op = SharedPrefixAttention(c, 32, batch, tokens)
    clean, clean_lse = op.run(q, ptab, 1024, tab, lengths, with_lse=True)
    assert bool(torch.isfinite(clean).all())
    for seq, head, token in ((9, 2, own - 1), (0, 0, own - 2), (40, 7, own - 3), (63, 5, own - 1), (17, 0, own - 1)):
        page, at = int(tab[seq, token // 64]), token % 64
        old = c.v[page, 0, at, head, 11].clone()
        c.v[page, 0, at, head, 11] = bad
        got, lse = op.run(q, ptab, 1024, tab, lengths, with_lse=True)
        op.status()
        c.v[page, 0, at, head, 11] = old
        sees = torch.zeros(batch, tokens, 32, dtype=torch.bool, device="cuda")
        sees[seq, token - (own - tokens):, 4 * head:4 * head + 4] = True
        assert not bool(torch.isfinite(got[sees]).all(-1).any())
        assert torch.equal(got[~sees], clean[~sees]) and torch.equal(lse[~sees], clean_lse[~sees])


@pytest.mark.parametrize("dim,q_heads,heads", [(64, 16, 8), (128, 32, 8), (256, 8, 4)])
def test_sequences_of_many_lengths(dim, q_heads, heads):
    """Lengths of 16 to 512 tokens, so that a CTA's ragged tiles follow one another at every distance: the last value of each sequence in turn."""
    from pi05_megakernel_b200.shared import SharedPrefixAttention
    batch, tokens, group = 32, 8, q_heads // heads
    c, ptab, tab, lengths, rnd = filled("bf16", batch, tokens, heads, dim, 500, 512, seed=1)
    lengths.copy_(16 * (1 + torch.randperm(batch, generator=torch.Generator().manual_seed(2))))
    q = rnd(batch, tokens, q_heads, dim)
    op = SharedPrefixAttention(c, q_heads, batch, tokens)
    clean = op.run(q, ptab, 500, tab, lengths)
    assert bool(torch.isfinite(clean).all())
    for seq, n in enumerate(lengths.tolist()):
        head, page, at = seq % heads, int(tab[seq, (n - 1) // 64]), (n - 1) % 64
        old = c.v[page, 0, at, head, 0].clone()
        c.v[page, 0, at, head, 0] = float("nan")
        got = op.run(q, ptab, 500, tab, lengths)
        c.v[page, 0, at, head, 0] = old
        sees = torch.zeros(batch, tokens, q_heads, dtype=torch.bool, device="cuda")
        sees[seq, tokens - 1, group * head:group * (head + 1)] = True
        assert bool(torch.isnan(got[sees]).all()) and torch.equal(got[~sees], clean[~sees]), seq
    op.status()


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dim", [64, 256])
def test_cleared_scales_do_not_meet_later_copies(fmt, dim):
    """Runs of many more tiles than there are buffers for scales, every third tile with scales that do not count (NaN in memory) and are cleared in place: the
    same outputs whatever memory holds there, time after time."""
    from pi05_megakernel_b200.shared import SharedPrefixAttention
    batch, heads, own = 96, 8, 130
    c, ptab, tab, lengths, rnd = filled(fmt, batch, 1, heads, dim, 640, own, seed=3)
    q = rnd(batch, 1, 16, dim)
    op = SharedPrefixAttention(c, 16, batch)
    want, want_lse = op.run(q, ptab, 640, tab, lengths, with_lse=True)
    assert bool(torch.isfinite(want).all())
    for n in ("k", "v"):
        getattr(c, n + "_scale")[tab[:, 2].long(), :, :, own - 128:] = float("nan")
    for _ in range(40):
        got, lse = op.run(q, ptab, 640, tab, lengths, with_lse=True)
        assert torch.equal(got, want) and torch.equal(lse, want_lse)
    op.status()


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_keys_with_infinities(dim):
    """BF16: a key counts by its score.  -infinity: as if it were masked, bit for bit, and zeros where no other key is left; +infinity: NaN."""
    from pi05_megakernel_b200.shared import SharedPrefixAttention
    c, ptab, tab, lengths, rnd = filled("bf16", 2, 1, 2, dim, 150, 20, seed=4)
    q = rnd(2, 1, 4, dim)
    q[..., 3] = torch.tensor([-1.0, -2.0, 1.0, 0.5], device="cuda")      # heads 0 and 1 see -infinity, 2 and 3 +infinity
    op = SharedPrefixAttention(c, 4, 2)
    for token in (0, 64, 149):
        page, at = int(ptab[token // 64]), token % 64
        old = c.k[page, 0, at].clone()
        valid = torch.ones(150, dtype=torch.bool, device="cuda")
        valid[token] = False
        want, want_lse = op.run(q, ptab, 150, tab, lengths, valid=valid, with_lse=True)
        c.k[page, 0, at, :, 3] = float("inf")
        got, lse = op.run(q, ptab, 150, tab, lengths, with_lse=True)
        c.k[page, 0, at] = old
        assert torch.equal(got[:, :, :2], want[:, :, :2]) and torch.equal(lse[:, :, :2], want_lse[:, :, :2])
        assert bool(torch.isnan(got[:, :, 2:]).all())
    c.k[int(ptab[0]), 0, 0, :, 3] = float("inf")
    got, lse = op.run(q, ptab, 1, with_lse=True)
    assert bool((got[:, :, :2] == 0).all()) and bool((lse[:, :, :2] == -float("inf")).all()) and bool(torch.isnan(got[:, :, 2:]).all())
    op.status()

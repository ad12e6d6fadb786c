"""Attention out of an 8-bit cache whose values have scales of very different sizes, and with the bound of its own roundings, against the definition in 64 bits.

Tolerance, per element, with p the probabilities, s the values' scales and c their codes:
  * the output is rounded to BF16: 2^-8 of it;
  * a probability times its value's scale is rounded to FP16: 2^-11 of it, so 2^-11 of sum p |v|; where the product is one of FP16's subnormals half a step of them
    instead, 2^-25 where the largest product of the row is at least 2^7: 2^-32 of max p s, times |c|, for every key (2^-31: the logarithm is approximate);
  * a score is an FP32 sum of head_dim products: dev = (head_dim + 8) 2^-24 scale max sum |q k|, and 2^-17 for the exponential and its argument, whose
    reference is up to 128 (half a step: 2^-18); e^(+-dev) in a probability and in their sum: 3 dev of sum p |v|;
  * the sums over N keys are FP32, sixteen keys at a time: (N / 16 + 16) 2^-22 of sum p |v|.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def rows(c, n, table, count, layer):
    """Codes [count, heads, dim] and scales [count, heads] of a table's first tokens in 64 bits on the host."""
    t = table.long().cpu()
    codes = getattr(c, n)[:, layer].float().double().cpu()[t].reshape(-1, c.kv_heads, c.head_dim)[:count]
    scales = getattr(c, n + "_scale")[:, layer].double().cpu()[t].transpose(1, 2).reshape(-1, c.kv_heads)[:count]
    return codes, scales


def check(c, got, q, ptab, prefix, tab, lengths, layer, causal=True):
    """Outputs and log-sum-exp against the definition, every query."""
    (o, z), scale = got, c.head_dim ** -0.5
    o, z, qd = o.double().cpu(), z.double().cpu(), q.double().cpu()
    b, t, hq, d = q.shape
    group = hq // c.kv_heads
    shared = {n: rows(c, n, ptab, prefix, layer) for n in ("k", "v")} if prefix else None
    for i in range(b):
        n = int(lengths[i])
        own = {m: rows(c, m, tab[i], n, layer) for m in ("k", "v")}
        part = {m: tuple(torch.cat((a, w)) for a, w in zip(shared[m], own[m])) if prefix else own[m] for m in ("k", "v")}
        keys = prefix + n
        for h in range(c.kv_heads):
            k, (code, s) = part["k"][0][:, h] * part["k"][1][:, h, None], (part["v"][0][:, h], part["v"][1][:, h])
            v, qh = code * s[:, None], qd[i, :, group * h:group * (h + 1)].reshape(t * group, d)
            x = scale * qh @ k.T
            if causal:
                late = torch.arange(keys)[None] > keys - t + torch.arange(t).repeat_interleave(group)[:, None]
                x = torch.where(late & (torch.arange(keys) >= prefix), torch.full_like(x, -math.inf), x)
            lse = torch.logsumexp(x, 1)
            p = torch.exp(x - lse[:, None])
            dev = (d + 8) * 2.0 ** -24 * scale * (qh.abs() @ k.abs().T).amax(1, keepdim=True) + 2.0 ** -17
            want, size = p @ v, p @ v.abs()
            seen = torch.isfinite(x).double()
            tol = 2.0 ** -8 * want.abs() + (2.0 ** -11 + 3 * dev + (keys / 16 + 16) * 2.0 ** -22) * size \
                + 2.0 ** -31 * (p * s).amax(1, keepdim=True) * (seen @ code.abs())
            mine = o[i, :, group * h:group * (h + 1)].reshape(t * group, d)
            worst = ((mine - want).abs() / tol).nan_to_num(1e9).max()
            assert float(worst) <= 1, (i, h, float(worst))
            zz = z[i, :, group * h:group * (h + 1)].reshape(-1)
            assert bool(((zz - lse).abs() <= 2 * dev[:, 0] + 2.0 ** -22 * lse.abs()).all())


def build(fmt, batch, prefix, own, heads, dim, page=32, seed=0):
    from pi05_megakernel_b200.cache import KvCache
    g = torch.Generator().manual_seed(seed)
    pp, op = -(-prefix // page), -(-own // page)
    c = KvCache(pp + batch * op, 2, page, heads, dim, fmt)
    order = torch.randperm(c.pages, generator=g).int().cuda()
    ptab, tab = order[:pp].contiguous(), order[pp:].view(batch, op).contiguous()
    rnd = lambda *s: torch.randn(*s, generator=g).to(torch.bfloat16).cuda()
    if prefix:
        c.write(rnd(1, 2, prefix, heads, dim), rnd(1, 2, prefix, heads, dim), ptab[None])
    k, v = rnd(batch, 2, own, heads, dim), rnd(batch, 2, own, heads, dim)
    c.write(k, v, tab)
    c.status()
    return c, ptab, tab, torch.full((batch,), own, dtype=torch.int32, device="cuda"), rnd, k, v


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dim,heads,prefix,own", [(64, 2, 40, 30), (128, 4, 0, 50), (256, 1, 200, 70)])
def test_large_values_that_a_query_does_not_see(fmt, dim, heads, prefix, own):
    """The last token's values 2^r times the others': the queries before it get the same bits whatever r is, and all of them what the definition says."""
    from pi05_megakernel_b200.shared import SharedPrefixAttention
    batch, tokens = 3, 4
    c, ptab, tab, lengths, rnd, k, v = build(fmt, batch, prefix, own, heads, dim)
    q = rnd(batch, tokens, 2 * heads, dim)
    op = SharedPrefixAttention(c, 2 * heads, batch, tokens)
    before = None
    for r in (0, 8, 16, 20, 24, 30, 32, 60, -24):
        big = (v.float() * torch.cat((torch.ones(own - 1), torch.tensor([2.0 ** r]))).cuda()[None, None, :, None, None]).to(torch.bfloat16)
        c.write(k, big, tab)
        got = op.run(q, ptab if prefix else None, prefix, tab, lengths, layer=1, with_lse=True)
        op.status()
        check(c, got, q, ptab, prefix, tab, lengths, 1)
        if before is None:
            before = got
        assert torch.equal(got[0][:, :-1], before[0][:, :-1]) and torch.equal(got[1][:, :-1], before[1][:, :-1]), r


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("tokens", [1, 3])
def test_large_values_that_hardly_count(fmt, dim, tokens):
    """One token of the prefix and one of the sequence with values 2^r times the others' and scores far below theirs: from negligible to all of the output."""
    from pi05_megakernel_b200.shared import SharedPrefixAttention
    batch, prefix, own, far = 2, 300, 40, 20.0
    c, ptab, tab, lengths, rnd, k, v = build(fmt, batch, prefix, own, 1, dim, seed=1)
    q = rnd(batch, tokens, 4, dim)
    q[..., 0] = 4.0
    low = torch.zeros(1, 2, 1, 1, dim, dtype=torch.bfloat16, device="cuda")
    low[..., 0] = -far * dim ** 0.5 / 4.0                                 # a score of -20 beside scores of about 1: e^-20 = 2^-29
    op = SharedPrefixAttention(c, 4, batch, tokens)
    place = lambda at: torch.tensor([at], dtype=torch.int32, device="cuda")
    for r in (0, 12, 20, 24, 29, 34, 44, 70):
        big = (rnd(1, 2, 1, 1, dim).float() * 2.0 ** r).to(torch.bfloat16)
        c.write(low, big, ptab[None], starts=place(130))
        c.write(low, big, tab[:1], starts=place(7))
        got = op.run(q, ptab, prefix, tab, lengths, layer=1, with_lse=True)
        op.status()
        check(c, got, q, ptab, prefix, tab, lengths, 1)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_values_of_zeros_and_of_every_size(fmt):
    """Scales from 2^-70 to 2^70 in one tile, zeros among them; and nothing but zeros."""
    from pi05_megakernel_b200.shared import SharedPrefixAttention
    batch, prefix, own, dim = 2, 150, 64, 128
    c, ptab, tab, lengths, rnd, k, v = build(fmt, batch, prefix, own, 2, dim, seed=2)
    q = rnd(batch, 2, 4, dim)
    op = SharedPrefixAttention(c, 4, batch, 2)
    size = torch.exp2((torch.arange(prefix) * 37 % 141 - 70).float()).cuda()
    size[::9] = 0
    c.write(rnd(1, 2, prefix, 2, dim), (rnd(1, 2, prefix, 2, dim).float() * size[None, None, :, None, None]).to(torch.bfloat16), ptab[None])
    got = op.run(q, ptab, prefix, tab, lengths, layer=1, with_lse=True)
    check(c, got, q, ptab, prefix, tab, lengths, 1)
    zero = torch.zeros(1, 2, prefix, 2, dim, dtype=torch.bfloat16, device="cuda")
    c.write(rnd(1, 2, prefix, 2, dim), zero, ptab[None])
    got = op.run(q, ptab, prefix, tab, lengths, layer=1, with_lse=True)
    check(c, got, q, ptab, prefix, tab, lengths, 1)
    c.write(k, torch.zeros_like(v), tab)
    got = op.run(q, ptab, prefix, tab, lengths, layer=1, with_lse=True)
    assert bool((got[0] == 0).all()) and bool(torch.isfinite(got[1]).all())
    op.status()


CASES = [
    # batch, tokens, q_heads, heads, dim, prefix, own, page, causal
    (4, 1, 8, 1, 256, 200, 20, 64, True),
    (2, 50, 8, 1, 256, 97, 61, 16, False),
    (5, 3, 8, 2, 128, 70, 33, 32, True),
    (9, 1, 12, 4, 128, 333, 130, 48, True),
    (2, 9, 7, 1, 64, 1, 90, 128, False),
    (20, 2, 8, 1, 256, 1100, 300, 64, True),
    (1, 1, 1, 1, 64, 4000, 1, 112, True),
    (24, 2, 32, 8, 64, 3000, 900, 32, True),
    (40, 1, 32, 8, 128, 2500, 400, 64, True),
]


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("batch,tokens,q_heads,heads,dim,prefix,own,page,causal", CASES)
def test_within_its_own_roundings(fmt, batch, tokens, q_heads, heads, dim, prefix, own, page, causal):
    from pi05_megakernel_b200.shared import SharedPrefixAttention
    c, ptab, tab, lengths, rnd, k, v = build(fmt, batch, prefix, own, heads, dim, page, seed=own)
    q = 2 * rnd(batch, tokens, q_heads, dim)
    op = SharedPrefixAttention(c, q_heads, batch, tokens)
    got = op.run(q, ptab, prefix, tab, lengths, layer=1, causal=causal, with_lse=True)
    op.status()
    check(c, got, q, ptab, prefix, tab, lengths, 1, causal)

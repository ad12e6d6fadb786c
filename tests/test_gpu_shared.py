"""Attention of several sequences over one shared prefix and their own tokens, against the definition in 64 bits on the values that the cache holds.

Tolerance, per element: the output is rounded to BF16 (half a step, 2^-8 of it), the probabilities are rounded to BF16 before the product with
the values (2^-8 of sum p |v| at most), and a score is an FP32 sum of head_dim products: with d = (head_dim + 8) 2^-24 scale max_j sum |q k_j|, what
e^(+-d) makes of a probability and of their sum, and 2^-18 for the exponential, its argument and the sums.
"""
import math

import pytest
import torch

from pi05_megakernel_b200 import _lib

pytestmark = pytest.mark.gpu


def values(c, n, layer):
    """The pool's values of a layer in 64 bits on the host: [pages, page_tokens, heads, dim]."""
    x = getattr(c, n)[:, layer].float().double().cpu()
    return x if c.format == "bf16" else x * getattr(c, n + "_scale")[:, layer].double().cpu().transpose(1, 2)[..., None]


def attend(c, q, prefix_table, prefix, table, lengths, layer, valid, causal, scale):
    """Outputs, log-sum-exp, and the tolerances of both."""
    b, t, hq, d = q.shape
    kv, vv = values(c, "k", layer), values(c, "v", layer)
    h, page = kv.shape[2], kv.shape[1]
    q = q.double().cpu()
    flat = lambda pool, tab, n: pool[tab.long().cpu()].reshape(-1, h, d)[:n]
    seen = torch.ones(prefix, dtype=torch.bool) if valid is None else valid.cpu()
    out, lse = torch.zeros(b, t, hq, d, dtype=torch.float64), torch.full((b, t, hq), -math.inf, dtype=torch.float64)
    tol, ltol = torch.zeros_like(out), torch.zeros_like(lse)
    for i in range(b):
        n = 0 if table is None else max(0, min(int(lengths[i]), table.shape[1] * page))
        parts = [(flat(kv, prefix_table, prefix)[seen], flat(vv, prefix_table, prefix)[seen])] if prefix else []
        base = int(seen.sum()) if prefix else 0
        if n:
            parts.append((flat(kv, table[i], n), flat(vv, table[i], n)))
        if not parts:
            continue
        k, v = torch.cat([p[0] for p in parts]), torch.cat([p[1] for p in parts])
        for j in range(t):
            last = base + (max(0, min(n, n - t + j + 1)) if causal else n)
            if last == 0:
                continue
            for a in range(hq):
                g = a // (hq // h)
                x = scale * (k[:last, g] @ q[i, j, a])
                z = torch.logsumexp(x, 0)
                p = torch.exp(x - z)
                out[i, j, a] = p @ v[:last, g]
                lse[i, j, a] = z
                dev = (d + 8) * 2.0 ** -24 * abs(scale) * float((k[:last, g].abs() @ q[i, j, a].abs()).max()) + 2.0 ** -18
                tol[i, j, a] = 2.0 ** -8 * out[i, j, a].abs() + (2.0 ** -8 + 3 * dev) * (p @ v[:last, g].abs())
                ltol[i, j, a] = 2 * dev + 2.0 ** -22 * abs(float(z))
    return out, lse, tol, ltol


def build(fmt, batch, prefix, own, page, heads, dim, layers=2, layer=1, seed=0, junk=True):
    """A cache whose pages are dealt out of order, and the tables; places that no length reaches hold NaN where the format has it."""
    from pi05_megakernel_b200.cache import KvCache
    g = torch.Generator().manual_seed(seed)
    pp, op = -(-prefix // page), -(-own // page)
    pages = pp + batch * op + 1
    c = KvCache(pages, layers, page, heads, dim, fmt)
    if junk:
        for n in ("k", "v"):
            getattr(c, n).view(torch.uint8).fill_(0xff)                   # a NaN of BF16 and of e4m3
            if fmt != "bf16":
                getattr(c, n + "_scale").fill_(float("nan"))
    order = torch.randperm(pages, generator=g).int().cuda()
    ptab, tab = order[:pp].contiguous(), order[pp:pp + batch * op].view(batch, op).contiguous()
    rnd = lambda *s: torch.randn(*s, generator=g).to(torch.bfloat16).cuda()
    if prefix:
        c.write(rnd(1, layers, prefix, heads, dim), rnd(1, layers, prefix, heads, dim), ptab[None])
    lengths = torch.zeros(batch, dtype=torch.int32)
    if own:
        lengths = torch.tensor([own * i // max(1, batch - 1) for i in range(batch)]).int() if batch > 1 else torch.tensor([own]).int()
        c.write(rnd(batch, layers, own, heads, dim), rnd(batch, layers, own, heads, dim), tab, counts=lengths.cuda())
    c.status()
    return c, ptab, tab, lengths.cuda(), rnd


def check(got, want):
    (o, z), (out, lse, tol, ltol) = got, want
    o, z = o.double().cpu(), z.double().cpu()
    none = torch.isinf(lse)
    assert torch.equal(torch.isinf(z) & (z < 0), none)
    assert bool((o[none] == 0).all())
    bad = ~((o - out).abs() <= tol)                                       # (a NaN is bad too)
    assert not bool(bad.any()), (int(bad.sum()), float((o - out).abs().max()), float(((o - out).abs() / tol.clamp_min(1e-30)).max()))
    assert bool((((z - lse).abs() <= ltol) | none).all()), float((z - lse).abs()[~none].max())


CASES = [
    # fmt, batch, tokens, q_heads, heads, dim, prefix, own, page, causal, masked
    ("bf16", 1, 1, 8, 1, 256, 1, 0, 16, True, False),
    ("bf16", 1, 1, 8, 1, 256, 0, 1, 16, True, False),
    ("bf16", 4, 1, 8, 1, 256, 200, 20, 64, True, True),
    ("int8", 4, 1, 8, 1, 256, 200, 20, 64, True, True),
    ("e4m3", 4, 1, 8, 1, 256, 200, 20, 64, True, True),
    ("bf16", 3, 50, 8, 1, 256, 131, 50, 64, False, True),
    ("int8", 2, 50, 8, 1, 256, 97, 61, 16, False, False),
    ("bf16", 5, 3, 8, 2, 128, 70, 33, 32, True, False),
    ("int8", 5, 3, 8, 2, 128, 70, 33, 32, True, True),
    ("e4m3", 17, 1, 12, 4, 128, 333, 130, 48, True, False),
    ("bf16", 33, 1, 4, 4, 64, 65, 7, 16, True, False),
    ("int8", 3, 7, 14, 2, 64, 129, 64, 16, True, False),
    ("e4m3", 2, 9, 7, 1, 64, 1, 90, 128, False, False),
    ("bf16", 2, 130, 2, 1, 128, 30, 140, 16, True, False),
    ("bf16", 1, 1, 64, 1, 128, 500, 0, 64, True, True),
    ("e4m3", 20, 2, 8, 1, 256, 1100, 300, 64, True, False),
    ("bf16", 16, 1, 16, 2, 128, 2500, 5, 64, True, False),
    ("int8", 1, 1, 1, 1, 64, 4000, 1, 112, True, False),
    # runs of many tiles in a CTA, of rows that fill their tiles and of a few
    ("bf16", 40, 1, 32, 8, 128, 4000, 700, 64, True, False),
    ("e4m3", 24, 2, 32, 8, 64, 3000, 900, 32, True, True),
    ("int8", 60, 1, 32, 8, 128, 2500, 400, 64, True, False),
    ("bf16", 30, 3, 16, 8, 256, 1500, 500, 64, True, False),
]


@pytest.mark.parametrize("fmt,batch,tokens,q_heads,heads,dim,prefix,own,page,causal,masked", CASES)
def test_against_the_definition(fmt, batch, tokens, q_heads, heads, dim, prefix, own, page, causal, masked):
    from pi05_megakernel_b200.shared import SharedPrefixAttention
    c, ptab, tab, lengths, rnd = build(fmt, batch, prefix, own, page, heads, dim, seed=prefix + own)
    valid = None
    if masked:
        valid = torch.rand(prefix, generator=torch.Generator().manual_seed(1)) < 0.7
        bad = (~valid).nonzero().flatten()
        for n in ("k", "v"):                                              # what a masked place holds does not matter: infinities, in a BF16 cache
            if fmt == "bf16":
                getattr(c, n)[ptab.cpu().long()[bad // page], 1, bad % page] = float("inf")
    q = 2 * rnd(batch, tokens, q_heads, dim)
    op = SharedPrefixAttention(c, q_heads, batch, tokens)
    args = dict(layer=1, valid=None if valid is None else valid.cuda(), causal=causal)
    own_args = (tab, lengths) if own else (None, None)
    got = op.run(q, ptab if prefix else None, prefix, *own_args, with_lse=True, **args)
    op.status()
    clean = c
    if masked and fmt == "bf16":                                          # (the definition leaves masked keys out, so it may read them)
        clean = type(c).wrap(torch.nan_to_num(c.k.float(), 0, 0, 0).to(torch.bfloat16), torch.nan_to_num(c.v.float(), 0, 0, 0).to(torch.bfloat16))
    check(got, attend(clean, q, ptab, prefix, *own_args, 1, valid, causal, dim ** -0.5))
    again = op.run(q, ptab if prefix else None, prefix, *own_args, with_lse=True, **args)
    assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])


@pytest.mark.parametrize("fmt", ["bf16", "int8", "e4m3"])
@pytest.mark.parametrize("dim", [64, 256])
def test_queries_without_keys(fmt, dim):
    """No valid prefix token and no own one: zeros; more queries than own tokens: the first ones see none."""
    from pi05_megakernel_b200.shared import SharedPrefixAttention
    c, ptab, tab, lengths, rnd = build(fmt, 3, 70, 20, 16, 1, dim)
    lengths.copy_(torch.tensor([0, 2, 20]))
    q = rnd(3, 5, 4, dim)
    valid = torch.zeros(70, dtype=torch.bool)
    op = SharedPrefixAttention(c, 4, 3, 5)
    for causal in (True, False):
        got = op.run(q, ptab, 70, tab, lengths, layer=1, valid=valid.cuda(), causal=causal, with_lse=True)
        op.status()
        check(got, attend(c, q, ptab, 70, tab, lengths, 1, valid, causal, dim ** -0.5))
    got = op.run(q, None, 0, with_lse=True)
    assert bool((got[0] == 0).all()) and bool((got[1] == -math.inf).all())


def test_large_scores_and_growing_maxima():
    """Scores of hundreds, rising along the keys, so that the softmax's reference moves in every tile; one key far above the rest."""
    from pi05_megakernel_b200.shared import SharedPrefixAttention
    c, ptab, tab, lengths, rnd = build("bf16", 2, 700, 90, 64, 1, 256)
    ramp = torch.linspace(0.1, 30, 700)[None, None, :, None, None]
    q = rnd(2, 1, 8, 256)
    k = (q[:1, :, :1].cpu().float().view(1, 1, 1, 1, 256) * ramp * 0.5).to(torch.bfloat16).expand(1, 2, 700, 1, 256).contiguous()
    c.write(k.cuda(), rnd(1, 2, 700, 1, 256), ptab[None])
    op = SharedPrefixAttention(c, 8, 2)
    for scale in (256 ** -0.5, 1.0):
        got = op.run(q, ptab, 700, tab, lengths, layer=1, scale=scale, with_lse=True)
        op.status()
        check(got, attend(c, q, ptab, 700, tab, lengths, 1, None, True, scale))


@pytest.mark.parametrize("fmt", ["bf16", "int8"])
def test_strides(fmt):
    """Queries as a slice of a projection's output, outputs into a larger tensor, tables cut from larger ones."""
    from pi05_megakernel_b200.shared import SharedPrefixAttention
    c, ptab, tab, lengths, rnd = build(fmt, 3, 100, 40, 16, 1, 256)
    qkv = rnd(2, 3, 2560)                                                 # [tokens][sequences][q | k | v]
    q = qkv[..., :2048].view(2, 3, 8, 256).transpose(0, 1)
    wide = torch.full((3, 9), -7, dtype=torch.int32, device="cuda")
    wide[:, 2:2 + tab.shape[1]] = tab
    big = torch.full((3, 4, 8, 512), 3.0, dtype=torch.bfloat16, device="cuda")
    out = big[:, 1:3, :, 256:]
    op = SharedPrefixAttention(c, 8, 5, 4)
    got = op.run(q, ptab, 100, wide[:, 2:2 + tab.shape[1]], lengths, layer=1, out=out, with_lse=True)
    op.status()
    assert got[0] is out
    check(got, attend(c, q, ptab, 100, tab, lengths, 1, None, True, 1 / 16))
    assert bool((big[:, [0, 3]] == 3).all()) and bool((big[:, 1:3, :, :256] == 3).all())


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
def test_bad_tables(fmt):
    """A bad page makes what sees it NaN and nothing else; lengths out of range are cut; both are reported."""
    from pi05_megakernel_b200.shared import SharedPrefixAttention
    c, ptab, tab, lengths, rnd = build(fmt, 3, 100, 40, 16, 1, 128)
    q = rnd(3, 1, 4, 128)
    op = SharedPrefixAttention(c, 4, 3)
    good = op.run(q, ptab, 100, tab, lengths, layer=1)
    wrong = tab.clone()
    wrong[2, 1] = c.pages
    got = op.run(q, ptab, 100, wrong, lengths, layer=1)
    with pytest.raises(_lib.EngineError, match="page out of range in sequence 2") as info:
        op.status()
    assert info.value.code == _lib.ERR_PAGE_TABLE
    assert torch.equal(got[:2], good[:2]) and bool(torch.isnan(got[2]).all())
    lost = ptab.clone()
    lost[3] = -1
    assert bool(torch.isnan(op.run(q, lost, 100, tab, lengths, layer=1)).all())
    with pytest.raises(_lib.EngineError, match="page out of range in the shared prefix"):
        op.status()
    wrong[2, 1], wrong[2, 2] = tab[2, 1], 1 << 30                         # behind the sequence's last token: not looked at
    short = torch.tensor([0, 3, 32], dtype=torch.int32, device="cuda")
    check(op.run(q, ptab, 100, wrong, short, layer=1, with_lse=True), attend(c, q, ptab, 100, tab, short, 1, None, True, 128 ** -0.5))
    op.status()
    for bad, cut in (([0, 20, 10 ** 6], [0, 20, tab.shape[1] * 16]), ([-5, 20, 40], [0, 20, 40])):
        n = torch.tensor(bad, dtype=torch.int32, device="cuda")
        got = op.run(q, ptab, 100, tab[:, :2] if bad[2] > 40 else tab, n, layer=1, with_lse=True)
        with pytest.raises(_lib.EngineError, match="start or length out of range"):
            op.status()
        cut = [min(x, 32) for x in cut] if bad[2] > 40 else cut
        check(got, attend(c, q, ptab, 100, tab, torch.tensor(cut), 1, None, True, 128 ** -0.5))


def test_a_key_that_is_not_a_number():
    """A quantised key with a NaN (its scale is one) makes the queries that see it NaN, and only those."""
    from pi05_megakernel_b200.shared import SharedPrefixAttention
    c, ptab, tab, lengths, rnd = build("int8", 2, 40, 20, 16, 1, 64)
    bad = rnd(1, 2, 1, 1, 64)
    bad[0, 1, 0, 0, 5] = float("nan")
    c.write(bad, rnd(1, 2, 1, 1, 64), tab[1:2], starts=torch.tensor([18], dtype=torch.int32, device="cuda"))
    q = rnd(2, 4, 3, 64)
    got = SharedPrefixAttention(c, 3, 2, 4).run(q, ptab, 40, tab, lengths, layer=1)     # query t of sequence 1 sees own tokens up to 16 + t
    assert bool(torch.isfinite(got[0]).all()) and bool(torch.isfinite(got[1, :2]).all()) and bool(torch.isnan(got[1, 2:]).all())


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_values_that_are_not_numbers_stay_with_those_that_see_them(dim, bad):
    """BF16: keys and values that are not numbers, at tokens that only some of a sequence's queries see, reach those and nobody else, whichever group of
    warps has the tile."""
    from pi05_megakernel_b200.shared import SharedPrefixAttention
    tokens, q_heads = 70, 3
    c, ptab, tab, lengths, rnd = build("bf16", 2, 100, 300, 16, 1, dim, junk=False)
    lengths.copy_(torch.tensor([300, 250]))
    q = rnd(2, tokens, q_heads, dim)
    op = SharedPrefixAttention(c, q_heads, 2, tokens)
    clean = op.run(q, ptab, 100, tab, lengths, layer=1)
    for token in (299, 290, 256, 255, 232):                               # of sequence 0, whose queries stand at 230 .. 299
        for pool in (c.k, c.v):
            page, at = int(tab[0, token // 16]), token % 16
            old = pool[page, 1, at].clone()
            pool[page, 1, at, 0, dim - 3] = bad
            got = op.run(q, ptab, 100, tab, lengths, layer=1)
            op.status()
            first = token - 230                                           # the first query that sees it
            assert torch.equal(got[1], clean[1]) and torch.equal(got[0, :first], clean[0, :first])
            if pool is c.v or bad != bad:
                assert not bool(torch.isfinite(got[0, first:]).all(-1).any())
            pool[page, 1, at] = old
    assert torch.equal(op.run(q, ptab, 100, tab, lengths, layer=1), clean)


def test_python_refusals():
    from pi05_megakernel_b200.shared import SharedPrefixAttention
    c, ptab, tab, lengths, rnd = build("int8", 2, 40, 20, 16, 2, 64)
    with pytest.raises(ValueError):
        SharedPrefixAttention(c, 3, 2)
    with pytest.raises(ValueError):
        SharedPrefixAttention(c, 4, 0)
    op = SharedPrefixAttention(c, 4, 2, 2)
    q = rnd(2, 2, 4, 64)
    ok = torch.ones(40, dtype=torch.bool, device="cuda")
    for bad in (lambda: op.run(q.float(), ptab, 40), lambda: op.run(q[:, :, :2], ptab, 40), lambda: op.run(q.repeat(2, 1, 1, 1), ptab, 40),
                lambda: op.run(q.repeat(1, 2, 1, 1), ptab, 40), lambda: op.run(q, None, 40), lambda: op.run(q, ptab, 49), lambda: op.run(q, ptab, -1),
                lambda: op.run(q, ptab, 40, tab), lambda: op.run(q, ptab, 40, tab[:1], lengths), lambda: op.run(q, ptab, 40, tab, lengths.long()),
                lambda: op.run(q, ptab.long(), 40), lambda: op.run(q, ptab, 40, layer=2), lambda: op.run(q, ptab, 40, valid=ok[:39]),
                lambda: op.run(q, ptab, 40, valid=ok.int()), lambda: op.run(q, ptab, 40, out=q[:1]), lambda: op.run(q.cpu(), ptab, 40),
                lambda: op.run(rnd(2, 2, 64, 4).transpose(2, 3), ptab, 40), lambda: op.run(rnd(2, 2, 4, 68)[..., :64], ptab, 40)):
        with pytest.raises(ValueError):
            bad()
    c.status()


def test_graph_replays_follow_the_lengths():
    """One captured step, replayed while the sequences grow (a write, then attention), equals the same calls made one by one."""
    from pi05_megakernel_b200.shared import SharedPrefixAttention
    c, ptab, tab, lengths, rnd = build("e4m3", 3, 300, 100, 16, 1, 256)
    op = SharedPrefixAttention(c, 8, 3)
    q, k, v = rnd(3, 1, 8, 256), rnd(3, 1, 1, 1, 256), rnd(3, 1, 1, 1, 256)
    starts = torch.tensor([0, 40, 77], dtype=torch.int32, device="cuda")
    lengths.copy_(starts + 1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        c.write(k, v, tab, starts=starts, layer=1)
        out, lse = op.run(q, ptab, 300, tab, lengths, layer=1, with_lse=True)
    for step in range(4):
        q.copy_(rnd(3, 1, 8, 256))
        k.copy_(rnd(3, 1, 1, 1, 256))
        v.copy_(rnd(3, 1, 1, 1, 256))
        graph.replay()
        torch.cuda.synchronize()
        want = attend(c, q, ptab, 300, tab, lengths, 1, None, True, 1 / 16)
        check((out, lse), want)
        again = op.run(q, ptab, 300, tab, lengths, layer=1, with_lse=True)
        assert torch.equal(again[0], out) and torch.equal(again[1], lse)
        starts += 1
        lengths += 1
    op.status()


def test_two_calls_at_once():
    """Two operators over one cache, each with its workspace, on two streams."""
    from pi05_megakernel_b200.shared import SharedPrefixAttention
    c, ptab, tab, lengths, rnd = build("int8", 4, 900, 60, 64, 1, 256)
    ops = [SharedPrefixAttention(c, 8, 4) for _ in range(2)]
    qs = [rnd(4, 1, 8, 256) for _ in range(2)]
    want = [op.run(q, ptab, 900, tab, lengths, layer=1) for op, q in zip(ops, qs)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(20):
        got = []
        for op, q, s in zip(ops, qs, streams):
            with torch.cuda.stream(s):
                got.append(op.run(q, ptab, 900, tab, lengths, layer=1))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    c.status()


def test_expanded_outputs_are_refused():
    from pi05_megakernel_b200.shared import SharedPrefixAttention
    c, ptab, tab, lengths, rnd = build("bf16", 2, 40, 20, 16, 2, 64)
    op, q = SharedPrefixAttention(c, 4, 2, 2), rnd(2, 2, 4, 64)
    for out in (q[:1].clone().expand(2, -1, -1, -1), q[:, :1].clone().expand(-1, 2, -1, -1)):
        with pytest.raises(ValueError):
            op.run(q, ptab, 40, tab, lengths, out=out)
    # queries may be expanded: they are only read
    assert torch.equal(op.run(q[:1].expand(2, -1, -1, -1), ptab, 40), op.run(q[:1].repeat(2, 1, 1, 1), ptab, 40))
    c.status()

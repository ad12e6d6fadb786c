"""Pools that something else has filled: e4m3 codes that are NaN make their rows NaN, read back and attended to, and nothing else."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("code", [0x7f, 0xff])
def test_codes_that_are_not_numbers(dim, code):
    from pi05_megakernel_b200.cache import KvCache
    from pi05_megakernel_b200.shared import SharedPrefixAttention
    g = torch.Generator().manual_seed(dim)
    pages, page, heads, own = 5, 16, 2, 30
    made = KvCache(pages, 2, page, heads, dim, "e4m3")
    table = torch.tensor([[3, 1], [4, 0]], dtype=torch.int32, device="cuda")
    rnd = lambda *s: torch.randn(*s, generator=g).to(torch.bfloat16).cuda()
    made.write(rnd(2, 2, own, heads, dim), rnd(2, 2, own, heads, dim), table)
    made.status()
    lengths = torch.full((2,), own, dtype=torch.int32, device="cuda")
    q = rnd(2, 4, 4, dim)
    attend = lambda c: SharedPrefixAttention(c, 4, 2, 4).run(q, None, 0, table, lengths, layer=1, with_lse=True)
    want, clean = made.read(table, own), attend(made)
    for which in ("k", "v"):
        pools = [t.clone() for t in (made.k, made.v, made.k_scale, made.v_scale)]
        codes = pools[0 if which == "k" else 1].view(torch.uint8)
        codes[1, 1, 12, 1, dim - 1] = code                                # token 28 of sequence 0, layer 1, head 1
        codes[2] = code                                                   # a page of nobody's
        c = KvCache.wrap(*pools)
        got = c.read(table, own)
        for n, a, b in (("k", got[0], want[0]), ("v", got[1], want[1])):
            lost = torch.zeros(a.shape[:-1], dtype=torch.bool, device="cuda")
            lost[0, 1, 28, 1] = n == which
            assert bool(torch.isnan(a[lost]).all()) and torch.equal(a[~lost], b[~lost])
        o, lse = attend(c)
        sees = torch.zeros(2, 4, 4, dtype=torch.bool, device="cuda")
        sees[0, 2:, 2:] = True                                            # queries stand at tokens 26 .. 29
        assert bool(torch.isnan(o[sees]).all()) and torch.equal(o[~sees], clean[0][~sees]) and torch.equal(lse[~sees], clean[1][~sees])
        c.status()


def test_pools_without_them_stay_as_they_are():
    """Every code that is a number, in pools of several steps' size (of one byte: also the other formats)."""
    from pi05_megakernel_b200.cache import KvCache
    codes = torch.arange(256, dtype=torch.int64)
    codes = codes[(codes & 127) != 127]
    for pages, page, heads, dim in ((3, 16, 2, 64), (2100, 64, 2, 256)):
        n = pages * page * heads * dim
        k = codes.repeat(n // len(codes) + 1)[:n].to(torch.uint8).cuda().view(torch.float8_e4m3fn).view(pages, 1, page, heads, dim)
        scale = torch.rand(pages, 1, heads, page, device="cuda")
        one, two = scale.clone(), scale.clone()
        KvCache.wrap(k, k.clone(), one, two)
        assert torch.equal(one, scale) and torch.equal(two, scale)
    k.view(torch.uint8)[[0, 1023, 1024, 2099], 0, 5, 1, 7] = 0xff
    KvCache.wrap(k, k, one, two)
    want = torch.zeros_like(scale, dtype=torch.bool)
    want[[0, 1023, 1024, 2099], 0, 1, 5] = True
    assert torch.equal(torch.isnan(one), want) and torch.equal(torch.isnan(two), want)

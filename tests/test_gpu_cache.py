"""Rows into the pages of a cache and out of them, against the definition in 64 bits.

What the 8-bit formats hold is compared bit for bit: with BF16 inputs the quotient x peak / max|x| is a middle of two codes exactly or far from one,
so there is one right code.  A scale is one FP32 division (within half a step, 2^-24); what is read back is code x scale in FP32, rounded to BF16:
within 2^-24 and then half a BF16 step, 2^-8 (a little more than that in all).
"""
import pytest
import torch

from pi05_megakernel_b200 import _lib

pytestmark = pytest.mark.gpu
PEAK = {"int8": 127.0, "e4m3": 448.0}


def e4m3_values():
    codes = torch.arange(127, dtype=torch.float64)
    e, m = codes.div(8, rounding_mode="floor"), codes % 8
    return torch.where(e == 0, m * 2.0 ** -9, (8 + m) * torch.exp2(e - 10))


def encode(x, fmt):
    """Codes (as the numbers that they are) and scales of rows in 64 bits."""
    x = x.double()
    a = x.abs().amax(-1, keepdim=True)
    ok = torch.isfinite(a) & (a > 0)
    y = torch.where(ok, x * PEAK[fmt] / torch.where(ok, a, torch.ones_like(a)), torch.zeros_like(x))
    if fmt == "int8":
        codes = torch.round(y)
    else:
        grid = e4m3_values()
        hi = torch.bucketize(y.abs(), grid).clamp(1, 126)
        up, down = grid[hi] - y.abs(), y.abs() - grid[hi - 1]
        codes = torch.copysign(grid[torch.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, hi - 1)], y)
    scale = torch.where(torch.isfinite(a), a / PEAK[fmt], torch.full_like(a, float("nan")))
    return codes, scale[..., 0]


def make(fmt, pages, layers, page, heads, dim, fill=None):
    from pi05_megakernel_b200.cache import KvCache
    c = KvCache(pages, layers, page, heads, dim, fmt)
    if fill is not None:
        for t in (c.k, c.v):
            t.view(torch.uint8).fill_(fill)
    return c


def held(c, n):
    """What the pool holds, as numbers: codes (or BF16 values) and scales in 64 bits on the host, tokens by heads."""
    codes = getattr(c, n).float().double().cpu()
    scale = None if c.format == "bf16" else getattr(c, n + "_scale").double().cpu().transpose(2, 3)
    return codes, scale


def check_held(c, n, p, at, layer, rows):
    """The pool's rows of page p, places at .. are those that `rows` [layers, tokens, heads, dim] encode to."""
    codes, scale = held(c, n)
    k = rows.shape[1]
    got = codes[p, layer:layer + rows.shape[0], at:at + k]
    if c.format == "bf16":
        assert torch.equal(got, rows.double())
        return
    want, s = encode(rows, c.format)
    assert torch.equal(got, want), (got - want).abs().max()
    sg = scale[p, layer:layer + rows.shape[0], at:at + k]
    assert torch.equal(torch.isnan(sg), torch.isnan(s))
    fine = ~torch.isnan(s)
    assert bool(((sg - s).abs()[fine] <= 2.0 ** -24 * s[fine] + 2.0 ** -150).all())


CASES = [
    # fmt, batch, layers, tokens, heads, dim, page, ragged
    ("int8", 1, 1, 1, 1, 256, 64, False),
    ("e4m3", 4, 1, 1, 1, 256, 16, False),
    ("bf16", 3, 2, 33, 2, 64, 16, True),
    ("int8", 3, 2, 65, 4, 64, 48, True),
    ("e4m3", 2, 3, 130, 8, 128, 64, True),
    ("int8", 1, 18, 101, 1, 256, 64, False),
    ("bf16", 2, 2, 128, 1, 256, 128, False),
    ("e4m3", 5, 1, 17, 3, 256, 32, True),
    ("int8", 7, 1, 31, 5, 128, 16, True),
]


@pytest.mark.parametrize("fmt,batch,layers,tokens,heads,dim,page,ragged", CASES)
def test_write_and_read(fmt, batch, layers, tokens, heads, dim, page, ragged):
    g = torch.Generator().manual_seed(tokens * 31 + dim)
    per = -(-(tokens + 5) // page)
    pages, first = 2 + batch * per, 1                                     # a layer of the cache stays behind
    table = 1 + torch.randperm(pages - 2, generator=g)[:batch * per].view(batch, per).int()
    starts = torch.tensor([i % 6 for i in range(batch)]).int()
    counts = torch.tensor([tokens * i // max(1, batch - 1) for i in range(batch)]).int() if ragged else None
    k, v = (torch.randn(batch, layers, tokens, heads, dim, generator=g).to(torch.bfloat16) for _ in range(2))
    c = make(fmt, pages, layers + first, page, heads, dim, fill=0x3b)
    before = {n: held(c, n)[0].clone() for n in ("k", "v")}
    tab, dev = table.cuda(), lambda t: None if t is None else t.cuda()
    c.write(k.cuda(), v.cuda(), tab, starts=starts.cuda(), counts=dev(counts), layer=first)
    c.status()
    touched = torch.zeros(before["k"].shape[:3], dtype=torch.bool)
    for n, rows in (("k", k), ("v", v)):
        for b in range(batch):
            for t in range(tokens if counts is None else int(counts[b])):
                pos = int(starts[b]) + t
                p, at = int(table[b, pos // page]), pos % page
                touched[p, first:, at] = True
                if t in (0, tokens // 2, tokens - 1) or tokens < 40:
                    check_held(c, n, p, at, first, rows[b, :, t:t + 1])
        assert torch.equal(held(c, n)[0][~touched], before[n][~touched])  # everything else as it was
    rk, rv = c.read(tab, tokens, starts=starts.cuda(), counts=dev(counts), layer=first)
    c.status()
    for n, rows, got in (("k", k, rk.cpu()), ("v", v, rv.cpu())):
        assert got.shape == rows.shape and got.dtype == torch.bfloat16
        has = torch.ones(batch, tokens, dtype=torch.bool) if counts is None else torch.arange(tokens) < counts[:, None]
        has = has[:, None, :, None, None].expand(rows.shape)
        assert bool((got[~has] == 0).all())
        if fmt == "bf16":
            assert torch.equal(got[has], rows[has])
        else:
            codes, scale = encode(rows, fmt)
            want = codes * scale[..., None]
            assert bool(((got.double() - want).abs() <= (2.0 ** -8 + 2.0 ** -22) * want.abs())[has].all())


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_rows_at_the_borders(fmt, dim):
    """Rows whose quotients are exactly between two codes, of zeros, of the smallest and the largest numbers, and with infinities and NaN."""
    g = torch.Generator().manual_seed(9)
    top = torch.cat([torch.arange(128, 256) * 2.0 ** -7, torch.tensor([2.0 ** -133, 2.0 ** -126, 1.5 * 2.0 ** -127, 2.0 ** -100, 3.3895314e38, 2.0 ** 127, 1e30, 1e-30])])
    rows = torch.empty(len(top) + 4, dim)
    for i, a in enumerate(top):
        x = torch.randint(-(1 << 8), (1 << 8) + 1, (dim,), generator=g) * 2.0 ** -8     # multiples of a / 256: a / 2, a / 254-ths of BF16 and so on
        rows[i] = x * a
        rows[i, 0], rows[i, 1], rows[i, 2] = a, a / 2, -a / 2
    rows[len(top)] = 0
    rows[len(top) + 1] = torch.randn(dim, generator=g)
    rows[len(top) + 1, dim - 1] = float("inf")
    rows[len(top) + 2] = torch.randn(dim, generator=g)
    rows[len(top) + 2, 3] = float("nan")
    rows[len(top) + 3] = torch.randn(dim, generator=g)
    rows[len(top) + 3, 5], rows[len(top) + 3, 6] = float("-inf"), float("nan")
    x = rows.to(torch.bfloat16).view(1, 1, -1, 1, dim)
    n = x.shape[2]
    c = make(fmt, 1, 1, -(-n // 16) * 16, 1, dim)
    table = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    c.write(x.cuda(), x.flip(-1).contiguous().cuda(), table)
    c.status()
    check_held(c, "k", 0, 0, 0, x[0])
    check_held(c, "v", 0, 0, 0, x[0].flip(-1))
    got = c.read(table, n)[0].cpu()[0, 0, :, 0]
    assert bool(torch.isnan(got[-3:]).all()) and bool((got[len(top)] == 0).all()) and bool(torch.isfinite(got[:-3]).all())


def test_strided_inputs_and_outputs():
    """Keys and values as slices of one projection's output [tokens, q | k | v], and outputs into a larger tensor with the layers outside."""
    g = torch.Generator().manual_seed(4)
    qkv = torch.randn(6, 5, 2560, generator=g).to(torch.bfloat16).cuda()  # 6 sequences x 5 tokens
    k = qkv[..., 2048:2304].view(6, 1, 5, 1, 256)
    v = qkv[..., 2304:2560].view(6, 1, 5, 1, 256)
    c = make("bf16", 8, 3, 16, 1, 256)
    table = torch.tensor([[7], [2], [5], [1], [0], [4]], dtype=torch.int32, device="cuda")
    c.write(k, v, table, layer=2)
    big = torch.full((3, 6, 5, 2, 256), 7.0, dtype=torch.bfloat16, device="cuda")
    outs = tuple(big[1:2, :, :, i:i + 1].transpose(0, 1) for i in range(2))
    c.read(table, 5, layer=2, layers=1, out=outs)
    c.status()
    assert torch.equal(big[1, :, :, 0], k[:, 0, :, 0]) and torch.equal(big[1, :, :, 1], v[:, 0, :, 0])
    assert bool((big[0] == 7).all()) and bool((big[2] == 7).all())
    wide = torch.zeros(6, 9, dtype=torch.int32, device="cuda")            # a table cut from a larger one
    wide[:, :1] = table
    again = c.read(wide[:, :1], 5, layer=2, layers=1)
    assert torch.equal(again[0], k)


@pytest.mark.parametrize("fmt", ["bf16", "int8"])
def test_rows_that_begin_on_16_bytes_only(fmt):
    """Rows at odd multiples of 16 bytes, in and out: the same as aligned ones."""
    g = torch.Generator().manual_seed(6)
    wide = torch.randn(2, 1, 7, 3, 136, generator=g).to(torch.bfloat16).cuda()
    k, v = wide[..., :128], wide[..., 8:]                                 # heads 272 bytes apart; v behind 16
    c = make(fmt, 3, 1, 16, 3, 128)
    table = torch.tensor([[2], [1]], dtype=torch.int32, device="cuda")
    c.write(k, v, table)
    want = c.read(table, 7)
    for b, p in enumerate((2, 1)):
        check_held(c, "k", p, 0, 0, k[b].cpu())
        check_held(c, "v", p, 0, 0, v[b].cpu())
    out = torch.zeros(2, 2, 1, 7, 3, 136, dtype=torch.bfloat16, device="cuda")
    c.read(table, 7, out=(out[0][..., 8:], out[1][..., 8:]))
    c.status()
    assert torch.equal(out[0][..., 8:], want[0]) and torch.equal(out[1][..., 8:], want[1]) and bool((out[..., :8] == 0).all())


def test_bad_pages_and_positions_are_left_out():
    c = make("int8", 4, 1, 16, 1, 64, fill=0x11)
    k = torch.randn(4, 1, 16, 1, 64).to(torch.bfloat16).cuda()
    table = torch.tensor([[2], [4], [-1], [3]], dtype=torch.int32, device="cuda")
    c.write(k, k, table)
    with pytest.raises(_lib.EngineError, match="page out of range in sequence [12]$") as info:
        c.status()
    assert info.value.code == _lib.ERR_PAGE_TABLE
    c.status()                                                            # read once, then cleared
    check_held(c, "k", 2, 0, 0, k[0].cpu())
    check_held(c, "v", 3, 0, 0, k[3].cpu())
    assert bool((c.k[:2].view(torch.uint8) == 0x11).all())
    got = c.read(table, 16)[0]
    assert bool(torch.isnan(got[1:3]).all()) and bool(torch.isfinite(got[0]).all())
    with pytest.raises(_lib.EngineError, match="page out of range"):
        c.status()
    before = c.k.clone()
    for starts in ([1, 0, 0, 0], [-1, 0, 0, 0], [2 ** 31 - 1, 0, 0, 0]):
        st = torch.tensor(starts, dtype=torch.int32, device="cuda")
        ok = torch.tensor([[2], [1], [0], [3]], dtype=torch.int32, device="cuda")
        c.write(k, k, ok, starts=st, counts=torch.tensor([16, 0, 0, 0], dtype=torch.int32, device="cuda"))
        with pytest.raises(_lib.EngineError, match="start or length out of range in sequence 0"):
            c.status()
        assert bool((c.k[[0, 1, 3]] == before[[0, 1, 3]]).all())
        assert bool(torch.isnan(c.read(ok, 16, starts=st)[0][0]).any())
        with pytest.raises(_lib.EngineError, match="start or length"):
            c.status()
    # a bad entry that no row needs is not looked at
    c.write(k, k, table, counts=torch.tensor([3, 0, 0, 1], dtype=torch.int32, device="cuda"))
    c.status()


def test_python_refusals():
    c = make("int8", 4, 2, 16, 2, 64)
    k = torch.zeros(2, 2, 8, 2, 64, dtype=torch.bfloat16, device="cuda")
    t = torch.zeros(2, 1, dtype=torch.int32, device="cuda")
    for bad in (lambda: c.write(k.float(), k.float(), t), lambda: c.write(k, k[:1], t), lambda: c.write(k[..., :32], k[..., :32], t),
                lambda: c.write(k, k, t.long()), lambda: c.write(k, k, t[:1]), lambda: c.write(k, k, t, layer=1), lambda: c.write(k.cpu(), k.cpu(), t),
                lambda: c.write(k, k.transpose(2, 1).contiguous().transpose(2, 1), t), lambda: c.write(k, k, t, counts=t[:, 0].long()),
                lambda: c.write(k, k, t, starts=t[:1, 0]), lambda: c.read(t, 8, out=(k, k), layer=1), lambda: c.read(t, 9, out=(k, k))):
        with pytest.raises(ValueError):
            bad()
    c.status()


def test_graph_and_streams():
    """A captured write and read follow what the tables and inputs hold at the replay, on a stream of their own."""
    c = make("e4m3", 6, 1, 16, 1, 128)
    k, v = (torch.randn(2, 1, 3, 1, 128).to(torch.bfloat16).cuda() for _ in range(2))
    table = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32, device="cuda")
    starts = torch.tensor([14, 2], dtype=torch.int32, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        c.write(k, v, table, starts=starts)
        out = c.read(table, 3, starts=starts)
    for step in range(3):
        k.copy_(torch.randn(k.shape))
        v.copy_(torch.randn(k.shape))
        table.copy_(torch.tensor([[step, 5], [4, (step + 1) % 3]]))
        starts.copy_(torch.tensor([13 + step, 16 - step]))
        graph.replay()
        torch.cuda.synchronize()
        for got, rows in zip(out, (k, v)):
            codes, scale = encode(rows.cpu(), "e4m3")
            want = codes * scale[..., None]
            assert bool(((got.cpu().double() - want).abs() <= (2.0 ** -8 + 2.0 ** -22) * want.abs()).all())
    c.status()


def test_many_rows_behind_32_bits_of_elements():
    """The last pages of a pool whose elements do not count in 32 bits."""
    pages, page = 140, 65536                                              # 140 x 65536 x 1 x 256: 2.3e9 elements of one byte
    from pi05_megakernel_b200.cache import KvCache
    c = KvCache(pages, 1, page, 1, 256, "int8")
    k = torch.randn(1, 1, 40, 1, 256).to(torch.bfloat16)
    table = torch.tensor([[pages - 1]], dtype=torch.int32, device="cuda")
    starts = torch.tensor([page - 40], dtype=torch.int32, device="cuda")
    c.write(k.cuda(), k.cuda(), table, starts=starts)
    got = c.read(table, 40, starts=starts)[1].cpu()
    c.status()
    codes, scale = encode(k, "int8")
    want = codes * scale[..., None]
    assert bool(((got.double() - want).abs() <= (2.0 ** -8 + 2.0 ** -22) * want.abs()).all())
    assert int(c.k[-1, 0, :page - 40].count_nonzero()) == 0 and int(c.k[:-1].view(torch.int64).count_nonzero()) == 0


def test_expanded_outputs_are_refused():
    c = make("int8", 4, 2, 16, 2, 64)
    t = torch.zeros(2, 1, dtype=torch.int32, device="cuda")
    one = torch.zeros(1, 2, 8, 2, 64, dtype=torch.bfloat16, device="cuda").expand(2, -1, -1, -1, -1)
    with pytest.raises(ValueError):
        c.read(t, 8, out=(one, one.clone().expand_as(one)))
    with pytest.raises(ValueError):
        c.read(t, 8, out=(one, one))
    c.status()

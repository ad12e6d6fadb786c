"""Outputs whose rows lie on one another, on the queries or, keys on values, are refused; those that only share a buffer are not."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def made(fmt="int8", heads=2, dim=64):
    from pi05_megakernel_b200.cache import KvCache
    g = torch.Generator().manual_seed(0)
    c = KvCache(6, 2, 16, heads, dim, fmt)
    table = torch.tensor([[3, 1], [5, 2]], dtype=torch.int32, device="cuda")
    rnd = lambda *s: torch.randn(*s, generator=g).to(torch.bfloat16).cuda()
    c.write(rnd(2, 2, 20, heads, dim), rnd(2, 2, 20, heads, dim), table)
    return c, table, rnd


def test_reads():
    c, table, rnd = made()
    want = c.read(table, 20)
    shape = want[0].shape
    at = lambda *st, offset=0: torch.zeros(20000, dtype=torch.bfloat16, device="cuda").as_strided(shape, (*st, 1), offset)
    dense = at(5120, 2560, 128, 64)
    for out in ((dense, dense), (at(5120, 2560, 128, 8), at(5120, 2560, 128, 8)), (at(5120, 2560, 64, 64), at(5120, 2560, 64, 64)),
                (at(2504, 2560, 128, 64), at(2504, 2560, 128, 64)), (dense, dense.view(-1)[:].as_strided(shape, dense.stride(), 64))):
        with pytest.raises(ValueError, match="different places"):
            c.read(table, 20, out=out)
    both = torch.zeros(2, 2, 20, 2, 2, 64, dtype=torch.bfloat16, device="cuda")
    for pair in ((both[..., 0, :], both[..., 1, :]), (both[..., 1, :], both[..., 0, :])):       # keys and values of a head side by side
        got = c.read(table, 20, out=pair)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    inside = torch.zeros(2, 2, 20, 2, 64, dtype=torch.bfloat16, device="cuda")
    swapped = tuple(inside.clone().permute(3, 1, 2, 0, 4) for _ in range(2))                    # batch inside, heads outside
    got = c.read(table, 20, out=swapped)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    # one sequence twice over: keys and values may lie anywhere when they are written
    c.write(want[0][:1].expand(2, -1, -1, -1, -1), want[0][:1].expand(2, -1, -1, -1, -1), table)
    assert torch.equal(c.read(table, 20)[0][0], c.read(table, 20)[1][1])
    c.status()


def test_attention():
    from pi05_megakernel_b200.shared import SharedPrefixAttention
    c, table, rnd = made("bf16")
    lengths = torch.tensor([20, 13], dtype=torch.int32, device="cuda")
    op = SharedPrefixAttention(c, 4, 2, 3)
    q = rnd(2, 3, 4, 64)
    want = op.run(q, None, 0, table, lengths)
    run = lambda q, out: op.run(q, None, 0, table, lengths, out=out)
    room = torch.zeros(4000, dtype=torch.bfloat16, device="cuda")
    for st in ((768, 256, 8), (768, 192, 64), (704, 256, 64), (64, 256, 64)):
        with pytest.raises(ValueError, match="different places"):
            run(q, room.as_strided((2, 3, 4, 64), (*st, 1)))
    with pytest.raises(ValueError, match="over those of q"):
        run(q, q)
    buffer = torch.zeros(2, 3, 3, 4, 64, dtype=torch.bfloat16, device="cuda")                   # [batch][tokens][q | out | spare]
    buffer[:, :, 0] = q
    got = run(buffer[:, :, 0], buffer[:, :, 1])
    assert torch.equal(got, want) and torch.equal(buffer[:, :, 0], q) and bool((buffer[:, :, 2] == 0).all())
    flat = buffer.view(2, 3, 768)
    with pytest.raises(ValueError, match="over those of q"):              # outputs half a row behind the queries
        run(buffer[:, :, 0], flat[:, :, 32:288].view(2, 3, 4, 64))
    with pytest.raises(ValueError, match="over those of q"):              # shifted by a token, of which the last is the queries' no more
        run(buffer[:, :2, 0], buffer[:, 1:, 0])
    q1 = rnd(1, 3, 4, 64)
    same = q1.expand(2, -1, -1, -1)                                       # queries that are only read may be expanded
    assert torch.equal(run(same, torch.zeros_like(q)), run(same.contiguous(), None))
    op.status()

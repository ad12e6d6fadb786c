"""Tables without pages: sequences that have no tokens yet, and lengths that say otherwise."""
import pytest
import torch

from pi05_megakernel_b200 import _lib

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", ["bf16", "int8"])
def test_tables_without_pages(fmt):
    from pi05_megakernel_b200.cache import KvCache
    from pi05_megakernel_b200.shared import SharedPrefixAttention
    g = torch.Generator().manual_seed(0)
    rnd = lambda *s: torch.randn(*s, generator=g).to(torch.bfloat16).cuda()
    c = KvCache(3, 1, 16, 2, 64, fmt)
    prefix = torch.tensor([2, 0], dtype=torch.int32, device="cuda")
    c.write(rnd(1, 1, 20, 2, 64), rnd(1, 1, 20, 2, 64), prefix[None])
    before = c.k.clone()
    empty = torch.zeros(3, 0, dtype=torch.int32, device="cuda")
    none, some = torch.zeros(3, dtype=torch.int32, device="cuda"), torch.tensor([0, 2, 0], dtype=torch.int32, device="cuda")
    q = rnd(3, 1, 4, 64)
    op = SharedPrefixAttention(c, 4, 3)
    want = op.run(q, prefix, 20)
    assert torch.equal(op.run(q, prefix, 20, empty, none), want)
    op.status()
    assert torch.equal(op.run(q, prefix, 20, empty, some), want)          # cut to what there is, and reported
    with pytest.raises(_lib.EngineError, match="start or length out of range in sequence 1"):
        op.status()
    k = rnd(3, 1, 4, 2, 64)
    c.write(k, k, empty, counts=none)
    assert all(bool((t == 0).all()) for t in c.read(empty, 4, counts=none))
    c.status()
    c.write(k, k, empty, counts=some)
    with pytest.raises(_lib.EngineError, match="start or length out of range in sequence 1"):
        c.status()
    got = c.read(empty, 4, counts=some)[0]
    with pytest.raises(_lib.EngineError, match="start or length out of range in sequence 1"):
        c.status()
    assert bool(torch.isnan(got[1, :, :2]).all()) and bool((got[1, :, 2:] == 0).all()) and bool((got[[0, 2]] == 0).all())
    assert torch.equal(c.k.view(torch.uint8), before.view(torch.uint8))

"""A prefill of some layers into a cache leaves the others' pages as they were, and a cache that does not fit is refused before anything runs."""
import pytest
import torch

from pi05_megakernel_b200 import fixture as FX

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def prefill():
    from pi05_megakernel_b200.prefill import Pi05Prefill
    geo = FX.PrefillGeometry(tokens=40)
    dev = {k: v.cuda() for k, v in FX.make_prefill_inputs(geo, 6, "full").items()}
    pre = Pi05Prefill(geo, "cuda")
    pre.bind(dev)
    yield pre, dev
    pre.close()


@pytest.mark.parametrize("fmt", ["bf16", "int8", "e4m3"])
@pytest.mark.parametrize("given", [False, True])
def test_layers_that_do_not_run(prefill, fmt, given):
    from pi05_megakernel_b200.cache import KvCache
    pre, dev = prefill
    cache = KvCache(4, 18, 16, 1, 256, fmt)
    table = torch.tensor([2, 0, 3], dtype=torch.int32, device="cuda")
    pools = [cache.k, cache.v] + ([] if fmt == "bf16" else [cache.k_scale, cache.v_scale])
    for p in pools:
        p.view(torch.uint8).fill_(0x3d)
    before = [p.clone() for p in pools]
    out = tuple(torch.full((18, 40, 1, 256), 5.0, dtype=torch.bfloat16, device="cuda") for _ in range(2)) if given else None
    k, v = pre.run(dev["embeddings"], dev["valid"], 3, out=out, cache=cache, table=table)
    pre.status()
    for p, was in zip(pools, before):
        assert torch.equal(p[:, 3:].view(torch.uint8), was[:, 3:].view(torch.uint8))
    # and a cache of just those layers holds the same
    small = KvCache(4, 3, 16, 1, 256, fmt)
    pre.run(dev["embeddings"], dev["valid"], 3, cache=small, table=table)
    for a, b in zip(cache.read(table[None], 40, layers=3), small.read(table[None], 40)):
        assert torch.equal(a, b)
    if fmt == "bf16":
        assert torch.equal(small.read(table[None], 40)[0][0], k[:3]) and torch.equal(small.read(table[None], 40)[1][0], v[:3])
    cache.status()
    small.status()


def test_refused_before_it_runs(prefill):
    from pi05_megakernel_b200.cache import KvCache
    pre, dev = prefill
    table = torch.tensor([2, 0, 3], dtype=torch.int32, device="cuda")
    out = tuple(torch.full((18, 40, 1, 256), 5.0, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    run = lambda cache, table, **more: pre.run(dev["embeddings"], dev["valid"], out=out, cache=cache, table=table, **more)
    fits = KvCache(4, 18, 16, 1, 256)
    for bad in (lambda: run(KvCache(4, 17, 16, 1, 256), table), lambda: run(KvCache(4, 2, 16, 1, 256), table, layers=3), lambda: run(KvCache(4, 18, 16, 2, 256), table),
                lambda: run(KvCache(4, 18, 16, 1, 128), table), lambda: run(fits, table.long()), lambda: run(fits, table[None]), lambda: run(fits, table.cpu()),
                lambda: run(fits, None), lambda: run(None, table)):
        with pytest.raises(ValueError):
            bad()
    assert all(bool((t == 5).all()) for t in out)

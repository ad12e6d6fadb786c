"""The cache's operators as they are used together: a prefilled prompt goes into the pages of a cache, action chunks run on what is read back from them, and
new tokens of several sequences step behind the shared prompt.

The chunk on a cached prefix is the chunk on the tensors that ``KvCache.read`` gives, bit for bit.  A step is held to the reference harness's band (twice the
BF16 eager path's own error against FP32, plus its tolerances), with the keys and values that the cache holds; the tokens' own keys and values of layer 0,
which depend on one projection and one norm only, to 4e-3 as in the prefill's tests.
"""
import pytest
import torch
import torch.nn.functional as F

from oracle import pi05_oracle as O
from pi05_megakernel_b200 import fixture as FX

pytestmark = pytest.mark.gpu
LAYERS = 3


def prefilled(tokens, fmt, pages, page=16, layers=LAYERS, seed=5):
    from pi05_megakernel_b200.cache import KvCache
    from pi05_megakernel_b200.prefill import Pi05Prefill
    inputs = FX.make_prefill_inputs(FX.PrefillGeometry(tokens=tokens), seed, "pad")
    dev = {k: v.cuda() for k, v in inputs.items()}
    pre = Pi05Prefill(FX.PrefillGeometry(tokens=tokens), "cuda")
    pre.bind(dev)
    cache = KvCache(pages, 18, page, 1, 256, fmt)
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(3)).int().cuda()
    n = -(-tokens // page)
    k, v = pre.run(dev["embeddings"], dev["valid"], layers, cache=cache, table=order[:n])
    pre.status()
    cache.status()
    return inputs, dev, pre, cache, order[:n].contiguous(), order[n:].contiguous(), k, v


def test_prefill_into_a_cache():
    """What comes back from the pages is what the prefill returned (BF16), or its quantisation."""
    for fmt, tol in (("bf16", 0.0), ("int8", 1 / 127), ("e4m3", 2.0 ** -4)):
        *_, cache, table, _, k, v = prefilled(50, fmt, 6, layers=18 if fmt == "bf16" else 2)
        rk, rv = cache.read(table[None], 50)
        for got, want in ((rk[0].float(), k.float()), (rv[0].float(), v.float())):
            # half a step of the code (int8: of the row's maximum; e4m3: of the element, half its smallest step near zero) and half a BF16 step
            top = want.abs().amax(-1, keepdim=True)
            bound = top * 0.5 * tol + want.abs() * 2.0 ** -8 if fmt != "e4m3" else want.abs() * (tol + 2.0 ** -7) + top * 2.0 ** -10 / 448
            assert bool(((got - want).abs() <= (bound * 1.001 if fmt != "bf16" else 0)).all())


@pytest.mark.parametrize("fmt,batch", [("bf16", 1), ("int8", 1), ("e4m3", 3)])
def test_chunk_on_a_cached_prefix(fmt, batch):
    """Bit for bit the chunk on the tensors that the cache reads back as; later launches follow the pages and the table."""
    from pi05_megakernel_b200.arm import CachedPrefix, Pi05Arm
    from pi05_megakernel_b200.cache import KvCache
    geo = FX.Geometry(prefix=100)
    stacked, _ = FX.make_batch(geo, 77, batch, "cuda", ["pad"] * batch)
    if batch == 1:
        stacked = {k: v[0] if k in FX.OBSERVATION else v for k, v in stacked.items()}
    cache = KvCache(4 * batch, 18, 32, 1, 256, fmt)
    table = torch.randperm(4 * batch, generator=torch.Generator().manual_seed(2)).int().view(batch, 4).cuda()
    pk, pv = (stacked[n].view(batch, 18, 100, 1, 256) for n in ("prefix_k", "prefix_v"))
    cache.write(pk, pv, table)
    arm, dense = (Pi05Arm(geo, "b200-s2-l3", "cuda", batch=batch) for _ in range(2))
    arm.bind(stacked, kv_pages=CachedPrefix(cache, table))
    for turn in range(2):
        arm.launch()
        arm.status()
        k, v = cache.read(table, 100)
        dense.bind({**stacked, "prefix_k": k if batch > 1 else k[0], "prefix_v": v if batch > 1 else v[0]})
        dense.launch()
        dense.status()
        assert torch.equal(arm.outputs()["actions"], dense.outputs()["actions"]) and bool(torch.isfinite(arm.outputs()["actions"]).all())
        cache.write(pk.flip(2), pv.flip(2), table)
    cache.status()
    with pytest.raises(ValueError):
        arm.bind(stacked, kv_pages=CachedPrefix(cache, table[:, :3].contiguous()))
    with pytest.raises(ValueError):
        CachedPrefix(KvCache(2, 18, 16, 2, 256, fmt), table)
    arm.bind(stacked)                                                     # and the dense tensors again
    arm.launch()
    dense.bind(stacked)
    dense.launch()
    assert torch.equal(arm.outputs()["actions"], dense.outputs()["actions"])
    arm.close()
    dense.close()


def step_oracle(v, x, positions, kv, sees, valid, widen):
    """The layers over tokens [batch, tokens, 2048] with the keys and values of the cache: kv[layer] = (prefix k, prefix v, own k, own v), own ones
    [batch, capacity, 256]; query (b, t) sees valid prefix tokens and the first sees[b][t] own ones."""
    cast = O._cast(widen)
    w = (lambda name, layer: v[name][layer].float()) if widen else (lambda name, layer: v[name][layer])
    batch, tokens = x.shape[:2]
    x = cast(x).reshape(batch * tokens, -1)
    flat = positions.reshape(-1)
    own = None
    for layer in range(len(kv)):
        n = O.rms_gemma(x, v["ln1"][layer], cast)
        q = O.rope((n @ w("lq", layer).T).view(-1, 8, 256), flat, cast)
        if layer == 0:
            own = (O.rope((n @ w("lk", 0).T).view(-1, 1, 256), flat, cast)[:, 0], n @ w("lv", 0).T)
        pk, pv, ok, ov = (cast(t) for t in kv[layer])
        mixed = []
        for i in range(batch * tokens):
            b, t = divmod(i, tokens)
            k, c = torch.cat((pk[valid], ok[b, :sees[b][t]])), torch.cat((pv[valid], ov[b, :sees[b][t]]))
            scores = (q[i] @ k.T) * 256 ** -0.5
            mixed.append((cast(F.softmax(scores, -1, dtype=torch.float32)) @ c).reshape(-1))
        x = x + torch.stack(mixed) @ w("lo", layer).T
        n = O.rms_gemma(x, v["ln2"][layer], cast)
        x = x + (F.gelu(n @ w("lg", layer).T, approximate="tanh") * (n @ w("lu", layer).T)) @ w("ld", layer).T
    return x.view(batch, tokens, -1), own


@pytest.mark.parametrize("fmt", ["bf16", "int8"])
def test_steps_behind_a_prefilled_prompt(fmt):
    """Three candidates: a first step of three tokens each, then one of a single token, in place and captured."""
    from pi05_megakernel_b200.shared import SharedPrefixAttention
    inputs, dev, pre, cache, ptab, rest, _, _ = prefilled(70, fmt, 12)
    batch, count = 3, int(inputs["valid"].sum())
    tab = rest[:6].view(batch, 2).contiguous()
    attention = SharedPrefixAttention(cache, 8, batch, 4)
    g = torch.Generator().manual_seed(8)
    lengths = torch.zeros(batch, dtype=torch.int32, device="cuda")
    done = torch.tensor([0, 0, 0])
    for tokens, captured in ((3, False), (1, False), (1, True)):
        x = torch.randn(batch, tokens, 2048, generator=g).to(torch.bfloat16)
        positions = (count + done[:, None] + torch.arange(tokens)).int()
        lengths += tokens
        args = (x.cuda(), positions.cuda(), attention, ptab, 70, tab, lengths, dev["valid"])
        if captured:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                hidden = pre.step(*args, layers=LAYERS)
            graph.replay()
        else:
            hidden = pre.step(*args, layers=LAYERS)
        pre.status()
        cache.status()
        done += tokens
        pk, pv = (t[0, :, :, 0].cpu() for t in cache.read(ptab[None], 70, layers=LAYERS))
        ok, ov = (t[:, :, :, 0].transpose(0, 1).cpu() for t in cache.read(tab, 32, layers=LAYERS))
        kv = [(pk[i], pv[i], ok[i], ov[i]) for i in range(LAYERS)]
        sees = [[int(done[b]) - tokens + t + 1 for t in range(tokens)] for b in range(batch)]
        want, own = step_oracle(inputs, x, positions.long(), kv, sees, inputs["valid"], False)
        exact, _ = step_oracle(inputs, x, positions.long(), kv, sees, inputs["valid"], True)
        d = O.band(want.float(), hidden.cpu().float(), exact.float())
        assert d["pass"], d
        if fmt == "bf16":
            for got, ref in ((ok[0], own[0]), (ov[0], own[1])):
                got = torch.stack([got[b, int(done[b]) - tokens:int(done[b])] for b in range(batch)]).reshape(-1, 256)
                assert float((got.float() - ref.float()).norm() / ref.float().norm()) < 4e-3
    pre.close()


def test_step_refusals():
    from pi05_megakernel_b200 import _lib
    from pi05_megakernel_b200.cache import KvCache
    from pi05_megakernel_b200.prefill import Pi05Prefill
    from pi05_megakernel_b200.shared import SharedPrefixAttention
    inputs, dev, pre, cache, ptab, rest, _, _ = prefilled(20, "int8", 6, layers=1)
    attention = SharedPrefixAttention(cache, 8, 3, 8)
    x = torch.zeros(3, 1, 2048, dtype=torch.bfloat16, device="cuda")
    pos = torch.zeros(3, 1, dtype=torch.int32, device="cuda")
    tab, n = rest[:3].view(3, 1).contiguous(), torch.ones(3, dtype=torch.int32, device="cuda")
    for bad in (lambda: pre.step(x.float(), pos, attention, ptab, 20, tab, n), lambda: pre.step(x, pos.long(), attention, ptab, 20, tab, n),
                lambda: pre.step(x, pos[:2], attention, ptab, 20, tab, n), lambda: pre.step(x, pos, attention, ptab, 33, tab, n),
                lambda: pre.step(x, pos, attention, ptab, 20, None, None), lambda: pre.step(x[:, :, :1024], pos, attention, ptab, 20, tab, n),
                lambda: pre.step(x, pos, SharedPrefixAttention(KvCache(6, 18, 16, 1, 128), 8, 3), ptab, 20, tab, n),
                lambda: pre.run(dev["embeddings"], dev["valid"], cache=cache)):
        with pytest.raises(ValueError):
            bad()
    many = torch.zeros(3, 8, 2048, dtype=torch.bfloat16, device="cuda")   # 24 tokens on a handle for 20
    with pytest.raises(_lib.EngineError, match="at most as many tokens"):
        pre.step(many, pos.expand(3, 8).contiguous(), attention, ptab, 20, tab, n * 8)
    with pytest.raises(_lib.EngineError, match="layers"):                 # a cache of one layer
        pre.step(x, pos, SharedPrefixAttention(KvCache(6, 1, 16, 1, 256), 8, 3), ptab, 20, tab, n, layers=2)
    with pytest.raises(_lib.EngineError):
        Pi05Prefill(FX.PrefillGeometry(tokens=20), "cuda").step(x, pos, attention, ptab, 20, tab, n)
    pre.close()

"""The cache operators and the attention over a shared prefix, as cases that can be timed and compared.

Three kinds of call:

* ``write``      keys and values of ``batch`` sequences x ``layers`` layers x ``tokens`` tokens go into the pages of a cache
                 (``KvCache.write``): BF16 as they are, or 8-bit codes with one FP32 scale per token and head;
* ``read``       the same rows out of their pages as BF16 (``KvCache.read``), zeros behind a sequence's last token;
* ``attention``  ``tokens`` queries of each of ``batch`` sequences over one prefix of ``prefix`` tokens that all of them share and
                 up to ``own`` tokens of their own (``SharedPrefixAttention.run``): outputs and log-sum-exp.

Keys and values have unit variance, queries are twice as wide (attention neither flat nor one-hot); lengths are spread evenly over their range
and dealt to the sequences by the seed; pages are dealt out of order.  Page 0 of every pool is in no table (a spare page).
"""
import math

import torch

own = False

DEV = "cuda" if torch.cuda.is_available() else "cpu"
PEAK = {"int8": 127.0, "e4m3": 448.0}
STORED = {"bf16": torch.bfloat16, "int8": torch.int8, "e4m3": torch.float8_e4m3fn}
LARGEST_ROWS = 16 * 4 * 2048 * 8 * 128          # elements of keys that a write or read case may have
LARGEST_FLOPS = 3.5e11                          # of an attention case
LARGEST_OWN = 64 * 1024 * 8 * 128               # elements of the own keys of an attention case


def _rows(name, kind, batch, layers, tokens, kv_heads, dim, fmt, page, ragged):
    return {"name": name, "kind": kind, "batch": batch, "layers": layers, "tokens": tokens, "kv_heads": kv_heads, "dim": dim, "format": fmt,
            "page": page, "ragged": ragged}


def _attention(name, batch, tokens, q_heads, kv_heads, dim, prefix, own_tokens, fmt, page, causal=True, masked=False):
    return {"name": name, "kind": "attention", "batch": batch, "tokens": tokens, "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim,
            "prefix": prefix, "own_tokens": own_tokens, "format": fmt, "page": page, "causal": causal, "masked": masked}


def listed():
    return [
        # one new token of four candidates in one layer: what a step pays per layer, all latency
        _rows("write-step-b4-int8", "write", 4, 1, 1, 1, 256, "int8", 64, False),
        # a prefilled observation, three cameras and a full prompt, all layers at once
        _rows("write-prefix-968-int8", "write", 1, 18, 968, 1, 256, "int8", 64, False),
        # a padded batch of long prompts, grouped heads, four layers
        _rows("write-b16-2048-e4m3", "write", 16, 4, 2048, 8, 128, "e4m3", 64, True),
        # the cache of one observation as the action chunk takes it
        _rows("read-prefix-968-int8", "read", 1, 18, 968, 1, 256, "int8", 64, False),
        # sixteen observations of up to 968 tokens for one launch of chunks
        _rows("read-b16-968-e4m3", "read", 16, 18, 968, 1, 256, "e4m3", 128, True),
        # pages of another pool, unquantised, narrow heads, an odd length
        _rows("read-b3-301-bf16", "read", 3, 5, 301, 4, 64, "bf16", 16, True),
        # a step of four candidates behind one observation
        _attention("step-b4-p968", 4, 1, 8, 1, 256, 968, 48, "bf16", 64, masked=True),
        # a step of sixteen candidates, longer texts, 8-bit cache
        _attention("step-b16-p968-int8", 16, 1, 8, 1, 256, 968, 200, "int8", 64),
        # a long history shared by an odd number of candidates, small pages
        _attention("step-b13-p30001-int8", 13, 1, 8, 1, 256, 30001, 77, "int8", 16),
        # eight action chunks sampled for one observation: 50 tokens that see each other
        _attention("chunk-b8-p968", 8, 50, 8, 1, 256, 968, 50, "bf16", 64, causal=False, masked=True),
        # a serving batch behind one system prompt, grouped heads of 128
        _attention("step-b64-p16384", 64, 1, 32, 8, 128, 16384, 1024, "bf16", 64),
        # drafted tokens checked in one pass: eight queries a sequence, grouped heads, 8-bit cache
        _attention("draft-b32-p8192-e4m3", 32, 8, 32, 8, 128, 8192, 512, "e4m3", 64),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    fmt, dim, page = rng.choice(("bf16", "int8", "e4m3")), rng.choice((64, 128, 256)), rng.choice((16, 32, 48, 64, 128))
    kv_heads = rng.choice((1, 1, 2, 4, 8))
    if rng.random() < 0.5:
        c = _rows("", rng.choice(("write", "read")), _log(rng, 1, 16), _log(rng, 1, 18), _log(rng, 1, 2048), kv_heads, dim, fmt, page, rng.random() < 0.5)
        while c["batch"] * c["layers"] * c["tokens"] * kv_heads * dim > LARGEST_ROWS:
            c["tokens"] = c["tokens"] * 2 // 3
    else:
        batch, group = _log(rng, 1, 64), rng.choice((1, 2, 4, 7, 8))
        tokens = rng.choice((1, 1, 1, 2, rng.randint(3, 16), 50))
        prefix, most = rng.choice((_log(rng, 1, 32768), _log(rng, 1, 32768), _log(rng, 1, 2048))), rng.choice((tokens, _log(rng, tokens, 1024)))
        c = _attention("", batch, tokens, group * kv_heads, kv_heads, dim, prefix, most, fmt, page, rng.random() < 0.7, rng.random() < 0.3)
        while c["batch"] > 1 and (4.0 * c["batch"] * tokens * group * kv_heads * dim * (prefix + most) > LARGEST_FLOPS / 8 or
                                  c["batch"] * most * kv_heads * dim > LARGEST_OWN):
            c["batch"] = c["batch"] * 2 // 3
    del c["name"]
    return c


def _spread(n, lo, hi):
    """n lengths from lo to hi, evenly."""
    return [lo + (hi - lo) * i // max(1, n - 1) if n > 1 else hi for i in range(n)]


def _counts(case):
    return _spread(case["batch"], case["tokens"] // 3, case["tokens"]) if case["ragged"] else [case["tokens"]] * case["batch"]


def _lengths(case):
    # own tokens, the ones that the queries belong to among them
    return _spread(case["batch"], min(case["tokens"], case["own_tokens"]), case["own_tokens"])


def _valid_count(case):
    return case["prefix"] - (case["prefix"] // 7 if case["masked"] else 0)


def _quantise(x, fmt):
    """Codes and scales of rows x [.., dim] in float32: code = x * peak / max|x|, rounded once from 64 bits."""
    amax = x.abs().amax(-1, keepdim=True)
    y = x.double() * PEAK[fmt] / amax.double()
    y = torch.where(amax > 0, y, torch.zeros_like(y))
    codes = torch.round(y).to(torch.int8) if fmt == "int8" else y.float().to(torch.float8_e4m3fn)
    return codes, (amax / PEAK[fmt]).squeeze(-1)


def _pool(g, pages, layers, page, heads, dim, fmt):
    """A pool in use: every page holds rows of some sequence, of one that is gone where no table names it."""
    out = []
    for _ in range(2):
        x = torch.randn((pages, layers, page, heads, dim), generator=g, device=DEV).to(torch.bfloat16)
        if fmt == "bf16":
            out.append((x, None))
        else:
            codes, scale = _quantise(x.float(), fmt)
            out.append((codes, scale.transpose(2, 3).contiguous()))       # scales: [pages, layers, heads, page]
    return out


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    b, page, fmt, heads, dim = case["batch"], case["page"], case["format"], case["kv_heads"], case["dim"]
    deal = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)[torch.randperm(len(v), generator=g, device=DEV)]
    s = dict(case)
    if case["kind"] == "attention":
        t, p_pages, o_pages = case["tokens"], -(-case["prefix"] // page), -(-case["own_tokens"] // page)
        layers = 2
        pages = 1 + p_pages + b * o_pages
        order = 1 + torch.randperm(pages - 1, generator=g, device=DEV).to(torch.int32)
        s["prefix_table"], s["table"] = order[:p_pages].contiguous(), order[p_pages:].view(b, o_pages).contiguous()
        s["lengths"] = deal(_lengths(case))
        s["q"] = (2 * torch.randn((b, t, case["q_heads"], dim), generator=g, device=DEV)).to(torch.bfloat16)
        s["valid"] = None
        if case["masked"]:
            s["valid"] = torch.zeros(case["prefix"], dtype=torch.bool, device=DEV)
            s["valid"][torch.randperm(case["prefix"], generator=g, device=DEV)[:_valid_count(case)]] = True
        (s["k"], s["k_scale"]), (s["v"], s["v_scale"]) = _pool(g, pages, layers, page, heads, dim, fmt)
    else:
        layers, t = case["layers"], case["tokens"]
        per = -(-t // page)
        pages = 1 + b * per
        s["table"] = (1 + torch.randperm(pages - 1, generator=g, device=DEV).to(torch.int32)).view(b, per).contiguous()
        s["counts"] = deal(_counts(case)) if case["ragged"] else None
        if case["kind"] == "write":
            s["new_k"], s["new_v"] = (torch.randn((b, layers, t, heads, dim), generator=g, device=DEV).to(torch.bfloat16) for _ in range(2))
            for n in ("k", "v"):
                s[n] = torch.zeros((pages, layers, page, heads, dim), dtype=STORED[fmt], device=DEV)
                s[n + "_scale"] = None if fmt == "bf16" else torch.zeros((pages, layers, heads, page), device=DEV)
        else:
            (s["k"], s["k_scale"]), (s["v"], s["v_scale"]) = _pool(g, pages, layers, page, heads, dim, fmt)
    if own:
        from pi05_megakernel_b200.cache import KvCache
        s["cache"] = KvCache.wrap(s["k"], s["v"], s["k_scale"], s["v_scale"])
        if case["kind"] == "attention":
            from pi05_megakernel_b200.shared import SharedPrefixAttention
            s["op"] = SharedPrefixAttention(s["cache"], q_heads=case["q_heads"], max_batch=b, max_tokens=case["tokens"])
    return s


def _places(s):
    """Page and place in the page of token t of sequence b: [batch, tokens] each, and whether the sequence has that token."""
    t = torch.arange(s["tokens"], device=DEV)
    pages = s["table"].long()[:, t // s["page"]]
    has = torch.ones_like(pages, dtype=torch.bool) if s["counts"] is None else t[None] < s["counts"][:, None]
    return pages, (t % s["page"])[None].expand_as(pages), has


def _write(s):
    pages, at, has = _places(s)
    pages = torch.where(has, pages, torch.zeros_like(pages))             # a token that a sequence lacks: into the spare page
    for n in ("k", "v"):
        rows = s["new_" + n].transpose(1, 2)                              # [batch, tokens, layers, heads, dim]
        if s["format"] == "bf16":
            s[n].view(torch.int16)[pages, :, at] = rows.view(torch.int16)
        else:
            codes, scale = _quantise(rows.float(), s["format"])
            s[n].view(torch.int8)[pages, :, at] = codes.view(torch.int8)
            s[n + "_scale"].transpose(2, 3)[pages, :, at] = scale


def _values(s, n, pages, at, layers=slice(None)):
    """Rows of the pool in float32: [.., layers, heads, dim] for pages and places of any shape."""
    rows = s[n].view(torch.int8 if s["format"] != "bf16" else torch.int16)[pages, layers, at].view(STORED[s["format"]]).float()
    return rows if s["format"] == "bf16" else rows * s[n + "_scale"].transpose(2, 3)[pages, layers, at][..., None]


def _read(s):
    pages, at, has = _places(s)
    out = []
    for n in ("k", "v"):
        rows = _values(s, n, pages, at)
        out.append(torch.where(has[..., None, None, None], rows, torch.zeros_like(rows)).transpose(1, 2).to(torch.bfloat16).contiguous())
    return out


def _attend(s):
    b, t, hq, h, d, page = s["batch"], s["tokens"], s["q_heads"], s["kv_heads"], s["dim"], s["page"]
    at = torch.arange(s["prefix"], device=DEV)
    pp, pa = s["prefix_table"].long()[at // page], at % page
    j = torch.arange(s["own_tokens"], device=DEV)
    op, oa = s["table"].long()[:, j // page], (j % page)[None].expand(b, -1)
    q = s["q"].float().view(b, t, h, hq // h, d)
    kp, vp = (_values(s, n, pp, pa, 1) for n in ("k", "v"))               # [prefix, heads, dim]
    ko, vo = (_values(s, n, op, oa, 1) for n in ("k", "v"))               # [batch, own, heads, dim]
    x = torch.cat((torch.einsum("bthgd,phd->bthgp", q, kp), torch.einsum("bthgd,bnhd->bthgn", q, ko)), -1) * d ** -0.5
    last = s["lengths"].long()[:, None] - (t - 1 - torch.arange(t, device=DEV) if s["causal"] else torch.zeros(t, dtype=torch.int64, device=DEV))
    sees = (j < last[..., None])[:, :, None, None]                        # [batch, tokens, 1, 1, own]
    shared = torch.ones(s["prefix"], dtype=torch.bool, device=DEV) if s["valid"] is None else s["valid"]
    sees = torch.cat((shared.expand(*sees.shape[:-1], -1), sees), -1)
    x = torch.where(sees, x, torch.full_like(x, -math.inf))
    top = x.amax(-1, keepdim=True)
    e = torch.exp(x - torch.where(top > -math.inf, top, torch.zeros_like(top)))
    total = e.sum(-1, keepdim=True)
    p = e / torch.where(total > 0, total, torch.ones_like(total))
    o = torch.einsum("bthgp,phd->bthgd", p[..., :s["prefix"]], vp) + torch.einsum("bthgn,bnhd->bthgd", p[..., s["prefix"]:], vo)
    return [o.reshape(b, t, hq, d).to(torch.bfloat16), (top + torch.log(total)).reshape(b, t, hq)]


def run(state):
    s = state
    if s["kind"] == "write":
        if own:
            s["cache"].write(s["new_k"], s["new_v"], s["table"], counts=s["counts"])
        else:
            _write(s)
        # what the pages hold now: codes are compared as they are, scales beside them (the spare page is nobody's)
        return [s["k"][1:], s["v"][1:]] + ([] if s["format"] == "bf16" else [s["k_scale"][1:], s["v_scale"][1:]])
    if s["kind"] == "read":
        return list(s["cache"].read(s["table"], s["tokens"], counts=s["counts"])) if own else _read(s)
    if own:
        return list(s["op"].run(s["q"], s["prefix_table"], s["prefix"], s["table"], s["lengths"], layer=1, valid=s["valid"], causal=s["causal"],
                                with_lse=True))
    return _attend(s)


def work(case):
    stored = case["dim"] * (2 if case["format"] == "bf16" else 1) + (0 if case["format"] == "bf16" else 4)      # a key's row
    if case["kind"] != "attention":
        rows = 2 * sum(_counts(case)) * case["layers"] * case["kv_heads"]
        written = rows if case["kind"] == "write" else 2 * case["batch"] * case["tokens"] * case["layers"] * case["kv_heads"]
        return {"bytes": rows * stored + written * case["dim"] * 2, "flops": 0}
    b, t, hq = case["batch"], case["tokens"], case["q_heads"]
    keys = _valid_count(case) + sum(_lengths(case))
    pairs = b * t * _valid_count(case)
    for n in _lengths(case):
        pairs += sum(max(0, n - (t - 1 - i)) for i in range(t)) if case["causal"] else n * t
    return {"bytes": 2 * keys * case["kv_heads"] * stored + b * t * hq * (4 * case["dim"] + 4), "flops": 4 * hq * case["dim"] * pairs}


# ------------------------------------------------------------------------------------------------ from the definitions, in 64 bits
def _nearest_e4m3(y):
    """The e4m3 value nearest to y, the one with an even last bit from the middle."""
    codes = torch.arange(127, dtype=torch.float64, device=y.device)
    e, m = torch.div(codes, 8, rounding_mode="floor"), codes % 8
    grid = torch.where(e == 0, m * 2.0 ** -9, (8 + m) * torch.exp2(e - 10))
    a = y.abs()
    hi = torch.bucketize(a, grid).clamp(1, 126)                           # grid[hi - 1] < a <= grid[hi]
    up, down = grid[hi] - a, a - grid[hi - 1]
    take = torch.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, hi - 1)
    return torch.copysign(grid[take], y)


def exact(case, seed):
    s = prepare(case, seed)
    b, t, h, d, page, fmt = case["batch"], case["tokens"], case["kv_heads"], case["dim"], case["page"], case["format"]
    if case["kind"] == "write":
        out, scales = [], []
        count = [t] * b if s["counts"] is None else s["counts"].tolist()
        for n in ("k", "v"):
            rows = s["new_" + n].double()
            if fmt != "bf16":
                a = rows.abs().amax(-1, keepdim=True)
                y = torch.where(a > 0, rows / torch.where(a > 0, a, torch.ones_like(a)) * PEAK[fmt], torch.zeros_like(rows))
                # a quotient that is a middle in the definition is one here too: x / a * peak is off it by an ulp of 64 bits
                y = torch.round(y * 2.0 ** 40) * 2.0 ** -40
                pool = torch.zeros(s[n].shape, dtype=torch.float64, device=DEV)
                scale = torch.zeros(s[n + "_scale"].shape, dtype=torch.float64, device=DEV)
                rows = torch.round(y) if fmt == "int8" else _nearest_e4m3(y)
            else:
                pool = torch.zeros(s[n].shape, dtype=torch.float64, device=DEV)
            for i in range(b):
                for first in range(0, count[i], page):
                    k, p = min(page, count[i] - first), int(s["table"][i, first // page])
                    pool[p, :, :k] = rows[i, :, first:first + k]
                    if fmt != "bf16":
                        scale[p, :, :, :k] = (a[i, :, first:first + k, :, 0] / PEAK[fmt]).transpose(1, 2)
            out.append(pool[1:].to(torch.int8) if fmt == "int8" else pool[1:])
            if fmt != "bf16":
                scales.append(scale[1:])
        return out + scales

    def value(n, p, layers):
        v = s[n][p, layers].double()
        return v if fmt == "bf16" else v * s[n + "_scale"][p, layers].double().transpose(-1, -2)[..., None]

    if case["kind"] == "read":
        out = []
        count = [t] * b if s["counts"] is None else s["counts"].tolist()
        for n in ("k", "v"):
            o = torch.zeros((b, case["layers"], t, h, d), dtype=torch.float64, device=DEV)
            for i in range(b):
                for first in range(0, count[i], page):
                    k = min(page, count[i] - first)
                    o[i, :, first:first + k] = value(n, int(s["table"][i, first // page]), slice(None))[:, :k]
            out.append(o)
        return out

    g = case["q_heads"] // h
    o = torch.zeros((b, t, case["q_heads"], d), dtype=torch.float64, device=DEV)
    lse = torch.full((b, t, case["q_heads"]), -math.inf, dtype=torch.float64, device=DEV)
    flat = lambda n, pages, length: torch.cat([value(n, int(p), 1) for p in pages.tolist()], 0)[:length] if length else torch.zeros((0, h, d), dtype=torch.float64, device=DEV)
    kp, vp = flat("k", s["prefix_table"], case["prefix"]), flat("v", s["prefix_table"], case["prefix"])
    if s["valid"] is not None:
        kp, vp = kp[s["valid"]], vp[s["valid"]]
    for i, length in enumerate(s["lengths"].tolist()):
        ko, vo = flat("k", s["table"][i], length), flat("v", s["table"][i], length)
        for c in range(h):
            q = s["q"][i, :, c * g:(c + 1) * g].double().reshape(t * g, d)
            x = torch.cat((q @ kp[:, c].T, q @ ko[:, c].T), 1) / math.sqrt(d)
            if case["causal"]:
                late = torch.arange(length, device=DEV)[None] > length - t + torch.arange(t, device=DEV)[:, None]
                x[:, kp.shape[0]:][late.repeat_interleave(g, 0)] = -math.inf
            if x.shape[1] == 0:
                continue
            z = torch.logsumexp(x, 1)
            p = torch.where(z[:, None] > -math.inf, torch.exp(x - z[:, None]), torch.zeros_like(x))
            o[i, :, c * g:(c + 1) * g] = (p[:, :kp.shape[0]] @ vp[:, c] + p[:, kp.shape[0]:] @ vo[:, c]).view(t, g, d)
            lse[i, :, c * g:(c + 1) * g] = z.view(t, g)
    return [o, lse]

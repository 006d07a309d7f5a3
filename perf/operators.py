"""The operators of serving many edit requests at once, as measurable cases.

Four operators, each in a plain form (elementary torch operations in fp32) and
as the framework's kernels:

* store: K/V rows quantised to INT8 (one scale per token and head) as they are
  written into a request's prefix cache, and the written rows read back;
* read: cached rows back to bf16 (what an attention over bf16 K/V consumes);
* attend: queries over [quantised cached prefix, fresh bf16 tokens], with
  per-request lengths, a key mask and shared K/V heads;
* adapt: low-rank adapters, one per request, beside a shared projection.
"""
import math
import sys

import torch

own = False
D = 128   # head dimension of every attention in this framework


def _api():
    if "qwen-image-2.1-accel_b200" not in sys.path:
        sys.path.insert(0, "qwen-image-2.1-accel_b200")
    from qwen_image_accel_b200.kernels import kv_cache, lora
    return kv_cache, lora


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # sixteen requests add one token each to their caches
        {"name": "store one token", "op": "store", "requests": 16, "tokens": 1, "kv_heads": 32, "capacity": 4608,
         "start": 4229},
        # the prefix of two edit requests (four condition images and their text) after its prefill, one layer
        {"name": "store two prefixes", "op": "store", "requests": 2, "tokens": 8325, "kv_heads": 32, "capacity": 8448,
         "start": 0},
        # a text-only prefix ahead of the quantised attention of one decode step
        {"name": "read a text prefix", "op": "read", "requests": 1, "tokens": 333, "kv_heads": 32, "capacity": 512,
         "ragged": False},
        # one condition image each for four requests whose prompts differ in length
        {"name": "read four prefixes", "op": "read", "requests": 4, "tokens": 4229, "kv_heads": 32, "capacity": 4608,
         "ragged": True},
        # one new token of one request against its prefix: the latency case
        {"name": "attend one token", "op": "attend", "requests": 1, "queries": 1, "fresh": 1, "cached": 4229,
         "heads": 32, "kv_heads": 32, "ragged": False, "masked": False},
        # one new token each of sixteen requests with long prefixes and shared K/V heads: the cache's bytes count
        {"name": "attend long prefixes", "op": "attend", "requests": 16, "queries": 1, "fresh": 1, "cached": 16391,
         "heads": 32, "kv_heads": 8, "ragged": True, "masked": False},
        # a block of prompt tokens for four requests, padded prompts masked
        {"name": "attend a text block", "op": "attend", "requests": 4, "queries": 77, "fresh": 77, "cached": 1111,
         "heads": 32, "kv_heads": 32, "ragged": True, "masked": True},
        # the target tokens of two 512x512 images in one denoising step, one layer, padded prompts masked
        {"name": "attend 512x512 targets", "op": "attend", "requests": 2, "queries": 1024, "fresh": 1024,
         "cached": 1357, "heads": 32, "kv_heads": 32, "ragged": False, "masked": True},
        # the target tokens of one 1024x1024 image over one condition image of that size
        {"name": "attend a 1024x1024 target", "op": "attend", "requests": 1, "queries": 4096, "fresh": 4096,
         "cached": 4229, "heads": 32, "kv_heads": 32, "ragged": False, "masked": False},
        # one token each of 32 requests through the output projection, eight adapters and none in use
        {"name": "adapt one token", "op": "adapt", "requests": 32, "tokens": 1, "width": 4096, "out": 4096,
         "adapters": 8, "rank": 64},
        # the prompt rows of four requests through the down projection
        {"name": "adapt text rows", "op": "adapt", "requests": 4, "tokens": 77, "width": 12288, "out": 4096,
         "adapters": 4, "rank": 16},
        # the target tokens of four 1024x1024 images through the stacked q|k|v projection
        {"name": "adapt image rows", "op": "adapt", "requests": 4, "tokens": 4096, "width": 4096, "out": 12288,
         "adapters": 4, "rank": 64},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["store", "read", "attend", "attend", "attend", "adapt", "adapt"])
    if op in ("store", "read"):
        kvh = rng.choice([4, 8, 24, 32])
        req = _log(rng, 1, 16)
        tokens = _log(rng, 1, max(1, 2 * 8325 * 32 // (req * kvh)) if req * kvh * 20000 > 2 * 8325 * 32 else 20000)
        start = 0 if op == "read" else rng.choice([0, _log(rng, 1, 3000)])
        case = {"op": op, "requests": req, "tokens": tokens, "kv_heads": kvh,
                "capacity": start + tokens + rng.choice([0, 1, 127])}
        case.update({"start": start} if op == "store" else {"ragged": rng.random() < 0.5})
        return case
    if op == "attend":
        heads, kvh = rng.choice([(32, 32), (32, 32), (24, 24), (32, 8), (16, 4), (12, 4), (8, 1)])
        req = _log(rng, 1, 16)
        queries = _log(rng, 1, 4096) if rng.random() < 0.7 else 1
        most = 4096 * 8325 * 32 // (req * queries * heads)         # no more products than the largest listed case
        cached = _log(rng, 1, max(1, min(20000, most, 16 * 16391 * 8 // (req * kvh))))
        fresh = rng.choice([queries, queries, 0, 1])
        if req * queries * heads * (cached + fresh) > 4096 * 8325 * 32:
            req, fresh = 1, min(fresh, 1)
        return {"op": op, "requests": req, "queries": queries, "fresh": fresh, "cached": cached, "heads": heads,
                "kv_heads": kvh, "ragged": rng.random() < 0.5, "masked": rng.random() < 0.5}
    width, out = rng.choice([(4096, 4096), (4096, 12288), (12288, 4096), (64, 4096), (4096, 64), (1000, 2056)])
    req = _log(rng, 1, 64)
    tokens = _log(rng, 1, max(1, min(16384, 16384 // req)))
    return {"op": op, "requests": req, "tokens": tokens, "width": width, "out": out, "adapters": _log(rng, 1, 16),
            "rank": _log(rng, 1, 128)}


# ------------------------------------------------------------------ what a case fixes beside its sizes
def _lengths(c, cached):
    """Tokens held per request: all alike, or down to half of the longest."""
    n = c["requests"]
    return [cached - (b * cached) // (2 * n) if c["ragged"] else cached for b in range(n)]


def _ranks(c):
    return [max(1, c["rank"] >> (i % 3)) for i in range(c["adapters"])]


def _ids(c):
    """One adapter per request; one request in (adapters + 1) has none."""
    return [(5 * b + 1) % (c["adapters"] + 1) - 1 for b in range(c["requests"])]


# ------------------------------------------------------------------ inputs
def _rows(g, *shape):
    """K/V rows: unit channels with a few large ones, token norms that vary."""
    x = torch.randn(*shape, device="cuda", generator=g)
    x = x * (0.5 + torch.rand(*shape[:-1], 1, device="cuda", generator=g))
    x[..., 5::37] *= 4
    return x.to(torch.bfloat16)


def _filled_cache(g, c, cached, capacity):
    """A cache as earlier calls left it: codes and scales of `cached` tokens."""
    shape = (c["requests"], c["kv_heads"], capacity)
    s = {"lengths": torch.tensor(_lengths(c, cached), dtype=torch.int32, device="cuda")}
    for t in "kv":
        codes = torch.randn(*shape, D, device="cuda", generator=g).mul_(42).round_().clamp_(-127, 127)
        s[t + "_codes"] = codes.to(torch.int8)
        s[t + "_scales"] = (0.015 + 0.015 * torch.rand(*shape, device="cuda", generator=g))
        del codes
    return s


def _inputs(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n = c["requests"]
    if c["op"] == "store":
        # views of a joint sequence that is longer than what is stored, as the prefill holds it
        joint = c["tokens"] + 64
        shape = (n, c["kv_heads"], c["capacity"])
        s = {t: _rows(g, n, joint, c["kv_heads"], D)[:, :c["tokens"]] for t in "kv"}
        for t in "kv":
            s[t + "_codes"] = torch.zeros(*shape, D, dtype=torch.int8, device="cuda")
            s[t + "_scales"] = torch.zeros(*shape, device="cuda")
        s["lengths"] = torch.full((n,), c["start"], dtype=torch.int32, device="cuda")
        return s
    if c["op"] == "read":
        return _filled_cache(g, c, c["tokens"], c["capacity"])
    if c["op"] == "attend":
        s = _filled_cache(g, c, c["cached"], c["cached"] + 59)
        s["q"] = (1.2 * torch.randn(n, c["queries"], c["heads"], D, device="cuda", generator=g)).to(torch.bfloat16)
        s["k"] = s["v"] = s["key_valid"] = None
        if c["fresh"]:
            s["k"], s["v"] = (_rows(g, n, c["fresh"], c["kv_heads"], D) for _ in range(2))
        if c["masked"]:
            s["key_valid"] = torch.rand(n, c["cached"] + c["fresh"], device="cuda", generator=g) < 0.9
        return s
    r = c["rank"]
    s = {"x": torch.randn(n, c["tokens"], c["width"], device="cuda", generator=g).to(torch.bfloat16),
         "base": torch.randn(n, c["tokens"], c["out"], device="cuda", generator=g).to(torch.bfloat16),
         "a": torch.randn(c["adapters"], r, c["width"], device="cuda", generator=g) / math.sqrt(c["width"]),
         "b": torch.randn(c["adapters"], c["out"], r, device="cuda", generator=g) * 0.3,
         "scales": 0.5 + torch.rand(c["adapters"], device="cuda", generator=g),
         "ids": torch.tensor(_ids(c), dtype=torch.int32, device="cuda")}
    used = torch.arange(r, device="cuda") < torch.tensor(_ranks(c), device="cuda")[:, None]
    s["a"] = (s["a"] * used[:, :, None]).to(torch.bfloat16)
    s["b"] = (s["b"] * used[:, None, :]).to(torch.bfloat16)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if own:
        # the handles that a server keeps: a layer's cache around its tensors, the adapters of a projection
        kv_cache, lora = _api()
        if case["op"] == "adapt":
            s["weights"] = lora.LoraWeights([(s["a"][i, :r], s["b"][i, :, :r], float(s["scales"][i]))
                                             for i, r in enumerate(_ranks(case))])
        else:
            extent = {"store": case.get("start"), "read": case.get("tokens"), "attend": case.get("cached")}[case["op"]]
            s["cache"] = kv_cache.QuantizedKV.from_tensors(s["k_codes"], s["v_codes"], s["k_scales"], s["v_scales"],
                                                           s["lengths"], extent)
    return s


# ------------------------------------------------------------------ one pass
def run(s):
    c = s["case"]
    return (_run_own if own else _run_plain)(c["op"], c, s)


def _run_own(op, c, s):
    kv_cache, lora = _api()
    if op == "store":
        kv_cache.kv_cache_write(s["cache"], s["k"], s["v"], start=c["start"])
        k, v = kv_cache.kv_cache_read(s["cache"], first=c["start"], tokens=c["tokens"])
        w = slice(c["start"], c["start"] + c["tokens"])
        return {"k": k, "v": v, "k_scales": s["k_scales"][:, :, w], "v_scales": s["v_scales"][:, :, w],
                "lengths": s["lengths"]}
    if op == "read":
        k, v = kv_cache.kv_cache_read(s["cache"], tokens=c["tokens"])
        return {"k": k, "v": v}
    if op == "attend":
        return kv_cache.cached_attention(s["q"], s["cache"], s["k"], s["v"], key_valid=s["key_valid"])
    return lora.lora_add(s["x"], s["base"], s["weights"], s["ids"])


def _read_back(codes, scales, lengths, first, n):
    """Rows [first, first + n) as bf16 [requests, n, heads, 128]; zeros past a request's length."""
    w = slice(first, first + n)
    x = codes[:, :, w].float() * scales[:, :, w, None]
    held = torch.arange(first, first + n, device=x.device) < lengths[:, None]
    return torch.where(held[:, None, :, None], x, 0.0).to(torch.bfloat16).transpose(1, 2)


def _run_plain(op, c, s):
    if op == "store":
        w = slice(c["start"], c["start"] + c["tokens"])
        s["lengths"].fill_(c["start"] + c["tokens"])
        for t in "kv":
            x = s[t].float().transpose(1, 2)
            amax = x.abs().amax(-1)
            inverse = torch.where(amax > 0, 127.0 / amax, 0.0)
            s[t + "_codes"][:, :, w] = (x * inverse[..., None]).round().clamp(-127, 127).to(torch.int8)
            s[t + "_scales"][:, :, w] = amax / 127.0
        return {"k": _read_back(s["k_codes"], s["k_scales"], s["lengths"], c["start"], c["tokens"]),
                "v": _read_back(s["v_codes"], s["v_scales"], s["lengths"], c["start"], c["tokens"]),
                "k_scales": s["k_scales"][:, :, w], "v_scales": s["v_scales"][:, :, w], "lengths": s["lengths"]}
    if op == "read":
        return {t: _read_back(s[t + "_codes"], s[t + "_scales"], s["lengths"], 0, c["tokens"]) for t in "kv"}
    if op == "attend":
        n, sq, h, kvh, p = c["requests"], c["queries"], c["heads"], c["kv_heads"], c["cached"]
        valid = torch.arange(p, device="cuda") < s["lengths"][:, None]
        k, v = (s[t + "_codes"][:, :, :p].float() * s[t + "_scales"][:, :, :p, None] for t in "kv")
        if c["fresh"]:
            valid = torch.cat([valid, valid.new_ones(n, c["fresh"])], 1)
            k, v = (torch.cat([x, s[t].float().transpose(1, 2)], 2) for x, t in ((k, "k"), (v, "v")))
        if s["key_valid"] is not None:
            valid = valid & s["key_valid"]
        q = s["q"].float().view(n, sq, kvh, h // kvh, D).permute(0, 2, 3, 1, 4).reshape(n, kvh, -1, D)
        score = (q @ k.transpose(2, 3)).mul_(D ** -0.5).masked_fill_(~valid[:, None, None, :], -math.inf)
        top = score.amax(-1, keepdim=True).clamp_(min=-1e30)
        weight = score.sub_(top).exp_()
        total = weight.sum(-1, keepdim=True)
        o = (weight @ v) / torch.where(total > 0, total, 1.0)
        return o.view(n, kvh, h // kvh, sq, D).permute(0, 3, 1, 2, 4).reshape(n, sq, h, D).to(torch.bfloat16)
    ids = s["ids"].long()
    at = ids.clamp(min=0)
    scale = torch.where(ids >= 0, s["scales"][at], 0.0)
    low = s["x"].float() @ s["a"][at].float().transpose(1, 2)
    return (s["base"].float() + (low * scale[:, None, None]) @ s["b"][at].float().transpose(1, 2)).to(torch.bfloat16)


# ------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    c = case
    s = _inputs(case, seed)
    if c["op"] == "store":
        got = {"lengths": None}
        for t in "kv":
            x = s[t].double()
            step = x.abs().max(dim=-1).values / 127
            codes = torch.round(x / torch.where(step > 0, step, torch.ones_like(step))[..., None])
            got[t] = codes * step[..., None]
            got[t + "_scales"] = step.permute(0, 2, 1)
        return got
    if c["op"] == "read":
        got = {}
        for t in "kv":
            x = torch.einsum("bhsd,bhs->bshd", s[t + "_codes"].double(), s[t + "_scales"].double())[:, :c["tokens"]]
            for b, held in enumerate(_lengths(c, c["tokens"])):
                x[b, held:] = 0
            got[t] = x
        return got
    if c["op"] == "attend":
        if c["requests"] * c["queries"] * c["heads"] * (c["cached"] + c["fresh"]) > 6e8:
            return None                                    # minutes of fp64 products
        out = torch.zeros(c["requests"], c["queries"], c["heads"], D, dtype=torch.float64, device="cuda")
        share = c["heads"] // c["kv_heads"]
        for b, held in enumerate(_lengths(c, c["cached"])):
            for h in range(c["kv_heads"]):
                part = {}
                for t in "kv":
                    x = s[t + "_codes"][b, h, :held].double() * s[t + "_scales"][b, h, :held].double()[:, None]
                    part[t] = torch.cat([x, s[t][b, :, h].double()]) if c["fresh"] else x
                if c["masked"]:
                    keep = torch.cat([s["key_valid"][b, :held], s["key_valid"][b, c["cached"]:]])
                    part = {t: x[keep] for t, x in part.items()}
                if not part["k"].shape[0]:
                    continue
                q = s["q"][b, :, h * share:(h + 1) * share].double()
                weight = torch.softmax(torch.einsum("qgd,kd->qgk", q, part["k"]) / math.sqrt(D), dim=-1)
                out[b, :, h * share:(h + 1) * share] = torch.einsum("qgk,kd->qgd", weight, part["v"])
        return out
    y = s["base"].double()
    for b, i in enumerate(_ids(c)):
        if i >= 0:
            low = torch.einsum("sw,rw->sr", s["x"][b].double(), s["a"][i].double())
            y[b] += s["scales"][i].double() * torch.einsum("sr,or->so", low, s["b"][i].double())
    return y


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    c = case
    n = c["requests"]
    if c["op"] == "store":
        rows = 2 * n * c["tokens"] * c["kv_heads"]
        # bf16 rows in, codes and scales out; codes and scales in, bf16 rows out
        return {"bytes": rows * (2 * D + (D + 4) + (D + 4) + 2 * D), "flops": rows * D * 5}
    if c["op"] == "read":
        held = 2 * sum(_lengths(c, c["tokens"])) * c["kv_heads"]
        return {"bytes": held * (D + 4) + 2 * n * c["tokens"] * c["kv_heads"] * 2 * D, "flops": held * D}
    if c["op"] == "attend":
        held = sum(_lengths(c, c["cached"]))
        keys = held + n * c["fresh"]
        size = 2 * 2 * n * c["queries"] * c["heads"] * D                       # q in, out
        size += 2 * c["kv_heads"] * (held * (D + 4) + n * c["fresh"] * 2 * D)   # the cache, the fresh rows
        size += n * (c["cached"] + c["fresh"]) if c["masked"] else 0
        return {"bytes": size, "flops": 4 * c["queries"] * c["heads"] * D * keys}
    ranks, ids = _ranks(c), _ids(c)
    size = 2 * n * c["tokens"] * 2 * c["out"]
    size += sum(2 * c["tokens"] * c["width"] for i in ids if i >= 0)
    size += sum(2 * ranks[i] * (c["width"] + c["out"]) for i in set(ids) if i >= 0)
    return {"bytes": size, "flops": sum(2 * c["tokens"] * ranks[i] * (c["width"] + c["out"]) for i in ids if i >= 0)}

"""What stands between a model's projections when several contexts decode
together: rotary positions, the paged cache of keys and values, the attention
that reads it, and the moves of its pages.

Each case is one pass through the package's public entry points (`own` true)
or through the same mathematics in elementary torch operations (`own` false).
The families:

  rope    rope: positions applied to (or, inverse, the gradient taken back
          through) every head of a batch of tokens
  append  cache_append: the new tokens' q and k rotated, k and v written to
          their pages
  attend  paged_attention: chunks of new tokens over the cached ones
  pages   cache_fork, cache_reserve and cache_release of contexts that share a
          prompt; cache_compact of a scattered cache
"""
import importlib.util
import math
import os
import sys

import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _package():
    """The package of the working folder (its folder's name is no identifier)."""
    if "nimllm_amd" not in sys.modules:
        root = os.path.join(os.getcwd(), "nim.llm_amd")
        spec = importlib.util.spec_from_file_location(
            "nimllm_amd", os.path.join(root, "__init__.py"), submodule_search_locations=[root])
        mod = importlib.util.module_from_spec(spec)
        sys.modules["nimllm_amd"] = mod
        spec.loader.exec_module(mod)
    return sys.modules["nimllm_amd"]


# ---------------------------------------------------------------- the cases


def listed():
    return [
        # one decoded token's queries, a width of 2048 in 32 heads: the smallest call
        {"name": "rope_one_token", "family": "rope", "tokens": 1, "heads": 32, "dim": 64, "rot": 64, "type": "f32",
         "layout": "interleaved", "scaling": "factors", "far": 8000, "inverse": False},
        # the gradient of a long batch's queries, part of each head, far positions
        {"name": "rope_gradient_8191", "family": "rope", "tokens": 8191, "heads": 32, "dim": 128, "rot": 96,
         "type": "bf16", "layout": "half", "scaling": "yarn", "far": 1000000, "inverse": True},
        # one token each of a small serving batch, fp32 projections, fp16 cache
        {"name": "append_24_tokens", "family": "append", "seqs": 24, "new": 1, "ctx": 4000, "heads": 32, "kv": 8,
         "dim": 128, "rot": 128, "page": 16, "type": "f32", "cache": "f16", "layout": "half", "scaling": "none"},
        # the prompts of three contexts, ragged
        {"name": "append_prompts", "family": "append", "seqs": 3, "new": 2777, "ctx": 2777, "heads": 32, "kv": 8,
         "dim": 128, "rot": 128, "page": 64, "type": "bf16", "cache": "bf16", "layout": "interleaved",
         "scaling": "linear"},
        # one chat context, the reference's own fp32 cache: latency
        {"name": "attend_chat_517", "family": "attend", "seqs": 1, "new": 1, "ctx": 517, "heads": 32, "kv": 8, "dim": 64,
         "page": 16, "type": "f32", "cache": "f32", "window": 0},
        # one token of one long context: few rows, a long axis
        {"name": "attend_long_131071", "family": "attend", "seqs": 1, "new": 1, "ctx": 131071, "heads": 32, "kv": 8,
         "dim": 128, "page": 64, "type": "f32", "cache": "f16", "window": 0},
        # a serving batch of ragged contexts, one token each
        {"name": "attend_64x16k", "family": "attend", "seqs": 64, "new": 1, "ctx": 16384, "heads": 32, "kv": 8,
         "dim": 128, "page": 16, "type": "bf16", "cache": "bf16", "window": 0},
        # a chunk of a long prompt, fp32 queries over an fp16 cache
        {"name": "attend_chunk_2048x16k", "family": "attend", "seqs": 1, "new": 2048, "ctx": 16384, "heads": 32, "kv": 8,
         "dim": 128, "page": 64, "type": "f32", "cache": "f16", "window": 0},
        # whole prompts from the start, 16-bit throughout
        {"name": "attend_prompts_2x4001", "family": "attend", "seqs": 2, "new": 4001, "ctx": 4001, "heads": 32, "kv": 8,
         "dim": 64, "page": 32, "type": "bf16", "cache": "bf16", "window": 0},
        # a mixed batch: one context reads its prompt while the others decode, a sliding window
        {"name": "attend_mixed_window", "family": "attend", "seqs": 17, "new": 509, "ctx": 8000, "heads": 28, "kv": 4,
         "dim": 128, "page": 16, "type": "f32", "cache": "bf16", "window": 4096, "mixed": True},
        # 48 continuations of one prompt begin, take their next tokens and end
        {"name": "pages_fork_48", "family": "pages", "op": "fork", "layers": 16, "pages": 4096, "page": 16, "kv": 8,
         "dim": 64, "seqs": 64, "ctx": 1003, "cache": "f16", "count": 48},
        # a scattered cache moved together
        {"name": "pages_compact_8192", "family": "pages", "op": "compact", "layers": 16, "pages": 8192, "page": 32,
         "kv": 8, "dim": 128, "seqs": 48, "ctx": 4000, "cache": "bf16", "count": 0},
    ]


def _spread(rng, lo, hi):
    """A whole number, even in its logarithm over lo .. hi."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    family = rng.choice(["rope", "append", "attend", "attend", "attend", "pages"])
    c = {"family": family}
    heads, kv = rng.choice([(32, 8), (32, 32), (16, 8), (28, 4), (14, 2), (8, 1), (40, 8), (9, 3)])
    if family == "rope":
        dim = rng.choice([64, 80, 96, 128, 256])
        c.update(tokens=_spread(rng, 1, 8191), heads=heads, dim=dim, rot=rng.choice([dim, dim // 2, dim // 4 * 2 - 2]),
                 type=rng.choice(["f32", "f16", "bf16"]), layout=rng.choice(["interleaved", "half"]),
                 scaling=rng.choice(["none", "linear", "factors", "yarn"]), far=_spread(rng, 100, 1000000),
                 inverse=rng.random() < 0.5)
        c["tokens"] = min(c["tokens"], 8191 * 32 * 128 // (heads * dim))
        return c
    c.update(heads=heads, kv=kv, dim=rng.choice([64, 64, 80, 96, 128, 128, 128, 256]),
             page=rng.choice([8, 16, 16, 32, 64, 256]))
    if family == "pages":
        c.pop("heads")
        c.update(op=rng.choice(["fork", "compact"]), layers=_spread(rng, 1, 32), seqs=_spread(rng, 2, 64),
                 ctx=_spread(rng, 1, 4000), cache=rng.choice(["f32", "f16", "bf16"]))
        c["count"] = rng.randrange(0, c["seqs"]) if c["op"] == "fork" else 0
        size = 2 if c["cache"] != "f32" else 4
        most = 8192 * 32 * 8 * 128 * 16 * 2 // (c["layers"] * c["page"] * c["kv"] * c["dim"] * size)
        c["ctx"] = max(1, min(c["ctx"], most // (2 * c["seqs"]) * c["page"]))
        c["pages"] = 2 * c["seqs"] * (-(-c["ctx"] // c["page"]) + 2) + rng.randrange(64)
        return c
    t = rng.choice(["f32", "f32", "f16", "bf16"])
    c.update(type=t, cache=rng.choice(["f32", "f16", "bf16"]) if t == "f32" else t)
    if family == "append":
        c.update(seqs=_spread(rng, 1, 64), new=_spread(rng, 1, 2777), layout=rng.choice(["interleaved", "half"]),
                 rot=rng.choice([c["dim"], c["dim"] // 2]), scaling=rng.choice(["none", "linear", "factors", "yarn"]))
        c["new"] = max(1, min(c["new"], 3 * 2777 * 48 * 128 // (c["seqs"] * (heads + 2 * kv) * c["dim"])))
        c["ctx"] = c["new"] + _spread(rng, 1, 4000)
        return c
    c["window"] = rng.choice([0, 0, _spread(rng, 16, 4096)])
    kind = rng.choice(["single", "few", "chunk", "mixed"])
    if kind in ("single", "few"):  # at most the bytes of 64 contexts of 16384
        c.update(seqs=_spread(rng, 1, 64), new=1 if kind == "single" else _spread(rng, 2, 9), ctx=_spread(rng, 9, 131071))
        c["ctx"] = max(9, min(c["ctx"], 64 * 16384 * 2 * 8 * 128 // (c["seqs"] * (4 if c["cache"] == "f32" else 2) *
                                                                    kv * c["dim"])))
        c["ctx"] = max(9, min(c["ctx"], 2 ** 28 // (c["seqs"] * c["new"] * heads)))
    else:  # at most the products of 2048 tokens over 16384, a quarter of them on fp32
        c.update(seqs=_spread(rng, 1, 5), new=_spread(rng, 10, 2048), mixed=kind == "mixed")
        most = 2048 * 16384 * 32 * 128 // (c["seqs"] * heads * c["dim"] * (4 if c["cache"] == "f32" else 1))
        c["ctx"] = max(c["new"], min(_spread(rng, c["new"], 16384), most // c["new"]))
        c["new"] = max(1, min(c["new"], most // c["ctx"]))
    return c


# ---------------------------------------------------------------- the sizes


def _lens(c):
    """Each context's length with its new tokens: the longest is ctx, the others
    between a quarter of it and all of it."""
    n = c["seqs"]
    return [max(_new(c)[i], c["ctx"] if i == 0 else int(c["ctx"] * (0.25 + 0.75 * ((i * 0.6180339887) % 1.0))))
            for i in range(n)]


def _new(c):
    """Each context's new tokens: ragged where there are many; in a mixed batch
    the first context reads a chunk and the others decode."""
    n, new = c["seqs"], c.get("new", 0)
    if c.get("mixed"):
        return [new] + [1] * (n - 1)
    if new < 16:
        return [new] * n
    return [min(new, c["ctx"]) if i == 0 else max(1, int(new * (0.3 + 0.7 * ((i * 0.6180339887) % 1.0)))) for i in range(n)]


def _starts(new):
    s = [0]
    for v in new:
        s.append(s[-1] + v)
    return s


# ---------------------------------------------------------------- the inputs


def _frequencies(c):
    """Each pair's angle per position, in 64 bits, and the amplitude, as a
    program has them from its model's file."""
    r = c["rot"]
    j = torch.arange(r // 2, dtype=torch.float64)
    f = 500000.0 ** (-2.0 * j / r)
    if c["scaling"] == "linear":
        return f / 4.0, 1.0
    if c["scaling"] == "factors":  # low frequencies stretched, a smooth step between
        wave = 2.0 * math.pi / f
        blend = ((8192.0 / wave - 1.0) / 3.0).clamp(0.0, 1.0)
        return f / (8.0 / (1.0 + 7.0 * blend)), 1.0
    if c["scaling"] == "yarn":
        place = [r * math.log(4096.0 / (b * 2.0 * math.pi)) / (2.0 * math.log(500000.0)) for b in (32.0, 1.0)]
        lo, hi = max(math.floor(place[0]), 0), min(math.ceil(place[1]), r - 1)
        ramp = ((j - lo) / max(hi - lo, 0.001)).clamp(0.0, 1.0)
        return f / 16.0 * ramp + f * (1.0 - ramp), 0.1 * math.log(16.0) + 1.0
    return f, 1.0


def prepare(case, seed):
    c = dict(case)
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, dtype=torch.float32, spread=1.0):
        return (torch.randn(shape, generator=gen, device="cuda") * spread).to(dtype)

    if c["family"] == "rope":
        f, amp = _frequencies(c)
        return {"case": c, "freqs": f.cuda(), "amp": amp,
                "x": normal(c["tokens"], c["heads"], c["dim"], dtype=_TYPES[c["type"]]),
                "positions": torch.randint(0, c["far"], (c["tokens"],), generator=gen, device="cuda", dtype=torch.int32)}
    lens, new = _lens(c), _new(c)
    per = -(-(max(lens) + 64) // c["page"])
    need = [-(-n // c["page"]) for n in lens]
    if c["family"] == "pages":
        pages = c["pages"]
        live = lens[:c["seqs"] - c["count"]]  # the last slots are empty: forks go there
        lens = live + [0] * c["count"]
        need = [-(-n // c["page"]) for n in lens]
    else:
        pages = sum(need) + 5
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    table = torch.full((c["seqs"], per), -1, dtype=torch.int32, device="cuda")
    refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    refs[order[:at].long()] = 1
    s = {"case": c, "table": table, "lens": torch.tensor(lens, dtype=torch.int32, device="cuda"),
         "starts": torch.tensor(_starts(new), dtype=torch.int32, device="cuda"), "max_new": max(new), "max_len": max(lens)}
    cache = _TYPES[c["cache"]]
    if c["family"] == "pages":
        s["kv"] = torch.empty((c["layers"], pages, 2, c["kv"], c["page"], c["dim"]), dtype=cache, device="cuda")
        for layer in s["kv"]:
            layer.copy_(normal(*layer.shape))
        s["refs"] = refs
        s["src"] = torch.randint(0, max(1, len(live)), (c["count"],), generator=gen, device="cuda", dtype=torch.int32)
        s["dst"] = torch.arange(len(live), c["seqs"], device="cuda", dtype=torch.int32)
        s["counts"] = torch.randint(1, 40, (c["seqs"],), generator=gen, device="cuda", dtype=torch.int32)
        return s
    s["kv"] = normal(pages, 2, c["kv"], c["page"], c["dim"], dtype=cache)
    tokens, t = sum(new), _TYPES[c["type"]]
    # queries wider than keys: rows whose weight gathers on some of the keys
    s["q"] = normal(tokens, c["heads"], c["dim"], dtype=t, spread=1.0 if c["family"] == "append" else 2.0)
    if c["family"] == "append":
        s["k"], s["v"] = (normal(tokens, c["kv"], c["dim"], dtype=t) for _ in range(2))
        f, s["amp"] = _frequencies(c)
        s["freqs"] = f.cuda()
    return s


# ---------------------------------------------------------------- one pass


def run(state):
    s, c = state, state["case"]
    if c["family"] == "rope":
        return _rope_own(s, c) if own else _rope(s["x"], s["positions"], s, c, -1.0 if c["inverse"] else 1.0)
    if c["family"] == "append":
        return _append_own(s, c) if own else _append(s, c)
    if c["family"] == "attend":
        return _attend_own(s, c) if own else _attend(s, c)
    if c["op"] == "fork":
        return _fork_own(s, c) if own else _fork(s, c)
    return _compact_own(s, c) if own else _compact(s, c)


def _rope_own(s, c):
    m = _package()
    plan = m.RopePlan(s["freqs"], c["layout"] == "interleaved", s["amp"])
    return m.rope(s["x"], s["positions"], plan, inverse=c["inverse"])


def _append_own(s, c):
    m = _package()
    plan = m.RopePlan(s["freqs"], c["layout"] == "interleaved", s["amp"])
    q = m.cache_append(s["kv"], s["table"], s["lens"], s["starts"], s["k"], s["v"], q=s["q"], plan=plan)
    return q, s["kv"]


def _attend_own(s, c):
    return _package().paged_attention(s["q"], s["kv"], s["table"], s["lens"], s["starts"], s["max_new"], s["max_len"],
                                      window=c["window"], lse=True)


def _fork_own(s, c):
    m = _package()
    table, lens, refs = s["table"].clone(), s["lens"].clone(), s["refs"].clone()
    a = m.cache_fork(s["kv"], table, lens, refs, s["src"], s["dst"])
    b = m.cache_reserve(table, lens, refs, c["page"], s["counts"])
    grown = table.clone(), lens.clone(), refs.clone()
    e = m.cache_release(table, lens, refs, s["dst"], c["page"])
    return grown, (table, lens, refs), (a, b, e), s["kv"]


def _compact_own(s, c):
    table, refs = s["table"].clone(), s["refs"].clone()
    return _package().cache_compact(s["kv"], table, refs), table, refs, s["kv"]


def _rope(x, positions, s, c, sign):
    angle = positions.double()[:, None] * s["freqs"][None, :]
    cos, sin = (angle.cos() * s["amp"]).float()[:, None, :], (angle.sin() * (s["amp"] * sign)).float()[:, None, :]
    y = x.float().clone()
    part = y[..., :c["rot"]]
    if c["layout"] == "interleaved":
        a, b = part[..., 0::2], part[..., 1::2]
    else:
        a, b = part[..., :c["rot"] // 2], part[..., c["rot"] // 2:]
    first, second = a * cos - b * sin, b * cos + a * sin
    a.copy_(first)
    b.copy_(second)
    return y.to(x.dtype)


def _places(s, tokens):
    """Each token's context and position."""
    at = torch.arange(tokens, device="cuda")
    seq = torch.bucketize(at, s["starts"][1:].long(), right=True)
    new = (s["starts"][1:] - s["starts"][:-1]).long()
    return seq, s["lens"].long()[seq] - new[seq] + at - s["starts"].long()[seq]


def _append(s, c):
    seq, pos = _places(s, s["q"].shape[0])
    q, k = (_rope(x, pos, s, c, 1.0) if x.dtype == torch.float32 else _rope(x.float(), pos, s, c, 1.0)
            for x in (s["q"], s["k"]))
    page = s["table"].long()[seq, pos // c["page"]]
    kv = s["kv"]
    kv[page, 0, :, pos % c["page"]] = k.to(kv.dtype)
    kv[page, 1, :, pos % c["page"]] = s["v"].to(kv.dtype)
    return q.to(s["q"].dtype), kv


def _attend(s, c):
    q, kv, n, wide = s["q"], s["kv"], c["seqs"], s["max_new"]
    per, group = kv.shape[2], q.shape[1] // kv.shape[2]
    new = (s["starts"][1:] - s["starts"][:-1]).long()
    at = torch.arange(wide, device="cuda")
    row = (s["starts"][:-1].long()[:, None] + at).clamp_max(q.shape[0] - 1)               # [n, wide]
    real = at < new[:, None]
    pos = s["lens"].long()[:, None] - new[:, None] + at
    key = torch.arange(s["max_len"], device="cuda")
    page = s["table"].long()[:, key // c["page"]].clamp_min(0)                             # [n, keys]
    there = (key < s["lens"][:, None])[:, None, :, None]
    k = kv[page, 0, :, key % c["page"]].permute(0, 2, 1, 3).float()                       # [n, kv, keys, d]
    v = kv[page, 1, :, key % c["page"]].permute(0, 2, 1, 3).float()
    k, v = torch.where(there, k, 0.0), torch.where(there, v, 0.0)
    x = q[row].float().reshape(n, wide, per, group, -1).permute(0, 2, 3, 1, 4).reshape(n, per, group * wide, -1)
    sees = key <= pos[..., None]                                                          # [n, wide, keys]
    if c["window"]:
        sees &= key > pos[..., None] - c["window"]
    score = torch.matmul(x, k.transpose(2, 3).contiguous()).mul_(1.0 / math.sqrt(c["dim"]))
    score = score.view(n, per, group, wide, -1).masked_fill_(~sees[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    top = torch.where(torch.isfinite(top), top, 0.0)
    p = score.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.view(n, per, group * wide, -1), v).view(n, per, group, wide, -1) / total.clamp_min(1e-37)
    lse = (top + total.log()).squeeze(-1)
    return (out.permute(0, 3, 1, 2, 4).reshape(n, wide, q.shape[1], -1)[real].to(q.dtype),
            lse.permute(0, 3, 1, 2).reshape(n, wide, q.shape[1])[real])


def _free(refs, count):
    """The `count` lowest pages that nobody holds."""
    return torch.nonzero(refs == 0).reshape(-1)[:count]


def _fork(s, c):
    table, lens, refs, kv, ps = s["table"].clone(), s["lens"].clone(), s["refs"].clone(), s["kv"], c["page"]
    src, dst = s["src"].long(), s["dst"].long()
    # full pages are shared, the last partial one is the new context's own copy
    full, part = lens[src].long() // ps, lens[src].long() % ps > 0
    at = torch.arange(table.shape[1], device="cuda")
    shared = at < full[:, None]
    refs.index_add_(0, table[src][shared].long(), torch.ones_like(table[src][shared]))
    took = _free(refs, int(part.sum()))
    table[dst] = torch.where(shared, table[src], -1)
    last = table[src[part], full[part]].long()
    table[dst[part], full[part]] = took.to(torch.int32)
    refs[took] = 1
    kv[:, took] = kv[:, last]
    lens[dst] = lens[src]
    # pages for the tokens to come, context by context
    have, want = -(-lens.long() // ps), -(-(lens + s["counts"]).long() // ps)
    more = (at >= have[:, None]) & (at < want[:, None])
    took = _free(refs, int(more.sum()))
    table[more] = took.to(torch.int32)
    refs[took] = 1
    lens += s["counts"]
    grown = table.clone(), lens.clone(), refs.clone()
    # the forks end
    gone = table[dst]
    refs.index_add_(0, gone[gone >= 0].long(), -torch.ones_like(gone[gone >= 0]))
    table[dst] = -1
    lens[dst] = 0
    fine = torch.zeros(1, dtype=torch.int32, device="cuda")
    return grown, (table, lens, refs), (fine, fine.clone(), fine.clone()), kv


def _compact(s, c):
    table, refs, kv = s["table"].clone(), s["refs"].clone(), s["kv"]
    held = refs > 0
    live = int(held.sum())
    src = torch.nonzero(held[live:]).reshape(-1) + live
    dst = torch.nonzero(~held[:live]).reshape(-1)
    kv[:, dst] = kv[:, src]
    place = torch.arange(refs.shape[0], device="cuda", dtype=torch.int32)
    place[src] = dst.to(torch.int32)
    table = torch.where(table >= 0, place[table.long().clamp_min(0)], table)
    refs[dst] = refs[src]
    refs[src] = 0
    return torch.tensor([live], dtype=torch.int32, device="cuda"), table, refs, kv


# ---------------------------------------------------------------- what a pass cannot do without


def _pairs(c):
    """The (query, key) pairs that are visible, and the keys that any query of
    their context sees, over all contexts."""
    pairs = keys = 0
    for n, new in zip(_lens(c), _new(c)):
        w = c["window"] or n
        first = n - new  # the first new token's position
        short = max(0, min(new, w - first))  # queries that see every key before them
        pairs += short * first + short * (short + 1) // 2 + (new - short) * w
        keys += n - max(0, first + 1 - w)
    return pairs, keys


def work(case):
    c = dict(case)
    size = {"f32": 4, "f16": 2, "bf16": 2}
    if c["family"] == "rope":
        n = c["tokens"] * c["heads"]
        return {"bytes": 2 * n * c["dim"] * size[c["type"]] + 4 * c["tokens"] + 4 * c["rot"], "flops": 3.0 * n * c["rot"]}
    row = c["kv"] * c["dim"] * size[c["cache"]]  # one token's keys (or values) in the cache
    if c["family"] == "pages":
        held = [-(-n // c["page"]) for n in _lens(c)]
        if c["op"] == "compact":
            # a live page above the live count moves: as many as the free pages below it, by expectation
            moved, words = sum(held) * (1.0 - sum(held) / c["pages"]), 4 * (2 * c["pages"] + 2 * c["seqs"] * max(held))
        else:
            moved, words = c["count"], 4 * (6 * c["pages"] + 10 * c["seqs"] * (max(held) + 4))
        return {"bytes": 2.0 * moved * c["layers"] * 2 * c["page"] * row + words, "flops": 0.0}
    tokens, t = sum(_new(c)), size[c["type"]]
    if c["family"] == "append":
        b = tokens * c["dim"] * t * (2 * c["heads"] + 2 * c["kv"]) + 2 * tokens * row
        return {"bytes": b + 8 * c["seqs"], "flops": 3.0 * tokens * (c["heads"] + c["kv"]) * c["rot"]}
    pairs, keys = _pairs(c)
    b = 2 * tokens * c["heads"] * c["dim"] * t + 4 * tokens * c["heads"] + 2 * keys * row + 4 * keys // c["page"]
    return {"bytes": b, "flops": 4.0 * c["dim"] * c["heads"] * pairs}


# ---------------------------------------------------------------- the definition in 64 bits


def _turned(x, positions, freqs, amp, c, sign=1.0):
    """Each pair as a complex number times amp * e^(i sign position f)."""
    x = x.double()
    r = c["rot"]
    turn = torch.polar(torch.full_like(freqs, amp).expand(positions.numel(), -1).contiguous(),
                       sign * positions.double()[:, None] * freqs)[:, None, :]
    head, rest = x[..., :r], x[..., r:]
    shape = head.shape[:-1]
    if c["layout"] == "interleaved":
        z = torch.view_as_complex(head.reshape(*shape, r // 2, 2).contiguous()) * turn
        return torch.cat([torch.view_as_real(z).reshape(*shape, r), rest], -1)
    z = torch.complex(head[..., :r // 2].contiguous(), head[..., r // 2:].contiguous()) * turn
    return torch.cat([z.real, z.imag, rest], -1)


def exact(case, seed):
    c = dict(case)
    if c["family"] == "pages":
        return None  # whole numbers and copies
    s = prepare(c, seed)
    if c["family"] == "rope":
        return _turned(s["x"], s["positions"], s["freqs"], s["amp"], c, -1.0 if c["inverse"] else 1.0)
    lens, new = _lens(c), _new(c)
    table, ps = s["table"].long(), c["page"]
    if c["family"] == "append":
        pos = torch.cat([torch.arange(n - k, n) for n, k in zip(lens, new)]).cuda()
        q, k = (_turned(s[x], pos, s["freqs"], s["amp"], c) for x in "qk")
        kv, at = s["kv"].double(), 0
        for i, (n, m) in enumerate(zip(lens, new)):
            p = torch.arange(n - m, n, device="cuda")
            page = table[i, p // ps]
            kv[page, 0, :, p % ps] = k[at:at + m]
            kv[page, 1, :, p % ps] = s["v"][at:at + m].double()
            at += m
        return q, kv
    per, d = c["kv"], c["dim"]
    group = c["heads"] // per
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.empty(s["q"].shape[:2], dtype=torch.float64, device="cuda")
    at = 0
    for i, (n, m) in enumerate(zip(lens, new)):
        p = torch.arange(n, device="cuda")
        rows = s["kv"][table[i, p // ps], :, :, p % ps].double()  # [n, 2, kv, d]
        mine = torch.arange(n - m, n, device="cuda")
        gone = p[None, :] > mine[:, None]
        if c["window"]:
            gone |= p[None, :] <= mine[:, None] - c["window"]
        for h in range(c["heads"]):
            k, v = rows[:, 0, h // group], rows[:, 1, h // group]
            score = (s["q"][at:at + m, h].double() @ k.t().contiguous() / math.sqrt(d)).masked_fill(gone, -math.inf)
            l = torch.logsumexp(score, 1)
            out[at:at + m, h] = torch.exp(score - l[:, None]) @ v
            lse[at:at + m, h] = l
        at += m
    return out, lse

"""What lets more contexts decode together than a 16-bit cache has room for:
keys and values in 8 or 4 bits, attention over them, and beam search, which
multiplies contexts and moves them about.

Each case is one pass through the package's public entry points (`own` true)
or through the same mathematics in elementary torch operations (`own` false).
The families:

  write    cache_append of new tokens into pages of Q8_0 or Q4_0 blocks, and
           cache_read of what they became
  read     cache_read: whole contexts as rows again
  attend   paged_attention: chunks of new tokens over such pages
  beams    beam_select: the best continuations of each group of beams
  reorder  cache_reorder: every context becomes what its parent was

A block is 32 elements of a head, an fp16 factor d and a whole number c each:
Q8_0 d c with -127 .. 127, Q4_0 d c with -8 .. 7.
"""
import importlib.util
import math
import os
import sys

import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_BITS = {"q8_0": 8, "q4_0": 4}


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
        # one token each of a small serving batch, fp32 projections: latency
        {"name": "write_24_tokens_q4", "family": "write", "seqs": 24, "new": 1, "ctx": 4000, "heads": 32, "kv": 8,
         "dim": 128, "page": 16, "type": "f32", "cache": "q4_0"},
        # the prompts of three contexts, ragged
        {"name": "write_prompts_q8", "family": "write", "seqs": 3, "new": 2777, "ctx": 2777, "heads": 32, "kv": 8,
         "dim": 128, "page": 64, "type": "bf16", "cache": "q8_0"},
        # one context taken out of the cache
        {"name": "read_one_517_q8", "family": "read", "seqs": 1, "new": 517, "ctx": 517, "heads": 32, "kv": 8, "dim": 64,
         "page": 16, "type": "f32", "cache": "q8_0"},
        # a batch of contexts taken out, to go on in 16 bits
        {"name": "read_16x4000_q4", "family": "read", "seqs": 16, "new": 4000, "ctx": 4000, "heads": 32, "kv": 8,
         "dim": 128, "page": 32, "type": "bf16", "cache": "q4_0"},
        # one chat context, one token: latency
        {"name": "attend_chat_517_q8", "family": "attend", "seqs": 1, "new": 1, "ctx": 517, "heads": 32, "kv": 8,
         "dim": 64, "page": 16, "type": "f32", "cache": "q8_0", "window": 0},
        # one token of one long context: few rows, a long axis
        {"name": "attend_long_131071_q4", "family": "attend", "seqs": 1, "new": 1, "ctx": 131071, "heads": 32, "kv": 8,
         "dim": 128, "page": 64, "type": "f32", "cache": "q4_0", "window": 0},
        # a serving batch of ragged contexts, one token each
        {"name": "attend_64x16k_q4", "family": "attend", "seqs": 64, "new": 1, "ctx": 16384, "heads": 32, "kv": 8,
         "dim": 128, "page": 16, "type": "bf16", "cache": "q4_0", "window": 0},
        # a chunk of a long prompt, fp32 queries
        {"name": "attend_chunk_2048x16k_q4", "family": "attend", "seqs": 1, "new": 2048, "ctx": 16384, "heads": 32,
         "kv": 8, "dim": 128, "page": 64, "type": "f32", "cache": "q4_0", "window": 0},
        # four beams of one chat
        {"name": "beams_4x32000", "family": "beams", "groups": 1, "beams": 4, "vocab": 32000, "ended": 0.0},
        # a batch of translations, some of whose beams have ended
        {"name": "beams_64x8x128256", "family": "beams", "groups": 64, "beams": 8, "vocab": 128256, "ended": 0.2},
        # the same chat's contexts follow their beams
        {"name": "reorder_4x517", "family": "reorder", "groups": 1, "beams": 4, "layers": 16, "page": 16, "kv": 8,
         "dim": 64, "ctx": 517, "own": 60, "cache": "f16"},
        # and the batch's
        {"name": "reorder_64x8x1003", "family": "reorder", "groups": 64, "beams": 8, "layers": 16, "page": 16, "kv": 8,
         "dim": 64, "ctx": 1003, "own": 90, "cache": "f16"},
    ]


def _spread(rng, lo, hi):
    """A whole number, even in its logarithm over lo .. hi."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    family = rng.choice(["write", "read", "attend", "attend", "attend", "beams", "beams", "reorder"])
    c = {"family": family}
    if family == "beams":
        c.update(groups=_spread(rng, 1, 64), beams=rng.choice([1, 2, 3, 4, 5, 8, 12, 16, 32]),
                 vocab=rng.choice([_spread(rng, 100, 262144), 32000, 50257, 128256, 151936]),
                 ended=rng.choice([0.0, 0.2, 0.5]))
        c["groups"] = max(1, min(c["groups"], 64 * 8 * 128256 // (c["beams"] * c["vocab"])))
        return c
    heads, kv = rng.choice([(32, 8), (32, 32), (16, 8), (28, 4), (14, 2), (8, 1), (40, 8), (9, 3)])
    c.update(heads=heads, kv=kv, dim=rng.choice([32, 64, 64, 96, 128, 128, 128, 192, 256]),
             page=rng.choice([16, 16, 32, 64, 256]))
    if family == "reorder":
        c.pop("heads")
        c.update(groups=_spread(rng, 1, 64), beams=rng.choice([2, 3, 4, 5, 8]), layers=_spread(rng, 1, 32),
                 ctx=_spread(rng, 1, 2000), own=_spread(rng, 1, 200), cache=rng.choice(["f32", "f16", "bf16"]))
        size = 4 if c["cache"] == "f32" else 2
        page = c["layers"] * c["page"] * c["kv"] * c["dim"] * 2 * size
        most = 6500 * 16 * 16 * 8 * 64 * 2 * 2 // page  # pages of the largest listed case's bytes
        per = -(-c["ctx"] // c["page"]) + 1 + c["beams"] * (-(-c["own"] // c["page"]) + 2)
        c["groups"] = max(1, min(c["groups"], most // per))
        return c
    c.update(type=rng.choice(["f32", "f32", "f16", "bf16"]), cache=rng.choice(["q8_0", "q4_0", "q4_0"]))
    if family == "write":
        c.update(seqs=_spread(rng, 1, 64), new=_spread(rng, 1, 2777))
        c["new"] = max(1, min(c["new"], 3 * 2777 * 8 * 128 // (c["seqs"] * kv * c["dim"])))
        c["ctx"] = c["new"] + _spread(rng, 1, 4000)
        return c
    if family == "read":
        c.update(seqs=_spread(rng, 1, 64), new=_spread(rng, 1, 8000))
        c["new"] = c["ctx"] = max(1, min(c["new"], 16 * 4000 * 8 * 128 // (c["seqs"] * kv * c["dim"])))
        return c
    c["window"] = rng.choice([0, 0, _spread(rng, 16, 4096)])
    kind = rng.choice(["single", "few", "chunk", "mixed"])
    if kind in ("single", "few"):  # at most the bytes of 64 contexts of 16384
        c.update(seqs=_spread(rng, 1, 64), new=1 if kind == "single" else _spread(rng, 2, 9), ctx=_spread(rng, 9, 131071))
        c["ctx"] = max(9, min(c["ctx"], 64 * 16384 * 8 * 128 // (c["seqs"] * kv * c["dim"])))
        c["ctx"] = max(9, min(c["ctx"], 2 ** 28 // (c["seqs"] * c["new"] * heads)))
    else:  # at most the products of 2048 tokens over 16384
        c.update(seqs=_spread(rng, 1, 5), new=_spread(rng, 10, 2048), mixed=kind == "mixed")
        most = 2048 * 16384 * 32 * 128 // (c["seqs"] * heads * c["dim"])
        c["ctx"] = max(c["new"], min(_spread(rng, c["new"], 16384), most // c["new"]))
        c["new"] = max(1, min(c["new"], most // c["ctx"]))
    return c


# ---------------------------------------------------------------- the sizes


def _lens(c):
    """Each context's length with its new tokens: the longest is ctx, the others
    between a quarter of it and all of it."""
    return [max(_new(c)[i], c["ctx"] if i == 0 else int(c["ctx"] * (0.25 + 0.75 * ((i * 0.6180339887) % 1.0))))
            for i in range(c["seqs"])]


def _new(c):
    """Each context's new tokens: ragged where there are many; in a mixed batch
    the first context reads a chunk and the others decode."""
    n, new = c["seqs"], c["new"]
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


# ---------------------------------------------------------------- a page of blocks
#
# For each kv head: keys' codes [page, row bytes], their factors [groups, page],
# values' codes, their factors.  Where element d of a row's codes lies (the
# order in which the matrix cores take a key's and a value's elements):


def _places(dim, bits, value):
    """(byte, shift) of each element of a row of codes."""
    d = torch.arange(dim, device="cuda")
    groups, x, in_block = dim // 32, d // 32, d % 32
    if not value:  # a quarter of each block side by side with the other blocks' same quarter
        quarter, e = in_block // 8, d % 8
        unit = quarter * groups + x
        if bits == 8:
            return unit * 8 + e, torch.zeros_like(d)
        nibble = e // 2 + 4 * (e % 2)
        return unit * 4 + nibble // 2, 4 * (nibble % 2)
    half, i = in_block // 16, d % 16  # four blocks' bytes side by side, then two's, then one's
    fours = groups // 4 * 4
    wide = torch.where(x < fours, 4, torch.where(x < fours + (groups & 2), 2, 1))
    first = torch.where(x < fours, x // 4 * 4, torch.where(x < fours + (groups & 2), fours, x))
    at = first * 16 + i * wide + x - first
    return (at * 2 + half, torch.zeros_like(d)) if bits == 8 else (at, 4 * half)


def _parts(c):
    """Bytes of a head's codes, of its factors, and of a page."""
    bits = _BITS[c["cache"]]
    codes, factors = c["page"] * c["dim"] * bits // 8, c["page"] * c["dim"] // 32 * 2
    return codes, factors, c["kv"] * 2 * (codes + factors)


def _blocks(x, bits):
    """(codes, factors) of rows [..., dim] in fp32."""
    b = x.unflatten(-1, (-1, 32))
    if bits == 8:
        t = b.abs().amax(-1) * (1.0 / 127.0)
    else:
        t = torch.maximum(b.amax(-1) * (1.0 / 7.0), b.amin(-1) * (-1.0 / 8.0))
    d = t.clamp_max(65504.0).half()
    step = torch.where(d > 0, 1.0 / d.float(), 0.0)
    lo, hi = (-127, 127) if bits == 8 else (-8, 7)
    return torch.round(b * step[..., None]).clamp(lo, hi).flatten(-2), d


def _packed(codes, bits, value):
    """Rows of codes as bytes."""
    byte, shift = _places(codes.shape[-1], bits, value)
    c = (codes + 2 ** (bits - 1)).to(torch.uint8)
    out = torch.zeros((*codes.shape[:-1], codes.shape[-1] * bits // 8), dtype=torch.uint8, device="cuda")
    out[..., byte[shift == 0]] = c[..., shift == 0]
    if bits == 4:
        out[..., byte[shift == 4]] |= c[..., shift == 4] << 4
    return out


def _values(pages, c):
    """fp32 keys and values [..., kv, page, dim] of pages of bytes [..., page bytes]."""
    bits, (codes, factors, _) = _BITS[c["cache"]], _parts(c)
    head = pages.unflatten(-1, (c["kv"], 2, codes + factors))

    def half(k):
        byte, shift = _places(c["dim"], bits, k == 1)
        rows = head[..., k, :codes].unflatten(-1, (c["page"], -1))[..., byte]
        whole = ((rows >> shift.to(torch.uint8)) & (2 ** bits - 1)).float() - 2 ** (bits - 1)
        d = head[..., k, codes:].contiguous().view(torch.float16).unflatten(-1, (-1, c["page"])).transpose(-1, -2)
        return (whole.unflatten(-1, (-1, 32)) * d.float()[..., None]).flatten(-2)

    return half(0), half(1)


# ---------------------------------------------------------------- the inputs


def prepare(case, seed):
    c = dict(case)
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, dtype=torch.float32, spread=1.0):
        return (torch.randn(shape, generator=gen, device="cuda") * spread).to(dtype)

    if c["family"] == "beams":
        return _beam_inputs(c, gen, normal)
    if c["family"] == "reorder":
        return _reorder_inputs(c, gen, normal)
    lens, new = _lens(c), _new(c)
    per = -(-(max(lens) + 64) // c["page"])
    need = [-(-n // c["page"]) for n in lens]
    pages = sum(need) + 5
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    table = torch.full((c["seqs"], per), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    s = {"case": c, "table": table, "lens": torch.tensor(lens, dtype=torch.int32, device="cuda"),
         "starts": torch.tensor(_starts(new), dtype=torch.int32, device="cuda"), "max_new": max(new), "max_len": max(lens)}
    bits, (codes, factors, size) = _BITS[c["cache"]], _parts(c)
    kv = torch.empty((pages, size), dtype=torch.uint8, device="cuda")
    step = max(1, 2 ** 26 // (c["kv"] * c["page"] * c["dim"] * 2))
    for p in range(0, pages, step):
        head = kv[p:p + step].unflatten(-1, (c["kv"], 2, codes + factors))
        for k in range(2):
            x, d = _blocks(normal(head.shape[0], c["kv"], c["page"], c["dim"]), bits)
            head[:, :, k, :codes] = _packed(x, bits, k == 1).flatten(-2)
            head[:, :, k, codes:] = d.transpose(-1, -2).contiguous().flatten(-2).view(torch.uint8)
    s["kv"] = kv
    tokens, t = sum(new), _TYPES[c["type"]]
    s["tokens"] = tokens
    if c["family"] == "write":
        s["k"], s["v"] = (normal(tokens, c["kv"], c["dim"], dtype=t) for _ in range(2))
    if c["family"] == "attend":  # queries wider than keys: rows whose weight gathers on some of the keys
        s["q"] = normal(tokens, c["heads"], c["dim"], dtype=t, spread=2.0)
    return s


def _beam_inputs(c, gen, normal):
    """Logits whose mass lies on some tens of ids, as a language model's do;
    beams that have come apart by a few nats."""
    rows = c["groups"] * c["beams"]
    s = {"case": c, "logits": normal(rows, c["vocab"], spread=3.0)}
    top = torch.randint(0, c["vocab"], (rows, 24), generator=gen, device="cuda")
    s["logits"].scatter_add_(1, top, normal(rows, 24, spread=3.0).abs_().add_(4.0))
    s["scores"] = normal(c["groups"], c["beams"], spread=2.0).sub_(30.0)
    s["ended"] = (torch.rand(rows, generator=gen, device="cuda") < c["ended"]).view(c["groups"], c["beams"]).int()
    s["eog"] = torch.cat([top[:1, 0], torch.randint(0, c["vocab"], (2,), generator=gen, device="cuda")]).int()
    return s


def _reorder_inputs(c, gen, normal):
    """Each group's beams share their prompt's full pages and have grown pages of
    their own; a beam's parent is a better beam more often than a worse one."""
    g, w, ps = c["groups"], c["beams"], c["page"]
    shared, n = c["ctx"] // ps, c["ctx"] + c["own"]
    mine = -(-n // ps) - shared
    pages = g * (shared + w * mine) + g * w + 3
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    table = torch.full((g * w, -(-n // ps) + 4), -1, dtype=torch.int32, device="cuda")
    table.view(g, w, -1)[:, :, :shared] = order[:g * shared].view(g, 1, shared)
    table[:, shared:shared + mine] = order[g * shared:g * (shared + w * mine)].view(g * w, mine)
    refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
    refs[order[:g * shared].long()] = w
    refs[order[g * shared:g * (shared + w * mine)].long()] = 1
    u = torch.rand((g, w), generator=gen, device="cuda")
    best = (u * u * w).long().clamp_max(w - 1)
    kv = torch.empty((c["layers"], pages, 2, c["kv"], ps, c["dim"]), dtype=_TYPES[c["cache"]], device="cuda")
    for layer in kv:
        layer.copy_(normal(*layer.shape))
    return {"case": c, "kv": kv, "table": table, "refs": refs,
            "lens": torch.full((g * w,), n, dtype=torch.int32, device="cuda"),
            "parents": (best + torch.arange(g, device="cuda")[:, None] * w).int()}


# ---------------------------------------------------------------- one pass


def run(state):
    s, c = state, state["case"]
    if c["family"] == "write":
        return _write_own(s, c) if own else _write(s, c)
    if c["family"] == "read":
        return _read_own(s, c) if own else _read(s, c, _TYPES[c["type"]])
    if c["family"] == "attend":
        return _attend_own(s, c) if own else _attend(s, c)
    if c["family"] == "beams":
        return _beams_own(s, c) if own else _beams(s, c)
    return _reorder_own(s, c) if own else _reorder(s, c)


def _format(c):
    return _package().PageFormat(c["cache"], c["kv"], c["page"], c["dim"])


def _write_own(s, c):
    m, f = _package(), _format(c)
    m.cache_append(s["kv"], s["table"], s["lens"], s["starts"], s["k"], s["v"], fmt=f)
    return m.cache_read(s["kv"], s["table"], s["lens"], s["starts"], s["tokens"], fmt=f)


def _read_own(s, c):
    return _package().cache_read(s["kv"], s["table"], s["lens"], s["starts"], s["tokens"], dtype=_TYPES[c["type"]],
                                 fmt=_format(c))


def _attend_own(s, c):
    return _package().paged_attention(s["q"], s["kv"], s["table"], s["lens"], s["starts"], s["max_new"], s["max_len"],
                                      window=c["window"], lse=True, fmt=_format(c))


def _beams_own(s, c):
    return _package().beam_select(s["logits"], s["scores"], ended=s["ended"], eog=s["eog"])


def _reorder_own(s, c):
    table, lens, refs = s["table"].clone(), s["lens"].clone(), s["refs"].clone()
    status = _package().cache_reorder(s["kv"], table, lens, refs, s["parents"].view(-1))
    return status, table, lens, refs, s["kv"]


def _tokens(s):
    """Each token's context and position."""
    at = torch.arange(s["tokens"], device="cuda")
    seq = torch.bucketize(at, s["starts"][1:].long(), right=True)
    new = (s["starts"][1:] - s["starts"][:-1]).long()
    return seq, s["lens"].long()[seq] - new[seq] + at - s["starts"].long()[seq]


def _write(s, c):
    bits, (codes, factors, _) = _BITS[c["cache"]], _parts(c)
    seq, pos = _tokens(s)
    page, place = s["table"].long()[seq, pos // c["page"]], pos % c["page"]
    heads = s["kv"].unflatten(-1, (c["kv"], 2, codes + factors))
    rows = heads[..., :codes].unflatten(-1, (c["page"], -1))  # [pages, kv, 2, page, row bytes]
    scales = heads[..., codes:].unflatten(-1, (c["dim"] // 32, c["page"], 2))

    def put(x, k):
        x, d = _blocks(x.float(), bits)
        rows[page, :, k, place] = _packed(x, bits, k == 1)
        scales[page, :, k, :, place] = d[..., None].view(torch.uint8)

    put(s["k"], 0)
    put(s["v"], 1)
    return _read(s, c, torch.float32)


def _read(s, c, dtype):
    bits, (codes, factors, _) = _BITS[c["cache"]], _parts(c)
    seq, pos = _tokens(s)
    page, place = s["table"].long()[seq, pos // c["page"]], pos % c["page"]
    heads = s["kv"].unflatten(-1, (c["kv"], 2, codes + factors))
    rows = heads[..., :codes].unflatten(-1, (c["page"], -1))
    scales = heads[..., codes:].unflatten(-1, (c["dim"] // 32, c["page"], 2))

    def get(k):
        byte, shift = _places(c["dim"], bits, k == 1)
        row = rows[page, :, k, place][..., byte]
        whole = ((row >> shift.to(torch.uint8)) & (2 ** bits - 1)).float() - 2 ** (bits - 1)
        d = scales[page, :, k, :, place].contiguous().view(torch.float16).float()
        return (whole.unflatten(-1, (-1, 32)) * d).flatten(-2).to(dtype)

    return get(0), get(1)


def _attend(s, c):
    q, n, wide, per = s["q"], c["seqs"], s["max_new"], c["kv"]
    group = c["heads"] // per
    new = (s["starts"][1:] - s["starts"][:-1]).long()
    at = torch.arange(wide, device="cuda")
    row = (s["starts"][:-1].long()[:, None] + at).clamp_max(q.shape[0] - 1)               # [n, wide]
    real = at < new[:, None]
    pos = s["lens"].long()[:, None] - new[:, None] + at
    used = -(-s["max_len"] // c["page"])
    k, v = _values(s["kv"][s["table"][:, :used].long().clamp_min(0)], c)                   # [n, used, kv, page, d]
    key = torch.arange(used * c["page"], device="cuda")
    there = (key < s["lens"][:, None])[:, None, :, None]
    k, v = (torch.where(there, x.transpose(1, 2).flatten(2, 3), 0.0) for x in (k, v))      # [n, kv, keys, d]
    x = q[row].float().reshape(n, wide, per, group, -1).permute(0, 2, 3, 1, 4).reshape(n, per, group * wide, -1)
    sees = (key <= pos[..., None]) & (key < s["lens"][:, None, None])                      # [n, wide, keys]
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


def _beams(s, c):
    """In 64 bits: candidates of different beams are compared."""
    g, w, v = c["groups"], c["beams"], c["vocab"]
    x = s["logits"].double()
    x = x - x.amax(-1, keepdim=True)
    x = x.sub_(x.exp().sum(-1, keepdim=True).log()).view(g, w, v).add_(s["scores"].double()[..., None])
    over = s["ended"].bool()
    x.masked_fill_(over[..., None], -math.inf)  # an ended beam stands for itself
    x[..., 0] = torch.where(over, s["scores"].double(), x[..., 0])
    x = x.view(g, w * v)
    least = x.topk(w, -1).values[:, -1:]
    same = x == least
    room = w - (x > least).sum(-1, keepdim=True)
    at = ((x > least) | (same & (same.cumsum(-1) <= room))).nonzero()[:, 1].view(g, w)  # the lowest of equals
    score, order = x.gather(1, at).sort(dim=-1, descending=True, stable=True)
    at = at.gather(1, order)
    beam = at // v
    done = over.gather(1, beam)
    token = torch.where(done, -1, at % v).int()
    parents = (beam + torch.arange(g, device="cuda")[:, None] * w).int()
    return parents, token, score.float(), (done | torch.isin(token, s["eog"])).int()


def _reorder(s, c):
    table, lens, refs, kv, ps = s["table"], s["lens"], s["refs"].clone(), s["kv"], c["page"]
    src = s["parents"].view(-1).long()
    slots = torch.arange(src.shape[0], device="cuda")
    n = lens.long()[src]
    full, part = n // ps, n % ps > 0
    # the parent's partial page stays with the parent, else with its first child
    first = torch.full_like(src, src.shape[0]).scatter_reduce(0, src, slots, "amin")
    keeps = torch.where(src[src] == src, src == slots, first[src] == slots)
    at = torch.arange(table.shape[1], device="cuda")
    new = torch.where(at < (full + (part & keeps))[:, None], table[src], -1)
    ones = torch.ones_like(table)
    refs.index_add_(0, table.clamp_min(0).view(-1).long(), (-ones * (table >= 0)).view(-1))
    refs.index_add_(0, new.clamp_min(0).view(-1).long(), (ones * (new >= 0)).view(-1))
    copies = torch.nonzero(part & ~keeps).reshape(-1)
    took = torch.nonzero(refs == 0).reshape(-1)[:copies.shape[0]]
    last = table[src[copies], full[copies]].long()
    new[copies, full[copies]] = took.to(torch.int32)
    refs[took] = 1
    kv[:, took] = kv[:, last]
    return torch.zeros(1, dtype=torch.int32, device="cuda"), new, n.to(torch.int32), refs, kv


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
    if c["family"] == "beams":  # one exponential and two sums each; ended rows are not read
        n = c["groups"] * c["beams"] * c["vocab"] * (1.0 - c["ended"])
        return {"bytes": 4.0 * n + 28 * c["groups"] * c["beams"], "flops": 3.0 * n}
    if c["family"] == "reorder":
        # beams that are not the first child of their parent, by expectation over the skewed choice
        w, n = c["beams"], c["ctx"] + c["own"]
        used = sum(1.0 - (1.0 - (math.sqrt((i + 1) / w) - math.sqrt(i / w))) ** w for i in range(w))
        copies = c["groups"] * (w - used) * (n % c["page"] > 0)
        page = 2 * c["kv"] * c["page"] * c["dim"] * size[c["cache"]]
        return {"bytes": 2.0 * copies * c["layers"] * page + 4 * c["groups"] * w * (2 * (n // c["page"]) + 4), "flops": 0.0}
    row = c["kv"] * (c["dim"] * _BITS[c["cache"]] // 8 + c["dim"] // 32 * 2)  # one token's keys (or values) in the cache
    tokens = sum(_new(c))
    if c["family"] == "write":  # rows read, blocks written and read, fp32 rows written
        n = tokens * c["kv"] * c["dim"]
        return {"bytes": 2 * n * size[c["type"]] + 4 * tokens * row + 8 * n, "flops": 8.0 * n}
    if c["family"] == "read":
        n = tokens * c["kv"] * c["dim"]
        return {"bytes": 2 * tokens * row + 2 * n * size[c["type"]], "flops": 2.0 * n}
    pairs, keys = _pairs(c)
    b = 2 * tokens * c["heads"] * c["dim"] * size[c["type"]] + 4 * tokens * c["heads"] + 2 * keys * row + 4 * keys // c["page"]
    return {"bytes": b, "flops": 4.0 * c["dim"] * c["heads"] * pairs}


# ---------------------------------------------------------------- the definition in 64 bits


def _plain_rows(kv, pages, places, c, k):
    """One context's keys (k 0) or values (1) in float64, [tokens, kv, dim],
    element by element of a row."""
    bits, dim, groups = _BITS[c["cache"]], c["dim"], c["dim"] // 32
    codes, factors, _ = _parts(c)
    out = torch.empty((pages.shape[0], c["kv"], dim), dtype=torch.float64, device="cuda")
    flat = kv.view(-1)
    start = pages[:, None] * kv.shape[1] + (torch.arange(c["kv"], device="cuda") * 2 + k)[None, :] * (codes + factors)
    row = start + (places * (dim * bits // 8))[:, None]
    for d in range(dim):
        x = d // 32
        if k == 0:
            unit, nibble = d % 32 // 8 * groups + x, d % 8 // 2 + d % 2 * 4
            at, shift = (unit * 8 + d % 8, 0) if bits == 8 else (unit * 4 + nibble // 2, nibble % 2 * 4)
        else:
            plane, wide = 0, 4
            while plane + wide > groups or x >= plane + wide:
                if plane + wide > groups:
                    wide //= 2
                else:
                    plane += wide
            at = plane * 16 + d % 16 * wide + x - plane
            at, shift = (at * 2 + d % 32 // 16, 0) if bits == 8 else (at, d % 32 // 16 * 4)
        code = (flat[row + at].long() >> shift) % 2 ** bits - 2 ** (bits - 1)
        there = start + codes + (x * c["page"] + places[:, None]) * 2
        half = (flat[there].long() | flat[there + 1].long() << 8).to(torch.int16).view(torch.float16)
        out[:, :, d] = code.double() * half.double()
    return out


def _held(x, c):
    """What blocks of fp32 elements become, in float64."""
    b = x.reshape(-1, 32)
    high, low = b.max(1).values, b.min(1).values
    if c["cache"] == "q8_0":
        d, most = (torch.maximum(high, -low) * (1.0 / 127.0)).half(), (127, 127)
    else:
        d, most = torch.maximum(high * (1.0 / 7.0), low * (-1.0 / 8.0)).half(), (8, 7)
    code = (b * d.float().reciprocal().nan_to_num(posinf=0.0)[:, None]).round()
    code = torch.minimum(torch.maximum(code, torch.full_like(code, -most[0])), torch.full_like(code, most[1]))
    return (code.double() * d.double()[:, None]).reshape(x.shape)


def exact(case, seed):
    c = dict(case)
    if c["family"] == "reorder":
        return None  # whole numbers and copies
    s = prepare(c, seed)
    if c["family"] == "write":  # what decides factors and codes is fp32, their product is not rounded
        return tuple(_held(s[x].float(), c) for x in "kv")
    if c["family"] == "beams":
        g, w, v = c["groups"], c["beams"], c["vocab"]
        out = torch.empty((g, w), dtype=torch.float64, device="cuda")
        for i in range(g):
            all_ = []
            for b in range(w):
                start = s["scores"][i, b].double()
                row = torch.log_softmax(s["logits"][i * w + b].double(), -1) + start
                all_.append(start.reshape(1) if s["ended"][i, b] else row)
            out[i] = torch.cat(all_).sort(descending=True).values[:w]
        return None, None, out, None
    lens, new = _lens(c), _new(c)
    table, ps = s["table"].long(), c["page"]
    if c["family"] == "read":
        parts = []
        for k in range(2):
            rows = []
            for i, (n, m) in enumerate(zip(lens, new)):
                p = torch.arange(n - m, n, device="cuda")
                rows.append(_plain_rows(s["kv"], table[i, p // ps], p % ps, c, k))
            parts.append(torch.cat(rows))
        return tuple(parts)
    group, d = c["heads"] // c["kv"], c["dim"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.empty(s["q"].shape[:2], dtype=torch.float64, device="cuda")
    at = 0
    for i, (n, m) in enumerate(zip(lens, new)):
        p = torch.arange(n, device="cuda")
        keys, values = (_plain_rows(s["kv"], table[i, p // ps], p % ps, c, k) for k in range(2))
        mine = torch.arange(n - m, n, device="cuda")
        gone = p[None, :] > mine[:, None]
        if c["window"]:
            gone |= p[None, :] <= mine[:, None] - c["window"]
        for h in range(c["heads"]):
            k, v = keys[:, h // group].contiguous(), values[:, h // group].contiguous()
            score = (s["q"][at:at + m, h].double() @ k.t().contiguous() / math.sqrt(d)).masked_fill(gone, -math.inf)
            l = torch.logsumexp(score, 1)
            out[at:at + m, h] = torch.exp(score - l[:, None]) @ v
            lse[at:at + m, h] = l
        at += m
    return out, lse

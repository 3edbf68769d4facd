"""Pages of blocks (Q8_0, Q4_0) written, read back and attended over, against
their definitions (tests/quant_ref.py)."""
import math
import random

import numpy as np
import pytest
import torch

import attention_ref as A
import quant_ref as R

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
NAME = {F32: "f32", F16: "f16", BF16: "bf16"}
KINDS = ["q8_0", "q4_0"]


def say(*a):
    print(*a, flush=True)


def near(got, want, bound, what=""):
    """|got - want| within the bound; NaN in `want` is not looked at."""
    g, w, b = (np.asarray(torch.as_tensor(x).double().cpu()) for x in (got, want, bound))
    live = ~np.isnan(w)
    with np.errstate(invalid="ignore"):
        ok = (g[live] == w[live]) | (np.abs(g[live] - w[live]) <= b[live])
        worst = np.nanmax(np.where(ok, 0, np.abs(g[live] - w[live]) / np.maximum(b[live], 1e-300))) if ok.size else 0
    assert ok.all(), f"{what}: {np.count_nonzero(~ok)} of {ok.size} off, worst {worst} bounds"


class Made:
    """One layer of blocks with random contents (random bytes where no context
    is), its tables, and the chunks of a call."""

    def __init__(self, pkg, kind, lens, new, heads, kv_heads, d, page, dtype, seed=0, slots=None, spread=2.0, slack=3,
                 contents=None):
        g, rng, gen = torch.Generator().manual_seed(seed), random.Random(seed), np.random.default_rng(seed)
        self.kind, self.lens_l, self.new, self.page, self.d, self.kvh = kind, list(lens), list(new), page, d, kv_heads
        self.fmt = pkg.PageFormat(kind, kv_heads, page, d)
        per = max([-(-n // page) for n in lens] + [1]) + 1
        total = sum(-(-n // page) for n in lens) + slack
        order = list(range(total))
        rng.shuffle(order)
        self.raw = gen.integers(0, 256, (total, self.fmt.page_bytes), dtype=np.uint8)
        made = gen.standard_normal((total, 2, kv_heads, page, d)).astype(np.float32) if contents is None else contents(gen, (total, 2, kv_heads, page, d))
        kc, kd = R.blocks(made[:, 0], kind)
        vc, vd = R.blocks(made[:, 1], kind)
        packed = R.pack(kc, kd, vc, vd, kind)
        self.table_l = []
        bits = R.BITS[kind]
        codes, row = page * d * bits // 8, d * bits // 8
        for n in lens:
            mine = [order.pop() for _ in range(-(-n // page))]
            self.table_l.append(mine + [-1] * (per - len(mine)))
            for j, p in enumerate(mine):
                # the tokens that are there; the others keep bytes of any kind
                m = min(page, n - j * page)
                to, fr = (z.reshape(total, kv_heads * 2, -1)[p] for z in (self.raw, packed))
                to[:, :m * row] = fr[:, :m * row]
                for x in range(d // 32):
                    o = codes + x * page * 2
                    to[:, o:o + m * 2] = fr[:, o:o + m * 2]
        self.table = torch.tensor(self.table_l, dtype=torch.int32)
        self.lens = torch.tensor(self.lens_l, dtype=torch.int32)
        self.starts_l = [0]
        for n in new:
            self.starts_l.append(self.starts_l[-1] + n)
        self.starts = torch.tensor(self.starts_l, dtype=torch.int32)
        self.q = (torch.randn(self.starts_l[-1], heads, d, generator=g) * spread).to(dtype)
        self.slots_l = slots
        self.slots = None if slots is None else torch.tensor(slots, dtype=torch.int32)
        self.scale = d ** -0.5

    def values(self):
        return R.unpack(self.raw, self.kind, self.kvh, self.page, self.d)

    def kv_cuda(self):
        return torch.from_numpy(self.raw).cuda()

    def check(self, pkg, window=0, first=None, hints=True, what="", q=None, out=None, scale=None, **kw):
        scale = self.scale if scale is None else scale
        want, lse, ob, lb = R.attend(self.q, self.values(), self.kind, self.table_l, self.lens_l, self.starts_l, scale,
                                     window, first, self.slots_l)
        f = None if first is None else torch.tensor(first, dtype=torch.int32).cuda()
        got, l = pkg.paged_attention(self.q.cuda() if q is None else q, self.kv_cuda(), self.table.cuda(),
                                     self.lens.cuda(), self.starts.cuda(), max_new=max(self.new + [0]) if hints else 0,
                                     max_len=max(self.lens_l + [0]) if hints else 0, window=window, first=f, scale=scale,
                                     slots=None if self.slots is None else self.slots.cuda(), lse=True, out=out,
                                     fmt=self.fmt, **kw)
        near(got, want, ob, what + " out")
        near(l, lse, lb, what + " lse")
        return got, l


# ---------------------------------------------------------------- written and read


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=NAME.get)
@pytest.mark.parametrize("d,kv_heads,page", [(32, 1, 16), (64, 8, 16), (96, 3, 32), (128, 8, 64), (160, 2, 16), (192, 1, 32),
                                             (224, 1, 16), (256, 5, 16)])
def test_blocks_are_written_by_their_definition(pkg, kind, dtype, d, kv_heads, page):
    say(f"[write] {kind} {NAME[dtype]} d={d} kv={kv_heads} page={page}")
    m = Made(pkg, kind, [page + 5, 0, 3 * page, 7], [9, 0, 2 * page, 7], 1, kv_heads, d, page, F32, seed=d)
    g = torch.Generator().manual_seed(d)
    tokens = m.starts_l[-1]
    k, v = ((torch.randn(tokens, kv_heads, d, generator=g) * 3).to(dtype) for _ in range(2))
    want = m.raw.copy()
    for what, x in ((0, k), (1, v)):
        codes, f = R.blocks(x.float().numpy(), kind)
        bits = R.BITS[kind]
        per, row = page * d * bits // 8, d * bits // 8
        heads = want.reshape(want.shape[0], kv_heads, 2, -1)
        for i, n in enumerate(m.new):
            for j in range(n):
                pos, t = m.lens_l[i] - n + j, m.starts_l[i] + j
                p, at = m.table_l[i][pos // page], pos % page
                line = np.zeros((kv_heads, row), dtype=np.uint8)
                for e in range(d):
                    byte, shift = R.place(d, bits, what == 1, e)
                    line[:, byte] |= ((codes[t, :, e] + 2 ** (bits - 1)) << shift).astype(np.uint8)
                heads[p, :, what, at * row:(at + 1) * row] = line
                for x32 in range(d // 32):
                    o = per + (x32 * page + at) * 2
                    heads[p, :, what, o:o + 2] = np.ascontiguousarray(f[t, :, x32]).view(np.uint8).reshape(-1, 2)
    args = (m.table.cuda(), m.lens.cuda(), m.starts.cuda())
    kv = m.kv_cuda()
    pkg.cache_append(kv, *args, k.cuda(), v.cuda(), fmt=m.fmt)
    assert np.array_equal(kv.cpu().numpy(), want)
    # rows off 16 bytes, heads before tokens, pages apart
    wide = torch.zeros(kv_heads, tokens, 2 * d + 3, dtype=dtype, device="cuda")
    a, b = wide[..., 1:1 + d].permute(1, 0, 2), wide[..., 2 + d:2 + 2 * d].permute(1, 0, 2)
    a.copy_(k)
    b.copy_(v)
    far = torch.zeros(m.raw.shape[0], m.raw.shape[1] + 48, dtype=torch.uint8, device="cuda")
    part = far[:, :m.raw.shape[1]]
    part.copy_(m.kv_cuda())
    pkg.cache_append(part, *args, a, b, fmt=m.fmt)
    assert np.array_equal(part.cpu().numpy(), want)
    assert not far[:, m.raw.shape[1]:].any()
    # and back, in each type and into strided rows
    have = R.unpack(want, kind, kv_heads, page, d)
    back = np.stack([[have[m.table_l[i][pos // page], z, :, pos % page] for i, n in enumerate(m.new)
                      for pos in range(m.lens_l[i] - n, m.lens_l[i])] for z in (0, 1)])
    for to in (F32, F16, BF16):
        got = pkg.cache_read(kv, *args, tokens, dtype=to, fmt=m.fmt)
        for z in (0, 1):
            assert torch.equal(got[z].cpu(), torch.from_numpy(back[z]).to(F32).to(to)), (to, z)
        rows = [torch.full((tokens, kv_heads + 1, d + 1), 7.0, dtype=to, device="cuda") for _ in range(2)]
        pkg.cache_read(kv, *args, tokens, k=rows[0][:, :kv_heads, 1:], v=rows[1][:, :kv_heads, 1:], fmt=m.fmt)
        for z in (0, 1):
            assert torch.equal(rows[z][:, :kv_heads, 1:], got[z])
            assert bool((rows[z][:, kv_heads] == 7).all()) and bool((rows[z][..., 0] == 7).all())


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("dtype,d,rot", [(F32, 64, 64), (BF16, 128, 96), (F16, 96, 38), (F32, 32, 2)])
def test_blocks_of_turned_keys(pkg, kind, interleaved, dtype, d, rot):
    """q as nls_rope turns it; keys within half a step of the turned ones (and
    the turn's own error), values as without a plan."""
    m = Made(pkg, kind, [40, 21], [9, 21], 4, 2, d, 16, dtype, seed=rot)
    g = torch.Generator().manual_seed(1)
    tokens = m.starts_l[-1]
    k, v = (torch.randn(tokens, 2, d, generator=g).to(dtype) for _ in range(2))
    plan = pkg.rope_plan(rot, interleaved=interleaved, attn_factor=1.25)
    args = (m.table.cuda(), m.lens.cuda(), m.starts.cuda())
    pos = torch.tensor([m.lens_l[i] - n + j for i, n in enumerate(m.new) for j in range(n)], dtype=torch.int32)
    kv, plain = m.kv_cuda(), m.kv_cuda()
    q = pkg.cache_append(kv, *args, k.cuda(), v.cuda(), q=m.q.cuda(), plan=plan, fmt=m.fmt)
    assert torch.equal(q, pkg.rope(m.q.cuda(), pos.cuda(), plan))
    same = m.q.cuda()
    again = m.kv_cuda()
    assert pkg.cache_append(again, *args, k.cuda(), v.cuda(), q=same, plan=plan, out=same, fmt=m.fmt) is same
    assert torch.equal(same, q) and torch.equal(again, kv)
    pkg.cache_append(plain, *args, k.cuda(), v.cuda(), fmt=m.fmt)
    got, got_v = pkg.cache_read(kv, *args, tokens, fmt=m.fmt)
    assert torch.equal(got_v, pkg.cache_read(plain, *args, tokens, fmt=m.fmt)[1])
    freqs = plan.freqs.cpu().numpy()
    want = A.turn(k.double(), pos, freqs, 1.25, interleaved)
    off = A.turn_bound(k.double(), pos, freqs, 1.25, interleaved, F32)
    b = np.abs(want).reshape(tokens, 2, -1, 32)
    # the factor: the largest element over 127, 7 or 8, rounded to fp16; a code is
    # then within half a step, but a largest element cut at 127, 7 or -8 by as
    # much as that rounding took off the factor (2^-11 of it)
    d16 = b.max(-1, keepdims=True) / (127 if kind == "q8_0" else 7) * (1 + 2.0 ** -10) + 2.0 ** -24
    bound = (d16 * (0.5 + 2.0 ** -10 * (127 if kind == "q8_0" else 8)) + 0 * b).reshape(want.shape) + 2 * off
    near(got, want, bound, "turned")


@pytest.mark.parametrize("kind", KINDS)
def test_blocks_of_unusual_elements(pkg, kind):
    """Zeros, fp32's and fp16's least numbers, elements beyond what a factor
    holds, equal ones, one sign alone; and what is not finite spoils its block."""
    d, page = 64, 16
    m = Made(pkg, kind, [16], [16], 1, 1, d, page, F32)
    g = torch.Generator().manual_seed(4)
    k = torch.randn(16, 1, d, generator=g)
    k[0] = 0.0
    k[1] *= 1e-42
    k[2] *= 1e-8
    k[3] *= 1e30
    k[4] *= 3e5
    k[5] = 2.5
    k[6] = -2.5
    k[7] = k[7].abs()
    k[8] = -k[8].abs()
    k[9, 0, 3] = math.inf
    k[10, 0, 40] = -math.inf
    k[11, 0, 63] = math.nan
    k[12] = -0.0
    k[13] *= 5e-7
    v = k.flip(0).contiguous()
    args = (m.table.cuda(), m.lens.cuda(), m.starts.cuda())
    kv = m.kv_cuda()
    pkg.cache_append(kv, *args, k.cuda(), v.cuda(), fmt=m.fmt)
    for got, x in zip(pkg.cache_read(kv, *args, 16, fmt=m.fmt), (k, v)):
        want = R.values(*R.blocks(x.numpy(), kind))
        got = got.cpu().numpy().astype(np.float64)
        assert np.array_equal(np.isnan(got), np.isnan(want))
        assert np.array_equal(got[~np.isnan(want)], want[~np.isnan(want)])
    assert int(np.isnan(want).sum()) == 3 * 32


@pytest.mark.parametrize("cache", [F32, F16, BF16], ids=NAME.get)
@pytest.mark.parametrize("d,page,token_major", [(64, 16, False), (80, 4, False), (8, 1, False), (256, 32, True)])
def test_read_of_wide_caches(pkg, cache, d, page, token_major):
    g = torch.Generator().manual_seed(d)
    kvh, lens, new = 3, [37, 5], [11, 5]
    shape = (80, 2, page, kvh, d) if token_major else (80, 2, kvh, page, d)
    kv = torch.randn(shape, generator=g).to(cache).cuda()
    if token_major:
        kv = kv.permute(0, 1, 3, 2, 4)
    per = -(-max(lens) // page)
    order = torch.randperm(kv.shape[0], generator=g)[:2 * per].view(2, per).int()
    table, ln, st = order.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), torch.tensor([0, 11, 16], dtype=torch.int32).cuda()
    pos = [(i, n - c + j) for i, (n, c) in enumerate(zip(lens, new)) for j in range(c)]
    for to in (F32, F16, BF16):
        k, v = pkg.cache_read(kv, table, ln, st, 16, dtype=to)
        for z, got in ((0, k), (1, v)):
            want = torch.stack([kv[int(order[i, p // page]), z, :, p % page] for i, p in pos])
            assert torch.equal(got, want.to(F32).to(to))


@pytest.mark.parametrize("kind", KINDS + [None])
def test_what_has_no_place(pkg, kind):
    """Slots out of range, lengths short of their rows, bad pages and rows of no
    sequence: nothing is written, the sequences' rows read as 0 and others stay."""
    d, page, kvh = 64, 16, 2
    fmt = None if kind is None else pkg.PageFormat(kind, kvh, page, d)
    kv = torch.zeros(4, 2, kvh, page, d).cuda() if kind is None else torch.zeros(4, fmt.page_bytes, dtype=torch.uint8).cuda()
    table = torch.tensor([[0, -1], [9, 1], [2, 3]], dtype=torch.int32).cuda()
    lens = torch.tensor([20, 18, 3], dtype=torch.int32).cuda()  # slot 2: 3 tokens, 5 rows
    starts = torch.tensor([2, 8, 12, 17, 19], dtype=torch.int32).cuda()
    slots = torch.tensor([0, 1, 2, 7], dtype=torch.int32).cuda()
    x = torch.randn(24, kvh, d, generator=torch.Generator().manual_seed(0)).cuda()
    pkg.cache_append(kv, table, lens, starts, x, x, slots=slots, fmt=fmt)
    out = torch.full((24, kvh, d), 7.0).cuda()
    k, v = pkg.cache_read(kv, table, lens, starts, 24, k=out, v=out.clone(), slots=slots, fmt=fmt)
    want = torch.zeros(24, dtype=torch.bool)
    want[2:4] = want[10:12] = want[14:17] = True  # positions 14, 15; 16, 17; 0 .. 2
    rest = torch.zeros(24, dtype=torch.bool)
    rest[:2] = rest[19:] = True
    for got in (k, v):
        got = got.cpu()
        assert bool((got[rest] == 7).all())
        assert bool((got[~want & ~rest] == 0).all())
        if kind is None:
            assert torch.equal(got[want], x.cpu()[want])
        else:
            assert np.array_equal(got[want].double().numpy(), R.values(*R.blocks(x.cpu()[want].numpy(), kind)))


# ---------------------------------------------------------------- attention


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=NAME.get)
@pytest.mark.parametrize("heads,kv_heads,d", [(4, 4, 64), (8, 2, 128), (7, 1, 96), (6, 2, 32), (16, 1, 192), (4, 1, 256),
                                              (20, 1, 128), (40, 1, 64), (3, 1, 160), (2, 2, 224)])
def test_attention_heads(pkg, kind, dtype, heads, kv_heads, d):
    say(f"[attention] {kind} {NAME[dtype]} {heads}/{kv_heads} d={d}")
    m = Made(pkg, kind, [1, 33, 70, 257, 16], [1, 1, 1, 1, 1], heads, kv_heads, d, 16, dtype, seed=heads + d)
    m.check(pkg, what="one token")
    m = Made(pkg, kind, [61, 129], [3, 2], heads, kv_heads, d, 32, dtype, seed=heads + d + 1)
    m.check(pkg, what="a few tokens")


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [F32, BF16], ids=NAME.get)
@pytest.mark.parametrize("page", [16, 32, 64, 256, 4096])
def test_attention_pages(pkg, kind, dtype, page):
    m = Made(pkg, kind, [5, 64, 65, 300, 0], [1, 1, 1, 1, 0], 8, 2, 64, page, dtype, seed=page)
    m.check(pkg)
    m.check(pkg, window=37, what="window")
    m.check(pkg, first=[0, 3, 60, 299, 1], what="first")
    m.check(pkg, first=[5, 64, 70, 17, 0], window=20, what="some without keys")


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=NAME.get)
@pytest.mark.parametrize("d", [64, 96, 128, 256])
@pytest.mark.parametrize("lens,new", [([70, 200], [70, 33]), ([513], [129]), ([300, 41, 9], [1, 40, 9]), ([131], [131])])
def test_attention_chunks(pkg, kind, dtype, d, lens, new):
    say(f"[chunks] {kind} {NAME[dtype]} d={d} {lens} {new}")
    m = Made(pkg, kind, lens, new, 4, 2, d, 16, dtype, seed=sum(lens) + d)
    m.check(pkg)
    m.check(pkg, window=50, what="window")
    m.check(pkg, first=[17] * len(lens), hints=False, what="first")


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [F32, BF16], ids=NAME.get)
def test_attention_long_single_token(pkg, kind, dtype):
    m = Made(pkg, kind, [20011, 3000], [1, 1], 8, 2, 64, 64, dtype, seed=5)
    m.check(pkg)
    m.check(pkg, window=4000)
    m.check(pkg, hints=False)

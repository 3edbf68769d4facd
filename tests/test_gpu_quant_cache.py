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


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=NAME.get)
def test_attention_rows_without_keys(pkg, kind, dtype):
    """Empty slots, slots out of range, pages out of range, lengths of zero and
    shorter than their rows, first keys behind the context."""
    m = Made(pkg, kind, [40, 0, 70, 33], [3, 2, 20, 1, 4], 4, 2, 64, 16, dtype, seed=3, slots=[0, 1, 2, 7, 3])
    m.table_l[0][1] = -1
    m.table_l[2][2] = 10 ** 6
    m.table_l[3][0] = -(2 ** 31)
    m.table = torch.tensor(m.table_l, dtype=torch.int32)
    m.check(pkg)
    m.check(pkg, first=[41, 0, 69, 32], what="first")
    m.check(pkg, window=1, what="itself alone")
    m.lens_l[3] = 2  # four rows, two tokens
    m.lens = torch.tensor(m.lens_l, dtype=torch.int32)
    m.check(pkg, what="short")


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [F32, BF16], ids=NAME.get)
@pytest.mark.parametrize("lens,new,heads,d", [([100], [1], 4, 64), ([90], [3], 4, 128), ([150], [60], 8, 64), ([150], [90], 8, 128),
                                              ([120, 40], [70, 1], 4, 256)])
def test_attention_blocks_that_are_not_finite(pkg, kind, dtype, lens, new, heads, d):
    """A value's factor of NaN reaches that block of the rows that see its key, a
    key's all of them; others stay what they are."""
    m = Made(pkg, kind, lens, new, heads, 2, d, 16, dtype, seed=d)
    m.check(pkg)
    bits = R.BITS[kind]
    codes, half = 16 * d * bits // 8, 16 * d * bits // 8 + 16 * d // 32 * 2
    n, c = lens[0], new[0]
    for what, key, block in ((1, n - 1, 0), (1, n - max(1, c // 2), d // 32 - 1), (0, n - max(1, c // 3), 1), (1, 0, 1)):
        raw = m.raw.copy()
        page, place = m.table_l[0][key // 16], key % 16
        o = (0 * 2 + what) * half + codes + (block * 16 + place) * 2  # kv head 0
        raw[page, o:o + 2] = np.array([np.nan], dtype=np.float16).view(np.uint8)
        for window in (0, 20):
            want, wl, ob, lb = R.attend(m.q, m.values(), kind, m.table_l, m.lens_l, m.starts_l, m.scale, window)  # all finite
            got, lse = pkg.paged_attention(m.q.cuda(), torch.from_numpy(raw).cuda(), m.table.cuda(), m.lens.cuda(), m.starts.cuda(),
                                           max(new), max(lens), window=window, lse=True, fmt=m.fmt)
            got, lse = got.cpu(), lse.cpu()
            pos = torch.arange(n - c, n)
            sees = (pos >= key) & ((pos - key < window) if window else True)
            hit = torch.zeros(got.shape, dtype=torch.bool)
            if what == 0:
                hit[:c, :heads // 2] = sees[:, None, None]
                assert torch.equal(torch.isnan(lse[:c, :heads // 2]), sees[:, None].expand(-1, heads // 2))
            else:
                hit[:c, :heads // 2, block * 32:block * 32 + 32] = sees[:, None, None]
            assert bool(torch.isnan(got[hit]).all()), (what, key, block, window)
            near(got, np.where(hit, np.nan, want), ob, f"{what} {key} {block} {window} out")
            if what == 1:
                near(lse, wl, lb, f"{what} {key} {block} {window} lse")


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=NAME.get)
@pytest.mark.parametrize("spread", [1e-4, 30.0, "tokens", "blocks"])
@pytest.mark.parametrize("lens,new", [([300], [1]), ([200], [3]), ([150], [70])])
def test_attention_factors_of_any_size(pkg, kind, dtype, spread, lens, new):
    """Small and large values, factors that differ by 2^10 between tokens or
    blocks (what lies below 2^-38 of the largest is in the bound)."""

    def contents(gen, shape):
        x = gen.standard_normal(shape).astype(np.float32)
        if spread == "tokens":
            x *= 2.0 ** gen.integers(-10, 1, shape[:4] + (1,)).astype(np.float32)
        elif spread == "blocks":
            x *= np.repeat(2.0 ** gen.integers(-10, 1, shape[:4] + (shape[4] // 32,)).astype(np.float32), 32, -1)
        else:
            x[:, 1] *= np.float32(spread)
        return x

    Made(pkg, kind, lens, new, 4, 2, 128, 16, dtype, seed=7, contents=contents).check(pkg)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=NAME.get)
@pytest.mark.parametrize("lens,new", [([60], [1]), ([130], [40])])
def test_attention_scales(pkg, kind, dtype, lens, new):
    m = Made(pkg, kind, lens, new, 4, 1, 64, 16, dtype, seed=9)
    for scale in (0.0, -0.125, 1.0, 1e-30, 30.0):
        m.check(pkg, scale=scale, what=f"scale {scale}")


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [F32, BF16], ids=NAME.get)
@pytest.mark.parametrize("lens,new", [([90], [1]), ([150], [40])])
def test_attention_one_key_far_above_the_others(pkg, kind, dtype, lens, new):
    """Scores of up to 10^8: the row's largest has all the weight, whose value is
    then the row (twice the output's half step, and the weight's part)."""
    m = Made(pkg, kind, lens, new, 4, 2, 64, 16, dtype, seed=11)
    for scale in (1e4, 1e7):
        got, lse = pkg.paged_attention(m.q.cuda(), m.kv_cuda(), m.table.cuda(), m.lens.cuda(), m.starts.cuda(), max(new),
                                       max(lens), scale=scale, lse=True, fmt=m.fmt)
        v = m.values()
        at = np.arange(lens[0])
        k, x = (v[np.array(m.table_l[0])[at // 16], z, :, at % 16] for z in (0, 1))
        for t in range(new[0]):
            n = lens[0] - new[0] + t + 1
            for h in range(4):
                s = k[:n, h // 2] @ m.q[t, h].double().numpy() * scale
                order = np.argsort(s)
                # (what fp32 cannot tell apart: 80 products and sums of the row)
                noise = np.abs(k[:n, h // 2]) @ np.abs(m.q[t, h].double().numpy()) * scale * 80 * 2.0 ** -24
                if s[order[-1]] - s[order[-2]] < 2 * noise.max() + 120:
                    continue
                want = x[order[-1], h // 2]
                off = np.abs(got[t, h].double().cpu().numpy() - want)
                # (elements next to 0 beside larger ones of their block: the weight times
                # the factor is rounded, not the element)
                assert (off <= np.abs(want) * (2 * R.HALF[dtype] + 2.0 ** -11) + 1e-30).all()
                assert abs(float(lse[t, h]) - s[order[-1]]) <= noise.max() + 2.0 ** -22 * abs(s[order[-1]])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [F32, BF16], ids=NAME.get)
def test_attention_strided_rows_and_rows_of_no_sequence(pkg, kind, dtype):
    m = Made(pkg, kind, [70, 55], [40, 3], 6, 2, 64, 16, dtype, seed=6)
    tokens = m.starts_l[-1]
    base = torch.zeros(6, tokens + 5, 64 + 3, dtype=dtype, device="cuda")
    q = base.permute(1, 0, 2)[2:2 + tokens, :, 1:65]
    q.copy_(m.q.cuda())
    dest = torch.full((tokens + 5, 7, 67), 7.0, dtype=dtype, device="cuda")
    m.check(pkg, q=q, out=dest[2:2 + tokens, :6, 1:65])
    assert bool((dest[:2] == 7).all()) and bool((dest[2 + tokens:] == 7).all())
    assert bool((dest[:, 6] == 7).all()) and bool((dest[..., 0] == 7).all()) and bool((dest[..., 65:] == 7).all())
    # padding before, behind and as sequences of no rows
    starts = torch.tensor([2, 2, 42, 42, 45], dtype=torch.int32).cuda()
    slots = torch.tensor([1, 0, 0, 1], dtype=torch.int32).cuda()
    pad = torch.zeros(tokens + 5, 6, 64, dtype=dtype, device="cuda")
    pad[2:45] = m.q.cuda()
    out, l = torch.full_like(pad, 7.0), torch.full((tokens + 5, 6), 7.0, device="cuda")
    pkg.paged_attention(pad, m.kv_cuda(), m.table.cuda(), m.lens.cuda(), starts, 40, 70, slots=slots, out=out, lse=l, fmt=m.fmt)
    right, rl, ob, lb = R.attend(m.q, m.values(), kind, m.table_l, m.lens_l, m.starts_l, m.scale)
    near(out[2:45], right, ob, "padded")
    near(l[2:45], rl, lb, "padded lse")
    for x in (out, l):
        assert bool((x[:2] == 7).all()) and bool((x[45:] == 7).all())


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype,heads,kv_heads,d", [(F32, 8, 2, 128), (BF16, 8, 2, 64), (F16, 28, 4, 128), (F32, 4, 1, 256), (BF16, 6, 2, 96)])
def test_attention_mixed_batches(pkg, kind, dtype, heads, kv_heads, d):
    lens, new = [300, 41, 90, 700, 64, 5], [130, 1, 30, 1, 2, 5]
    m = Made(pkg, kind, lens, new, heads, kv_heads, d, 32, dtype, seed=d)
    m.check(pkg)
    m.check(pkg, window=100, what="window")
    m.check(pkg, hints=False, what="no hints")
    # hints that are wrong either way
    args = (m.q.cuda(), m.kv_cuda(), m.table.cuda(), m.lens.cuda(), m.starts.cuda())
    want, lse, ob, lb = R.attend(m.q, m.values(), kind, m.table_l, m.lens_l, m.starts_l, m.scale)
    for max_new, max_len in ((1, 10), (1, 1 << 40), (1 << 20, 64), (0, 700)):
        got, l = pkg.paged_attention(*args, max_new, max_len, lse=True, fmt=m.fmt)
        near(got, want, ob, f"hints {max_new} {max_len}")
        near(l, lse, lb, f"hints {max_new} {max_len} lse")


@pytest.mark.parametrize("kind", KINDS)
def test_attention_many_empty_sequences(pkg, kind):
    m = Made(pkg, kind, [100], [30], 4, 2, 64, 16, F32, seed=1)
    want, _, ob, _ = R.attend(m.q, m.values(), kind, m.table_l, m.lens_l, m.starts_l, m.scale)
    n = 3000
    starts = torch.cat([torch.zeros(n, dtype=torch.int32), torch.tensor([0, 30], dtype=torch.int32), torch.full((n,), 30, dtype=torch.int32)]).cuda()
    slots = torch.zeros(2 * n + 1, dtype=torch.int32).cuda()
    args = (m.kv_cuda(), m.table.cuda(), m.lens.cuda(), starts)
    got = pkg.paged_attention(m.q.cuda(), *args, 30, 100, slots=slots, fmt=m.fmt)
    near(got, want, ob)
    k, v = pkg.cache_read(*args, 30, slots=slots, fmt=m.fmt)
    assert torch.equal(k, pkg.cache_read(m.kv_cuda(), m.table.cuda(), m.lens.cuda(), m.starts.cuda(), 30, fmt=m.fmt)[0])


@pytest.mark.parametrize("kind", KINDS)
def test_far_pages(pkg, kind):
    """Offsets beyond 32 bits: pages 2^29 bytes apart."""
    fmt = pkg.PageFormat(kind, 2, 16, 64)
    apart, pages = 1 << 29, 12
    far = torch.zeros(apart * (pages - 1) + fmt.page_bytes, dtype=torch.uint8, device="cuda").as_strided((pages, fmt.page_bytes), (apart, 1))
    near_ = torch.zeros(pages, fmt.page_bytes, dtype=torch.uint8, device="cuda")
    g = torch.Generator().manual_seed(2)
    table = torch.tensor([[11, 9, 10, 8, 1]], dtype=torch.int32).cuda()
    lens, n = torch.tensor([75], dtype=torch.int32).cuda(), 75
    k, v = (torch.randn(n, 2, 64, generator=g).cuda() for _ in range(2))
    q = torch.randn(n, 4, 64, generator=g).cuda()
    starts = torch.tensor([0, n], dtype=torch.int32).cuda()
    out = []
    for kv in (far, near_):
        pkg.cache_append(kv, table, lens, starts, k, v, fmt=fmt)
        one = torch.tensor([0, 1], dtype=torch.int32).cuda()
        out.append([*pkg.cache_read(kv, table, lens, starts, n, fmt=fmt), pkg.paged_attention(q, kv, table, lens, starts, n, n, fmt=fmt),
                    pkg.paged_attention(q[:1], kv, table, lens, one, 1, n, fmt=fmt)])
    assert torch.equal(far, near_)
    for a, b in zip(*out):
        assert torch.equal(a, b) and bool(a.abs().sum() > 0)


# ---------------------------------------------------------------- streams, graphs, refusals


@pytest.mark.parametrize("kind", KINDS)
def test_step_captured_and_replayed(pkg, kind):
    """Append, read and attention of a chunk and of single tokens in one graph,
    replayed over other inputs between eager work."""
    m = Made(pkg, kind, [150, 60, 2100], [40, 1, 1], 4, 2, 64, 16, F32, seed=4)
    kv, table, lens, starts = m.kv_cuda(), m.table.cuda(), m.lens.cuda(), m.starts.cuda()
    g = torch.Generator().manual_seed(8)
    ins = [(torch.randn(42, 4, 64, generator=g).cuda(), torch.randn(42, 2, 64, generator=g).cuda(), torch.randn(42, 2, 64, generator=g).cuda())
           for _ in range(4)]
    q, k, v = (x.clone() for x in ins[0])
    plan = pkg.rope_plan(64)

    def step():
        turned = pkg.cache_append(kv, table, lens, starts, k, v, q=q, plan=plan, fmt=m.fmt)
        return (turned, *pkg.cache_read(kv, table, lens, starts, 42, fmt=m.fmt),
                *pkg.paged_attention(turned, kv, table, lens, starts, 40, 2100, lse=True, fmt=m.fmt))

    want = []
    for x in ins:
        for to, fr in zip((q, k, v), x):
            to.copy_(fr)
        want.append([y.clone() for y in step()])
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            got = step()
    torch.cuda.current_stream().wait_stream(stream)
    for again in range(2):
        for x, w in zip(ins, want):
            for to, fr in zip((q, k, v), x):
                to.copy_(fr)
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(got, w):
                assert torch.equal(a, b)
            torch.randn(1000, 1000, device="cuda").sum().item()


def test_two_streams_at_once_and_same_bits(pkg):
    made = [Made(pkg, k, [500, 3000], [40, 1], 8, 2, 128, 32, t, seed=s) for s, (k, t) in enumerate([("q4_0", F32), ("q8_0", BF16)])]
    args = [(m.q.cuda(), m.kv_cuda(), m.table.cuda(), m.lens.cuda(), m.starts.cuda(), 40, 3000) for m in made]
    want = [pkg.paged_attention(*a, fmt=m.fmt).clone() for m, a in zip(made, args)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in made]
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(pkg.paged_attention(*args[i], fmt=made[i].fmt))
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert all(torch.equal(x, w) for x in g)


def test_refused_calls(pkg):
    m = Made(pkg, "q4_0", [40], [3], 4, 2, 64, 16, F32)
    kv, table, lens, starts, q = m.kv_cuda(), m.table.cuda(), m.lens.cuda(), m.starts.cuda(), m.q.cuda()
    k = torch.zeros(3, 2, 64).cuda()
    bad = pkg.SamplerError, AssertionError
    for kw in (dict(kv=kv[:, :-16]), dict(kv=kv.view(kv.shape[0], -1, 16)), dict(kv=kv.cpu()), dict(fmt=pkg.PageFormat("q8_0", 2, 16, 64)),
               dict(fmt=pkg.PageFormat("q4_0", 2, 8, 64)), dict(fmt=pkg.PageFormat("q4_0", 2, 16, 60)), dict(fmt=pkg.PageFormat("q5_0", 2, 16, 64)),
               dict(fmt=pkg.PageFormat("q4_0", 2, 24, 64)), dict(fmt=pkg.PageFormat("q4_0", 0, 16, 64)), dict(fmt=pkg.PageFormat("q4_0", 2, 16, 288))):
        a = dict(kv=kv, fmt=m.fmt)
        a.update(kw)
        with pytest.raises(bad):
            pkg.paged_attention(q, a["kv"], table, lens, starts, fmt=a["fmt"])
        with pytest.raises(bad):
            pkg.cache_append(a["kv"], table, lens, starts, k, k, fmt=a["fmt"])
        with pytest.raises(bad):
            pkg.cache_read(a["kv"], table, lens, starts, 3, fmt=a["fmt"])
    for kw in (dict(k=k.double()), dict(k=k[:, :1]), dict(v=k[:2]), dict(k=k.int())):
        a = dict(k=k, v=k)
        a.update(kw)
        with pytest.raises(bad):
            pkg.cache_append(kv, table, lens, starts, a["k"], a["v"], fmt=m.fmt)
        with pytest.raises(bad):
            pkg.cache_read(kv, table, lens, starts, 3, k=a["k"], v=a["v"], fmt=m.fmt)
    with pytest.raises(bad):
        pkg.cache_read(kv, table, lens, starts, 3, dtype=torch.float64, fmt=m.fmt)
    with pytest.raises(bad):
        pkg.paged_attention(q[..., :32], kv, table, lens, starts, fmt=m.fmt)
    with pytest.raises(bad):
        pkg.paged_attention(q, kv, table, lens, starts, scale=math.inf, fmt=m.fmt)
    # nothing to do is no error
    none = torch.zeros(1, dtype=torch.int32).cuda()
    pkg.cache_append(kv, table, lens, none, k[:0], k[:0], fmt=m.fmt)
    assert pkg.cache_read(kv, table, lens, none, 0, fmt=m.fmt)[0].shape == (0, 2, 64)
    assert pkg.paged_attention(q[:0], kv, table, lens, none, fmt=m.fmt).shape == (0, 4, 64)


# ---------------------------------------------------------------- together


@pytest.mark.parametrize("kind", KINDS)
def test_pages_of_blocks_forked_compacted_and_copied(pkg, kind):
    """The calls that move whole pages move pages of blocks as they are."""
    heads, d, page, layers = 2, 64, 16, 2
    cache = pkg.PagedCache(layers, 20, page, heads, d, 4, 6, dtype=kind)
    ints = lambda x: torch.tensor(x, dtype=torch.int32).cuda()
    g = torch.Generator().manual_seed(3)
    lens = [40, 33, 0, 16]
    starts = ints([0, 40, 73, 73, 89])
    assert int(cache.reserve(ints(lens))) == pkg.PAGES_DONE
    rows = [[torch.randn(89, heads, d, generator=g).cuda() for _ in range(2)] for _ in range(layers)]
    for i, (k, v) in enumerate(rows):
        cache.append(i, k, v, starts)
    before = [cache.read(i, starts, 89) for i in range(layers)]
    for (k, v), (a, b) in zip(rows, before):
        for x, y in ((k, a), (v, b)):
            codes, f = R.blocks(x.cpu().numpy(), kind)
            assert np.array_equal(y.cpu().double().numpy(), R.values(codes, f))
    assert int(cache.fork(ints([0]), ints([2]))) == pkg.PAGES_DONE
    assert cache.lens.tolist() == [40, 33, 40, 16]
    assert int(cache.release(ints([0]))) == pkg.PAGES_DONE
    assert int(cache.compact()) == 7 and cache.refs.tolist() == [1] * 7 + [0] * 13
    again, slots = ints([0, 33, 73, 89]), ints([1, 2, 3])
    for i, (a, b) in enumerate(before):
        for x, y in zip(cache.read(i, again, 89, slots=slots), (a, b)):
            assert torch.equal(x, torch.cat([y[40:73], y[:40], y[73:]]))
    used = cache.kv[:, :7].clone()
    pkg.cache_copy_pages(cache.kv, ints([0, 6]), ints([19, 10]), fmt=cache.fmt)
    assert torch.equal(cache.kv[:, [19, 10]], used[:, [0, 6]]) and torch.equal(cache.kv[:, :7], used)


@pytest.mark.parametrize("kind,dtype", [("q8_0", F32), ("q4_0", F32), ("q4_0", BF16)])
def test_beam_search_over_blocks(pkg, kind, dtype):
    """Prompts read as chunks, then steps of beam search over one cache of blocks:
    room, append, attention, logits by an F32 head, the best continuations, the
    contexts that follow them; each step against definitions over the contexts'
    own tokens, and in the end every context read back."""
    groups, beams, heads, kvh, d, page, vocab, layers = 2, 4, 4, 2, 64, 16, 501, 2
    rows, steps, prompts = groups * beams, 9, [37, 19]
    g = torch.Generator().manual_seed(12)
    # a model of its own: a token's q, k and v by tables, the layers' outputs summed
    tq, tk, tv = (torch.randn(layers, vocab, n, d, generator=g).to(dtype).cuda() for n in (heads, kvh, kvh))
    head = (torch.randn(vocab, heads * d, generator=g) / 8).cuda()
    raw = head.view(torch.uint8).reshape(-1)
    eog = torch.tensor([3], dtype=torch.int32).cuda()
    cache = pkg.PagedCache(layers, 64, page, kvh, d, rows, 10, dtype=kind)

    def run(tokens, starts, slots, max_new):
        hidden = 0
        for i in range(layers):
            cache.append(i, tk[i][tokens], tv[i][tokens], starts, slots=slots)
            hidden = hidden + cache.attend(i, tq[i][tokens], starts, slots=slots, max_new=max_new).float()
        return hidden.reshape(len(tokens), -1)

    def defined(context):
        """The logits after a context, in float64, and their bound."""
        t = torch.tensor(context)
        n, total, bound = len(context), 0, 0
        for i in range(layers):
            kv = np.empty((1, 2, kvh, n, d))
            for z, x in ((0, tk), (1, tv)):
                kv[0, z] = np.swapaxes(R.values(*R.blocks(x[i].cpu()[t].float().numpy(), kind)), 0, 1)
            out, _, ob, _ = R.attend(tq[i].cpu()[t[-1:]], kv, kind, [[0]], [n], [0, 1], d ** -0.5)
            total, bound = total + out, bound + ob
        w = head.cpu().double().numpy()
        total, bound = total.reshape(-1), bound.reshape(-1)
        size = np.abs(w) @ np.abs(total)  # the sums of the layers and of the products
        return w @ total, np.abs(w) @ bound + size * (heads * d + 4) * 2.0 ** -24

    contexts = [torch.randint(0, vocab, (n,), generator=g).tolist() for n in prompts]
    slots = torch.tensor([0, beams], dtype=torch.int32).cuda()
    need = torch.zeros(rows, dtype=torch.int32)
    need[0], need[beams] = prompts
    assert int(cache.reserve(need.cuda())) == pkg.PAGES_DONE
    starts = torch.tensor([0, prompts[0], sum(prompts)], dtype=torch.int32).cuda()
    hidden = run(torch.tensor(sum(contexts, [])).cuda(), starts, slots, max(prompts))
    first = hidden[(starts[1:] - 1).long()]
    # every beam of a group starts as its first one; the others are worth nothing
    parents = (torch.arange(rows) // beams * beams).int().cuda()
    assert int(cache.reorder(parents)) == pkg.PAGES_DONE
    contexts = [list(contexts[r // beams]) for r in range(rows)]
    scores = torch.full((groups, beams), -math.inf).cuda()
    scores[:, 0] = 0
    ended = torch.zeros(groups, beams, dtype=torch.int32).cuda()
    logits = pkg.lm_head(raw, 0, vocab, heads * d, first.repeat_interleave(beams, 0), exact=True)
    one = torch.arange(rows + 1, dtype=torch.int32).cuda()
    for step in range(steps):
        say(f"[beam search] {kind} {NAME[dtype]} step {step}")
        old, was = scores.cpu().double().numpy(), ended.cpu().numpy().reshape(-1)
        parents, tokens, scores, ended = pkg.beam_select(logits, scores, ended=ended, eog=eog)
        p, t, s, e = (x.reshape(-1).cpu() for x in (parents, tokens, scores, ended))
        # what was chosen is worth what the definitions say, and nothing left out is worth more
        for k in range(groups):
            worth, bound = np.full((beams, vocab + 1), -np.inf), np.zeros((beams, vocab + 1))  # (last: itself)
            for b in range(beams):
                r = k * beams + b
                if was[r]:
                    worth[b, -1] = old[k, b]
                elif old[k, b] > -math.inf:
                    y, by = defined(contexts[r])
                    assert (np.abs(logits[r].cpu().double().numpy() - y) <= by).all()
                    top = y.max()
                    lse = top + math.log(np.exp(y - top).sum())
                    worth[b, :-1], bound[b, :-1] = old[k, b] + y - lse, by + by.max() + (np.abs(old[k, b]) + np.abs(y) + abs(lse) + 8) * 2.0 ** -20
            mine = [(int(p[k * beams + b]), int(t[k * beams + b])) for b in range(beams)]
            assert len(set(mine)) == beams and all(x // beams == k for x, _ in mine)
            for b, (x, v) in enumerate(mine):
                assert abs(float(s[k * beams + b]) - worth[x % beams, v]) <= bound[x % beams, v]
                assert int(e[k * beams + b]) == int(bool(was[x]) or v == 3) and bool(was[x]) == (v == -1)
            least = min(float(s[k * beams + b]) for b in range(beams))
            rest = worth - bound
            for x, v in mine:
                rest[x % beams, v] = -np.inf
            assert rest.max() <= least + bound.max()
        assert int(cache.reorder(parents.reshape(-1))) == pkg.PAGES_DONE
        contexts = [contexts[int(x)] + ([] if was[int(x)] else [int(v)]) for x, v in zip(p, t)]
        # the ended ones wait: no new token of theirs
        going = [r for r in range(rows) if not was[int(p[r])]]
        need = torch.zeros(rows, dtype=torch.int32)
        need[going] = 1
        assert int(cache.reserve(need.cuda())) == pkg.PAGES_DONE
        assert cache.lens.tolist() == [len(c) for c in contexts]
        at = torch.tensor(going).cuda()
        hidden = run(t[going].cuda().long(), one[:len(going) + 1], at.int(), 1)
        logits = torch.zeros(rows, vocab, device="cuda")
        logits[at] = pkg.lm_head(raw, 0, vocab, heads * d, hidden, exact=True)
    starts = torch.tensor(np.concatenate([[0], np.cumsum([len(c) for c in contexts])]), dtype=torch.int32).cuda()
    t = torch.tensor(sum(contexts, []))
    for i in range(layers):
        for got, x in zip(cache.read(i, starts, len(t)), (tk, tv)):
            assert np.array_equal(got.cpu().double().numpy(), R.values(*R.blocks(x[i].cpu()[t].float().numpy(), kind)))


@pytest.mark.parametrize("kind", KINDS)
def test_beam_step_captured_and_replayed(pkg, kind):
    """A step of beam search as one graph: room, append, attention, choice and the
    contexts that follow, replayed over several steps beside the same steps alone."""
    groups, beams, heads, kvh, d, page, vocab = 2, 3, 4, 2, 64, 16, 300
    rows = groups * beams
    g = torch.Generator().manual_seed(1)
    head = (torch.randn(vocab, heads * d, generator=g) / 4).cuda()
    table = torch.randn(vocab, heads + 2 * kvh, d, generator=g).cuda()
    one, need = torch.arange(rows + 1, dtype=torch.int32).cuda(), torch.ones(rows, dtype=torch.int32).cuda()

    def made():
        cache = pkg.PagedCache(1, 40, page, kvh, d, rows, 7, dtype=kind)
        cache.reserve(torch.full((rows,), 13, dtype=torch.int32).cuda())
        x = torch.randn(rows * 13, 2 * kvh, d, generator=torch.Generator().manual_seed(5)).cuda()
        cache.append(0, x[:, :kvh], x[:, kvh:], one * 13)
        return [cache, torch.arange(rows, dtype=torch.int32).cuda() + 7, torch.zeros(groups, beams).cuda()]

    def step(cache, tokens, scores):
        cache.reserve(need)
        x = table.index_select(0, tokens)
        cache.append(0, x[:, heads:heads + kvh], x[:, heads + kvh:], one)
        y = cache.attend(0, x[:, :heads], one, max_new=1, max_len=112)
        logits = pkg.lm_head(head.view(torch.uint8).reshape(-1), 0, vocab, heads * d, y.reshape(rows, -1))
        parents, chosen, worth, _ = pkg.beam_select(logits, scores)
        cache.reorder(parents.reshape(-1))
        tokens.copy_(chosen.reshape(-1))
        scores.copy_(worth)
        return parents, y

    alone, captured, spare = made(), made(), made()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step(*spare)  # (what the calls set up once)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            got = step(*captured)
    torch.cuda.current_stream().wait_stream(stream)
    for i in range(20):
        want = step(*alone)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip((*got, *captured[1:]), (*want, *alone[1:])):
            assert torch.equal(a, b), i
        assert torch.equal(captured[0].lens, alone[0].lens)
    starts = (torch.arange(rows + 1, dtype=torch.int32) * 33).cuda()
    for a, b in zip(captured[0].read(0, starts, rows * 33), alone[0].read(0, starts, rows * 33)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=NAME.get)
@pytest.mark.parametrize("d", [32, 96, 160, 192, 224])
def test_attention_of_every_number_of_blocks_in_parts(pkg, kind, dtype, d):
    """Heads that fill no tile, keys split over workgroups, rows with gaps behind
    them that stay as they are, blocks that are not finite in unseen places."""
    m = Made(pkg, kind, [2100, 1300], [1, 70], 4, 2, d, 16, dtype, seed=d)
    dest = torch.full((71, 5, d + 8), 7.0, dtype=dtype, device="cuda")
    m.check(pkg, out=dest[:, :4, :d])
    assert bool((dest[:, 4] == 7).all()) and bool((dest[..., d:] == 7).all())
    m.check(pkg, window=300, first=[1900, 1000], what="window")


# The outputs' bound where small weights add up: a weight times its factor is one
# part of eleven bits (2^-11, and its factor or weight another's at most), scores and
# exponentials in fp32 are some 2^-18 of it, and sums of that many equal terms in
# fp32 lose at most 16384 2^-24.
SMALL = 2.0 ** -10 + 2.0 ** -10 + 2.0 ** -16


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=NAME.get)
@pytest.mark.parametrize("value", [1.0, 1e-3, 1e-4, 4e-5, 7000.0])
def test_attention_many_small_weights_and_values(pkg, kind, dtype, value):
    """Some keys of nearly all the weight whose values are 0, four of any 256 so that
    whoever sums has one, and 16128 equal ones of 2^-14.5 each, whose values are all
    alike: rounded one by one the same way, their sum would be off by as much as each."""
    page, d, lens = 4096, 64, [16384]

    def contents(gen, shape):
        x = np.zeros(shape, dtype=np.float32)
        x[:, 1] = value
        for far in (7, 39, 71, 103):
            x[:, 0, :, far::256] = 1.0
            x[:, 1, :, far::256] = 0.0
        return x

    m = Made(pkg, kind, lens, [1], 4, 1, d, page, dtype, seed=3, contents=contents)
    m.q = torch.ones(1, 4, d, dtype=dtype)
    scale = 14.5 * math.log(2.0) / d / float(m.values()[m.table_l[0][0], 0, 0, 7, 0])
    say(f"[small weights] {kind} {NAME[dtype]} {value}")
    want, lse, _, lb = R.attend(m.q, m.values(), kind, m.table_l, m.lens_l, m.starts_l, scale)
    got, l = pkg.paged_attention(m.q.cuda(), m.kv_cuda(), m.table.cuda(), m.lens.cuda(), m.starts.cuda(), 1, 16384,
                                 scale=scale, lse=True, fmt=m.fmt)
    # (fp16 outputs have a least step: half of 2^-24)
    near(got, want, np.abs(want) * (SMALL + R.HALF[dtype]) + (2.0 ** -25 if dtype == F16 else 0), f"{kind} {value}")
    near(l, lse, lb, "lse")


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=NAME.get)
@pytest.mark.parametrize("d", [32, 128, 256])
@pytest.mark.parametrize("lens,new", [([2], [2]), ([8], [7]), ([4, 40], [3, 2])])
def test_attention_a_neighbour_that_is_not_finite(pkg, kind, dtype, d, lens, new):
    """The last token's values are NaN in every block, and the tokens before it have
    the only finite ones or by far the largest: rows that do not see it are as without it."""
    def contents(gen, shape):
        x = gen.standard_normal(shape).astype(np.float32)
        x[:, 1] *= 1e-3
        x[:, 1, :, min(lens) - 2] = 50.0
        x[:, 1, :, min(lens) - 1] = np.nan
        return x

    m = Made(pkg, kind, lens, new, 2, 1, d, 64, dtype, seed=d, contents=contents)
    say(f"[nan neighbour] {kind} {NAME[dtype]} d={d} {lens}")
    got, _ = m.check(pkg)
    assert torch.isfinite(got[:new[0] - 1].float()).all() and torch.isnan(got[new[0] - 1].float()).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype,rot,interleaved,off", [(F32, 64, False, 0), (BF16, 64, True, 0), (F16, 32, False, 1), (BF16, 0, False, 0)])
def test_many_tokens_are_written_and_read_as_few_are(pkg, kind, dtype, rot, interleaved, off):
    """A call of so many tokens that a workgroup takes several at a time, of ragged
    and empty sequences, against the same sequences in calls that do not."""
    d, kvh, heads, page, seqs, slots = 96, 2, 3, 16, 190, 200
    rng, g = random.Random(rot + off), torch.Generator().manual_seed(rot)
    new = [rng.choice([0, 0, 1, 2, 7, 19, 40]) for _ in range(seqs - 1)] + [600]
    cut = 90
    lens = [rng.randint(0, 60) for _ in range(slots)]
    slot_of = rng.sample(range(slots), seqs)
    slot_of[3], slot_of[5] = -1, slots + 4
    for i in range(seqs):
        if 0 <= slot_of[i] < slots and i % 7:
            lens[slot_of[i]] += new[i]  # else some are shorter than their rows
    per = 45
    table = [[rng.choice([-1, 10 ** 6]) if rng.random() < 0.05 else s * per + j for j in range(per)] for s in range(slots)]
    starts = [5]
    for n in new:
        starts.append(starts[-1] + n)
    tokens = starts[-1] + 9
    assert tokens > 2048
    fmt = pkg.PageFormat(kind, kvh, page, d)
    ints = lambda x: torch.tensor(x, dtype=torch.int32).cuda()
    rows = [torch.randn(tokens, h, d + off, generator=g).to(dtype).cuda()[..., off:] for h in (heads, kvh, kvh)]
    plan = pkg.rope_plan(rot, interleaved=interleaved) if rot else None
    tb, ln, sl = ints(table), ints(lens), ints(slot_of)
    fill = torch.randint(0, 120, (slots * per, fmt.page_bytes), dtype=torch.uint8, generator=g).cuda()  # (no factor is NaN)
    whole, parts = fill.clone(), fill.clone()
    out, k, v = (torch.full_like(x, 7) for x in rows)
    pkg.cache_append(whole, tb, ln, ints(starts), rows[1], rows[2], q=rows[0], plan=plan, slots=sl, out=out, fmt=fmt)
    pkg.cache_read(whole, tb, ln, ints(starts), tokens, k=k, v=v, slots=sl, fmt=fmt)
    out2, k2, v2 = (torch.full_like(x, 7) for x in rows)
    for a, b in ((0, cut), (cut, seqs)):
        lo, hi = (0 if a == 0 else starts[a]), (tokens if b == seqs else starts[b])
        assert hi - lo < 2048
        st, part = ints([s - lo for s in starts[a:b + 1]]), slice(lo, hi)
        pkg.cache_append(parts, tb, ln, st, rows[1][part], rows[2][part], q=rows[0][part], plan=plan, slots=sl[a:b], out=out2[part], fmt=fmt)
        pkg.cache_read(parts, tb, ln, st, hi - lo, k=k2[part], v=v2[part], slots=sl[a:b], fmt=fmt)
    assert torch.equal(whole, parts) and not torch.equal(whole, fill)
    for x, y in ((out, out2), (k, k2), (v, v2)):
        assert torch.equal(x, y) and bool((x[:5] == 7).all()) and bool((x[-9:] == 7).all())


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [F32, BF16], ids=NAME.get)
@pytest.mark.parametrize("max_new,max_len", [(1, 1), (1, 100000), (4096, 1), (7, 600)])
def test_attention_hints_that_are_wrong(pkg, kind, dtype, max_new, max_len):
    m = Made(pkg, kind, [700, 90, 1, 1300], [50, 3, 1, 1], 8, 2, 64, 32, dtype, seed=max_new)
    for window, first in ((0, None), (65, [3, 0, 0, 1200])):
        want, lse, ob, lb = R.attend(m.q, m.values(), kind, m.table_l, m.lens_l, m.starts_l, m.scale, window, first)
        f = None if first is None else torch.tensor(first, dtype=torch.int32).cuda()
        got, l = pkg.paged_attention(m.q.cuda(), m.kv_cuda(), m.table.cuda(), m.lens.cuda(), m.starts.cuda(), max_new=max_new,
                                     max_len=max_len, window=window, first=f, lse=True, fmt=m.fmt)
        near(got, want, ob, "out")
        near(l, lse, lb, "lse")


@pytest.mark.parametrize("kind,value", [("q8_0", 7.6e-6), ("q4_0", 4.2e-7), ("q4_0", 3e-6)])
def test_attention_factors_of_denormal_size(pkg, kind, value):
    """Values whose factors are the least that fp16 holds, and small weights: their
    product is 22 bits of fp32 queries' all the same."""
    d, n = 64, 512

    def contents(gen, shape):
        x = np.zeros(shape, dtype=np.float32)
        x[:, 0], x[:, 1] = -0.027, value
        for far in (7, 39, 71, 103):
            x[:, 0, :, far::256] = 1.0
            x[:, 1, :, far::256] = 0.0
        return x

    m = Made(pkg, kind, [n], [1], 4, 1, d, 512, F32, seed=3, contents=contents)
    m.q = torch.ones(1, 4, d)
    scale = 20.3 * math.log(2.0) / d / float(m.values()[m.table_l[0][0], 0, 0, 7, 0])
    want, _, _, _ = R.attend(m.q, m.values(), kind, m.table_l, m.lens_l, m.starts_l, scale)
    assert (want > 0).all()
    got = pkg.paged_attention(m.q.cuda(), m.kv_cuda(), m.table.cuda(), m.lens.cuda(), m.starts.cuda(), 1, n, scale=scale, fmt=m.fmt)
    # scores of 20 (in exponents of base 2): 64 products and sums, a rounding each of
    # factor, scale and exponent, 70 * 20 * 2^-24; exponentials, the two parts, and
    # sums of 512 terms in fp32
    near(got, want, np.abs(want) * (70 * 20 * 2.0 ** -24 + 2.0 ** -21 + 2 * 528 * 2.0 ** -24 + 2.0 ** -23), kind)

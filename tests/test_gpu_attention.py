"""Rotary positions, the paged cache and attention against their definitions in
float64 (tests/attention_ref.py), at the sizes, layouts and masks where they can
go wrong.  Counterpart: rope and attnTask over the dense cache of nimllm's
forward pass (src/nimllm/model.nim:300-302, :362-393, :446)."""
import math
import random
import sys

import numpy as np
import pytest
import torch

import attention_ref as R

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
PAIRS = [(F32, F32), (F32, F16), (F32, BF16), (F16, F16), (BF16, BF16)]
NAME = {F32: "f32", F16: "f16", BF16: "bf16"}


def say(*a):
    print(*a, flush=True)
    sys.stdout.flush()


def near(got, want, bound, what=""):
    """|got - want| within the bound element by element; infinities and zeros of
    rows without a key equal."""
    g, w, b = (np.asarray(torch.as_tensor(x).double().cpu()) for x in (got, want, bound))
    live = ~np.isnan(w)
    same = g[live] == w[live]
    with np.errstate(invalid="ignore"):
        off = np.abs(g[live] - w[live])
    ok = same | (off <= b[live])
    assert ok.all(), f"{what}: {np.count_nonzero(~ok)} of {ok.size} off, worst {np.nanmax(np.where(ok, 0, off / np.maximum(b[live], 1e-300)))} bounds"


# ---------------------------------------------------------------- rotary positions


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=NAME.get)
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("tokens,heads,d,rot", [(1, 1, 2, 2), (1, 32, 64, 64), (7, 3, 80, 38), (33, 5, 96, 48),
                                                (130, 8, 128, 128), (3, 2, 256, 192), (2, 3, 128, 0)])
def test_rope(pkg, dtype, interleaved, tokens, heads, d, rot):
    say(f"[rope] {NAME[dtype]} interleaved={interleaved} {tokens}x{heads}x{d} rot {rot}")
    g = torch.Generator().manual_seed(tokens * 1000 + d + rot)
    x = torch.randn(tokens, heads, d, generator=g).to(dtype)
    pos = torch.randint(-5, 1_000_000, (tokens,), generator=g, dtype=torch.int32)
    freqs = [10000.0 ** (-2.0 * j / max(rot, 1)) for j in range(rot // 2)]
    plan = pkg.RopePlan(torch.tensor(freqs, dtype=torch.float64).cuda(), interleaved, 1.25)
    for inverse in (False, True):
        want = R.turn(x.double(), pos, freqs, 1.25, interleaved, -1.0 if inverse else 1.0)
        bound = R.turn_bound(x.double(), pos, freqs, 1.25, interleaved, dtype)
        got = pkg.rope(x.cuda(), pos.cuda(), plan, inverse=inverse)
        near(got, want, bound, "fresh")
        assert torch.equal(got[..., rot:].cpu(), x[..., rot:])
        # in place, and from and to strided rows that start off 16 bytes
        y = x.cuda()
        assert pkg.rope(y, pos.cuda(), plan, inverse=inverse, out=y) is y
        assert torch.equal(y, got)
        wide = torch.zeros(heads, tokens, d + 3, dtype=dtype, device="cuda")
        part = wide.permute(1, 0, 2)[..., 1:1 + d]
        part.copy_(x.cuda())
        dest = torch.full((tokens, heads + 1, d + 1), 7.0, dtype=dtype, device="cuda")
        pkg.rope(part, pos.cuda(), plan, inverse=inverse, out=dest[:, :heads, :d])
        assert torch.equal(dest[:, :heads, :d], got)
        assert bool((dest[:, heads] == 7).all()) and bool((dest[..., d] == 7).all())


def test_rope_gradient(pkg):
    """The inverse is the transpose: <rope(x), g> = <x, inverse(g)>, and the
    gradient agrees with differences of the float64 definition."""
    g = torch.Generator().manual_seed(3)
    x, up = torch.randn(5, 2, 64, generator=g), torch.randn(5, 2, 64, generator=g)
    pos = torch.tensor([0, 1, 17, 4000, 131071], dtype=torch.int32)
    plan = pkg.rope_plan(48, interleaved=False, scaling="yarn", base=500000.0, factor=8.0, original_context=4096.0)
    freqs = plan.freqs.cpu().numpy()
    got = pkg.rope(up.cuda(), pos.cuda(), plan, inverse=True).cpu().double()
    bound = R.turn_bound(up.double(), pos, freqs, plan.amplitude, False, F32)
    near(got, R.turn(up.double(), pos, freqs, plan.amplitude, False, -1.0), bound, "formula")
    f = lambda z: float((torch.from_numpy(R.turn(z, pos, freqs, plan.amplitude, False)) * up.double()).sum())
    for t, h, i in [(0, 0, 0), (1, 1, 5), (2, 0, 24), (3, 1, 47), (4, 0, 60), (4, 1, 23)]:
        z = x.double().numpy().copy()
        z[t, h, i] += 1e-3
        a = f(z)
        z[t, h, i] -= 2e-3
        # linear: the difference is exact but for float64 sums of 640 terms
        assert abs((a - f(z)) / 2e-3 - float(got[t, h, i])) <= bound[t, h, i] + 640 * 2.0 ** -53 * 200 / 2e-3


def test_rope_plan_kinds(pkg):
    for kw in (dict(), dict(scaling="linear", factor=4.0), dict(scaling="yarn", factor=16.0, original_context=4096.0),
               dict(freq_factors=[1.0 + 0.1 * j for j in range(32)])):
        plan = pkg.rope_plan(64, **kw)
        freqs, amp = pkg.rope_frequencies(64, **kw)
        assert plan.freqs.tolist() == freqs and plan.amplitude == amp


# ---------------------------------------------------------------- the cache


class Made:
    """A cache of one layer with random contents, every place of it that no
    context holds NaN, and the chunks of a call."""

    def __init__(self, lens, new, heads, kv_heads, d, page, dtype, cache, seed=0, token_major=False, slots=None,
                 spread=2.0, slack=3):
        g = torch.Generator().manual_seed(seed)
        rng = random.Random(seed)
        self.lens_l, self.new, self.page = list(lens), list(new), page
        per = max([-(-n // page) for n in lens] + [1]) + 1
        total = sum(-(-n // page) for n in lens) + slack
        order = list(range(total))
        rng.shuffle(order)
        shape = (total, 2, page, kv_heads, d) if token_major else (total, 2, kv_heads, page, d)
        kv = torch.full(shape, math.nan, dtype=cache)
        if token_major:
            kv = kv.permute(0, 1, 3, 2, 4)
        self.table_l = []
        for n in lens:
            row = [order.pop() for _ in range(-(-n // page))]
            self.table_l.append(row + [-1] * (per - len(row)))
            for j in range(len(row)):
                m = min(page, n - j * page)
                kv[row[j], :, :, :m] = torch.randn(2, kv_heads, m, d, generator=g).to(cache)
        self.kv = kv
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

    def kv_cuda(self):
        """The cache on the GPU with its own strides."""
        out = torch.empty_strided(self.kv.shape, self.kv.stride(), dtype=self.kv.dtype, device="cuda")
        return out.copy_(self.kv)

    def check(self, pkg, window=0, first=None, hints=True, what="", q=None, out=None, **kw):
        want, lse, ob, lb = R.attend(self.q, self.kv, self.table_l, self.lens_l, self.starts_l, self.scale, window,
                                     first, self.slots_l)
        f = None if first is None else torch.tensor(first, dtype=torch.int32).cuda()
        got, l = pkg.paged_attention(self.q.cuda() if q is None else q, self.kv_cuda(), self.table.cuda(),
                                     self.lens.cuda(), self.starts.cuda(),
                                     max_new=max(self.new + [0]) if hints else 0,
                                     max_len=max(self.lens_l + [0]) if hints else 0, window=window, first=f,
                                     slots=None if self.slots is None else self.slots.cuda(), lse=True, out=out, **kw)
        near(got, want, ob, what + " out")
        near(l, lse, lb, what + " lse")
        return got, l


@pytest.mark.parametrize("dtype,cache", PAIRS, ids=lambda t: NAME[t])
@pytest.mark.parametrize("heads,kv_heads,d", [(4, 4, 64), (8, 2, 128), (7, 1, 80), (6, 2, 8), (16, 1, 96), (4, 1, 256),
                                              (20, 1, 64), (3, 3, 136)])
def test_attention_heads(pkg, dtype, cache, heads, kv_heads, d):
    """Single tokens and short chunks over every head layout, with and without
    what the caller knows of the lengths."""
    for lens, new in (([1, 37, 130], [1, 1, 1]), ([70, 5, 33], [3, 5, 0])):
        say(f"[attend] {NAME[dtype]}/{NAME[cache]} {heads}/{kv_heads}x{d} lens {lens} new {new}")
        m = Made(lens, new, heads, kv_heads, d, 16, dtype, cache, seed=heads * d)
        a = m.check(pkg, what="hints")
        b = m.check(pkg, hints=False, what="no hints")
        assert a[0].shape == b[0].shape


@pytest.mark.parametrize("dtype,cache", PAIRS, ids=lambda t: NAME[t])
@pytest.mark.parametrize("page,token_major", [(1, False), (8, True), (64, False), (256, True)])
def test_attention_pages(pkg, dtype, cache, page, token_major):
    """Pages of one token, pages that end inside a tile, and both orders of heads
    and tokens within a page; lengths around every power of two."""
    lens = [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257]
    say(f"[attend] pages of {page} {NAME[dtype]}/{NAME[cache]}")
    Made(lens, [1] * len(lens), 4, 2, 64, page, dtype, cache, seed=page, token_major=token_major).check(pkg)


@pytest.mark.parametrize("dtype,cache", PAIRS, ids=lambda t: NAME[t])
@pytest.mark.parametrize("lens,new", [([200], [200]), ([333, 64, 129], [77, 64, 1]), ([150, 1, 90], [128, 1, 33]),
                                      ([70, 0, 300, 41], [1, 0, 150, 41])])
def test_attention_chunks(pkg, dtype, cache, lens, new):
    for window, first in ((0, None), (50, None), (0, [3 + i for i in range(len(lens))]), (1, None)):
        say(f"[attend] chunks {NAME[dtype]}/{NAME[cache]} lens {lens} new {new} window {window} first {first}")
        Made(lens, new, 4, 2, 64, 16, dtype, cache, seed=sum(lens)).check(pkg, window=window, first=first)


@pytest.mark.parametrize("dtype,cache", PAIRS, ids=lambda t: NAME[t])
def test_attention_chunk_wide_heads(pkg, dtype, cache):
    for heads, kv_heads, d in ((6, 2, 128), (5, 1, 256), (3, 3, 72)):
        say(f"[attend] chunk {NAME[dtype]}/{NAME[cache]} {heads}/{kv_heads}x{d}")
        Made([190, 40], [101, 40], heads, kv_heads, d, 32, dtype, cache, seed=d).check(pkg, window=0)


@pytest.mark.parametrize("dtype,cache", PAIRS, ids=lambda t: NAME[t])
def test_attention_long_single_token(pkg, dtype, cache):
    """A long axis, split over workgroups and joined; a first key and a window
    inside it."""
    for window, first in ((0, None), (1000, None), (0, [4999, 0]), (0, [5001, 7])):
        say(f"[attend] long {NAME[dtype]}/{NAME[cache]} window {window} first {first}")
        Made([5001, 2900], [1, 1], 4, 1, 64, 64, dtype, cache, seed=9).check(pkg, window=window, first=first)


def test_attention_true_lengths_beyond_the_hints(pkg):
    m = Made([900, 700], [3, 40], 8, 2, 64, 16, F32, F16, seed=4)
    want, lse, ob, lb = R.attend(m.q, m.kv, m.table_l, m.lens_l, m.starts_l, m.scale)
    for max_new, max_len in ((1, 16), (1, 0), (0, 1), (43, 100000), (2, 300)):
        say(f"[attend] hints {max_new} {max_len}")
        got, l = pkg.paged_attention(m.q.cuda(), m.kv_cuda(), m.table.cuda(), m.lens.cuda(), m.starts.cuda(), max_new,
                                     max_len, lse=True)
        near(got, want, ob)
        near(l, lse, lb)


@pytest.mark.parametrize("dtype,cache", PAIRS, ids=lambda t: NAME[t])
def test_attention_rows_without_keys(pkg, dtype, cache):
    """Empty slots, slots shorter than their new tokens, a first key behind the
    row, slots out of range, pages out of range: zeros and -infinity."""
    m = Made([40, 0, 2, 30], [2, 3, 4, 20], 4, 2, 64, 16, dtype, cache, seed=1)
    m.check(pkg, what="short")
    m.check(pkg, first=[39, 0, 0, 25], what="first")
    m.check(pkg, first=[-7, 2 ** 31 - 1, 5, 2 ** 31 - 1], what="far first")
    m = Made([40, 30, 20], [2, 3, 18, 1], 4, 2, 64, 16, dtype, cache, seed=2, slots=[-1, 2, 1, 3])
    m.check(pkg, what="slots")
    m = Made([100, 90], [1, 50], 4, 2, 64, 16, dtype, cache, seed=3)
    for row, at, page in ((0, 2, -1), (1, 0, m.kv.shape[0]), (1, 3, 2 ** 31 - 1), (0, 6, -2 ** 31)):
        m.table_l[row][at] = page
    m.table = torch.tensor(m.table_l, dtype=torch.int32)
    m.check(pkg, what="pages")


@pytest.mark.parametrize("dtype,cache", PAIRS, ids=lambda t: NAME[t])
def test_attention_masked_values_do_not_reach_a_row(pkg, dtype, cache):
    """Infinities and NaN in the keys and values that only later rows of a chunk
    see, or that none sees: the other rows come out as without them."""
    for lens, new, bad in (([37, 60], [4, 2], [(0, 34), (0, 36), (1, 59)]), ([130, 90], [90, 60], [(0, 60), (0, 129), (1, 77)])):
        for value in (math.nan, math.inf):
            say(f"[attend] masked {value} {NAME[dtype]}/{NAME[cache]} lens {lens}")
            m = Made(lens, new, 4, 2, 64, 16, dtype, cache, seed=6)
            clean = R.attend(m.q, m.kv, m.table_l, m.lens_l, m.starts_l, m.scale)
            for s, j in bad:
                m.kv[m.table_l[s][j // 16], :, :, j % 16] = value
            got, lse = pkg.paged_attention(m.q.cuda(), m.kv_cuda(), m.table.cuda(), m.lens.cuda(), m.starts.cuda(),
                                           max(new), max(lens), lse=True)
            for i in range(2):
                firstbad = min(j for s, j in bad if s == i)
                n = max(0, firstbad - (lens[i] - new[i]))
                a = m.starts_l[i]
                near(got[a:a + n], clean[0][a:a + n], clean[2][a:a + n], f"seq {i}")
                near(lse[a:a + n], clean[1][a:a + n], clean[3][a:a + n], f"seq {i} lse")
                if math.isnan(value):
                    assert bool(torch.isnan(got[a + n:a + new[i]]).all())
    # behind a first key and outside a window
    m = Made([300], [40], 4, 2, 64, 16, dtype, cache, seed=8)
    clean = R.attend(m.q, m.kv, m.table_l, m.lens_l, m.starts_l, m.scale, 64, [240])
    for j in list(range(0, 200)) + [239]:
        m.kv[m.table_l[0][j // 16], :, :, j % 16] = math.nan
    got, lse = pkg.paged_attention(m.q.cuda(), m.kv_cuda(), m.table.cuda(), m.lens.cuda(), m.starts.cuda(), 40, 300,
                                   window=64, first=torch.tensor([240], dtype=torch.int32).cuda(), lse=True)
    near(got, clean[0], clean[2])
    near(lse, clean[1], clean[3])


@pytest.mark.parametrize("dtype,cache", PAIRS, ids=lambda t: NAME[t])
@pytest.mark.parametrize("lens,new", [([37, 60], [4, 2]), ([130, 90], [130, 60]), ([300], [300]), ([700, 40], [150, 1])])
def test_attention_infinite_values_reach_the_rows_that_see_them(pkg, dtype, cache, lens, new):
    """An infinity or NaN among the values alone: every row that sees its key is
    infinite or NaN there, in that element and no other, and the rows that do not
    see it come out as without it."""
    say(f"[attend] infinite values {NAME[dtype]}/{NAME[cache]} lens {lens} new {new}")
    m = Made(lens, new, 4, 2, 64, 16, dtype, cache, seed=9)
    want, _, bound, _ = R.attend(m.q, m.kv, m.table_l, m.lens_l, m.starts_l, m.scale)
    want, bound = want.clone(), bound.clone()
    sees = torch.zeros(want.shape, dtype=torch.bool)
    for s, j, h, e, value in ((0, 5, 0, 3, math.inf), (0, lens[0] - new[0] + new[0] // 2, 1, 40, math.nan),
                              (0, lens[0] - 1, 1, 63, -math.inf), (len(lens) - 1, 0, 0, 17, math.inf)):
        m.kv[m.table_l[s][j // 16], 1, h, j % 16, e] = value
        for t in range(new[s]):
            if lens[s] - new[s] + t >= j:
                sees[m.starts_l[s] + t, 2 * h:2 * h + 2, e] = True
    got = pkg.paged_attention(m.q.cuda(), m.kv_cuda(), m.table.cuda(), m.lens.cuda(), m.starts.cuda(), max(new),
                              max(lens)).double().cpu()
    assert not bool(torch.isfinite(got[sees]).any()), f"{int(torch.isfinite(got[sees]).sum())} of {int(sees.sum())} finite"
    want[sees] = math.nan
    near(got, want, bound)


def test_attention_scores_of_minus_infinity(pkg):
    """A key whose score is -infinity weighs nothing; a row with none else is
    empty."""
    m = Made([20, 3], [1, 1], 2, 1, 64, 16, F32, F32, seed=2)
    m.q[:] = m.q.abs()
    for j in (4, 5, 19):
        m.kv[m.table_l[0][j // 16], 0, :, j % 16] = -math.inf
    for j in range(3):
        m.kv[m.table_l[1][0], 0, :, j] = -math.inf
    got, lse = pkg.paged_attention(m.q.cuda(), m.kv_cuda(), m.table.cuda(), m.lens.cuda(), m.starts.cuda(), 1, 20,
                                   lse=True)
    want = R.attend(m.q, m.kv, m.table_l, m.lens_l, m.starts_l, m.scale)
    keep = [j for j in range(20) if j not in (4, 5, 19)]
    rows = torch.stack([m.kv[m.table_l[0][j // 16], :, :, j % 16] for j in keep]).double()
    for h in range(2):
        p = torch.softmax(rows[:, 0, 0] @ m.q[0, h].double() * m.scale, 0)
        near(got[0, h], p @ rows[:, 1, 0], torch.full((64,), 1e-5, dtype=torch.float64))
    assert bool((got[1] == 0).all()) and bool((lse[1] == -math.inf).all())
    del want


@pytest.mark.parametrize("dtype,cache", PAIRS, ids=lambda t: NAME[t])
@pytest.mark.parametrize("lens,new", [([150, 40], [150, 3]), ([400, 70], [100, 1])])
def test_attention_keys_of_minus_infinity(pkg, dtype, cache, lens, new):
    """Keys of -infinity under queries above 0 are as if they were not there; fp32
    queries over 16-bit keys may have NaN for them, and only in rows that see one."""
    say(f"[attend] keys of -infinity {NAME[dtype]}/{NAME[cache]} lens {lens}")
    m = Made(lens, new, 4, 2, 64, 1, dtype, cache, seed=12)
    m.q = m.q.abs() + 0.125
    gone = [(0, j) for j in (0, 1, 7, 63, 64, 100, lens[0] - 1)] + [(1, j) for j in range(0, 40, 2)]
    without = [list(r) for r in m.table_l]
    for s, j in gone:
        without[s][j] = -1
    want, lse, ob, lb = R.attend(m.q, m.kv, without, m.lens_l, m.starts_l, m.scale)
    for s, j in gone:
        m.kv[m.table_l[s][j], 0, :, 0] = -math.inf
    got, l = pkg.paged_attention(m.q.cuda(), m.kv_cuda(), m.table.cuda(), m.lens.cuda(), m.starts.cuda(), max(new),
                                 max(lens), lse=True)
    if dtype == F32 and cache != F32:
        # (the first key is -infinity: every row sees one)
        got, l = got.double().cpu(), l.double().cpu()
        want, lse = want.clone(), lse.clone()
        want[torch.isnan(got)], lse[torch.isnan(l)] = math.nan, math.nan
    near(got, want, ob)
    near(l, lse, lb)


def test_attention_large_scores(pkg):
    """Scores of hundreds, either sign, and queries beyond fp16's range: the
    maximum leaves before the exponential."""
    for dtype, cache in PAIRS:
        if dtype == F16:
            continue
        say(f"[attend] large {NAME[dtype]}/{NAME[cache]}")
        Made([300, 77], [1, 30], 4, 2, 64, 16, dtype, cache, seed=5, spread=100.0).check(pkg)
    m = Made([40], [2], 2, 1, 64, 16, F32, F16, seed=5, spread=1e6)
    m.scale = 64 ** -0.5 * 1e-5
    m.check(pkg, scale=m.scale, what="queries of 1e6")
    m = Made([40], [2], 2, 1, 64, 16, F32, F16, seed=5, spread=1e-9)
    m.scale = 64 ** -0.5 * 1e9
    m.check(pkg, scale=m.scale, what="queries of 1e-9")


@pytest.mark.parametrize("dtype,cache", PAIRS, ids=lambda t: NAME[t])
def test_attention_scales(pkg, dtype, cache):
    """Negative scales, zero (every key weighs the same), and scores of 10^8 and
    more, where a row goes to its largest score's value and stays finite."""
    for scale in (-0.2, 0.0):
        say(f"[attend] scale {scale} {NAME[dtype]}/{NAME[cache]}")
        m = Made([300, 90], [1, 40], 4, 2, 64, 16, dtype, cache, seed=21)
        m.scale = scale
        m.check(pkg, scale=scale)
    for scale in (1e8, 1e30, -1e30):
        say(f"[attend] scale {scale} {NAME[dtype]}/{NAME[cache]}")
        m = Made([300, 90], [1, 40], 4, 2, 64, 16, dtype, cache, seed=22)
        got = pkg.paged_attention(m.q.cuda(), m.kv_cuda(), m.table.cuda(), m.lens.cuda(), m.starts.cuda(), 40, 300,
                                  scale=scale).cpu()
        assert bool(torch.isfinite(got).all())
        seen = 0
        for i in range(2):
            for t in range(m.starts_l[i], m.starts_l[i + 1]):
                n = m.lens_l[i] - m.starts_l[i + 1] + t + 1
                rows = torch.stack([m.kv[m.table_l[i][j // 16], :, :, j % 16] for j in range(n)]).double()
                for h in range(4):
                    s = (rows[:, 0, h // 2] @ m.q[t, h].double()) * math.copysign(1.0, scale)
                    two = s.topk(min(2, n)).values
                    # products of 64 terms of up to 40: the fp32 scores are within 64 * 40 * 2^-23 of these
                    if n == 1 or float(two[0] - two[1]) > 1e-3:
                        assert torch.equal(got[t, h], rows[int(s.argmax()), 1, h // 2].to(dtype)), (i, t, h)
                        seen += 1
        assert seen > 100


def test_attention_strided_rows_and_rows_of_no_sequence(pkg):
    for dtype, cache in PAIRS:
        say(f"[attend] strided {NAME[dtype]}/{NAME[cache]}")
        m = Made([70, 90], [3, 40], 4, 2, 80, 16, dtype, cache, seed=3)
        n = m.q.shape[0]
        q = torch.zeros(4, n + 6, 83, dtype=dtype, device="cuda").permute(1, 0, 2)[..., 1:81]
        q[2:2 + n] = m.q.cuda()
        out = torch.full((n + 6, 5, 81), 7.0, dtype=dtype, device="cuda")
        lse = torch.full((n + 6, 4), 7.0, device="cuda")
        want, wl, ob, lb = R.attend(m.q, m.kv, m.table_l, m.lens_l, m.starts_l, m.scale)
        pkg.paged_attention(q, m.kv_cuda(), m.table.cuda(), m.lens.cuda(), (m.starts + 2).cuda(), 40, 90,
                            out=out[:, :4, :80], lse=lse)
        near(out[2:2 + n, :4, :80], want, ob)
        near(lse[2:2 + n], wl, lb)
        rest = out.clone()
        rest[2:2 + n, :4, :80] = 7.0
        assert bool((rest == 7).all()) and bool((lse[:2] == 7).all()) and bool((lse[2 + n:] == 7).all())


@pytest.mark.parametrize("dtype,cache", PAIRS, ids=lambda t: NAME[t])
def test_attention_one_sequence_among_padding(pkg, dtype, cache):
    """One sequence of few rows in a batch padded to many, split over its keys;
    a workspace of the caller's, and the same slot in two sequences."""
    m = Made([3000], [2], 4, 2, 64, 16, dtype, cache, seed=31)
    want, wl, ob, lb = R.attend(m.q, m.kv, m.table_l, m.lens_l, m.starts_l, m.scale)
    q = torch.zeros(40, 4, 64, dtype=dtype, device="cuda")
    q[5:7] = m.q.cuda()
    out, lse = torch.full_like(q, 7.0), torch.full((40, 4), 7.0, device="cuda")
    args = (m.kv_cuda(), m.table.cuda(), m.lens.cuda(), (m.starts + 5).cuda())
    need = pkg.paged_attention_workspace(q, *args, max_len=3000)
    assert need > 0
    work = torch.empty(need, dtype=torch.uint8, device="cuda")
    pkg.paged_attention(q, *args, max_len=3000, out=out, lse=lse, work=work)
    near(out[5:7], want, ob)
    near(lse[5:7], wl, lb)
    assert bool((out[:5] == 7).all()) and bool((out[7:] == 7).all()) and bool((lse[7:] == 7).all())
    # two sequences of one slot: each's rows are its last tokens
    m.starts_l, m.starts = [0, 1, 2], torch.tensor([0, 1, 2], dtype=torch.int32)
    m.new, m.slots_l, m.slots = [1, 1], [0, 0], torch.tensor([0, 0], dtype=torch.int32)
    m.check(pkg)


@pytest.mark.parametrize("dtype,cache", PAIRS, ids=lambda t: NAME[t])
@pytest.mark.parametrize("heads,kv_heads,d", [(8, 2, 80), (4, 2, 128), (6, 3, 200), (2, 1, 256), (20, 1, 128)])
def test_attention_mixed_batches(pkg, dtype, cache, heads, kv_heads, d):
    """Chunks and sequences of few rows in one call, all of them split over their
    keys, with a window and without."""
    say(f"[attend] mixed {NAME[dtype]}/{NAME[cache]} {heads}/{kv_heads} heads of {d}")
    lens, new = [1100, 40, 1300, 3, 900], [1, 40, 70, 3, 2]
    Made(lens, new, heads, kv_heads, d, 16, dtype, cache, seed=11).check(pkg, what="mixed")
    Made(lens, new, heads, kv_heads, d, 16, dtype, cache, seed=13).check(pkg, window=777, hints=False, what="window")


def test_attention_with_and_without_lse(pkg):
    m = Made([33, 5], [20, 1], 4, 2, 64, 16, F32, F16, seed=4)
    args = (m.q.cuda(), m.kv_cuda(), m.table.cuda(), m.lens.cuda(), m.starts.cuda())
    got, lse = pkg.paged_attention(*args, lse=True)
    mine = torch.full_like(lse, 7.0)
    again, same = pkg.paged_attention(*args, lse=mine)
    assert same is mine and torch.equal(mine, lse) and torch.equal(got, again)
    for none in (None, False):
        assert torch.equal(pkg.paged_attention(*args, lse=none), got)


@pytest.mark.parametrize("d", [64, 128])
def test_attention_many_empty_sequences(pkg, d):
    """Thousands of sequences of no rows around a chunk and single tokens, with
    hints of far longer contexts."""
    seqs, at = 4000, {3: (700, 90), 1999: (300, 1), 3999: (65, 20)}
    m = Made([n for n, _ in at.values()], [k for _, k in at.values()], 16, 8, d, 16, F32, BF16, seed=6)
    want, lse, ob, lb = R.attend(m.q, m.kv, m.table_l, m.lens_l, m.starts_l, m.scale)
    starts, slots = [0], []
    for s in range(seqs):
        starts.append(starts[-1] + at.get(s, (0, 0))[1])
        slots.append(sorted(at).index(s) if s in at else s % 5 - 1)
    ints = lambda v: torch.tensor(v, dtype=torch.int32).cuda()
    say(f"[attend] {seqs} sequences, heads of {d}")
    got, l = pkg.paged_attention(m.q.cuda(), m.kv_cuda(), m.table.cuda(), m.lens.cuda(), ints(starts), slots=ints(slots),
                                 max_new=90, max_len=700, lse=True)
    near(got, want, ob)
    near(l, lse, lb)
    wide = torch.full((3, 1 << 16), -1, dtype=torch.int32)  # room for contexts of a million tokens
    wide[:, :m.table.shape[1]] = m.table
    got, l = pkg.paged_attention(m.q.cuda(), m.kv_cuda(), wide.cuda(), m.lens.cuda(), ints(starts), slots=ints(slots), lse=True)
    near(got, want, ob)
    near(l, lse, lb)


def test_attention_far_pages(pkg):
    """A cache of more than 2^32 elements: the pages in use are its last ones."""
    m = Made([100, 70], [1, 50], 4, 2, 64, 16, F32, F16, seed=12)
    pages = (1 << 32) // (2 * 2 * 16 * 64) + 64
    far = torch.empty((pages, 2, 2, 16, 64), dtype=F16, device="cuda")
    off = pages - m.kv.shape[0]
    far[off:] = m.kv.cuda()
    want, wl, ob, lb = R.attend(m.q, m.kv, m.table_l, m.lens_l, m.starts_l, m.scale)
    table = torch.where(m.table >= 0, m.table + off, -1).cuda()
    got, lse = pkg.paged_attention(m.q.cuda(), far, table, m.lens.cuda(), m.starts.cuda(), 50, 100, lse=True)
    near(got, want, ob)
    near(lse, wl, lb)
    k = torch.randn(51, 2, 64, device="cuda")
    pkg.cache_append(far, table, m.lens.cuda(), m.starts.cuda(), k, k + 1)
    page = int(table[1][69 // 16])
    assert torch.equal(far[page, 0, :, 69 % 16], k[50].half()) and torch.equal(far[page, 1, :, 69 % 16], (k[50] + 1).half())


@pytest.mark.parametrize("dtype,cache", PAIRS, ids=lambda t: NAME[t])
@pytest.mark.parametrize("interleaved,rot,d", [(True, 64, 64), (False, 40, 80), (False, 128, 128), (True, 6, 72)])
def test_append(pkg, dtype, cache, interleaved, rot, d):
    say(f"[append] {NAME[dtype]}/{NAME[cache]} interleaved={interleaved} rot {rot} of {d}")
    lens, new = [37, 5, 0, 64, 20], [3, 5, 0, 17, 1]
    m = Made(lens, new, 4, 2, d, 16, dtype, cache, seed=rot)
    n = m.q.shape[0]
    g = torch.Generator().manual_seed(d)
    k, v = (torch.randn(n, 2, d, generator=g).to(dtype) for _ in range(2))
    plan = pkg.rope_plan(rot, interleaved=interleaved, base=500000.0)
    freqs = plan.freqs.cpu().numpy()
    pos = np.concatenate([np.arange(a - b, a) for a, b in zip(lens, new)])
    kv = m.kv_cuda()
    q = pkg.cache_append(kv, m.table.cuda(), m.lens.cuda(), m.starts.cuda(), k.cuda(), v.cuda(), q=m.q.cuda(), plan=plan)
    near(q, R.turn(m.q.double(), pos, freqs, 1.0, interleaved), R.turn_bound(m.q.double(), pos, freqs, 1.0, interleaved, dtype), "q")
    kw, kb = R.turn(k.double(), pos, freqs, 1.0, interleaved), R.turn_bound(k.double(), pos, freqs, 1.0, interleaved, cache)
    seq = [i for i, b in enumerate(new) for _ in range(b)]
    expect = m.kv.clone()
    got = kv.cpu()
    for t in range(n):
        page, off = m.table_l[seq[t]][pos[t] // 16], pos[t] % 16
        near(got[page, 0, :, off], kw[t], kb[t], "k")
        assert torch.equal(got[page, 1, :, off], v[t].to(cache))
        expect[page, :, :, off] = got[page, :, :, off]
    assert torch.equal(torch.nan_to_num(got.float(), 123.0), torch.nan_to_num(expect.float(), 123.0))
    # in place; without q; without a plan
    y = m.q.cuda()
    kv2 = m.kv_cuda()
    pkg.cache_append(kv2, m.table.cuda(), m.lens.cuda(), m.starts.cuda(), k.cuda(), v.cuda(), q=y, plan=plan, out=y)
    assert torch.equal(y, q) and torch.equal(torch.nan_to_num(kv2.float()), torch.nan_to_num(kv.float()))
    kv3 = m.kv_cuda()
    assert pkg.cache_append(kv3, m.table.cuda(), m.lens.cuda(), m.starts.cuda(), k.cuda(), v.cuda()) is None
    page = m.table_l[3][63 // 16]
    assert torch.equal(kv3[page, 0, :, 15].cpu(), k[24].to(cache))


def test_append_skips_what_has_no_place(pkg):
    """Slots out of range, pages out of range, positions beyond the table or
    before 0, rows of no sequence: nothing is written, the rest is."""
    m = Made([20, 18], [2, 2, 2, 3], 2, 1, 64, 16, F32, F32, seed=1, slots=[0, 5, -1, 1])
    m.table_l[1][1] = m.kv.shape[0]
    k = torch.randn(12, 1, 64)
    kv = m.kv_cuda()
    t = torch.tensor(m.table_l, dtype=torch.int32).cuda()
    pkg.cache_append(kv, t, m.lens.cuda(), m.starts.cuda(), k.cuda(), k.cuda(), slots=m.slots.cuda())
    expect = m.kv.clone()
    for row, j, tok in ((0, 18, 0), (0, 19, 1), (1, 15, 6)):
        expect[m.table_l[row][j // 16], :, :, j % 16] = k[tok]
    assert torch.equal(torch.nan_to_num(kv.cpu(), 123.0), torch.nan_to_num(expect, 123.0))
    # lengths beyond the table, and shorter than the new tokens
    kv = m.kv_cuda()
    lens = torch.tensor([m.table.shape[1] * 16 + 1, 1], dtype=torch.int32).cuda()
    starts = torch.tensor([0, 3, 6], dtype=torch.int32).cuda()
    t = torch.tensor([[0] * m.table.shape[1], [1] * m.table.shape[1]], dtype=torch.int32).cuda()
    pkg.cache_append(kv, t, lens, starts, k.cuda(), k.cuda())
    expect = m.kv.clone()
    expect[0, :, :, 14], expect[0, :, :, 15], expect[1, :, :, 0] = k[0], k[1], k[5]
    assert torch.equal(torch.nan_to_num(kv.cpu(), 123.0), torch.nan_to_num(expect, 123.0))


def test_append_converts_with_one_rounding(pkg):
    """fp32 to the cache's type: nearest, ties to even; beyond fp16's range inf."""
    x = torch.tensor([1.0, 1 + 2.0 ** -11, 1 + 3 * 2.0 ** -11, 65504.0, 65519.9, 65520.0, -1e30, 2.0 ** -24, 2.0 ** -26,
                      1 + 2.0 ** -8, 1 + 3 * 2.0 ** -8, 3e38, 0.1, -0.3, 1e-40, math.nan])
    for cache in (F16, BF16, F32):
        kv = torch.zeros((1, 2, 1, 1, 16), dtype=cache, device="cuda")
        one = lambda *v: torch.tensor(v, dtype=torch.int32).cuda()
        pkg.cache_append(kv, one(0).reshape(1, 1), one(1), one(0, 1), x.reshape(1, 1, 16).cuda(), x.reshape(1, 1, 16).cuda())
        want = x.to(cache)
        for part in kv[0, :, 0, 0].cpu():
            assert torch.equal(torch.nan_to_num(part.float(), 5.0), torch.nan_to_num(want.float(), 5.0))


# ---------------------------------------------------------------- pages


class Pages:
    """The page calls' rules on Python lists: who holds what, and each page's
    contents as a label."""

    def __init__(self, slots, per, pages, ps):
        self.table = [[-1] * per for _ in range(slots)]
        self.lens, self.refs, self.ps = [0] * slots, [0] * pages, ps
        self.label = list(range(1000, 1000 + pages))

    def free(self):
        return [p for p, r in enumerate(self.refs) if r == 0]

    def held(self, s):
        return -(-self.lens[s] // self.ps)

    def reserve(self, counts):
        if any(c < 0 for c in counts):
            return 3
        need = [-(-(n + c) // self.ps) - self.held(s) for s, (n, c) in enumerate(zip(self.lens, counts))]
        if any(self.held(s) + k > len(self.table[s]) for s, k in enumerate(need)):
            return 2
        free = self.free()
        if sum(need) > len(free):
            return 1
        for s, c in enumerate(counts):
            for j in range(need[s]):
                p = free.pop(0)
                self.table[s][self.held(s) + j], self.refs[p] = p, 1
            self.lens[s] += c
        return 0

    def fork(self, src, dst):
        n = len(self.lens)
        if any(not 0 <= x < n for x in src + dst) or len(set(dst)) < len(dst) or set(src) & set(dst):
            return 3
        if any(self.lens[d] for d in dst):
            return 3
        free = self.free()
        if sum(self.lens[s] % self.ps > 0 for s in src) > len(free):
            return 1
        for s, d in zip(src, dst):
            whole = self.lens[s] // self.ps
            for j in range(whole):
                self.table[d][j] = self.table[s][j]
                self.refs[self.table[s][j]] += 1
            if self.lens[s] % self.ps:
                p = free.pop(0)
                self.table[d][whole], self.refs[p], self.label[p] = p, 1, self.label[self.table[s][whole]]
            self.lens[d] = self.lens[s]
        return 0

    def release(self, slots):
        if any(not 0 <= s < len(self.lens) for s in slots):
            return 3
        for s in slots:
            for j in range(self.held(s)):
                self.refs[self.table[s][j]] -= 1
                self.table[s][j] = -1
            self.lens[s] = 0
        return 0

    def compact(self):
        live = sum(r > 0 for r in self.refs)
        src = [p for p in range(live, len(self.refs)) if self.refs[p] > 0]
        dst = [p for p in range(live) if self.refs[p] == 0]
        to = dict(zip(src, dst))
        for a, b in to.items():
            self.refs[b], self.refs[a], self.label[b] = self.refs[a], 0, self.label[a]
        self.table = [[to.get(p, p) for p in row] for row in self.table]
        return live


def _same(cache, model, what):
    assert cache.table.tolist() == model.table, what + " table"
    assert cache.lens.tolist() == model.lens, what + " lens"
    assert cache.refs.tolist() == model.refs, what + " refs"
    # every page of every layer holds its label, in all of its elements
    kv = cache.kv.float()
    want = (torch.tensor(model.label).float()[None, :] + 10000 * torch.arange(kv.shape[0])[:, None]).cuda()
    assert bool((kv == want[:, :, None, None, None, None]).all()), what + " contents"


@pytest.mark.parametrize("slots,per,pages,ps,layers,d", [(6, 5, 20, 4, 3, 8), (3, 70, 200, 1, 1, 8), (40, 9, 150, 16, 2, 64),
                                                         (5, 40, 5000, 8, 1, 16), (1, 1, 1, 4096, 1, 8),
                                                         (1100, 3, 2500, 2, 1, 8), (4, 50, 1 << 19, 1, 1, 8)])
def test_pages_follow_the_rules(pkg, slots, per, pages, ps, layers, d):
    """Random reserves, forks, releases and compactions, refused ones among them,
    against the rules on lists."""
    rng = random.Random(slots * pages)
    c = pkg.PagedCache(layers, pages, ps, 2, d, slots, per)
    model = Pages(slots, per, pages, ps)
    c.kv.copy_((torch.tensor(model.label).float()[None, :] + 10000 * torch.arange(layers)[:, None])
               .reshape(layers, pages, 1, 1, 1, 1).cuda().expand_as(c.kv))
    ints = lambda v: torch.tensor(v, dtype=torch.int32).cuda()
    seen = set()
    for step in range(40):
        op = rng.choice(["reserve", "reserve", "fork", "release", "compact"])
        say(f"[pages] {slots}x{per} of {pages}: step {step} {op}")
        if op == "reserve":
            top = rng.choice([1, ps, 3 * ps])
            counts = [rng.randrange(0, top + 1) if rng.random() < 0.3 else 0 for _ in range(slots)]
            if rng.random() < 0.1:
                counts[rng.randrange(slots)] = rng.choice([-1, 2 ** 31 - 1])
            got, want = c.reserve(ints(counts)), model.reserve(counts)
        elif op == "fork":
            full = [s for s in range(slots) if model.lens[s]] or [0]
            empty = [s for s in range(slots) if not model.lens[s]]
            rng.shuffle(empty)
            dst = empty[:rng.randrange(0, 6)]
            src = [rng.choice(full) for _ in dst]
            if dst and rng.random() < 0.2:
                i = rng.randrange(len(dst))
                if rng.random() < 0.5:
                    dst[i] = rng.choice([-1, slots, dst[0], full[0]])
                else:
                    src[i] = rng.choice([-1, slots, dst[0]])
            got, want = c.fork(ints(src), ints(dst)), model.fork(src, dst)
        elif op == "release":
            gone = [rng.randrange(slots) for _ in range(rng.randrange(0, max(2, slots // 4)))]
            gone += gone[:1]
            if rng.random() < 0.1:
                gone.append(rng.choice([-1, slots]))
            got, want = c.release(ints(gone)), model.release(gone)
        else:
            got, want = c.compact(), model.compact()
        assert int(got) == want, (step, op)
        seen.add((op, want if op != "compact" else 0))
        _same(c, model, f"step {step} {op}")
    assert ("reserve", 0) in seen and ("compact", 0) in seen


def test_pages_of_many_slots_at_once(pkg):
    """More forks and releases in one call than a workgroup has threads, against
    the rules on lists; then one too many for the pages."""
    slots, pages, ps = 2300, 1700, 4
    c = pkg.PagedCache(2, pages, ps, 1, 8, slots, 3)
    model = Pages(slots, 3, pages, ps)
    c.kv.copy_((torch.tensor(model.label).float()[None, :] + 10000 * torch.arange(2)[:, None])
               .reshape(2, pages, 1, 1, 1, 1).cuda().expand_as(c.kv))
    ints = lambda v: torch.tensor(v, dtype=torch.int32).cuda()
    rng = random.Random(8)
    counts = [7, 8, 1] + [0] * (slots - 3)
    assert int(c.reserve(ints(counts))) == model.reserve(counts) == 0
    dst = list(range(3, slots))
    rng.shuffle(dst)
    src = [rng.randrange(3) for _ in dst]
    say("[pages] 2297 forks")
    assert int(c.fork(ints(src), ints(dst))) == model.fork(src, dst) == 0
    _same(c, model, "forks")
    gone = [s for s in range(slots) if s % 3] + [5, 4]
    say("[pages] releases")
    assert int(c.release(ints(gone))) == model.release(gone) == 0
    _same(c, model, "releases")
    assert int(c.compact()) == model.compact()
    _same(c, model, "compact")
    src, dst = [0] * len(gone[:-2]), gone[:-2]
    say("[pages] too many forks")
    assert int(c.fork(ints(src), ints(dst))) == model.fork(src, dst) == 1
    _same(c, model, "too many")
    dst[-1] = dst[0]
    assert int(c.fork(ints(src), ints(dst))) == model.fork(src, dst) == 3
    _same(c, model, "twice")


def test_copy_pages(pkg):
    kv = torch.randn(3, 10, 2, 2, 16, 72, device="cuda").half()
    want = kv.clone()
    ints = lambda v: torch.tensor(v, dtype=torch.int32).cuda()
    want[:, [1, 2, 9]] = want[:, [5, 0, 5]]
    pkg.cache_copy_pages(kv, ints([5, 0, -1, 3, 5, 4]), ints([1, 2, 3, 10, 9, -5]))
    assert torch.equal(kv, want)
    pkg.cache_copy_pages(kv, ints([]), ints([]))
    assert torch.equal(kv, want)


@pytest.mark.parametrize("order", [(0, 1, 2, 3), (2, 0, 1, 3), (1, 2, 0, 3), (2, 1, 0, 3)])
@pytest.mark.parametrize("kv_heads,ps,d", [(3, 4, 8), (1, 8, 16), (5, 1, 8)])
def test_pages_in_any_dense_order(pkg, order, kv_heads, ps, d):
    """Pages whose (key or value, head, token) come in any order: copied, forked
    and compacted as the plain order is."""
    say(f"[pages] order {order} {kv_heads} x {ps} x {d}")
    sizes = (2, kv_heads, ps, d)
    back = [order.index(i) for i in range(4)]
    made = lambda: torch.zeros((2, 12) + tuple(sizes[i] for i in order), device="cuda").permute(0, 1, *[2 + i for i in back])
    g = torch.Generator().manual_seed(3)
    init = torch.randn((2, 12) + sizes, generator=g).cuda()
    ints = lambda v: torch.tensor(v, dtype=torch.int32).cuda()
    kv = made().copy_(init)
    assert kv.shape[2:] == sizes
    pkg.cache_copy_pages(kv, ints([3, 7]), ints([1, 0]))
    init[:, 1], init[:, 0] = init[:, 3].clone(), init[:, 7].clone()
    assert torch.equal(kv, init)
    c = pkg.PagedCache(2, 12, ps, kv_heads, d, 3, 8)
    c.kv = kv
    n = 2 * ps + ps // 2
    assert int(c.reserve(ints([1, n, 0]))) == 0
    assert int(c.fork(ints([1]), ints([2]))) == 0
    assert int(c.release(ints([0]))) == 0
    live = int(c.compact())
    assert live == -(-n // ps) + (n % ps != 0)
    for s in (1, 2):
        assert c.table[s, :-(-n // ps)].max() < live
        for j in range(n):
            # pages 1 .. were slot 1's when the contents were made
            assert torch.equal(kv[:, c.table[s, j // ps].item(), :, :, j % ps], init[:, 1 + j // ps, :, :, j % ps])


def test_pages_that_are_not_dense_are_refused(pkg):
    ints = torch.tensor([0], dtype=torch.int32).cuda()
    wide = torch.zeros(2, 12, 2, 3, 4, 16, device="cuda")
    for kv in (wide[..., :8], wide[:, :, :, :2], wide[:, :, :, :, ::2], wide[:, :, :, :1].expand(2, 12, 2, 3, 4, 16),
               wide.as_strided((2, 12, 2, 4, 1, 8), (768, 64, 8, 32, 8, 1))):
        with pytest.raises(AssertionError):
            pkg.cache_copy_pages(kv, ints, ints)


# ---------------------------------------------------------------- together


def _layer_step(pkg, m, cache, x, starts, counts, w, plan, dims, max_new, max_len):
    """One decoding step of a one-layer model: projections, cache, attention,
    output projection, logits."""
    heads, kv_heads, d, width, vocab = dims
    status = cache.reserve(counts)
    t = x.shape[0]
    q = pkg.lm_head(w["q"], 1, heads * d, width, x).view(t, heads, d)
    k = pkg.lm_head(w["k"], 1, kv_heads * d, width, x).view(t, kv_heads, d)
    v = pkg.lm_head(w["v"], 1, kv_heads * d, width, x).view(t, kv_heads, d)
    q = cache.append(0, k, v, starts, q=q, plan=plan, out=q)
    o = cache.attend(0, q, starts, max_new=max_new, max_len=max_len)
    y = x + pkg.lm_head(w["o"], 1, width, heads * d, o.view(t, heads * d))
    return status, pkg.lm_head(w["out"], 1, vocab, width, y)


def test_contexts_decode_together(pkg):
    """Three contexts of unlike prompts, then single tokens, a fork, a release
    and a compaction on the way: every step's logits agree with the whole
    forward recomputed in float64 without a cache."""
    heads, kv_heads, d, width, vocab = dims = (4, 2, 16, 64, 50)
    g = torch.Generator().manual_seed(5)
    half = {n: (torch.randn(r, c, generator=g) / math.sqrt(c)).half()
            for n, r, c in (("q", heads * d, width), ("k", kv_heads * d, width), ("v", kv_heads * d, width),
                            ("o", width, heads * d), ("out", vocab, width))}
    w = {n: x.contiguous().view(torch.uint8).reshape(-1).cuda() for n, x in half.items()}
    emb = torch.randn(vocab, width, generator=g)
    plan = pkg.rope_plan(d, interleaved=True)
    freqs = plan.freqs.cpu().numpy()
    cache = pkg.PagedCache(1, 40, 4, kv_heads, d, 5, 16, dtype=F32)
    cache.kv.fill_(math.nan)  # nothing of a place that was never written may matter
    ints = lambda v: torch.tensor(v, dtype=torch.int32).cuda()

    def whole(ids):
        """Logits of the last token, in float64."""
        x = emb[ids].double()
        n = len(ids)
        q, k, v = ((x @ half[c].double().t()).reshape(n, -1, d).numpy() for c in "qkv")
        pos = np.arange(n)
        q, k = R.turn(q, pos, freqs, 1.0, True), R.turn(k, pos, freqs, 1.0, True)
        o = np.zeros((heads, d))
        for h in range(heads):
            s = k[:, h // 2] @ q[-1, h] / math.sqrt(d)
            p = np.exp(s - s.max())
            o[h] = (p / p.sum()) @ v[:, h // 2]
        y = x[-1] + torch.from_numpy(o.reshape(-1)) @ half["o"].double().t()
        return y @ half["out"].double().t()

    rng = random.Random(1)
    text = {s: [rng.randrange(vocab) for _ in range(n)] for s, n in ((0, 9), (1, 1), (2, 6))}
    new = {s: list(t) for s, t in text.items()}
    for step in range(8):
        order = [s for s in range(5) if s in new]
        counts, rows, starts = [0] * 5, [], [0] * 6
        for s in range(5):
            rows += new.get(s, [])
            starts[s + 1] = len(rows)
            counts[s] = len(new.get(s, []))
        say(f"[together] step {step} slots {order}")
        st, logits = _layer_step(pkg, None, cache, emb[rows].cuda(), ints(starts), ints(counts), w, plan, dims,
                                 max(counts), max(len(t) for t in text.values()))
        assert int(st) == 0
        for s in order:
            got, want = logits[starts[s + 1] - 1].cpu().double(), whole(text[s])
            # fp32 sums of 64 terms in four projections in a row
            assert float((got - want).abs().max()) <= 4 * 64 * 2.0 ** -24 * float(want.abs().max()) * 8
        if step == 2:
            assert int(cache.fork(ints([0, 2]), ints([3, 4]))) == 0
            text[3], text[4] = list(text[0]), list(text[2])
        if step == 4:
            assert int(cache.release(ints([0, 1]))) == 0
            del text[0], text[1]
            cache.compact()
        new = {s: [rng.randrange(vocab)] for s in text}
        for s in new:
            text[s] += new[s]


def test_step_captured_and_replayed(pkg):
    """reserve, append and attention in a graph, replayed token after token with
    eager work between: each replay as the eager calls on a second cache."""
    heads, kv_heads, d, slots = 8, 2, 64, 3
    plan = pkg.rope_plan(d, interleaved=False)
    make = lambda: pkg.PagedCache(1, 60, 8, kv_heads, d, slots, 20, dtype=F16)
    a, b = make(), make()
    g = torch.Generator(device="cuda").manual_seed(2)
    starts = torch.tensor([0, 1, 2, 3], dtype=torch.int32).cuda()
    ones = torch.ones(slots, dtype=torch.int32, device="cuda")
    x = torch.randn(slots, heads + 2 * kv_heads, d, generator=g, device="cuda")

    def step(c, x):
        st = c.reserve(ones)
        q = c.append(0, x[:, heads:heads + kv_heads], x[:, heads + kv_heads:], starts, q=x[:, :heads], plan=plan)
        return st, c.attend(0, q, starts, max_new=1, max_len=160)

    pre = torch.tensor([30, 0, 7], dtype=torch.int32).cuda()
    for c in (a, b):
        assert int(c.reserve(pre)) == 0
        c.kv.normal_(generator=torch.Generator(device="cuda").manual_seed(4))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(b, x)  # kernels loaded before the capture
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    b.table.copy_(a.table), b.lens.copy_(a.lens), b.refs.copy_(a.refs), b.kv.copy_(a.kv)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        st, out = step(a, x)
    for i in range(20):
        say(f"[graph] replay {i}")
        x.normal_(generator=g)
        graph.replay()
        est, eout = step(b, x)
        torch.cuda.synchronize()
        assert int(st) == int(est) == 0
        assert torch.equal(out, eout) and torch.equal(a.kv, b.kv)
        assert torch.equal(a.table, b.table) and torch.equal(a.lens, b.lens) and torch.equal(a.refs, b.refs)


def test_two_streams_at_once(pkg):
    """Attention calls in flight on two streams, each with its own workspace."""
    ms = [Made([4000, 3000], [1, 1], 8, 2, 64, 16, F32, F16, seed=s) for s in (1, 2)]
    args = [(m.q.cuda(), m.kv_cuda(), m.table.cuda(), m.lens.cuda(), m.starts.cuda(), 1, 4000) for m in ms]
    alone = [pkg.paged_attention(*a).clone() for a in args]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in ms]
    got = [[], []]
    for _ in range(10):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(pkg.paged_attention(*args[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, alone[i]) for o in got[i])


def test_same_bits_every_time(pkg):
    for m in (Made([4000, 3000], [1, 1], 8, 2, 64, 16, F32, BF16, seed=1), Made([900, 500], [300, 9], 8, 2, 128, 16, BF16, BF16, seed=2)):
        args = (m.q.cuda(), m.kv_cuda(), m.table.cuda(), m.lens.cuda(), m.starts.cuda(), max(m.new), max(m.lens_l))
        a = pkg.paged_attention(*args)
        assert all(torch.equal(pkg.paged_attention(*args), a) for _ in range(3))


def test_refused_calls(pkg):
    """Python's own checks; the C ABI's are in tests/test_attention_cpu.py."""
    m = Made([20], [1], 4, 2, 64, 16, F32, F16, seed=1)
    base = [m.q.cuda(), m.kv_cuda(), m.table.cuda(), m.lens.cuda(), m.starts.cuda()]

    def refused(i, x, **kw):
        a = list(base)
        if i is not None:
            a[i] = x
        with pytest.raises((AssertionError, pkg.SamplerError)):
            pkg.paged_attention(*a, **kw)

    refused(0, base[0].double())
    refused(0, base[0].bfloat16())            # q of another 16-bit type than the cache
    refused(0, base[0][:, :3])                # heads no multiple of the cache's
    refused(0, base[0][..., :32])
    refused(0, base[0].cpu())
    refused(1, base[1].double())
    refused(2, base[2].long())
    refused(2, base[2].t())
    refused(3, base[3].long())
    refused(4, base[4].long())
    refused(None, None, window=-1)
    refused(None, None, max_new=-1)
    refused(None, None, scale=math.inf)
    refused(None, None, scale=math.nan)
    refused(None, None, lse=torch.empty(1, 4, 1, device="cuda"))
    refused(None, None, lse=torch.empty(1, 4, dtype=F16, device="cuda"))
    refused(None, None, first=torch.zeros(2, dtype=torch.int32, device="cuda"))
    refused(None, None, slots=torch.zeros(2, dtype=torch.int32, device="cuda"))
    refused(None, None, out=torch.empty(1, 1, 64, device="cuda").expand(1, 4, 64))  # heads on one place
    with pytest.raises(pkg.SamplerError):
        pkg.rope_plan(64, scaling="dynamic")
    with pytest.raises(AssertionError):
        pkg.rope(base[0], torch.zeros(2, dtype=torch.int32, device="cuda"), pkg.rope_plan(64))
    with pytest.raises(pkg.SamplerError):
        pkg.rope(base[0], torch.zeros(1, dtype=torch.int32, device="cuda"), pkg.rope_plan(66))
    # no tokens, no sequences
    none = torch.empty(0, 4, 64, device="cuda")
    assert pkg.paged_attention(none, *base[1:4], torch.zeros(2, dtype=torch.int32, device="cuda")).shape == (0, 4, 64)
    out = torch.full((1, 4, 64), 7.0, device="cuda")
    pkg.paged_attention(*base[:4], torch.zeros(1, dtype=torch.int32, device="cuda"), out=out)
    assert bool((out == 7).all())




def _goes_to_its_largest(pkg, m, scale):
    """Scores so far apart that a row is the value of its largest one, rows of
    near ties aside.  Returns how many rows were looked at."""
    got, lse = pkg.paged_attention(m.q.cuda(), m.kv_cuda(), m.table.cuda(), m.lens.cuda(), m.starts.cuda(), max(m.new),
                                   max(m.lens_l), scale=scale, lse=True)
    got, lse = got.cpu(), lse.cpu()
    assert bool(torch.isfinite(got).all()) and bool(torch.isfinite(lse).all())
    heads, kv_heads, d = m.q.shape[1], m.kv.shape[2], m.q.shape[2]
    seen = 0
    for i in range(len(m.new)):
        for t in range(m.starts_l[i], m.starts_l[i + 1]):
            n = m.lens_l[i] - m.starts_l[i + 1] + t + 1
            rows = torch.stack([m.kv[m.table_l[i][j // m.page], :, :, j % m.page] for j in range(n)]).double()
            for h in range(heads):
                k, v, x = rows[:, 0, h // (heads // kv_heads)], rows[:, 1, h // (heads // kv_heads)], m.q[t, h].double()
                s = (k @ x) * scale
                # an fp32 score may be off by this: d products and sums, the parts
                # of a query, the scale and log2 e.  (Sums of fp16 products are
                # aligned by the operands' exponents, and a denormal's is that of
                # 2^-14: 24 bits of it hold what 2^-14 times the query is held by.)
                size = k.abs().clamp(min=2.0 ** -14) if m.kv.dtype == F16 else k.abs()
                ds = float(((size @ x.abs()) * abs(scale)).max()) * ((d + 4) * 2.0 ** -24 + 2.0 ** -22)
                two = s.topk(min(2, n)).values
                # lse: the score's error, the whole number and logarithm it is made
                # of (2^-24 of it, four times), and the other keys' weights (at most n)
                assert abs(float(lse[t, h]) - float(two[0])) <= ds + 4 * abs(float(two[0])) * 2.0 ** -24 + math.log(n) + 1e-6
                if n > 1 and float(two[0] - two[1]) <= 2 * ds + 40:
                    continue
                # a weight of one key: 22 bits or more (fp32 queries) or 16 of it
                # enter the product, the quotient is rounded, then the output
                want = v[int(s.argmax())]
                bound = want.abs() * (2.0 ** -20 if m.q.dtype == F32 else 2 * R.HALF[m.q.dtype]) + n * math.exp(-40) * v.abs().max()
                near(got[t, h], want, bound + R.tiny(m.q.dtype), f"row {i} {t} {h}")
                seen += 1
    return seen


@pytest.mark.parametrize("dtype,cache", PAIRS, ids=lambda t: NAME[t])
@pytest.mark.parametrize("lens,new", [([300, 90], [1, 3]), ([1300, 60], [1, 2]), ([300, 90], [20, 40])])
def test_attention_scores_around_whole_fp32_numbers(pkg, dtype, cache, lens, new):
    """Scores of 10^6 to 10^9: fp32 holds whole numbers there, or every second to
    sixteenth one, and what is added to a maximum is rounded."""
    for scale in (1e5, 3e5, 1e6, 2e6, -2e6, 4e6, 8e6, 1.6e7):
        say(f"[attend] scale {scale} {NAME[dtype]}/{NAME[cache]} lens {lens} new {new}")
        m = Made(lens, new, 4, 2, 64, 16, dtype, cache, seed=22)
        assert _goes_to_its_largest(pkg, m, scale) > 10


@pytest.mark.parametrize("dtype,cache", PAIRS, ids=lambda t: NAME[t])
@pytest.mark.parametrize("lens,new", [([300, 90, 33], [20, 40, 2]), ([1300, 60], [1, 2])])
def test_attention_scores_next_to_zero(pkg, dtype, cache, lens, new):
    """Scales and queries down to the least fp32 numbers: every visible key weighs
    the same, in masked tiles too."""
    for scale, spread in ((1e-45, 2.0), (-1e-45, 2.0), (1e-41, 2.0), (1e-38, 2.0), (0.125, 1e-42), (0.125, 1e-44), (1e-20, 1e-30),
                          (1.0, 1e-36), (1e-45, 1e-44)):
        if dtype != F32 and spread < 1.0:
            continue
        say(f"[attend] scale {scale} queries of {spread} {NAME[dtype]}/{NAME[cache]} lens {lens}")
        m = Made(lens, new, 4, 2, 64, 16, dtype, cache, seed=22, spread=spread)
        m.scale = scale
        m.check(pkg, scale=scale)
        m.check(pkg, scale=scale, window=21)


@pytest.mark.parametrize("lens,new", [([300, 90, 33], [20, 40, 2]), ([1300, 60], [1, 2]), ([1300, 70], [50, 60])])
def test_attention_large_queries_over_zeros(pkg, lens, new):
    """Queries of 1e30 under a scale of 1e13: keys of zeros have scores of 0, and
    one of fp16's least numbers has a finite score that takes all of the weight."""
    say(f"[attend] large queries over zeros, lens {lens}")
    m = Made(lens, new, 4, 2, 64, 16, F32, F16, seed=23)
    m.q = m.q.abs() * 1e30 + 1e29
    m.kv[:, 0] = 0.0
    m.scale = 1e13
    m.check(pkg, scale=1e13, what="zeros")
    for s, n in enumerate(lens):
        m.kv[m.table_l[s][0], 0, :, 0] = 2.0 ** -24
    assert _goes_to_its_largest(pkg, m, 1e13) == 4 * sum(new)


@pytest.mark.parametrize("dtype,cache,heads,kv_heads,d", [(F32, F32, 4, 2, 128), (F32, F16, 8, 2, 128), (F32, BF16, 4, 1, 256),
                                                          (BF16, BF16, 8, 2, 64), (F16, F16, 4, 2, 256)])
def test_mixed_batches_captured_and_replayed(pkg, dtype, cache, heads, kv_heads, d):
    """Chunks and single tokens of wide heads, all split and joined, in two graphs
    of one set of tensors, replayed in turn with new inputs, other lengths and
    eager calls between: each replay as the eager call."""
    say(f"[graph] {NAME[dtype]}/{NAME[cache]} {heads}/{kv_heads} heads of {d}")
    m = Made([1500, 700, 40, 900], [1, 90, 40, 3], heads, kv_heads, d, 16, dtype, cache, seed=17)
    q, kv, table, lens, starts = m.q.cuda(), m.kv_cuda(), m.table.cuda(), m.lens.cuda(), m.starts.cuda()
    call = lambda window: pkg.paged_attention(q, kv, table, lens, starts, 90, 1500, window=window, lse=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(0), call(600)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for window in (0, 600):
        graphs.append((torch.cuda.CUDAGraph(), window))
        with torch.cuda.graph(graphs[-1][0]):
            graphs[-1] += (call(window),)
    g = torch.Generator(device="cuda").manual_seed(5)
    for i in range(12):
        say(f"[graph] replay {i}")
        q.copy_(torch.randn(q.shape, generator=g, device="cuda") * 2)
        lens[0] = 1500 - 100 * i
        lens[1] = 90 + 50 * i
        graph, window, got = graphs[i % 2]
        graph.replay()
        if i % 3 == 0:
            graphs[(i + 1) % 2][0].replay()
        want = call(window)
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_page_calls_captured_and_replayed(pkg):
    """A pool whose bitmap takes more LDS than a kernel has unasked: reserve, fork,
    release and compact in one graph, as the eager calls on a second cache."""
    make = lambda: pkg.PagedCache(1, 400000, 2, 1, 8, 12, 500, dtype=F16)
    a, b = make(), make()
    ints = lambda v: torch.tensor(v, dtype=torch.int32).cuda()
    grow, src, dst, gone = ints([3, 5, 0, 7] + [0] * 8), ints([0, 1]), ints([4, 5]), ints([4, 5, 0])

    def step(c):
        return c.reserve(grow), c.fork(src, dst), c.release(gone), c.compact()

    step(b)  # kernels loaded before the capture
    torch.cuda.synchronize()
    for x, y in ((b.table, a.table), (b.lens, a.lens), (b.refs, a.refs), (b.kv, a.kv)):
        x.copy_(y)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(a)
    for i in range(8):
        say(f"[graph] pages, replay {i}")
        noise = torch.randn(a.kv.shape, generator=torch.Generator(device="cuda").manual_seed(i), device="cuda").half()
        a.kv.copy_(noise), b.kv.copy_(noise)
        grow[6 + i % 4] = 1 + i
        graph.replay()
        want = step(b)
        torch.cuda.synchronize()
        assert [int(x) for x in got] == [int(x) for x in want] and [int(x) for x in got[:3]] == [0, 0, 0]
        assert torch.equal(a.table, b.table) and torch.equal(a.lens, b.lens) and torch.equal(a.refs, b.refs)
        assert torch.equal(a.kv, b.kv)


def test_forks_share_pages_and_attend_as_their_parent(pkg):
    """Contexts that share a prompt's pages: the same query has the same bits in
    each, for single tokens and chunks, whatever the others' tokens are."""
    cache = pkg.PagedCache(1, 400, 16, 2, 128, 24, 80, dtype=BF16)
    ints = lambda v: torch.tensor(v, dtype=torch.int32).cuda()
    g = torch.Generator(device="cuda").manual_seed(3)
    cache.kv.normal_(generator=g)
    assert int(cache.reserve(ints([1003] + [0] * 23))) == 0
    assert int(cache.fork(ints([0] * 23), ints(list(range(1, 24))))) == 0
    assert int((cache.refs > 1).sum()) == 1003 // 16 and int(cache.refs.max()) == 24
    for n in (1, 33):
        say(f"[forks] {n} tokens each")
        assert int(cache.reserve(ints([n] * 24))) == 0
        q, k, v = (torch.randn(n, h, 128, generator=g, device="cuda").bfloat16().repeat(24, 1, 1) for h in (8, 2, 2))
        starts = ints([n * i for i in range(25)])
        q = cache.append(0, k, v, starts, q=q, plan=pkg.rope_plan(128))
        out = cache.attend(0, q, starts, max_new=n, max_len=1100).view(24, n, 8, 128)
        assert all(torch.equal(out[i], out[0]) for i in range(24))
        alone = pkg.paged_attention(q[:n], cache.kv[0], cache.table[:1], cache.lens[:1], starts[:2], max_new=n, max_len=1100)
        # (split otherwise: the same sums in another order, bf16 weights rounded from other maxima)
        assert float((alone.float() - out[0].float()).abs().max()) <= 4 * R.HALF[BF16] * float(cache.kv.abs().max())


def test_rope_next_to_quarter_turns(pkg):
    """Angles next to whole quarters of a turn, where the sine or the cosine is
    next to 0: it is right to its own last places, as a table in 64 bits is."""
    quarter = math.pi / 2
    pos = torch.tensor([1, 2, 3, 5, 1001, 40002, 99999], dtype=torch.int32)
    freqs = [quarter * (1 + e) for e in (0.0, 3e-9, -1e-8, 5e-8, 1e-7, -4e-7, 1e-6, 2e-3)]
    plan = pkg.RopePlan(torch.tensor(freqs, dtype=torch.float64).cuda(), True, 1.0)
    x = torch.zeros(len(pos), 1, 16)
    x[..., 0::2] = 1.0  # turned: (cos, sin) of the angle
    got = pkg.rope(x.cuda(), pos.cuda(), plan).cpu().double().view(-1, 8, 2)
    angle = np.asarray(pos, dtype=np.float64)[:, None] * np.asarray(freqs)[None, :]
    want = torch.from_numpy(np.stack([np.cos(angle), np.sin(angle)], -1))
    # the float64 angle's product and reduction (2^-52 of it, twice), sine and
    # cosine to 4 units of 2^-24, the turn by what is behind 24 bits (its square's
    # half, 2^-47, a rounding more), the product with 1
    bound = torch.from_numpy(angle)[..., None] * 2.0 ** -51 + want.abs() * 8 * 2.0 ** -24 + 2.0 ** -46
    near(got, want, bound, "quarters")
    # and on the way into the cache, at positions behind others
    kv = torch.zeros((1, 2, 1, 8, 16), device="cuda")
    one = lambda *v: torch.tensor(v, dtype=torch.int32).cuda()
    q = pkg.cache_append(kv, one(0).reshape(1, 1), one(6), one(0, 5), x[:5].cuda(), x[:5].cuda(), q=x[:5].cuda(), plan=plan)
    angle = np.arange(1, 6)[:, None] * np.asarray(freqs)[None, :]
    want = torch.from_numpy(np.stack([np.cos(angle), np.sin(angle)], -1))
    bound = 2.0 ** -48 + want.abs() * 8 * 2.0 ** -24 + 2.0 ** -46
    near(q.cpu().double().view(-1, 8, 2), want, bound, "q")
    near(kv[0, 0, 0, 1:6].cpu().double().view(-1, 8, 2), want, bound, "k")

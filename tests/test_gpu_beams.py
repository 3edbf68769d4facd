"""Beam search: the selection over beams and vocabulary, the contexts that
follow it, and both together over a cache, against their definitions."""
import math
import random

import numpy as np
import pytest
import torch

import quant_ref as R

pytestmark = pytest.mark.gpu


def say(*a):
    print(*a, flush=True)


# ---------------------------------------------------------------- selection


def select(logits, scores, ended=None, eog=()):
    """The definition in float64, group by group: parents, tokens, scores, ended;
    and how near the nearest two candidates of different rows are among the
    first beams + 1."""
    groups, beams = scores.shape
    x = logits.astype(np.float64).reshape(groups, beams, -1)
    out = [np.zeros((groups, beams), dtype=t) for t in (np.int64, np.int64, np.float64, np.int64)]
    gap = math.inf
    for g in range(groups):
        all_ = []
        for b in range(beams):
            s = float(scores[g, b])
            if not s > -math.inf:
                continue
            if ended is not None and ended[g, b]:
                all_.append((-s, b, -1))
                continue
            row = np.where(np.isnan(x[g, b]), -np.inf, x[g, b])
            m = row.max()
            if m == -np.inf:
                continue
            d = np.where(row == m, 0.0, row - m)
            c = d - math.log(np.exp(d).sum()) + s
            near = np.argsort(-c, kind="stable")[:beams + 1]
            all_ += [(-c[v], b, int(v)) for v in near if c[v] > -np.inf]
        all_.sort()
        for one, two in zip(all_[:beams], all_[1:beams + 1]):
            if one[1] != two[1] and one[0] != two[0]:
                gap = min(gap, two[0] - one[0])
        for j in range(beams):
            if j < len(all_):
                c, b, v = all_[j]
                done = (ended is not None and bool(ended[g, b])) or v in eog
                out[0][g, j], out[1][g, j], out[2][g, j], out[3][g, j] = g * beams + b, v, -c, done
            else:
                out[0][g, j], out[1][g, j], out[2][g, j] = g * beams + j, -1, -math.inf
    return out, gap


# A row's sum: 32 terms of 2^-22 each one after another and 9 more sums in fp32,
# the rest in float64; then one rounding of the score.
LSE = 2.0 ** -22 + 41 * 2.0 ** -24


def check(pkg, logits, scores, ended=None, eog=(), **kw):
    (parents, tokens, worth, over), gap = select(logits, scores, ended, set(eog))
    assert gap > 2 * LSE, gap  # else the order were not decided
    to = lambda a, t: None if a is None else torch.from_numpy(np.ascontiguousarray(a, dtype=t)).cuda()
    got = pkg.beam_select(to(logits, np.float32), to(scores, np.float32), ended=to(ended, np.int32),
                          eog=to(list(eog), np.int32) if eog else None, **kw)
    p, t, s, e = (x.cpu().numpy() for x in got)
    assert np.array_equal(p, parents) and np.array_equal(t, tokens) and np.array_equal(e, over)
    live = np.isfinite(worth)
    assert np.array_equal(s[~live], worth[~live])
    assert (np.abs(s[live] - worth[live]) <= LSE + 2.0 ** -24 * np.abs(worth[live]) * (1 + LSE)).all()
    return got


def made(seed, groups, beams, vocab, spread=3.0):
    g = np.random.default_rng(seed)
    return (g.standard_normal((groups * beams, vocab)) * spread).astype(np.float32), \
        (g.standard_normal((groups, beams)) * 2 - 30).astype(np.float32)


@pytest.mark.parametrize("groups,beams,vocab", [(1, 1, 1), (1, 2, 1), (3, 4, 2), (2, 5, 7), (1, 4, 32000), (5, 3, 8191),
                                                (2, 8, 8192), (2, 8, 8193), (1, 64, 1000), (2, 16, 50257), (3, 2, 300),
                                                (1, 64, 50), (1, 7, 151936), (40, 2, 999), (1, 1, 100001)])
def test_selection(pkg, groups, beams, vocab):
    say(f"[beams] {groups}x{beams}x{vocab}")
    logits, scores = made(groups * 1000 + beams + vocab, groups, beams, vocab)
    check(pkg, logits, scores)
    rng = np.random.default_rng(1)
    ended = (rng.random((groups, beams)) < 0.4).astype(np.int32)
    check(pkg, logits, scores, ended)
    eog = sorted({0, vocab - 1, int(logits.reshape(-1, vocab)[0].argmax())})
    check(pkg, logits, scores, ended, eog)


def test_first_step(pkg):
    """One live beam a group: its best continuations, also beyond what the merge
    holds at a time."""
    for beams, vocab in ((4, 32000), (32, 128256), (64, 300001), (64, 70)):
        logits, scores = made(beams, 2, beams, vocab)
        scores[:] = -np.inf
        scores[0, 0] = scores[1, beams - 1] = 0.0
        check(pkg, logits, scores)


@pytest.mark.parametrize("beams,vocab", [(4, 3), (8, 5000), (64, 40000), (5, 20000)])
def test_equal_candidates_go_by_the_lowest(pkg, beams, vocab):
    logits, scores = np.zeros((2 * beams, vocab), dtype=np.float32), np.full((2, beams), -3.0, dtype=np.float32)
    check(pkg, logits, scores)
    logits[:, vocab // 2:] = 1.0
    check(pkg, logits, scores)
    logits[:, ::3] = 2.0  # many of them on each bound
    check(pkg, logits, scores)
    # ended beams worth as much as continuations of others
    logits[:] = -np.inf
    logits[:, vocab - 1] = 5.0
    check(pkg, logits, scores, np.tile(np.arange(beams) % 2, (2, 1)))


def test_unusual_logits_and_scores(pkg):
    beams, vocab = 4, 9001
    logits, scores = made(3, 6, beams, vocab)
    x = logits.reshape(6, beams, vocab)
    x[0, 0, ::2] = -np.inf
    x[0, 1] = -np.inf
    x[0, 2, 5:] = np.nan
    x[0, 3] = np.nan
    x[1, :, 1:] = -np.inf          # one candidate each
    x[2] = -np.inf                 # none
    x[3, 0, 77] = x[3, 0, 8500] = np.inf
    x[3, 1, :] = np.inf
    x[4, 2] = 3e38
    x[4, 3] = -3e38
    scores[5] = [np.nan, -np.inf, -1.0, 0.0]
    check(pkg, logits, scores)
    x[:, :, 4096:] = -np.inf       # a slice without any
    check(pkg, logits, scores)


def test_far_scores_and_steep_rows(pkg):
    logits, scores = made(9, 3, 6, 40000, spread=300.0)
    check(pkg, logits, scores)
    logits, scores = made(10, 3, 6, 40000, spread=1e-3)
    scores = scores * 1e4
    check(pkg, logits, scores)


def test_scores_and_ended_in_place(pkg):
    logits, scores = made(5, 7, 8, 12345)
    rng = np.random.default_rng(2)
    ended = (rng.random((7, 8)) < 0.3).astype(np.int32)
    want = check(pkg, logits, scores, ended, [5, 17])
    x, s, e = torch.from_numpy(logits).cuda(), torch.from_numpy(scores).cuda(), torch.from_numpy(ended).cuda()
    p, t = torch.empty_like(e), torch.empty_like(e)
    work = torch.empty(pkg.lib().nls_beam_workspace(7, 8, 12345), dtype=torch.uint8, device="cuda")
    got = pkg.beam_select(x.view(7, 8, -1), s, ended=e, eog=torch.tensor([5, 17], dtype=torch.int32).cuda(), out=(p, t, s, e), work=work)
    assert got[2] is s and got[3] is e
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_rows_off_16_bytes(pkg):
    logits, scores = made(6, 2, 3, 10007)
    want = check(pkg, logits, scores)
    far = torch.zeros(logits.size + 3, device="cuda")
    far[3:] = torch.from_numpy(logits).cuda().view(-1)
    got = pkg.beam_select(far[3:].view(6, 10007), torch.from_numpy(scores).cuda())
    for a, b in zip(got, want):
        assert torch.equal(a, b)


# ---------------------------------------------------------------- contexts follow


class Model:
    """The page tables by their rules, and what every place of every slot's
    context holds (a number per token, the same in all layers)."""

    def __init__(self, slots, per, pages, ps):
        self.per, self.ps = per, ps
        self.table, self.lens, self.refs = [[-1] * per for _ in range(slots)], [0] * slots, [0] * pages
        self.held = [[] for _ in range(slots)]

    def lowest(self):
        return self.refs.index(0)

    def reserve(self, counts, tokens):
        for s, n in enumerate(counts):
            for j in range(-(-self.lens[s] // self.ps), -(-(self.lens[s] + n) // self.ps)):
                p = self.lowest()
                self.table[s][j], self.refs[p] = p, 1
            self.lens[s] += n
            self.held[s] = self.held[s] + tokens[s]

    def reorder(self, src):
        ps, slots = self.ps, range(len(src))
        refs, new, copies = list(self.refs), [], []
        first = {}
        for s in slots:
            if src[s] >= 0 and (src[s] not in first or src[s] == s):
                if first.get(src[s]) != src[s]:
                    first[src[s]] = s
        for s in slots:
            for p in self.table[s]:
                if p >= 0:
                    refs[p] -= 1
        for s in slots:
            row = [-1] * self.per
            if src[s] >= 0:
                n = self.lens[src[s]]
                keep = -(-n // ps) if first[src[s]] == s else n // ps
                row[:keep] = self.table[src[s]][:keep]
                for p in row[:keep]:
                    refs[p] += 1
                if n % ps and first[src[s]] != s:
                    copies.append((s, n // ps))
            new.append(row)
        if refs.count(0) < len(copies):
            return 1
        for s, j in copies:
            p = refs.index(0)
            new[s][j], refs[p] = p, 1
        self.lens = [self.lens[p] if p >= 0 else 0 for p in src]
        self.held = [list(self.held[p]) if p >= 0 else [] for p in src]
        self.table, self.refs = new, refs
        return 0

    def same(self, c):
        assert c.lens.tolist() == self.lens
        assert c.table.tolist() == self.table
        assert c.refs.tolist() == self.refs


def put(c, m, counts):
    """The new tokens' numbers into every layer of the cache."""
    starts = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    x = [t for s, n in enumerate(counts) for t in m.held[s][len(m.held[s]) - n:]]
    kvh, d = (c.fmt.kv_heads, c.fmt.head_dim) if c.fmt else (c.kv.shape[3], c.kv.shape[5])
    k = torch.tensor(x, dtype=torch.float32).view(-1, 1, 1).expand(-1, kvh, d).contiguous().cuda()
    for layer in range(c.kv.shape[0]):
        c.append(layer, k + layer, -k, torch.from_numpy(starts).cuda())


def holds(c, m):
    """Every context is what its history says, in every layer."""
    starts = torch.from_numpy(np.concatenate([[0], np.cumsum(m.lens)]).astype(np.int32)).cuda()
    want = np.array([t for h in m.held for t in h], dtype=np.float32)
    for layer in range(c.kv.shape[0]):
        k, v = (x.cpu().numpy() for x in c.read(layer, starts, len(want)))
        for got, w in ((k, want + layer), (v, -want)):
            if c.fmt:  # equal elements of a block: one factor, one code
                w = R.values(*R.blocks(np.repeat(w[:, None], 32, 1), c.fmt.kind))[:, 0]
            else:
                w = torch.from_numpy(w).to(c.kv.dtype).double().numpy()
            assert (got == w[:, None, None]).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32, "q8_0", "q4_0"], ids=str)
@pytest.mark.parametrize("slots,per,pages,ps,layers", [(4, 6, 30, 16, 2), (12, 9, 120, 16, 1), (1, 3, 4, 32, 3), (33, 4, 140, 16, 1)])
def test_contexts_follow(pkg, dtype, slots, per, pages, ps, layers):
    rng = random.Random(slots)
    c = pkg.PagedCache(layers, pages, ps, 2, 32, slots, per, dtype=dtype)
    m = Model(slots, per, pages, ps)
    for step in range(25):
        counts = [rng.choice([0, 1, 1, 2, 5, ps]) if n + ps <= per * ps else 0 for n in m.lens]
        need = sum(-(-(n + k) // ps) - -(-n // ps) for n, k in zip(m.lens, counts))
        if m.refs.count(0) >= need:
            m.reserve(counts, [[float(rng.randint(1, 99)) for _ in range(k)] for k in counts])
            assert c.reserve(torch.tensor(counts, dtype=torch.int32).cuda()).item() == 0
            put(c, m, counts)
        kind = step % 5
        src = [rng.randrange(slots) for _ in range(slots)]
        if kind == 1:
            src = [s if rng.random() < 0.7 else rng.randrange(-1, slots) for s in range(slots)]
        elif kind == 2:
            src = [slots - 1 - s for s in range(slots)]  # all change places
        elif kind == 3:
            src = [rng.randrange(slots)] * slots         # all go on from one
        elif kind == 4 and step > 20:
            src = [-1] * slots
        say(f"[reorder] step {step} {src}")
        st = m.reorder(src)
        got = c.reorder(torch.tensor(src, dtype=torch.int32).cuda()).item()
        assert got == st
        m.same(c)
        holds(c, m)


def test_reorder_does_all_or_nothing(pkg):
    c = pkg.PagedCache(1, 5, 16, 1, 32, 3, 4)
    c.reserve(torch.tensor([20, 5, 5], dtype=torch.int32).cuda())  # 4 of 5 pages
    state = [x.clone() for x in (c.table, c.lens, c.refs, c.kv)]
    same = lambda: all(torch.equal(a, b) for a, b in zip(state, (c.table, c.lens, c.refs, c.kv)))
    go = lambda *src: c.reorder(torch.tensor(src, dtype=torch.int32).cuda()).item()
    for src in ((0, 1, 3), (-2, 1, 2), (0, 1, 1 << 30)):
        assert go(*src) == pkg.PAGES_BAD_ENTRY and same()
    c.refs[4] = 1  # held by someone else
    state[2] = c.refs.clone()
    assert go(0, 0, 2) == pkg.PAGES_DONE  # slot 1's page serves the copy
    assert c.refs.tolist() == [2, 1, 1, 1, 1] and c.lens.tolist() == [20, 20, 5]
    state = [x.clone() for x in (c.table, c.lens, c.refs, c.kv)]
    assert go(0, 1, 0) == pkg.PAGES_DONE
    assert c.refs.tolist() == [3, 1, 1, 1, 1]
    c.lens[1] = -1
    state = [x.clone() for x in (c.table, c.lens, c.refs, c.kv)]
    assert go(0, 0, 0) == pkg.PAGES_BAD_ENTRY and same()
    c.lens[1] = 4 * 16 + 1
    state[1] = c.lens.clone()
    assert go(0, 0, 0) == pkg.PAGES_BAD_ENTRY and same()
    # none left: two contexts with partial pages, all pages held
    c = pkg.PagedCache(1, 3, 16, 1, 32, 3, 2)
    c.reserve(torch.tensor([5, 5, 0], dtype=torch.int32).cuda())
    c.refs[2] = 7
    state = [x.clone() for x in (c.table, c.lens, c.refs, c.kv)]
    assert go(0, 1, 1) == pkg.PAGES_NONE_LEFT and same()
    assert go(0, -1, 0) == pkg.PAGES_DONE and c.refs.tolist() == [1, 1, 7]


def test_reorder_many_slots(pkg):
    """More slots than the plan's threads, long rows, pages shared by many."""
    slots, per, ps = 2500, 7, 16
    c = pkg.PagedCache(1, 9000, ps, 1, 32, slots, per, dtype="q4_0")
    m = Model(slots, per, 9000, ps)
    rng = random.Random(8)
    counts = [rng.choice([0, 3, 16, 40]) for _ in range(slots)]
    m.reserve(counts, [[float(rng.randint(1, 99)) for _ in range(k)] for k in counts])
    assert c.reserve(torch.tensor(counts, dtype=torch.int32).cuda()).item() == 0
    put(c, m, counts)
    for _ in range(2):
        src = [rng.randrange(max(-1, s // 8 * 8 - 1), min(slots, s // 8 * 8 + 8)) for s in range(slots)]
        assert m.reorder(src) == 0
        assert c.reorder(torch.tensor(src, dtype=torch.int32).cuda()).item() == 0
        m.same(c)
        holds(c, m)


def test_reorder_over_the_most_pages(pkg):
    """524288 pages, contexts on the last ones, copies onto the lowest free one."""
    pages = 1 << 19
    c = pkg.PagedCache(1, pages, 1, 1, 8, 3, 5, dtype=torch.float16)
    c.page_size = 1
    c.refs.fill_(1)
    c.refs[pages - 3] = 0
    c.refs[7] = 0
    c.table[0, :2] = torch.tensor([pages - 1, pages - 2], dtype=torch.int32)
    c.lens[0] = 2
    assert c.reorder(torch.tensor([0, 0, -1], dtype=torch.int32).cuda()).item() == pkg.PAGES_DONE
    assert c.table.tolist() == [[pages - 1, pages - 2, -1, -1, -1]] * 2 + [[-1] * 5] and c.lens.tolist() == [2, 2, 0]
    assert c.refs[pages - 2:].tolist() == [2, 2]
    # pages of 2 tokens: the partial last one is copied to page 7
    wide = torch.randn(1, pages, 2, 1, 2, 8, device="cuda", dtype=torch.float16)
    before = wide[:, pages - 2].clone()
    table, lens = c.table.clone(), torch.tensor([3, 0, 0], dtype=torch.int32).cuda()
    table[1] = -1
    refs = c.refs.clone()
    refs[pages - 2:] = 1
    parents = torch.tensor([0, 0, 0], dtype=torch.int32).cuda()
    assert pkg.cache_reorder(wide, table, lens, refs, parents).item() == pkg.PAGES_DONE
    assert table[:, :3].tolist() == [[pages - 1, pages - 2, -1], [pages - 1, 7, -1], [pages - 1, pages - 3, -1]]
    assert torch.equal(wide[:, 7], before) and torch.equal(wide[:, pages - 3], before)
    assert refs[pages - 3:].tolist() == [1, 1, 3] and int(refs[7]) == 1 and lens.tolist() == [3] * 3


@pytest.mark.parametrize("slots,pages", [(5, 18), (2100, 4208), (5, 70001)])
def test_reorder_leaves_pages_that_others_hold(pkg, slots, pages):
    """Pages of contexts that end here, with more on their counts than the entries
    that let them go (a caller's own, or of slots outside of the given rows): no copy
    takes them, and the counts go down by what was let go."""
    ps, per = 16, 3
    c = pkg.PagedCache(2, pages, ps, 1, 32, slots, per, dtype=torch.float32)
    counts = [20, 18, 16, 32, 7] + [0] * (slots - 5)
    assert c.reserve(torch.tensor(counts, dtype=torch.int32).cuda()).item() == pkg.PAGES_DONE
    # 0: pages 0, 1; 1: pages 2, 3; 2: page 4; 3: pages 5, 6; 4: page 7
    c.kv.normal_()
    c.refs[2] = 2                  # one more holder
    c.refs[3] = 5
    c.refs[8:] = 1
    c.refs[pages - 3] = 0
    c.table[3, 0] = 4              # page 4 by two slots: 2 and 3 (page 5 is free then)
    c.refs[4], c.refs[5] = 2, 1    # 5: only someone else
    kv = c.kv.clone()
    parents = [0, 0, 0, 0, 0] + [-1] * (slots - 5)
    if slots > 2050:
        parents[2050] = 0
    # copies for slots 1, 2, 3, 4 (and 2050): the pages that were slot 2's and 3's alone
    # (4, held twice and let go twice, and 6), slot 4's, the free one, and no other
    n = sum(p == 0 for p in parents) - 1
    st = c.reorder(torch.tensor(parents, dtype=torch.int32).cuda()).item()
    if n > 4:
        assert st == pkg.PAGES_NONE_LEFT and torch.equal(c.kv, kv) and c.lens.tolist() == counts
        parents[2050] = -1
        st = c.reorder(torch.tensor(parents, dtype=torch.int32).cuda()).item()
    assert st == pkg.PAGES_DONE
    fresh = [4, 6, 7, pages - 3]
    assert c.table[:5].tolist() == [[0, 1, -1]] + [[0, p, -1] for p in fresh]
    assert c.refs[:8].tolist() == [5, 1, 1, 4, 1, 1, 1, 1] and int(c.refs[pages - 3]) == 1
    assert c.lens.tolist() == [20] * 5 + [0] * (slots - 5)
    kv[:, fresh] = kv[:, 1:2]
    assert torch.equal(c.kv, kv)


def test_reorder_of_some_rows_of_a_table(pkg):
    """Rows 2 and on of a table whose first two slots share pages with them."""
    c = pkg.PagedCache(1, 9, 16, 2, 32, 6, 3, dtype="q8_0")
    assert c.reserve(torch.tensor([37, 0, 0, 0, 5, 0], dtype=torch.int32).cuda()).item() == pkg.PAGES_DONE
    c.kv.random_(0, 255)
    to = lambda *x: torch.tensor(x, dtype=torch.int32).cuda()
    assert c.fork(to(0, 0), to(2, 3)).item() == pkg.PAGES_DONE  # pages 0, 1 three times; 2, 4, 5 theirs; slot 4: 3
    assert c.table.tolist()[:5] == [[0, 1, 2], [-1] * 3, [0, 1, 4], [0, 1, 5], [3, -1, -1]]
    kv = c.kv.clone()
    # slots 2 and 3 end, 4 and 5 go on from 4, with a copy
    st = pkg.cache_reorder(c.kv, c.table[2:], c.lens[2:], c.refs, to(-1, -1, 2, 2), fmt=c.fmt)
    assert st.item() == pkg.PAGES_DONE
    assert c.table.tolist() == [[0, 1, 2], [-1] * 3, [-1] * 3, [-1] * 3, [3, -1, -1], [4, -1, -1]]
    assert c.refs.tolist() == [1, 1, 1, 1, 1, 0, 0, 0, 0] and c.lens.tolist() == [37, 0, 0, 0, 5, 5]
    kv[:, 4] = kv[:, 3]
    assert torch.equal(c.kv, kv)


def test_sums_of_a_row_across_lanes(pkg):
    """One logit of weight 1 and 255 of 2^-26, no two within a thread's run: a lane
    that adds another's 2^-26 to its 1 in fp32 loses them one by one."""
    vocab = 1024
    logits = np.full((1, vocab), -np.inf, dtype=np.float32)
    logits[0, ::4] = -26 * math.log(2.0)
    logits[0, 0] = 0.0
    (parents, tokens, worth, over), _ = select(logits, np.zeros((1, 1), dtype=np.float32))
    assert -4e-6 < worth[0, 0] < -3e-6
    got = pkg.beam_select(torch.from_numpy(logits).cuda(), torch.zeros(1, 1, device="cuda"))
    assert got[0].item() == 0 and got[1].item() == 0
    # an exponential: its argument of 18 rounded twice (2 * 18 * 2^-24) and two units of its own
    assert abs(got[2].item() - worth[0, 0]) <= abs(worth[0, 0]) * (36 * 2.0 ** -24 + 2.0 ** -22 + 2.0 ** -24)


def test_equal_candidates_of_unequal_logits_beyond_the_lists(pkg):
    """Logits that are equal beside the rest of a candidate, in float64, and more
    candidates than the merge holds: the lowest ids come first all the same."""
    beams, vocab = 64, 40000
    logits, scores = np.zeros((beams, vocab), dtype=np.float32), np.full((1, beams), -3.0, dtype=np.float32)
    far = np.arange(1000, 1010)
    logits[:, far] = 1e-20
    p, t, s, e = (x.cpu().numpy() for x in pkg.beam_select(torch.from_numpy(logits).cuda(), torch.from_numpy(scores).cuda()))
    # a row's 64 largest logits: the ten, and the lowest 54 of the others
    assert np.array_equal(t[0], np.concatenate([np.arange(54), far])) and (p == 0).all() and (e == 0).all()
    want = -3.0 - math.log(vocab)
    assert (np.abs(s - want) <= LSE + 2.0 ** -24 * abs(want)).all()


@pytest.mark.parametrize("groups,beams,vocab", [(2, 48, 32000), (2, 56, 128256), (3, 64, 8000), (2, 64, 32000), (1, 64, 128256),
                                                (1, 33, 262144)])
def test_selection_of_many_beams(pkg, groups, beams, vocab):
    """Ordinary logits with as many beams as overflow the slices' lists and the
    merge's."""
    logits, scores = made(groups + beams + vocab, groups, beams, vocab)
    say(f"[beams] {groups}x{beams}x{vocab}")
    check(pkg, logits, scores)
    # beams of one score, as after a first step, and logits whose mass is on a few ids
    g = np.random.default_rng(beams)
    scores = (g.standard_normal((groups, beams)) * 0.1 - 3).astype(np.float32)
    logits[:, g.integers(0, vocab, 300)] += np.abs(g.standard_normal(300) * 4).astype(np.float32)
    check(pkg, logits, scores, (g.random((groups, beams)) < 0.2).astype(np.int32), [5, 7])

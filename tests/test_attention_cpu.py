"""nimllm_attention.h without a GPU: the rotary frequencies against their
formulas, the index arithmetic of the paged cache, and every refusal of the C
ABI, which comes before any device work (the pointers here are no memory)."""
import ctypes
import math
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
OK, INVALID = 0, 1


def test_index_arithmetic(tmp_path):
    exe = str(tmp_path / "paged_check")
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-fsanitize=address,undefined", "-fno-sanitize-recover=all",
                    os.path.join(ROOT, "tests", "paged_check.cpp"), "-o", exe], check=True)
    out = subprocess.run([exe], check=True, capture_output=True, text=True).stdout
    assert out.startswith("ok"), out


@pytest.mark.parametrize("dim,base", [(2, 10000.0), (64, 10000.0), (128, 500000.0), (38, 1e6)])
def test_rope_frequencies(pkg, dim, base):
    plain = [base ** (-2.0 * j / dim) for j in range(dim // 2)]
    close = lambda a, b: all(abs(x - y) <= 4 * 2.0 ** -52 * abs(y) * 16 for x, y in zip(a, b)) and len(a) == len(b)
    f, amp = pkg.rope_frequencies(dim, base=base)
    assert close(f, plain) and amp == 1.0
    f, amp = pkg.rope_frequencies(dim, base=base, scaling="linear", factor=4.0, attn_factor=0.5)
    assert close(f, [x / 4.0 for x in plain]) and amp == 0.5
    factors = [1.0 + j for j in range(dim // 2)]
    f, amp = pkg.rope_frequencies(dim, base=base, freq_factors=factors)
    assert close(f, [x / y for x, y in zip(plain, factors)])
    f, amp = pkg.rope_frequencies(dim, base=base, scaling="yarn", factor=8.0, original_context=4096.0)
    assert abs(amp - (0.1 * math.log(8.0) + 1.0)) < 1e-15
    for j, (x, y) in enumerate(zip(f, plain)):
        turns = 4096.0 * y / (2 * math.pi)  # over the original context
        assert y / 8.0 * (1 - 1e-12) <= x <= y * (1 + 1e-12)
        if turns >= 64.0:
            assert abs(x - y) <= 1e-12 * y, j
        if turns <= 0.5 and j >= 2:
            assert abs(x - y / 8.0) <= 1e-12 * y, j
    assert pkg.rope_frequencies(0) == ([], 1.0)


def test_rope_frequencies_refusals(pkg):
    bad = [dict(dim=63), dict(dim=-2), dict(dim=64, base=0.0), dict(dim=64, base=math.inf), dict(dim=64, base=math.nan),
           dict(dim=64, scaling="linear", factor=0.0), dict(dim=64, scaling="linear", factor=math.nan),
           dict(dim=64, scaling="yarn", factor=4.0), dict(dim=64, scaling="yarn", factor=4.0, original_context=math.inf),
           dict(dim=64, scaling="yarn", factor=4.0, original_context=4096.0, beta_fast=0.0),
           dict(dim=64, scaling="yarn", factor=4.0, original_context=4096.0, base=1.0),
           dict(dim=64, attn_factor=math.nan), dict(dim=64, scaling="other"),
           dict(dim=4, freq_factors=[1.0, 0.0]), dict(dim=4, freq_factors=[math.nan, 1.0])]
    for kw in bad:
        with pytest.raises(pkg.SamplerError):
            pkg.rope_frequencies(**kw)
    amp = ctypes.c_double()
    s = pkg.NlsRopeScaling(7, 10000.0, 1.0, 0, 32, 1, 1, None)
    assert pkg.lib().nls_rope_frequencies(ctypes.byref(s), 0, None, ctypes.byref(amp)) == INVALID
    assert pkg.lib().nls_rope_frequencies(None, 0, None, ctypes.byref(amp)) == INVALID


AT = 1 << 20  # an address; nothing reads it


def _cache(pkg, **kw):
    f = dict(d_kv=AT, type=1, pages=10, page_size=16, kv_heads=2, head_dim=64, page_stride=2 * 2 * 16 * 64,
             value_offset=2 * 16 * 64, head_stride=16 * 64, token_stride=64, d_table=AT, table_stride=5, slots=3,
             max_pages=5, d_lens=AT)
    f.update(kw)
    return pkg.NlsPagedKv(**f)


BAD_CACHES = [dict(d_kv=None), dict(d_kv=AT + 8), dict(type=2), dict(type=-1), dict(pages=0), dict(page_size=0),
              dict(page_size=24), dict(page_size=8192), dict(kv_heads=0), dict(head_dim=0), dict(head_dim=60),
              dict(head_dim=264), dict(page_stride=-8), dict(page_stride=4), dict(page_stride=8), dict(value_offset=8),
              dict(value_offset=1028), dict(head_stride=8), dict(token_stride=8), dict(token_stride=1 << 50), dict(page_stride=1 << 30),
              dict(d_table=None), dict(d_table=AT + 2), dict(table_stride=4), dict(table_stride=-1), dict(slots=0),
              dict(max_pages=0), dict(d_lens=None), dict(d_lens=AT + 1)]
BAD_CHUNKS = [dict(seqs=-1), dict(tokens=-1), dict(d_starts=None), dict(d_starts=AT + 2), dict(d_slots=AT + 1)]
BAD_HEADS = [dict(d=None), dict(d=AT + 1), dict(token_stride=-1), dict(head_stride=-1), dict(head_stride=1 << 50)]
OVERLAPS = [dict(head_stride=32), dict(token_stride=0), dict(token_stride=64, head_stride=64), dict(token_stride=200),
            dict(head_stride=400, token_stride=64)]


def _chunks(pkg, **kw):
    f = dict(seqs=2, tokens=9, d_starts=AT, d_slots=None)
    f.update(kw)
    return pkg.NlsChunks(**f)


def _heads(pkg, **kw):
    f = dict(d=AT, token_stride=256, head_stride=64)
    f.update(kw)
    return pkg.NlsHeads(**f)


def test_attention_refusals(pkg):
    L = pkg.lib()

    def call(c=None, ch=None, type=0, q=None, out=None, heads=4, scale=0.125, window=0, first=None, lse=None, max_new=1,
             max_len=80, work=AT, work_bytes=1 << 40):
        return L.nls_paged_attention(c or _cache(pkg), ch or _chunks(pkg), type, q or _heads(pkg), out or _heads(pkg),
                                     heads, scale, window, first, lse, max_new, max_len, work, work_bytes, None)

    for kw in BAD_CACHES:
        assert call(c=_cache(pkg, **kw)) == INVALID, kw
    for kw in BAD_CHUNKS:
        assert call(ch=_chunks(pkg, **kw)) == INVALID, kw
    for kw in BAD_HEADS:
        assert call(q=_heads(pkg, **kw)) == INVALID, kw
        assert call(out=_heads(pkg, **kw)) == INVALID, kw
    for kw in OVERLAPS:
        assert call(out=_heads(pkg, **kw)) == INVALID, kw
    for kw in (dict(type=30), dict(type=8), dict(heads=0), dict(heads=3), dict(heads=-2), dict(heads=1 << 20),
               dict(scale=math.inf), dict(scale=math.nan), dict(window=-1), dict(ch=_chunks(pkg, tokens=1 << 24)), dict(first=AT + 2), dict(lse=AT + 1),
               dict(max_new=-1), dict(max_len=-1)):
        assert call(**kw) == INVALID, kw
    need = L.nls_paged_attention_workspace(_cache(pkg), _chunks(pkg), 4, 1, 1 << 20, 0)
    if need:
        long = dict(max_len=1 << 20)
        assert call(work=None, **long) == INVALID
        assert call(work=AT + 16, **long) == INVALID
        assert call(work_bytes=need - 1, **long) == INVALID
    assert L.nls_paged_attention(None, _chunks(pkg), 0, _heads(pkg), _heads(pkg), 4, 1.0, 0, None, None, 1, 1, AT, 1 << 40,
                                 None) == INVALID
    assert L.nls_paged_attention(_cache(pkg), None, 0, _heads(pkg), _heads(pkg), 4, 1.0, 0, None, None, 1, 1, AT, 1 << 40,
                                 None) == INVALID
    assert L.nls_last_error()
    # nothing to do is no error
    assert call(ch=_chunks(pkg, tokens=0, d_starts=None)) == OK
    assert call(ch=_chunks(pkg, seqs=0, d_starts=None)) == OK
    for kw in (dict(tokens=0), dict(seqs=0)):
        assert L.nls_paged_attention_workspace(_cache(pkg), _chunks(pkg, **kw), 4, 1, 1 << 20, 0) == 0
    # a table of more places than a context has tokens counts as its longest context
    for tokens, heads, max_new in ((1 << 20, 32, 0), (3, 4, 1), (900, 4, 0)):
        ch = _chunks(pkg, seqs=3, tokens=tokens)
        size = lambda max_len, **kw: L.nls_paged_attention_workspace(_cache(pkg, page_size=4096, **kw), ch, heads, max_new,
                                                                     max_len, 0)
        assert size(0, max_pages=1 << 20) == size(1 << 40, max_pages=1 << 20) == size(0x7fffff00, max_pages=1 << 20)
    assert L.nls_paged_attention_workspace(_cache(pkg, page_size=4096, max_pages=1 << 20), _chunks(pkg, seqs=1, tokens=1 << 20),
                                           32, 0, 0, 0) == 0
    # the workspace's own checks
    for kw in (dict(kv_heads=0), dict(head_dim=300), dict(page_size=5), dict(max_pages=0)):
        assert L.nls_paged_attention_workspace(_cache(pkg, **kw), _chunks(pkg), 4, 1, 100, 0) == 0
    assert L.nls_paged_attention_workspace(_cache(pkg), _chunks(pkg), 3, 1, 100, 0) == 0
    assert L.nls_paged_attention_workspace(None, _chunks(pkg), 4, 1, 100, 0) == 0


def test_append_and_rope_refusals(pkg):
    L = pkg.lib()
    plan = pkg.NlsRopePlan(AT, 64, 1, 1.0)
    bad_plans = [pkg.NlsRopePlan(None, 64, 1, 1.0), pkg.NlsRopePlan(AT + 4, 64, 1, 1.0), pkg.NlsRopePlan(AT, 63, 1, 1.0),
                 pkg.NlsRopePlan(AT, 66, 1, 1.0), pkg.NlsRopePlan(AT, -2, 1, 1.0)]

    def append(c=None, ch=None, plan=plan, type=0, q=None, out=None, heads=4, k=None, v=None):
        h = lambda x: x or _heads(pkg)
        return L.nls_cache_append(c or _cache(pkg), ch or _chunks(pkg), plan, type, h(q), h(out), heads, h(k), h(v), None)

    for kw in BAD_CACHES:
        assert append(c=_cache(pkg, **kw)) == INVALID, kw
    for kw in BAD_CHUNKS:
        assert append(ch=_chunks(pkg, **kw)) == INVALID, kw
    for kw in BAD_HEADS:
        for name in ("q", "out", "k", "v"):
            assert append(**{name: _heads(pkg, **kw)}) == INVALID, (name, kw)
    for kw in OVERLAPS:
        assert append(out=_heads(pkg, **kw)) == INVALID, kw
    for p in bad_plans:
        assert append(plan=p) == INVALID
    assert append(type=30) == INVALID and append(type=14) == INVALID and append(heads=-1) == INVALID
    assert append(out=_heads(pkg, token_stride=512)) == INVALID  # in place with other strides
    assert append(ch=_chunks(pkg, tokens=0)) == OK

    def rope(plan=plan, type=0, x=None, y=None, tokens=3, heads=4, dim=64, pos=AT):
        return L.nls_rope(plan, type, x or _heads(pkg), y or _heads(pkg), tokens, heads, dim, pos, 0, None)

    for kw in BAD_HEADS:
        assert rope(x=_heads(pkg, **kw)) == INVALID and rope(y=_heads(pkg, **kw)) == INVALID, kw
    for kw in OVERLAPS[:-1]:
        assert rope(y=_heads(pkg, **kw)) == INVALID, kw
    for p in bad_plans:
        assert rope(plan=p) == INVALID
    for kw in (dict(type=3), dict(tokens=-1), dict(tokens=1 << 24), dict(heads=-1), dict(dim=0), dict(dim=257), dict(pos=None), dict(pos=AT + 2),
               dict(y=_heads(pkg, token_stride=512))):
        assert rope(**kw) == INVALID, kw
    assert L.nls_rope(None, 0, _heads(pkg), _heads(pkg), 1, 1, 64, AT, 0, None) == INVALID
    assert rope(tokens=0) == OK and rope(heads=0) == OK


def test_page_call_refusals(pkg):
    L = pkg.lib()

    def tables(**kw):
        f = dict(d_table=AT, table_stride=5, slots=3, max_pages=5, d_lens=AT, d_refs=AT, pages=10, page_size=16)
        f.update(kw)
        return pkg.NlsPageTables(**f)

    def pool(**kw):
        f = dict(d_kv=AT, layers=2, page_bytes=4096, layer_stride=40960, page_stride=4096)
        f.update(kw)
        return pkg.NlsPagePool(**f)

    big = 1 << 30
    bad_tables = [dict(d_table=None), dict(d_table=AT + 2), dict(table_stride=4), dict(slots=0), dict(max_pages=0),
                  dict(d_refs=None), dict(d_refs=AT + 1), dict(pages=0), dict(pages=(1 << 19) + 1), dict(slots=(1 << 16) + 1), dict(page_size=3),
                  dict(page_size=0), dict(page_size=8192), dict(slots=1 << 16, max_pages=1 << 16, table_stride=1 << 16)]
    bad_pools = [dict(d_kv=None), dict(d_kv=AT + 8), dict(layers=0), dict(page_bytes=0), dict(page_bytes=24),
                 dict(layer_stride=8), dict(page_stride=2048), dict(page_stride=-16), dict(layer_stride=2048)]
    reserve = lambda t, c=AT, st=AT, w=AT, n=big: L.nls_cache_reserve(t, c, st, w, n, None)
    fork = lambda p, t, a=AT, b=AT, n=2, st=AT, w=AT, wb=big: L.nls_cache_fork(p, t, a, b, n, st, w, wb, None)
    release = lambda t, s=AT, n=2, st=AT, w=AT, wb=big: L.nls_cache_release(t, s, n, st, w, wb, None)
    compact = lambda p, t, live=AT, w=AT, wb=big: L.nls_cache_compact(p, t, live, w, wb, None)
    for kw in bad_tables:
        t = tables(**kw)
        assert reserve(t) == fork(pool(), t) == release(t) == compact(pool(), t) == INVALID, kw
    t = tables(d_lens=None)
    assert reserve(t) == fork(pool(), t) == release(t) == INVALID
    for kw in bad_pools:
        p = pool(**kw)
        assert fork(p, tables()) == compact(p, tables()) == L.nls_cache_copy_pages(p, 10, AT, AT, 1, None) == INVALID, kw
    t = tables()
    need = L.nls_cache_workspace(t, 2)
    assert need > 0 and need % 256 == 0
    for w, n in ((None, big), (AT + 16, big), (AT, need - 256)):
        assert reserve(t, w=w, n=n) == fork(pool(), t, w=w, wb=n) == release(t, w=w, wb=n) == INVALID
        assert compact(pool(), t, w=w, wb=n) == INVALID
    assert reserve(t, c=None) == reserve(t, st=None) == reserve(t, c=AT + 2) == INVALID
    assert fork(pool(), t, a=None) == fork(pool(), t, b=None) == fork(pool(), t, n=-1) == fork(pool(), t, n=4) == INVALID
    assert fork(pool(), t, st=AT + 1) == INVALID
    assert release(t, s=None) == release(t, n=-1) == release(t, st=None) == INVALID
    assert compact(pool(), t, live=None) == INVALID
    copy = lambda pages=10, a=AT, b=AT, n=2: L.nls_cache_copy_pages(pool(), pages, a, b, n, None)
    assert copy(pages=0) == copy(a=None) == copy(b=AT + 1) == copy(n=-1) == INVALID
    assert copy(n=0) == OK
    assert L.nls_cache_workspace(None, 0) == 0 and L.nls_cache_workspace(t, -1) == 0


def test_scales_beyond_the_exponents_base_are_refused(pkg):
    """A scale that is finite, but infinite in exponents of base 2, would make a
    score of 0 NaN."""
    call = lambda scale: pkg.lib().nls_paged_attention(_cache(pkg), _chunks(pkg), 0, _heads(pkg), _heads(pkg), 4, scale, 0, None,
                                                       None, 1, 80, None, 0, None)
    for scale in (2.4e38, -2.4e38, 3.4e38):
        assert call(scale) == INVALID, scale
        assert b"log2" in pkg.lib().nls_last_error()
    # (below the limit the call goes on to its other checks: its rows are none)
    none = _chunks(pkg, tokens=0, d_starts=None)
    for scale in (2.3e38, -2.3e38, 1e-45, 0.0):
        assert pkg.lib().nls_paged_attention(_cache(pkg), none, 0, _heads(pkg), _heads(pkg), 4, scale, 0, None, None, 1, 80, None,
                                             0, None) == OK


@pytest.mark.parametrize("chunks,heads,max_new,max_len", [
    (dict(seqs=2, tokens=2), 4, 1, 0),                  # single tokens, the keys split over workgroups
    (dict(seqs=2, tokens=2), 4, 1, 1 << 15),
    (dict(seqs=2, tokens=2), 4, 0, 0),
    (dict(seqs=1, tokens=90), 4, 0, 0),                 # one chunk
    (dict(seqs=2, tokens=90), 4, 80, 40000),            # a chunk and few rows
    (dict(seqs=2, tokens=90), 32, 0, 0)])
@pytest.mark.parametrize("head_dim", [64, 128, 256])
def test_attention_workspace_refusals(pkg, chunks, heads, max_new, max_len, head_dim):
    """Calls whose parts wait in the workspace: none, a misaligned one and one a
    byte too short are refused before any device work."""
    L = pkg.lib()
    c = _cache(pkg, max_pages=4096, table_stride=4096, head_dim=head_dim, head_stride=16 * head_dim, token_stride=head_dim,
               value_offset=2 * 16 * head_dim, page_stride=4 * 16 * head_dim)
    ch = _chunks(pkg, **chunks)
    rows = _heads(pkg, token_stride=heads * head_dim, head_stride=head_dim)
    need = L.nls_paged_attention_workspace(c, ch, heads, max_new, max_len, 0)
    assert need > 0 and need % 256 == 0
    call = lambda work, size: L.nls_paged_attention(c, ch, 0, rows, rows, heads, 0.125, 0, None, None, max_new, max_len, work,
                                                    size, None)
    for work, size in ((None, need), (AT, need - 1), (AT, 0), (AT + 16, need), (AT + 128, 1 << 40)):
        assert call(work, size) == INVALID, (work, size)
        assert b"workspace" in L.nls_last_error()
    # a window shortens what is split, and with it the workspace
    assert L.nls_paged_attention_workspace(c, ch, heads, max_new, max_len, 64) < need


_REFUSED = '''
import importlib.util, sys
import torch
spec = importlib.util.spec_from_file_location("nimllm_amd", sys.argv[1], submodule_search_locations=[])
m = importlib.util.module_from_spec(spec)
sys.modules["nimllm_amd"] = m
spec.loader.exec_module(m)
if __debug__:
    sys.exit("run with -O")


class OnGpu(torch.Tensor):
    """Host memory that says it is device 0's; nothing is launched."""
    def get_device(self):
        return 0


launched = []
m._launch = lambda device, what, *args: launched.append(what)
gpu = lambda t: t.as_subclass(OnGpu)
ints = lambda n, dtype=torch.int32: gpu(torch.zeros(n, dtype=dtype))
real = lambda *shape, dtype=torch.float32: gpu(torch.zeros(shape, dtype=dtype))
kv, table, lens, starts = real(6, 2, 2, 16, 64), ints((3, 4)), ints(3), ints(3)
q, k = real(5, 4, 64), real(5, 2, 64)
pool, refs = real(1, 6, 2, 2, 16, 64), ints(6)
plan = m.RopePlan(gpu(torch.ones(32, dtype=torch.float64)))
attend = dict(q=q, kv=kv, table=table, lens=lens, starts=starts, out=q.clone())
append = dict(kv=kv, table=table, lens=lens, starts=starts, k=k, v=k, q=q, plan=plan, out=q)
calls = {
    m.rope: (dict(x=q, positions=ints(5), plan=plan, out=q), [
        dict(positions=ints(4)), dict(positions=ints(5, torch.int64)), dict(positions=gpu(torch.zeros(10, dtype=torch.int32)[::2])),
        dict(positions=torch.zeros(5, dtype=torch.int32)), dict(out=real(5, 4, 32)), dict(out=real(5, 4, 64, dtype=torch.float16)),
        dict(x=torch.zeros(5, 4, 64), out=torch.zeros(5, 4, 64)), dict(plan=m.RopePlan(real(32))),
        dict(plan=m.RopePlan(torch.ones(32, dtype=torch.float64))), dict(x=gpu(torch.zeros(5, 64, 4).transpose(1, 2)))]),
    m.paged_attention: (attend, [
        dict(first=ints(2)), dict(slots=ints(3)), dict(lens=ints(2)), dict(lens=ints(3, torch.int64)), dict(table=ints((3, 4), torch.int64)),
        dict(table=gpu(torch.zeros((4, 3), dtype=torch.int32).t())), dict(starts=ints(0)), dict(starts=torch.zeros(3, dtype=torch.int32)),
        dict(q=real(5, 4, 32), out=real(5, 4, 32)), dict(out=real(4, 4, 64)), dict(lse=real(5, 3)), dict(lse=real(5, 4, dtype=torch.float16)),
        dict(lse=torch.zeros(5, 4)), dict(kv=real(6, 1, 2, 16, 64)), dict(kv=torch.zeros(6, 2, 2, 16, 64)), dict(max_len=64, work=torch.zeros(1 << 20)),
        dict(kv=gpu(torch.zeros(6, 2, 2, 64, 16).transpose(3, 4)))]),
    m.cache_append: (append, [
        dict(v=real(4, 2, 64)), dict(k=real(5, 1, 64), v=real(5, 1, 64)), dict(k=real(5, 2, 32), v=real(5, 2, 32)), dict(q=real(4, 4, 64), out=real(4, 4, 64)),
        dict(out=real(5, 3, 64)), dict(q=None), dict(v=real(5, 2, 64, dtype=torch.float16)), dict(slots=ints(1)), dict(lens=ints(4))]),
    m.cache_reserve: (dict(table=table, lens=lens, refs=refs, page_size=16, counts=ints(3)), [
        dict(counts=ints(2)), dict(counts=ints(3, torch.int64)), dict(lens=ints(2)), dict(refs=ints(6, torch.int64))]),
    m.cache_fork: (dict(kv=pool, table=table, lens=lens, refs=refs, src=ints(1), dst=ints(1)), [
        dict(dst=ints(2)), dict(refs=ints(5)), dict(kv=pool[..., :32]), dict(lens=ints(2))]),
    m.cache_release: (dict(table=table, lens=lens, refs=refs, slots=ints(2), page_size=16), [
        dict(slots=ints(2, torch.int64)), dict(lens=ints(4)), dict(slots=torch.zeros(2, dtype=torch.int32))]),
    m.cache_compact: (dict(kv=pool, table=table, refs=refs), [dict(refs=ints(7)), dict(kv=pool[:, :, :, :1])]),
    m.cache_copy_pages: (dict(kv=pool, src=ints(2), dst=ints(2)), [
        dict(src=ints(3)), dict(kv=torch.zeros(1, 6, 2, 2, 16, 64)), dict(kv=pool[..., ::2])]),
}
bad = []
for call, (good, wrong) in calls.items():
    call(**good)
    if not launched:
        bad.append((call.__name__, "the right call was not made"))
    for i, kw in enumerate(wrong):
        del launched[:]
        try:
            call(**{**good, **kw})
            bad.append((call.__name__, i, sorted(kw), "was taken"))
        except (AssertionError, m.SamplerError):
            pass
        if launched:
            bad.append((call.__name__, i, sorted(kw), "was launched"))
    del launched[:]
try:
    m.rope_frequencies(64, freq_factors=[1.0] * 31)
    bad.append("freq_factors")
except AssertionError:
    pass
print(bad or "all refused")
'''


@pytest.mark.parametrize("flag", ["-O", "-OO"])
def test_python_refusals_without_asserts(tmp_path, flag):
    """What the C ABI cannot see is refused by the Python entry points under
    python -O as well."""
    script = tmp_path / "refused.py"
    script.write_text(_REFUSED)
    done = subprocess.run([sys.executable, flag, str(script), os.path.join(ROOT, "nim.llm_amd", "__init__.py")],
                          capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and done.stdout.strip() == "all refused", done.stdout + done.stderr[-2000:]


def test_numbers_beyond_32_bits_are_refused(pkg, monkeypatch):
    """ctypes would cut them: a window of 2^32 + 5 would be one of 5."""
    import torch

    class OnGpu(torch.Tensor):
        def get_device(self):
            return 0

    launched = []
    monkeypatch.setattr(pkg, "_launch", lambda device, what, *args: launched.append(what))
    ints = lambda *n: torch.zeros(n, dtype=torch.int32).as_subclass(OnGpu)
    real = lambda *n: torch.zeros(n).as_subclass(OnGpu)
    q, args = real(2, 4, 64), (real(6, 2, 2, 16, 64), ints(3, 4), ints(3), ints(3))
    for kw in (dict(window=(1 << 32) + 5), dict(window=1 << 32), dict(window=1 << 31), dict(window=-(1 << 32)), dict(window=-1),
               dict(max_new=(1 << 32) + 1), dict(max_new=-1), dict(max_len=1 << 64), dict(max_len=-1)):
        with pytest.raises(AssertionError):
            pkg.paged_attention(q, *args, out=real(2, 4, 64), **kw)
        with pytest.raises(AssertionError):
            pkg.paged_attention_workspace(q, *args, **kw)
    for page in ((1 << 32) + 16, 0, -16, 8192):
        with pytest.raises(AssertionError):
            pkg.cache_reserve(ints(3, 4), ints(3), ints(6), page, ints(3))
        with pytest.raises(AssertionError):
            pkg.cache_release(ints(3, 4), ints(3), ints(6), ints(1), page)
    assert not launched
    pkg.paged_attention(q, *args, out=real(2, 4, 64), window=(1 << 31) - 1, max_new=(1 << 31) - 1, max_len=(1 << 63) - 1)
    pkg.cache_reserve(ints(3, 4), ints(3), ints(6), 16, ints(3))
    assert launched == ["nls_paged_attention", "nls_cache_reserve"]

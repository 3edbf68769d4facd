"""Caches of blocks and beam search without a GPU: where blocks lie, and every
refusal of the C ABI, which comes before any device work (the pointers here are
no memory)."""
import math
import os
import subprocess

import numpy as np
import pytest

import quant_ref as R

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
OK, INVALID, EMPTY = 0, 1, 2
AT = 1 << 20  # an address; nothing reads it


def test_places_of_blocks(tmp_path):
    exe = str(tmp_path / "quant_check")
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-fsanitize=address,undefined", "-fno-sanitize-recover=all",
                    os.path.join(ROOT, "tests", "quant_check.cpp"), "-o", exe], check=True)
    lines = subprocess.run([exe], check=True, capture_output=True, text=True).stdout.split("\n")
    assert lines[-2:] == ["ok", ""]
    for line in lines[:-2]:
        kind, dim, k, e, byte, shift = map(int, line.split())
        assert R.place(dim, 8 if kind == 8 else 4, k == 1, e) == (byte, shift)
    assert len(lines) - 2 == 2 * 2 * sum(range(32, 257, 32))


@pytest.mark.parametrize("kind", ["q8_0", "q4_0"])
def test_blocks_by_hand(kind):
    """The definition itself, at elements whose codes are known."""
    x = np.zeros((1, 32), dtype=np.float32)
    assert R.blocks(x, kind)[1][0, 0] == 0 and not R.blocks(x, kind)[0].any()
    x[0, :3] = (1.0, -0.5, 0.25)
    c, d = R.blocks(x, kind)
    most = 127 if kind == "q8_0" else 7
    assert d[0, 0] == np.float16(np.float32(1.0) * (np.float32(1) / np.float32(most))) and c[0, 0] == most
    assert abs(c[0, 1] + most / 2) <= 1 and abs(c[0, 2] - most / 4) <= 1 and not c[0, 3:].any()
    if kind == "q4_0":
        x[0, 0] = -8.0
        c, d = R.blocks(x, kind)
        assert d[0, 0] == 1 and c[0, 0] == -8 and c[0, 1] == 0  # -0.5 to the even


def test_page_bytes(pkg):
    size = pkg.lib().nls_cache_page_bytes
    assert size(8, 3, 16, 64) == 3 * 2 * (16 * 64 + 16 * 2 * 2) == pkg.PageFormat("q8_0", 3, 16, 64).page_bytes
    assert size(2, 8, 4096, 256) == 8 * 2 * (4096 * 128 + 4096 * 8 * 2) == pkg.PageFormat("q4_0", 8, 4096, 256).page_bytes
    assert size(0, 2, 1, 8) == 2 * 2 * 8 * 4 and size(1, 2, 16, 80) == size(30, 2, 16, 80) == 2 * 2 * 16 * 80 * 2
    for bad in ((3, 1, 16, 64), (-1, 1, 16, 64), (8, 0, 16, 64), (8, 1, 8, 64), (8, 1, 24, 64), (8, 1, 8192, 64), (8, 1, 16, 0),
                (8, 1, 16, 48), (2, 1, 16, 288), (1, 1, 16, 4), (1, 1, 0, 64)):
        assert size(*bad) == -1, bad
    for bad in (("q5_0", 1, 16, 64), ("q4_0", -1, 16, 64), ("q4_0", 1 << 40, 16, 64), ("q4_0", 1, 1 << 33, 64), ("q4_0", 1, 16, 64 + (1 << 32))):
        with pytest.raises(pkg.SamplerError):
            pkg.PageFormat(*bad).page_bytes


def _cache(pkg, kind=2, **kw):
    f = dict(d_kv=AT, type=kind, pages=10, page_size=16, kv_heads=2, head_dim=64, page_stride=4 * (16 * 8 * kind * 2 + 64) if kind == 2 else 4 * (1024 + 64),
             value_offset=0, head_stride=0, token_stride=0, d_table=AT, table_stride=5, slots=3, max_pages=5, d_lens=AT)
    f.update(kw)
    return pkg.NlsPagedKv(**f)


BAD = [dict(d_kv=None), dict(d_kv=AT + 8), dict(pages=0), dict(page_size=8), dict(page_size=24), dict(head_dim=48), dict(head_dim=288),
       dict(kv_heads=0), dict(page_stride=-16), dict(page_stride=8), dict(page_stride=1024), dict(page_stride=4 * 1088 + 8),
       dict(page_stride=1 << 50), dict(value_offset=2048), dict(head_stride=1024), dict(token_stride=64), dict(table_stride=4),
       dict(d_table=None), dict(d_lens=None), dict(slots=0), dict(kv_heads=1 << 20, page_size=4096, head_dim=256, page_stride=1 << 39), dict(type=3)]


@pytest.mark.parametrize("kind", [8, 2])
def test_refusals_over_blocks(pkg, kind):
    L = pkg.lib()
    ch = lambda **kw: pkg.NlsChunks(**{**dict(seqs=2, tokens=9, d_starts=AT, d_slots=None), **kw})
    hd = lambda **kw: pkg.NlsHeads(**{**dict(d=AT, token_stride=256, head_stride=64), **kw})

    def attend(c=None, chunks=None, type=0, q=None, out=None, heads=4, scale=0.125):
        return L.nls_paged_attention(c or _cache(pkg, kind), chunks or ch(), type, q or hd(), out or hd(), heads, scale, 0, None, None, 1, 80,
                                     AT, 1 << 40, None)

    def append(c=None, chunks=None, type=0, k=None, v=None, plan=None):
        return L.nls_cache_append(c or _cache(pkg, kind), chunks or ch(), plan, type, hd(), hd(), 4, k or hd(), v or hd(), None)

    def read(c=None, chunks=None, type=0, k=None, v=None):
        return L.nls_cache_read(c or _cache(pkg, kind), chunks or ch(), type, k or hd(), v or hd(), None)

    for call in (attend, append, read):
        for kw in BAD:
            assert call(c=_cache(pkg, kind, **kw)) == INVALID, kw
        for kw in (dict(seqs=-1), dict(tokens=-1), dict(d_starts=None), dict(d_starts=AT + 2), dict(d_slots=AT + 1), dict(tokens=1 << 24)):
            assert call(chunks=ch(**kw)) == INVALID, kw
        for t in (8, 2, 3, -1):
            assert call(type=t) == INVALID
        for t in (0, 1, 30):  # any type of rows, none of them here
            assert call(type=t, chunks=ch(tokens=0, d_starts=None)) == OK
    for kw in (dict(d=None), dict(d=AT + 1), dict(token_stride=-1), dict(head_stride=1 << 50)):
        assert append(k=hd(**kw)) == append(v=hd(**kw)) == read(k=hd(**kw)) == read(v=hd(**kw)) == attend(q=hd(**kw)) == INVALID
    for kw in (dict(head_stride=32), dict(token_stride=0), dict(token_stride=100)):  # rows that overlap
        assert read(k=hd(**kw)) == read(v=hd(**kw)) == attend(out=hd(**kw)) == INVALID
    assert append(plan=pkg.NlsRopePlan(AT, 128, 1, 1.0)) == append(plan=pkg.NlsRopePlan(None, 64, 1, 1.0)) == INVALID
    assert attend(scale=math.inf) == attend(heads=3) == INVALID
    assert L.nls_cache_read(None, ch(), 0, hd(), hd(), None) == L.nls_cache_read(_cache(pkg, kind), None, 0, hd(), hd(), None) == INVALID
    # a wide cache is read by the same call, and refused by its own rules
    wide = dict(type=1, page_stride=2 * 2 * 16 * 64, value_offset=2 * 16 * 64, head_stride=16 * 64, token_stride=64)
    assert read(c=_cache(pkg, kind, **wide), chunks=ch(seqs=0, d_starts=None)) == OK
    assert read(c=_cache(pkg, kind, **{**wide, "token_stride": 8})) == INVALID


def test_beam_refusals(pkg):
    L = pkg.lib()

    def call(logits=AT, groups=3, beams=4, vocab=1000, scores=AT, ended=AT, eog=AT, n_eog=2, parents=AT, tokens=AT, out=AT, over=AT, work=AT,
             bytes=1 << 40):
        return L.nls_beam_select(logits, groups, beams, vocab, scores, ended, eog, n_eog, parents, tokens, out, over, work, bytes, None)

    for kw in (dict(groups=-1), dict(beams=0), dict(beams=65), dict(beams=-1), dict(vocab=-1), dict(vocab=1 << 29), dict(groups=1 << 23),
               dict(groups=1 << 17, vocab=1 << 24), dict(n_eog=-1), dict(logits=None), dict(scores=None), dict(eog=None), dict(parents=None),
               dict(tokens=None), dict(out=None), dict(work=None), dict(work=AT + 16), dict(bytes=8), dict(logits=AT + 2), dict(scores=AT + 1),
               dict(ended=AT + 2), dict(eog=AT + 3), dict(parents=AT + 2), dict(tokens=AT + 1), dict(out=AT + 2), dict(over=AT + 1)):
        assert call(**kw) == INVALID, kw
    assert call(vocab=0) == EMPTY
    assert call(groups=0, logits=None, work=None) == OK
    need = L.nls_beam_workspace(3, 4, 1000)
    assert need > 0 and call(bytes=need - 1) == INVALID
    assert L.nls_beam_workspace(3, 65, 1000) == L.nls_beam_workspace(-1, 4, 1000) == 0


def test_reorder_refusals(pkg):
    L = pkg.lib()
    pool = lambda **kw: pkg.NlsPagePool(**{**dict(d_kv=AT, layers=2, page_bytes=4096, layer_stride=40960, page_stride=4096), **kw})
    tabs = lambda **kw: pkg.NlsPageTables(**{**dict(d_table=AT, table_stride=5, slots=3, max_pages=5, d_lens=AT, d_refs=AT, pages=10, page_size=16), **kw})

    def call(p=None, t=None, src=AT, status=AT, work=AT, bytes=1 << 40):
        return L.nls_cache_reorder(p or pool(), t or tabs(), src, status, work, bytes, None)

    for kw in (dict(d_table=None), dict(d_lens=None), dict(d_refs=None), dict(slots=0), dict(slots=1 << 17), dict(pages=0), dict(pages=1 << 20),
               dict(max_pages=0), dict(page_size=24), dict(table_stride=4)):
        assert call(t=tabs(**kw)) == INVALID, kw
        assert L.nls_cache_reorder_workspace(tabs(**kw)) == 0
    for kw in (dict(d_kv=None), dict(d_kv=AT + 8), dict(layers=0), dict(page_bytes=8), dict(page_stride=2048), dict(layer_stride=16)):
        assert call(p=pool(**kw)) == INVALID, kw
    for kw in (dict(src=None), dict(src=AT + 2), dict(status=None), dict(status=AT + 1), dict(work=None), dict(work=AT + 64), dict(bytes=64)):
        assert call(**kw) == INVALID, kw
    need = L.nls_cache_reorder_workspace(tabs())
    assert need % 256 == 0 and need >= 4 * (2 + 5 * 3 + 15) and call(bytes=need - 1) == INVALID

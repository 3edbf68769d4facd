"""Pages of blocks by their definition: what the elements become, where their
bits lie, and attention over them in float64 with the error that the kernels'
arithmetic may make."""
import math

import numpy as np
import torch

HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}  # half a step, relative
BITS = {"q8_0": 8, "q4_0": 4}


def blocks(x, kind):
    """(codes int64 [..., dim], factors float16 [..., dim / 32]) of fp32 rows."""
    b = np.asarray(x, dtype=np.float32)
    b = b.reshape(*b.shape[:-1], b.shape[-1] // 32, 32)
    with np.errstate(all="ignore"):
        hi, lo = b.max(-1), b.min(-1)
        if kind == "q8_0":
            t, low, high = np.maximum(hi, -lo) * (np.float32(1) / np.float32(127)), -127, 127
        else:
            t, low, high = np.maximum(hi * (np.float32(1) / np.float32(7)), lo * np.float32(-0.125)), -8, 7
        d = np.minimum(t, np.float32(515.5 if kind == "q8_0" else 8188)).astype(np.float16)  # (fp16 holds d c)
        step = np.where(d > 0, np.float32(1) / d.astype(np.float32), np.float32(0)).astype(np.float32)
        c = np.clip(np.nan_to_num(np.rint(b * step[..., None]), nan=low, posinf=high, neginf=low), low, high)
        d = np.where(np.isfinite(b).all(-1), d, np.float16(np.nan))
    return c.astype(np.int64).reshape(np.shape(x)), d


def values(codes, d):
    """float64 values."""
    return (codes.reshape(*d.shape, 32) * d.astype(np.float64)[..., None]).reshape(codes.shape)


def place(dim, bits, value, e):
    """(byte, shift) of element e within a row's codes."""
    g, x, r = dim // 32, e // 32, e % 32
    if not value:
        unit = r // 8 * g + x
        if bits == 8:
            return unit * 8 + r % 8, 0
        n = r % 8 // 2 + 4 * (r % 2)
        return unit * 4 + n // 2, 4 * (n % 2)
    first, wide = 0, 4
    while x >= first + wide or first + wide > g:  # planes of four blocks, then two, then one
        if first + wide > g:
            wide //= 2
        else:
            first += wide
    at = first * 16 + r % 16 * wide + x - first
    return (2 * at + r // 16, 0) if bits == 8 else (at, r // 16 * 4)


def pack(kc, kd, vc, vd, kind):
    """uint8 [pages, page_bytes] of codes [pages, heads, tokens, dim] and factors
    [pages, heads, tokens, dim / 32]."""
    bits = BITS[kind]
    pages, heads, size, dim = kc.shape
    parts = []
    for value, c, d in ((False, kc, kd), (True, vc, vd)):
        row = np.zeros((pages, heads, size, dim * bits // 8), dtype=np.uint8)
        for e in range(dim):
            at, shift = place(dim, bits, value, e)
            row[..., at] |= ((c[..., e] + 2 ** (bits - 1)) << shift).astype(np.uint8)
        f = np.ascontiguousarray(np.swapaxes(d, -1, -2)).view(np.uint8)
        parts += [row.reshape(pages, heads, -1), f.reshape(pages, heads, -1)]
    return np.concatenate(parts, -1).reshape(pages, -1)


def unpack(raw, kind, heads, size, dim):
    """float64 [pages, 2, heads, size, dim] of uint8 [pages, page_bytes]."""
    bits, raw = BITS[kind], np.asarray(raw)
    codes, factors = size * dim * bits // 8, size * dim // 32 * 2
    h = raw.reshape(raw.shape[0], heads, 2, codes + factors)
    out = np.empty((raw.shape[0], 2, heads, size, dim))
    for k in range(2):
        row = h[:, :, k, :codes].reshape(-1, heads, size, dim * bits // 8).astype(np.int64)
        d = np.ascontiguousarray(h[:, :, k, codes:]).view(np.float16).reshape(-1, heads, dim // 32, size).astype(np.float64)
        for e in range(dim):
            at, shift = place(dim, bits, k == 1, e)
            with np.errstate(invalid="ignore"):
                out[:, k, :, :, e] = (((row[..., at] >> shift) & (2 ** bits - 1)) - 2 ** (bits - 1)) * d[:, :, e // 32]
    return out


def attend(q, kv, kind, table, lens, starts, scale, window=0, first=None, slots=None):
    """(out, lse, bound of out, bound of lse) in float64 for the rows that belong
    to a sequence, NaN elsewhere.  q: a CPU tensor of its own type; kv: unpack's."""
    pages, _, kvh, size, d = kv.shape
    heads, group, e32 = q.shape[1], q.shape[1] // kvh, 2.0 ** -24
    x = q.double().numpy()
    out = np.full(q.shape, np.nan)
    lse, ob, lb = np.full(q.shape[:2], np.nan), np.full(q.shape, np.nan), np.full(q.shape[:2], np.nan)
    most = 127 if kind == "q8_0" else 8
    # of a weight times a factor or a value: two parts each, or one of eleven bits
    # (few rows: of the weight times the factor; chunks: of the weight and of the value)
    part = 2.0 ** -10 if q.dtype == torch.bfloat16 else 2.0 ** -22
    for i in range(len(starts) - 1):
        a, b = starts[i], starts[i + 1]
        if a == b:
            continue
        s = i if slots is None else slots[i]
        n = int(lens[s]) if 0 <= s < len(lens) else 0
        f = max(0, int(first[s])) if first is not None and 0 <= s < len(lens) else 0
        keys = [j for j in range(f, n) if j // size < len(table[s]) and 0 <= table[s][j // size] < pages]
        at = np.array(keys, dtype=np.int64)
        page = np.array([table[s][j // size] for j in keys], dtype=np.int64)
        pos = n - (b - a) + np.arange(b - a)
        see = at[None, :] <= pos[:, None]
        if window:
            see &= at[None, :] > pos[:, None] - window
        some = see.any(1)
        for h in range(heads):
            k, v = (kv[page, z, h // group, at % size] for z in (0, 1))
            z = x[a:b, h]
            if not some.any():
                out[a:b, h], lse[a:b, h], ob[a:b, h], lb[a:b, h] = 0.0, -np.inf, 0.0, 0.0
                continue
            with np.errstate(invalid="ignore"):
                sc = np.where(see, z @ k.T * scale, -np.inf)
                # what a row does not see must not reach it, NaN times 0 neither
                sc = np.where(see, sc, -np.inf)
                top = np.where(some, sc.max(1), 0.0)
                w = np.exp(sc - top[:, None])
                total = w.sum(1)
            for t in range(b - a):
                if not some[t]:
                    out[a + t, h], lse[a + t, h], ob[a + t, h], lb[a + t, h] = 0.0, -np.inf, 0.0, 0.0
                    continue
                m = see[t]
                p, kt, vt = w[t, m] / total[t], np.abs(k[m]), v[m]
                out[a + t, h] = p @ vt
                lse[a + t, h] = l = top[t] + math.log(total[t])
                # A score: d products and sums, the queries' parts (2^-22 of each
                # product, and 2^-37 of the row's largest element), factors and
                # scale; then the exponent's argument, of the size of the score.
                zt = np.abs(z[t])
                ds = ((kt @ zt).max() * ((d + 8) * e32 + 2.0 ** -22) + kt.sum(1).max() * zt.max() * 2.0 ** -37) * abs(scale)
                ds += 4 * np.abs(sc[t, m]).max() * e32 + 4 * e32
                # A weight: its score's error twice, the exponential, its product
                # with the factor as parts; sums over the keys, joined parts
                # among them.  And fp16's least step, at 2^14 for the largest
                # weight times a power of two over the largest factor, per code;
                # for chunks, at 2^7 for a weight of 1, per value: half of 2^-24 2^-7.
                count = int(m.sum())
                dw = 2 * ds + 2.0 ** -21 + 2 * (count + 16) * e32
                mean = p @ np.abs(vt)
                big = np.abs(vt).max() * 2 if kind == "q8_0" else np.abs(vt).max() * 8
                ob[a + t, h] = (mean * (dw * (1 + dw) + part) + count * (2.0 ** -38 * big + 2.0 ** -32 * np.abs(vt).max())
                                + np.abs(out[a + t, h]) * HALF[q.dtype] * 2 + 1e-37 + (2.0 ** -25 if q.dtype == torch.float16 else 0))
                lb[a + t, h] = dw + abs(l) * 4 * e32
    return out, lse, ob, lb

"""The definitions of rotary positions and paged attention in float64, element
by element from the formulas, and the error that fp32 arithmetic may make.

Counterpart of rope and attnTask in nimllm's forward pass
(src/nimllm/model.nim:362-393, :446), for a cache in pages."""
import math

import numpy as np
import torch

HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}  # half a step, relative


def _np(x):
    """A float64 array of a tensor's or array's values."""
    return x.detach().cpu().double().numpy() if torch.is_tensor(x) else np.asarray(x, dtype=np.float64)


def turn(x, pos, freqs, amplitude, interleaved, sign=1.0):
    """x [tokens, heads, d] float64 with the first 2 len(freqs) elements turned."""
    x = _np(x)
    out = x.copy()
    r = 2 * len(freqs)
    ang = sign * _np(pos)[:, None] * _np(freqs)[None, :]
    # the reduction of a far angle in extended precision would differ by less
    # than 2^-53 of the angle
    c, s = np.cos(ang)[:, None, :] * amplitude, np.sin(ang)[:, None, :] * amplitude
    ia, ib = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    a, b = x[..., ia], x[..., ib]
    out[..., ia], out[..., ib] = a * c - b * s, b * c + a * s
    return out


def turn_bound(x, pos, freqs, amplitude, interleaved, dtype):
    """|result - turn| may be: the angle (float64 product, then rounded to fp32
    within [-pi, pi]: 2^-22), sine and cosine to 4 units of 2^-24 each, the
    amplitude's product, two products and a sum, one rounding to the type."""
    x, pos, freqs = np.abs(_np(x)), _np(pos), _np(freqs)
    r = 2 * len(freqs)
    ia, ib = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    far = float(np.max(np.abs(pos)) if len(pos) else 0) * float(np.max(freqs) if len(freqs) else 0)
    rel = 2.0 ** -22 + far * 2.0 ** -51 + 10 * 2.0 ** -24
    out = np.array(x)
    both = (x[..., ia] + x[..., ib]) * amplitude
    out[..., ia] = out[..., ib] = both
    b = out * HALF[dtype] * (1 + rel) + tiny(dtype)
    b[..., :r] += out[..., :r] * rel
    return b


def tiny(dtype):
    """Half of the smallest step of the type."""
    return {torch.float32: 2.0 ** -150, torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}[dtype]


def attend(q, kv, table, lens, starts, scale, window=0, first=None, slots=None):
    """(out, lse, bound of out, bound of lse) in float64 for the rows that belong
    to a sequence; NaN elsewhere.  q and kv: CPU tensors of their own types."""
    page_size, pages = kv.shape[3], kv.shape[0]
    heads, d = q.shape[1], q.shape[2]
    group = heads // kv.shape[2]
    out = torch.full(q.shape, math.nan, dtype=torch.float64)
    lse = torch.full(q.shape[:2], math.nan, dtype=torch.float64)
    ob, lb = out.clone(), lse.clone()
    e32 = 2.0 ** -24
    same = q.dtype == kv.dtype and q.dtype != torch.float32
    for i in range(len(starts) - 1):
        a, b = starts[i], starts[i + 1]
        s = i if slots is None else slots[i]
        n = int(lens[s]) if 0 <= s < len(lens) else 0
        where, keys = [], []
        for j in range(max(0, int(first[s]) if first is not None and 0 <= s < len(lens) else 0), n):
            p = int(table[s][j // page_size]) if j // page_size < len(table[s]) else -1
            if 0 <= p < pages:
                where.append((p, j % page_size))
                keys.append(j)
        if where:
            w = torch.tensor(where)
            rows = kv[w[:, 0], :, :, w[:, 1]].double()  # [keys, 2, kv heads, d]
        else:
            rows = torch.zeros((0, 2, kv.shape[2], d), dtype=torch.float64)
        keys = torch.tensor(keys, dtype=torch.int64)
        for t in range(a, b):
            pos = n - (b - a) + (t - a)
            see = keys <= pos
            if window:
                see &= keys > pos - window
            for h in range(heads):
                k, v = rows[see, 0, h // group], rows[see, 1, h // group]
                if k.shape[0] == 0:
                    out[t, h], lse[t, h], ob[t, h], lb[t, h] = 0.0, -math.inf, 0.0, 0.0
                    continue
                x = q[t, h].double()
                sc = (k @ x) * scale
                l = torch.logsumexp(sc, 0)
                p = torch.exp(sc - l)
                out[t, h], lse[t, h] = p @ v, l
                # A score: d products and sums (and, for fp32 queries, their
                # parts: 2^-22 of each product), the scale, and the exponent's
                # argument, of the size of the score.
                ds = (((k.abs() @ x.abs()) * abs(scale)).max() * ((d + 4) * e32 + 2.0 ** -22)
                      + 4 * sc.abs().max() * e32 + 4 * e32)
                # A weight: its score's error twice (the largest one's too), the
                # exponential, its parts or its rounding to the cache's type;
                # then a sum over the keys, joined parts among them.
                m = k.shape[0]
                dw = 2 * ds + 2.0 ** -21 + m * 2.0 ** -36 + 2 * (m + 16) * e32 + (HALF[kv.dtype] if same else 0.0)
                mean = p @ v.abs()
                ob[t, h] = mean * dw * (1 + dw) + out[t, h].abs() * HALF[q.dtype] * 2 + tiny(q.dtype) + 1e-37
                # (the sum of the weights may be taken after their rounding)
                lb[t, h] = dw + l.abs() * 4 * e32
    return out, lse, ob, lb

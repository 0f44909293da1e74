"""CPU oracle of the paged 8-bit KV cache.  TEST INFRASTRUCTURE ONLY: the
package never imports it.

No counterpart in the reference.  Restates, in numpy and float64, what
include/kvdec_paged8.h defines: one block at a time, one query row at a time.
A cache is a dict of k_pages, v_pages (uint8 bit patterns, head-major views
[num_pages, KVH, page_size, D] are taken with ``layout``) and k_scales,
v_scales [num_pages, KVH, page_size / block] float32; ``code`` is "int8" or
"e4m3".  ``tests/test_paged8_oracle.py`` pins it.
"""

from __future__ import annotations

import numpy as np

TOP = {"e4m3": 448.0, "int8": 127.0}
LOWEST = -100
NAN_CODE = 0x7F


def e4m3_table():
    """The value of each byte: sign, 4 exponent bits (bias 7), 3 mantissa bits."""
    b = np.arange(256)
    e, m = (b >> 3) & 15, b & 7
    v = np.where(e == 0, m * 2.0**-9, (8 + m) * 2.0**(e - 10.0))
    v = np.where((b & 0x7F) == NAN_CODE, np.nan, v)
    return np.where(b & 0x80, -v, v)


_E4M3 = e4m3_table()


def values(codes, code):
    """Code bytes as float64."""
    return _E4M3[codes] if code == "e4m3" else codes.view(np.int8).astype(np.float64)


def encode(x, code):
    """float64 values in the codes' range to the nearest code, ties to even;
    e4m3: anything not finite is the NaN code."""
    x = np.asarray(x, dtype=np.float64)
    if code == "int8":
        return np.rint(x).astype(np.int8).view(np.uint8)
    a = np.where(np.isfinite(x), np.abs(x), 0.0)
    e = np.maximum(np.frexp(a)[1] - 1, -6)                # values of exponent e lie 2^(e - 3) apart
    units = np.rint(a / np.exp2(e - 3.0))                 # 0..16
    e, units = np.where(units == 16, e + 1, e), np.where(units == 16, 8, units)
    bits = np.where(units < 8, units, (e + 7) * 8 + (units - 8)).astype(np.uint8)
    bits |= np.where(np.signbit(x), 0x80, 0).astype(np.uint8)
    return np.where(np.isfinite(x), bits, NAN_CODE).astype(np.uint8)


def need_scale(amax, code):
    """The least power of two >= 2^-100 that brings amax into the range."""
    if amax == 0:
        return np.float32(2.0**LOWEST)
    e = int(np.ceil(np.log2(amax / TOP[code])))
    while amax > TOP[code] * 2.0**e:
        e += 1
    while amax <= TOP[code] * 2.0**(e - 1):
        e -= 1
    return np.float32(2.0**max(e, LOWEST))


def _heads_first(pages, layout):
    return pages if layout == "HND" else pages.swapaxes(1, 2)


def _offsets(cu, B, T):
    return list(range(B + 1)) if cu is None else [0] + [min(max(int(c), 0), T) for c in cu[1:]]


def _len(seq_lens, b):
    return max(int(seq_lens[b]), 0)


def _place(table, b, pos, page_size, num_pages):
    """(page, row) of a position, or None where no page holds it."""
    if pos < 0 or pos >= table.shape[1] * page_size:
        return None
    p = int(table[b, pos // page_size])
    return (p, pos % page_size) if 0 <= p < num_pages else None


def write(cache, k, v, table, seq_lens, cu, code, layout="NHD"):
    """The cache after a call with rows k, v [T, KVH, D] (a new dict)."""
    out = {n: a.copy() for n, a in cache.items()}
    B, T = table.shape[0], k.shape[0]
    off = _offsets(cu, B, T)
    for name, x in (("k", np.asarray(k, np.float64)), ("v", np.asarray(v, np.float64))):
        pages, scales = _heads_first(out[name + "_pages"], layout), out[name + "_scales"]
        num_pages, KVH, ps, _ = pages.shape
        block = ps // scales.shape[2]
        for b in range(B):
            n = off[b + 1] - off[b]
            length = _len(seq_lens, b)
            p0 = length - n
            if n <= 0:
                continue
            for start in range(max(p0, 0) // block * block, length, block):
                at = _place(table, b, start, ps, num_pages)
                if at is None:
                    continue
                page, row = at
                r0, r1 = max(p0 - start, 0), min(length - start, block)
                new = x[off[b] + start + r0 - p0:off[b] + start + r1 - p0]
                for h in range(KVH):
                    y = new[:, h]
                    fin = np.isfinite(y)
                    s = need_scale(np.abs(y[fin]).max(initial=0.0), code)
                    old = scales[page, h, row // block]
                    if r0 > 0:
                        s = np.fmax(old, s)
                    rows = pages[page, h, row:row + block]
                    if code == "int8" and (not fin.all() or (r0 > 0 and np.isnan(old))):
                        scales[page, h, row // block] = np.nan
                        rows[r0:r1] = 0
                        continue
                    if r0 > 0 and s != old:
                        ratio = float(np.float32(old) / np.float32(s))
                        held = rows[:r0].copy()
                        again = encode(values(held, code) * ratio, code)
                        rows[:r0] = again
                    rows[r0:r1] = encode(y / float(s), code)
                    scales[page, h, row // block] = s
    return out


def _row(cache, name, page, row, layout, code):
    """[KVH, D] float64 values of a row."""
    pages, scales = _heads_first(cache[name + "_pages"], layout), cache[name + "_scales"]
    block = pages.shape[2] // scales.shape[2]
    return values(pages[page, :, row], code) * scales[page, :, row // block].astype(np.float64)[:, None]


def gather(cache, name, table, b, first, end, layout, code):
    """[end - first, KVH, D] values of a sequence's positions (no page: 0)."""
    pages = _heads_first(cache[name + "_pages"], layout)
    num_pages, KVH, ps, D = pages.shape
    out = np.zeros((end - first, KVH, D))
    for p in range(first, end):
        at = _place(table, b, p, ps, num_pages)
        if at is not None:
            out[p - first] = _row(cache, name, *at, layout, code)
    return out


def read(cache, table, seq_lens, cu, T, code, layout="NHD"):
    """k, v [T, KVH, D] in float64."""
    B = table.shape[0]
    ps = _heads_first(cache["k_pages"], layout).shape[2]
    off = _offsets(cu, B, T)
    got = []
    for name in "kv":
        KVH, D = _heads_first(cache[name + "_pages"], layout).shape[1::2]
        out = np.zeros((T, KVH, D))
        for b in range(B):
            length = _len(seq_lens, b)
            n = off[b + 1] - off[b]
            if n > 0:
                first = length - n
                lead = max(-first, 0)
                out[off[b] + lead:off[b + 1]] = gather(cache, name, table, b, first + lead, length, layout, code)
        got.append(out)
    return got


def attention(q, cache, table, seq_lens, cu, sm_scale, code, layout="NHD", window=None, sink=0):
    """[T, H, D] in float64."""
    q = np.asarray(q, np.float64)
    T, H, D = q.shape
    B = table.shape[0]
    ps = _heads_first(cache["k_pages"], layout).shape[2]
    KVH = _heads_first(cache["k_pages"], layout).shape[1]
    G = H // KVH
    off = _offsets(cu, B, T)
    o = np.zeros((T, H, D))
    for b in range(B):
        length = _len(seq_lens, b)
        n = off[b + 1] - off[b]
        if n <= 0 or length == 0:
            continue
        held = min(length, table.shape[1] * ps)   # no keys past the table
        kk = gather(cache, "k", table, b, 0, held, layout, code)
        vv = gather(cache, "v", table, b, 0, held, layout, code)
        for i in range(n):
            pos = length - n + i
            if pos < 0:
                continue
            p = np.arange(min(pos + 1, held))
            if window is not None:
                p = p[(p < sink) | (p > pos - window)]
            for h in range(H if len(p) else 0):
                x = kk[p, h // G] @ q[off[b] + i, h] * sm_scale
                w = np.exp(x - np.max(x)) if not np.isnan(x).any() else np.full_like(x, np.nan)
                o[off[b] + i, h] = w @ vv[p, h // G] / w.sum()
    return o

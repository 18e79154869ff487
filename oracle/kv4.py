"""The 4-bit (OCP MXFP4) cache in float64: its format, the rounding of a write and attention over
it, from the definitions (loops and tables, no code shared with the library)."""
from __future__ import annotations

import math

import numpy as np

PAGE = 16
E2M1 = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def quantize(x):
    """(codes, scales) of float rows (..., d): per 32 dims the scale byte 127 + e, e the exponent of
    the largest magnitude minus 2, one more from 7/4 of that power on (1 <= byte <= 252; 255 with a
    NaN or an infinity); codes = the nearest of +-E2M1 to x / 2^e, ties to the even code."""
    x = np.asarray(x, np.float64)
    b = x.reshape(-1, 32)
    codes = np.zeros(b.shape, np.uint8)
    scales = np.zeros(b.shape[0], np.uint8)
    mids = (E2M1[1:] + E2M1[:-1]) / 2
    for i, row in enumerate(b):
        top = np.abs(row).max() if np.isfinite(row).all() else np.inf
        if not np.isfinite(top):
            scales[i] = 255
            continue
        e = -200
        if top > 0:
            f, e = math.frexp(top)                       # top = f 2^e, 1/2 <= f < 1
            e = e - 1 + (f >= 0.875) - 2
        byte = min(max(127 + e, 1), 252)
        scales[i] = byte
        a = np.abs(row) / 2.0 ** (byte - 127)
        c = np.searchsorted(mids, a, side="left")        # a tie goes to the lower code
        tie = np.isin(a, mids) & (c % 2 == 1)            # ... or, if that is odd, the next one
        codes[i] = (c + tie) | np.where(np.signbit(row), 8, 0)
    return codes.reshape(x.shape), scales.reshape(*x.shape[:-1], x.shape[-1] // 32)


def values(codes, scales):
    """float64 values of codes (..., d) and scales (..., d / 32)."""
    c = np.asarray(codes).reshape(*np.shape(scales), 32)
    v = np.where(c & 8, -1.0, 1.0) * E2M1[c & 7]
    s = np.where(np.asarray(scales) == 255, np.nan, 2.0 ** (np.asarray(scales, np.float64) - 127))
    return (v * s[..., None]).reshape(np.shape(codes))


def held(x):
    """The float64 values that the cache holds for rows x."""
    return values(*quantize(x))


def _places(d):
    """Byte and nibble of each (token, dim): K codes, V codes; scale byte of each (token, block)."""
    w = min(d, 128)
    k, v = np.zeros((2, PAGE, d), int), np.zeros((2, PAGE, d), int)
    s = np.zeros((PAGE, d // 32), int)
    for t in range(PAGE):
        for i in range(d):
            k[:, t, i] = t * (d // 2) + i // 2, i % 2
            run = i % w // (w // 16)
            at = i % (w // 16)
            v[:, t, i] = (8 * d + i // w * 8 * w + t // 4 * 2 * w + run * (w // 8) + t % 4 * (w // 32) +
                          at // 2, at % 2)
        for b in range(d // 32):
            s[t, b] = 16 * d + 16 * b + t
    return k, v, s


def pack(k, v):
    """uint8 cache (pages, heads, 17 d) of float rows k, v (pages, heads, 16, d)."""
    n, h, _, d = np.shape(k)
    pk, pv, ps = _places(d)
    out = np.zeros((n, h, 17 * d), np.uint8)
    for x, place, off in ((k, pk, 0), (v, pv, d // 2)):
        codes, scales = quantize(x)
        for t in range(PAGE):
            for i in range(d):
                out[:, :, place[0, t, i]] |= codes[:, :, t, i] << np.uint8(4 * place[1, t, i])
            for b in range(d // 32):
                out[:, :, ps[t, b] + off] = scales[:, :, t, b]
    return out


def unpack(cache, d):
    """float64 K and V (pages, heads, 16, d) of a uint8 cache (pages, heads, 17 d)."""
    pk, pv, ps = _places(d)
    out = []
    for place, off in ((pk, 0), (pv, d // 2)):
        codes = cache[:, :, place[0]] >> (4 * place[1]) & 15
        out.append(values(codes, cache[:, :, ps + off]))
    return out


def rope(x, positions, inv_freq, style):
    """float64 rotary embedding of rows x (tokens, heads, d)."""
    x = np.asarray(x, np.float64)
    a = np.asarray(positions, np.float64)[:, None] * np.asarray(inv_freq, np.float64)
    c, s = np.cos(a)[:, None], np.sin(a)[:, None]
    y = np.empty_like(x)
    d = x.shape[-1]
    lo, hi = (slice(0, d // 2), slice(d // 2, d)) if style == 0 else (slice(0, d, 2), slice(1, d, 2))
    y[..., lo] = x[..., lo] * c - x[..., hi] * s
    y[..., hi] = x[..., hi] * c + x[..., lo] * s
    return y


def attend(q, k, v, seen, scale=None, cap=0.0, sinks=None):
    """float64 attention: q (rows, heads, d), k and v (keys, kv heads, d), seen (rows, keys). Also the
    largest sum of |q_i k_i| * scale over the keys that any row sees (what the scores' error goes by)."""
    q = np.asarray(q, np.float64)
    rows, hq, d = q.shape
    g = hq // k.shape[1]
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    out = np.zeros_like(q)
    size = 0.0
    for h in range(hq):
        kh, vh = k[:, h // g], v[:, h // g]
        s = q[:, h] @ kh.T * scale
        if kh.size and seen.any():
            size = max(size, float((np.abs(q[:, h]) @ np.abs(kh).T * scale)[seen].max()))
        if cap:
            s = cap * np.tanh(s / cap)
        s = np.where(seen, s, -np.inf)
        top = s.max(axis=1, initial=-np.inf)
        if sinks is not None:
            top = np.maximum(top, sinks[h])
        top = np.where(np.isfinite(top) | np.isnan(top), top, 0.0)
        p = np.exp(s - top[:, None])
        total = p.sum(axis=1) + (0.0 if sinks is None else np.exp(sinks[h] - top))
        o = np.where(seen, p, 0.0) @ np.where(seen.any(axis=0)[:, None], vh, 0.0)
        out[:, h] = np.where(total[:, None] == 0, 0.0, o / np.where(total == 0, 1.0, total)[:, None])
    return out, size


def decode(q, cache, indptr, indices, last, window=0, **kw):
    """attend for one query token per sequence over its pages; (outputs, largest score size, largest
    |v|)."""
    d = q.shape[2]
    out, size, big = np.zeros(q.shape), 0.0, 0.0
    used = sorted(set(int(i) for i in indices))
    at = {p: i for i, p in enumerate(used)}
    kk, vv = unpack(cache[used], d) if used else (np.zeros((0, cache.shape[1], PAGE, d)),) * 2
    for b in range(q.shape[0]):
        ids = [at[int(i)] for i in indices[indptr[b]:indptr[b + 1]]]
        n = PAGE * (len(ids) - 1) + int(last[b]) if ids else 0
        lo = max(0, n - window) if window else 0
        k, v = (x[ids].transpose(0, 2, 1, 3).reshape(-1, cache.shape[1], d)[lo:n] for x in (kk, vv))
        out[b:b + 1], s = attend(q[b:b + 1], k, v, np.ones((1, n - lo), bool), **kw)
        size = max(size, s)
        big = max(big, float(np.abs(v).max(initial=0.0)))
    return out, size, big


def grow(table, rows, cached, added, pages, num_tokens, capacity):
    """(table, kv_indptr, kv_indices, kv_last, q_indptr, slots, positions) of a step, request by
    request; kv_indices entries past the table's total are None."""
    table = np.array(table)
    blocks = table.shape[1]
    pages = list(pages)
    indptr, q_indptr, last, ids, slots, pos = [0], [0], [], [], [], []
    for r, c, n in zip(rows, cached, added):
        ok = 0 <= r < table.shape[0] and c >= 0 and n >= 0 and c + n <= PAGE * blocks
        n = max(int(n), 0)
        if ok:
            have, want = -(-int(c) // PAGE), -(-(int(c) + n) // PAGE)
            for i in range(have, want):
                table[r, i] = pages.pop(0) if pages else -1
            ids += [int(x) for x in table[r, :want]]
            last.append(int(c) + n - PAGE * (want - 1) if want else 0)
            for p in range(int(c), int(c) + n):
                page = int(table[r, p // PAGE])
                slots.append(PAGE * page + p % PAGE if 0 <= page < 2 ** 27 - 1 else -1)
                pos.append(p)
        else:
            last.append(0)
            slots += [-1] * n
            pos += [0] * n
        indptr.append(len(ids))
        q_indptr.append(q_indptr[-1] + n)
    slots, pos = (slots + [-1] * num_tokens)[:num_tokens], (pos + [0] * num_tokens)[:num_tokens]
    ids = (ids + [None] * capacity)[:capacity]
    return table, indptr, ids, last, q_indptr, slots, pos

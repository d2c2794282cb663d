"""CPU oracle (numpy, 64 bits) of the prompt side and the block-scaled e4m3 cache.

Each function restates one operator from its definition, row by row, and
shares nothing with the library.  Attention also returns the weighted sum of
|v| that its error bounds are made of.
"""

from __future__ import annotations

import math

import numpy as np

E4M3_MAX = 448.0
MIN_SCALE_EXP = -24


# ------------------------------------------------------------------ e4m3
def e4m3_values() -> np.ndarray:
    """The value of each of the 256 codes (sign, 4 exponent bits, 3 mantissa bits)."""
    out = np.empty(256)
    for c in range(256):
        s, e, m = -1.0 if c & 0x80 else 1.0, (c >> 3) & 15, c & 7
        if e == 15 and m == 7:
            out[c] = math.nan
        else:
            out[c] = s * (m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7))
    return out


_VALUES = e4m3_values()
_POSITIVE = _VALUES[:127]  # codes 0 .. 126: 0 to 448, ascending


def e4m3_encode(x: np.ndarray) -> np.ndarray:
    """Codes of the nearest values, ties to the even code; beyond 448 (infinities
    too) saturates, NaN stays NaN."""
    x = np.asarray(x, np.float64)
    a = np.minimum(np.abs(np.where(np.isnan(x), 0.0, x)), E4M3_MAX)
    hi = np.clip(np.searchsorted(_POSITIVE, a), 0, 126)
    lo = np.maximum(hi - 1, 0)
    up, down = _POSITIVE[hi] - a, a - _POSITIVE[lo]
    code = np.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    code = np.where(a == _POSITIVE[hi], hi, code)
    code = np.where(np.isnan(x), 127, code)
    return (code + np.where(np.signbit(x), 128, 0)).astype(np.uint8)


def e4m3_decode(codes: np.ndarray) -> np.ndarray:
    return _VALUES[np.asarray(codes, np.uint8)]


def least_scale(amax: float) -> float:
    """The least power of two >= 2^-24 that brings `amax` to 448 or below."""
    e = MIN_SCALE_EXP
    while amax > E4M3_MAX * 2.0 ** e:
        e += 1
    return 2.0 ** e


# ------------------------------------------------------------------ slots
def prompt_slots(cached, new, table, num_slots, page, free=None, free_count=0):
    """(table, slots, cu_seqlens, seq_lens, free_left, rows not served)."""
    table = np.array(table, np.int64)
    b, width = table.shape
    slots = np.full(num_slots, -1, np.int64)
    cu = np.zeros(b + 1, np.int64)
    seq = np.array(cached, np.int64)
    asked = taken = at = 0
    unserved = []
    for r in range(b):
        c, n = int(cached[r]), int(new[r])
        cu[r] = at
        fits = c >= 0 and n >= 0 and c + n <= width * page
        need = -(-(c + n) // page) - -(-c // page) if fits and free is not None else 0
        served = (fits and (need == 0 or asked + need <= free_count)
                  and (n <= 0 or at + n <= num_slots))
        if served:
            for j in range(need):
                table[r, -(-c // page) + j] = free[free_count - 1 - asked - j]
            if need:
                taken = asked + need
            for i in range(n):
                p = c + i
                slots[at + i] = table[r, p // page] * page + p % page
            seq[r] = c + n
        else:
            unserved.append(r)
            seq[r] = max(c, 0)
        asked += need
        at += max(n, 0)
    cu[b] = at
    return table, slots, cu, seq, free_count - taken, unserved


# ------------------------------------------------------------------ writes
def kv_write(x, pool, slots):
    """pool [P, H, page, 128] after writing tokens x [T, H, 128]."""
    pool = np.array(pool)
    page = pool.shape[2]
    for t, s in enumerate(slots):
        if 0 <= s < pool.shape[0] * page:
            pool[s // page, :, s % page] = x[t]
    return pool


def kv_write_fp8_block(x, codes, scales, slots):
    """(codes, scales) after the write: codes uint8 [P, H, page, 128], scales
    [P, H, page / block]."""
    codes, scales = np.array(codes), np.array(scales, np.float64)
    pages, heads, page, _ = codes.shape
    block = page // scales.shape[2]
    t = 0
    while t < len(slots):
        s = int(slots[t])
        if s < 0 or s >= pages * page:
            t += 1
            continue
        end = t
        while end < len(slots) and slots[end] >= 0 and slots[end] // block == s // block:
            end += 1
        p, g, kept = s // page, (s % page) // block, s % block
        for h in range(heads):
            run = np.asarray(x[t:end, h], np.float64)
            finite = np.abs(run[np.isfinite(run)])
            scale = least_scale(finite.max() if finite.size else 0.0)
            if kept:
                old = scales[p, h, g]
                if old >= scale:
                    scale = old
                else:
                    lo = g * block
                    part = e4m3_decode(codes[p, h, lo:lo + kept]) * (old / scale)
                    codes[p, h, lo:lo + kept] = e4m3_encode(part)
            scales[p, h, g] = scale
            for i in range(t, end):
                codes[p, h, slots[i] % page] = e4m3_encode(run[i - t] / scale)
        t = end
    return codes, scales


def dequantised(codes, scales):
    """Values [P, H, page, 128] of an e4m3 pool with block scales."""
    block = codes.shape[2] // scales.shape[2]
    return e4m3_decode(codes) * np.repeat(np.asarray(scales, np.float64), block, axis=2)[..., None]


# ------------------------------------------------------------------ attention
def _row(q, k, v):
    """One query over its visible keys: (output, log-sum-exp, sum of w |v|,
    largest sum of |q k| of a score)."""
    if len(k) == 0:
        return np.zeros(q.shape[-1]), -math.inf, np.zeros(q.shape[-1]), 0.0
    scale = 1.0 / math.sqrt(q.shape[-1])
    s = k @ q * scale
    m = s.max()
    w = np.exp(s - m)
    total = w.sum()
    w = w / total
    return w @ v, m + math.log(total), w @ np.abs(v), float((np.abs(k) @ np.abs(q)).max() * scale)


def prompt_attention(q, k, v, cu_q, cu_k):
    """(output, lse, sum of w |v|, score magnitude per row) in 64 bits; rows of
    no sequence are NaN."""
    q, k, v = (np.asarray(a, np.float64) for a in (q, k, v))
    tq, hq, d = q.shape
    g = hq // k.shape[1]
    out, mag = np.full((tq, hq, d), np.nan), np.full((tq, hq, d), np.nan)
    lse, size = np.full((tq, hq), np.nan), np.zeros((tq, hq))
    for b in range(len(cu_q) - 1):
        lq, lk = cu_q[b + 1] - cu_q[b], cu_k[b + 1] - cu_k[b]
        for i in range(lq):
            n = max(0, min(lk, i + 1 + lk - lq))
            ks = slice(cu_k[b], cu_k[b] + n)
            for h in range(hq):
                r = _row(q[cu_q[b] + i, h], k[ks, h // g], v[ks, h // g])
                t = cu_q[b] + i
                out[t, h], lse[t, h], mag[t, h], size[t, h] = r
    return out, lse, mag, size


def paged_decode(q, k_values, v_values, v_scales, table, seq_lens, q_indices=None,
                 out_indices=None, out_rows=None):
    """(output, sum of w |v|, score magnitude, keys * the largest w * 448 *
    V scale) of a decode step over dequantised pools; untouched output rows
    are NaN."""
    q = np.asarray(q, np.float64)
    hq, d = q.shape[1:]
    b, page, hkv = len(seq_lens), k_values.shape[2], k_values.shape[1]
    out = np.full((out_rows or b, hq, d), np.nan)
    mag, size, unit = out.copy(), np.zeros(out.shape[:2]), np.zeros(out.shape[:2])
    per_token = np.repeat(v_scales, page // v_scales.shape[2], axis=2)
    for r in range(b):
        n = max(0, min(int(seq_lens[r]), table.shape[1] * page))
        pages = table[r, :-(-n // page)]
        for h in range(hq):
            kv = h // (hq // hkv)
            k = k_values[pages, kv].reshape(-1, d)[:n]
            v = v_values[pages, kv].reshape(-1, d)[:n]
            o = r if out_indices is None else out_indices[r]
            query = q[r if q_indices is None else q_indices[r], h]
            out[o, h], lse, mag[o, h], size[o, h] = _row(query, k, v)
            if n:
                w = np.exp(k @ query / math.sqrt(d) - lse)
                unit[o, h] = n * E4M3_MAX * (w * per_token[pages, kv].reshape(-1)[:n]).max()
    return out, mag, size, unit

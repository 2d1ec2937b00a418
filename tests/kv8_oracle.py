"""64-bit oracle of the paged 8-bit key/value cache, from its definition.

e4m3: sign, 4 exponent bits (bias 7), 3 fraction bits; 0x7f and 0xff are NaN,
there are no infinities, the largest magnitude is 448.
"""

import numpy as np

E_MIN, E_MAX = -32, 63


def _table():
    t = np.empty(256)
    for c in range(256):
        s, e, f = c >> 7, c >> 3 & 15, c & 7
        v = f / 8 * 2.0 ** -6 if e == 0 else (1 + f / 8) * 2.0 ** (e - 7)
        t[c] = np.nan if c & 0x7f == 0x7f else -v if s else v
    return t


DECODE = _table()
_POS = DECODE[:0x7f]                       # 0 .. 448, ascending


def encode(x):
    """Nearest e4m3 code, ties to the even code, saturating; NaN -> 0x7f."""
    x = np.asarray(x, np.float64)
    a = np.minimum(np.abs(np.nan_to_num(x, nan=0.0, posinf=1e300, neginf=-1e300)), 448.0)
    hi = np.minimum(np.searchsorted(_POS, a), 0x7e)
    lo = np.maximum(hi - 1, 0)
    up, down = _POS[hi] - a, a - _POS[lo]
    code = np.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    code = np.where(np.signbit(x), code | 0x80, code)
    return np.where(np.isnan(x), 0x7f, code).astype(np.uint8)


def exponent(amax):
    """Least e in range with amax <= 448 * 2**e."""
    e = E_MIN
    while amax > 448.0 * 2.0 ** e and e < E_MAX:
        e += 1
    return e


def append(codes, exps, table, kv_lens, q_lens, k, v):
    """Codes and exponents after the new tokens' k, v [tokens, heads, d]."""
    codes, exps = codes.copy(), exps.copy()
    P = codes.shape[3]
    at = 0
    for b, (L, n) in enumerate(zip(kv_lens, q_lens)):
        for i in range((L - n) // P, -(-L // P) if n else 0):
            lo, hi = max(L - n, i * P), min(L, (i + 1) * P)
            page = table[b][i]
            for side, x in ((0, k), (1, v)):
                for h in range(codes.shape[2]):
                    new = x[at + lo - (L - n):at + hi - (L - n), h].astype(np.float64)
                    size = np.abs(new[np.isfinite(new)])
                    e = exponent(size.max() if size.size else 0.0)
                    old = lo - i * P
                    if old:
                        before = int(exps[page, side, h])
                        e = max(e, before)
                        if e > before:
                            held = DECODE[codes[page, side, h, :old]] * 2.0 ** (before - e)
                            codes[page, side, h, :old] = encode(held)
                    codes[page, side, h, old:old + hi - lo] = encode(new * 2.0 ** -e)
                    exps[page, side, h] = e
        at += n
    return codes, exps


def sees(L, n, window, sinks):
    """[n, L] truth: query i sees key j."""
    pos, key = np.arange(L - n, L)[:, None], np.arange(L)[None]
    ok = key <= pos
    if window:
        ok &= (pos - key < window) | (key < sinks)
    return ok


def held(codes, exps, table, b, L, h):
    """K and V [L, d] of sequence b, head h, as they are held."""
    P = codes.shape[3]
    pages = [table[b][i] for i in range(-(-L // P))]
    return [np.concatenate([DECODE[codes[p, side, h]] * 2.0 ** int(exps[p, side, h])
                            for p in pages])[:L] for side in (0, 1)]


def attend(codes, exps, table, kv_lens, q_lens, q, scale, window=0, sinks=0):
    """(out, bound) [tokens, heads, d] in 64 bits.  ``bound``: how far a kernel
    may be off that keeps scores, maxima, sums and outputs in f32 and rounds
    the weights once to f16 and the output not at all:

    * weights, f16: 2^-11 of the value; below f16's normal range 2^-25 of the
      largest weight, times 2^6 where the pages' exponents differ (the kernels
      scale weights by up to that), for each of L keys;
    * scores: queries below 2^-14 of their row's largest element are rounded
      by 2^-25 of it, and the D products and 4 further operations by 2^-23
      each (the sums need not round to nearest), of sum |q k|, which
      moves a weight by that share of itself, numerator and denominator alike;
    * L-term f32 sums of weights and products, 2^-23 a term.
    Each is a share of the largest |v| that the row sees."""
    H, D = codes.shape[2], codes.shape[4]
    G = q.shape[1] // H
    out = np.zeros(q.shape)
    bound = np.zeros(q.shape)
    at = 0
    for b, (L, n) in enumerate(zip(kv_lens, q_lens)):
        if n == 0:
            continue
        see = sees(L, n, window, sinks)
        for h in range(H):
            k, v = held(codes, exps, table, b, L, h)
            used = {int(exps[table[b][i], 1, h]) for i in range(-(-L // codes.shape[3]))}
            spread = 2.0 ** min(6, max(used) - min(used))
            for g in range(G):
                row = q[at:at + n, h * G + g].astype(np.float64)
                with np.errstate(invalid="ignore", over="ignore"):
                    s = row @ k.T * scale
                    s[~see] = -np.inf
                    size = (np.abs(row) @ np.abs(k).T) * abs(scale)
                    size += np.abs(row).max(1, keepdims=True) * np.abs(k).sum(1)[None] * abs(scale) * 2.0 ** -2
                    size = np.where(see, size, 0).max(1, keepdims=True)
                    p = np.exp(s - s.max(1, keepdims=True))
                    l = p.sum(1, keepdims=True)
                    for i in range(n):
                        w = see[i]
                        out[at + i, h * G + g] = p[i, w] @ v[w] / l[i]
                        top = np.nanmax(np.abs(v[w]))
                        bound[at + i, h * G + g] = top * (
                            2.0 ** -11 + L * spread * 2.0 ** -25 + 2 * size[i, 0] * (D + 4) * 2.0 ** -23
                            + 2 * L * 2.0 ** -23)
        at += n
    return out, bound


def close(got, want, bound, dtype):
    """Within the bound and the output's own rounding; NaN where it is NaN."""
    half = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11}[dtype]
    got = got.astype(np.float64)
    nan = np.isnan(want)
    tol = bound + half * (np.abs(want) + bound) + 2.0 ** -25
    return bool((np.isnan(got) == nan).all()) and bool((np.abs(got - want)[~nan] <= tol[~nan]).all())


def pool(rng, pages, heads, slots, dim, spread=3.0, dtype=None):
    """Filled pages: normal values times a factor of each page."""
    x = rng.standard_normal((pages, 2, heads, slots, dim))
    x *= 2.0 ** (spread * rng.random((pages, 2, heads, 1, 1)))
    exps = np.vectorize(exponent)(np.abs(x).max((3, 4))).astype(np.int8)
    codes = encode(x * 2.0 ** -exps.astype(float)[..., None, None])
    return codes, exps


def tables(rng, pages, lens, slots):
    """Distinct pages for each sequence, as rows of one table."""
    order = iter(rng.permutation(pages))
    width = max(1, max(-(-n // slots) for n in lens))
    t = np.zeros((len(lens), width), np.int32)
    for b, n in enumerate(lens):
        for i in range(-(-n // slots)):
            t[b, i] = next(order)
    return t

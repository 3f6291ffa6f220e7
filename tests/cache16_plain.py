"""Plain 64-bit statements of rotary positions, the paged cache in 16 bits and attention over prefixes that sequences share (calm_b200.seqops), with the bounds that their kernels'
roundings give."""
import math

import numpy as np

F32 = 2.0 ** -24  # half a step relative to a value


def rotate(x, pos, frequencies, gain, pairs):
    """x [tokens][heads][dim], pos [tokens] -> the turned rows and what fp32 may be off by before the last rounding.

    Bound, for each of the two products: the angle in turns is a 64-bit product of a 64-bit frequency over 2 pi (three roundings of 2^-53 of an angle of pos * f); its fraction, doubled, lies in
    [-1, 1] and is rounded to fp32 (2^-25 half turns, pi 2^-25 as an angle); sincospi is within a step of values up to 1 (2^-23 at most), times gain (2^-24), times the channel (2^-24); the
    difference adds 2^-24 of the result."""
    d = 2 * len(frequencies)
    angle = pos.astype(np.float64)[:, None] * frequencies
    cos, sin = (np.cos(angle) * gain)[:, None], (np.sin(angle) * gain)[:, None]
    off = np.abs(angle)[:, None] * 3 * 2.0 ** -53 + math.pi * 2.0 ** -25 + 2 * F32 + 2 * F32
    a, b = (x[..., :d // 2], x[..., d // 2:d]) if pairs == "halves" else (x[..., 0:d:2], x[..., 1:d:2])
    out, tol = x.copy(), np.zeros(x.shape)
    for at, p, q, s in (((0, a, b, -sin)), ((1, b, a, sin))):
        with np.errstate(invalid="ignore"):
            y = p * cos + q * s
            t = (np.abs(p) + np.abs(q)) * abs(gain) * off + F32 * np.abs(y)
        where = slice(at * (d // 2), (at + 1) * (d // 2)) if pairs == "halves" else slice(at, d, 2)
        out[..., where], tol[..., where] = y, t
    return out, tol


def rounded(want, tol, half, least):
    """What a result may be off by once it is rounded: half a step of the larger value that may be rounded, or of the type's smallest numbers."""
    return tol + half * (np.abs(want) + tol) + least


def positions(table, slot, page, pages, keys):
    """Page ids of the positions `keys` of a slot, -1 where there is none."""
    if not 0 <= slot < len(table):
        return np.full(len(keys), -1)
    at = keys // page
    ids = np.where(at < table.shape[1], table[slot, np.minimum(at, table.shape[1] - 1)], -1)
    return np.where((ids >= 0) & (ids < pages), ids, -1)


def attend(q, k, v, table, portions, groups, page, scale, window=0, softcap=0.0, sink=None, half=2.0 ** -8):
    """q [tokens][Hq][dim]; k, v [pages][heads][page][dim]; portions = (start, count, slot, position) of each sequence; groups = (first, sequences, positions) -> out (NaN where no sequence
    has a row) and a bound of what the kernel's arithmetic may add to it before the last rounding.

    Bound: products of 16-bit numbers are exact in fp32.  A score is a sum over dim in steps of 16 products.  The tensor core aligns a step's products and the running sum to the largest of the 17 and may cut
    each off at its 2^-23: per step 2^-23 of the running sum and 17 times that of the largest product.  Then factors, maximum and exponential (six roundings of the exponent, 2^-21).  Weights enter the second
    product with `half` of their own (fp16: or 2^-25 2^-10 of the largest).  A score's error d moves a weight by e^d; the numerator's sum and the denominator's add a rounding per 16 keys and per share."""
    T, Hq, D = q.shape
    pages, heads = k.shape[:2]
    group = Hq // heads
    of = {}
    for f, n, p in groups:
        for b in range(f, f + n):
            of[b] = (portions[f][2], p)
    out, tol = np.full(q.shape, math.nan), np.zeros(q.shape)
    for b, (st, n, slot, p0) in enumerate(portions):
        if n < 1 or p0 < 0 or st < 0 or st + n > T:
            continue
        first, shared = of.get(b, (slot, 0))
        keys = np.arange(p0 + n)
        ids = np.where(keys < shared, positions(table, first, page, pages, keys), positions(table, slot, page, pages, keys))
        good = ids >= 0
        if window:
            good &= keys > p0 - window
        keys, ids = keys[good], ids[good]
        pos = p0 + np.arange(n)
        seen = keys[None] <= pos[:, None]
        if window:
            seen &= keys[None] > pos[:, None] - window
        for h in range(Hq):
            x = q[st:st + n, h]
            if not len(keys):
                out[st:st + n, h] = 0.0
                continue
            kk, vv = k[ids, h // group, keys % page], v[ids, h // group, keys % page]
            # what some row does not see must not matter: rows of keys that no row sees are taken out above, others are masked below
            clean = np.where(np.isfinite(vv), vv, 0.0)
            with np.errstate(invalid="ignore", over="ignore"):
                s = x @ kk.T * scale
                mag = np.abs(x) @ np.abs(kk).T * abs(scale)
                big = np.abs(kk).max(1)[None] * np.abs(x).max(1)[:, None] * abs(scale)
                ds = ((D / 16 + 6) * mag + D / 16 * 17 * big) * 2.0 ** -23
                if softcap:
                    s = softcap * np.tanh(s / softcap)
                    ds = ds + softcap * 2.0 ** -21 + 4 * F32 * np.abs(s)  # (1 - t) / (1 + t), t = e^(-2 |x|): t and its difference from 1 within 2^-22, the quotient's reciprocal within 2^-23
                s = np.where(seen, s, -math.inf)
                m = s.max(1, keepdims=True)
                if sink is not None:
                    m = np.maximum(m, sink[h])
                base = np.where(np.isfinite(m), m, 0.0)
                ds = np.where(seen, ds + 6 * F32 * (np.abs(s - base) + np.abs(s)) + 2.0 ** -21, 0.0)
                w = np.where(seen, np.exp(s - np.where(m == -math.inf, 0.0, m)), 0.0)
                den = w.sum(1, keepdims=True) + (0.0 if sink is None else np.where(m == sink[h], 1.0, np.exp(sink[h] - m)) * (sink[h] != -math.inf))
                p = w / np.where(den == 0, 1.0, den)
                o = p @ clean
                for ch in np.unique(np.nonzero(~np.isfinite(vv))[1]):  # values that are not finite reach the rows that see them
                    bad = np.nonzero(~np.isfinite(vv[:, ch]))[0]
                    o[:, ch] += np.where(seen[:, bad] & (p[:, bad] > 0), p[:, bad] * vv[bad, ch][None], 0.0).sum(1)
                adds = (len(keys) / 16 + 200) * 2.0 ** -23
                spread = p @ np.abs(clean)
                cut = len(keys) / 16 * 17 * 2.0 ** -23 * (p[:, :, None] * np.abs(clean)[None]).max(1) if n * len(keys) * D < 3e7 else len(keys) / 16 * 17 * 2.0 ** -23 * p.max(1)[:, None] * np.abs(clean).max(0)
                t = (p * ds) @ np.abs(clean) + (p * ds).sum(1)[:, None] * np.abs(o) + (half + adds) * spread + adds * np.abs(o) + cut
                t = t + (2.0 ** -35 + 2.0 ** -111) * seen @ np.abs(clean)
            out[st:st + n, h], tol[st:st + n, h] = o, t
    return out, tol

"""Plain 64-bit statements of the operators on callers' memory (calm_b200.seqops), with the bounds that their kernels' roundings give."""
import math

import numpy as np
import torch

F32, BF16, F16 = 2.0 ** -24, 2.0 ** -8, 2.0 ** -11  # half a step relative to a value


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


# ---------------------------------------------------------------- beams

def beam_select(logits, scores, n):
    """logits [G][K][V], scores [G][K] (float64 numpy) -> tokens, parents, scores [G][n] and, per pick, what an fp32 log-sum may be off by."""
    G, K, V = logits.shape
    tok, par, best = np.full((G, n), -1), np.full((G, n), -1), np.full((G, n), -math.inf)
    for g in range(G):
        all_d = np.full((K, V), -math.inf)
        for b in range(K):
            x = np.where(np.isnan(logits[g, b]), -math.inf, logits[g, b])
            if not scores[g, b] > -math.inf or x.max() == -math.inf:
                continue
            m = x.max()
            with np.errstate(invalid="ignore"):
                diff = np.where(x == m, 0.0, x - m)
            all_d[b] = scores[g, b] + (diff - math.log(np.exp(diff).sum()))
        d = all_d.reshape(-1)
        order = np.argsort(-d, kind="stable")[:n]
        order = order[d[order] > -math.inf]
        k = len(order)
        tok[g, :k], par[g, :k], best[g, :k] = order % V, order // V, d[order]
    return tok, par, best


def log_sum_bound(V):
    """exp2f is within 2 steps (2^-22); its argument's rounding moves a term by y e^-y 2^-24 1.45 at most; then sums of 16, of a thread's tiles, of 256 threads and of
    slices, one rounding an addition.  A relative error of the sum is an absolute one of its logarithm."""
    return 2.0 ** -22 + F32 + (4 + math.ceil(V / 4096) + 8 + 8 + 4) * F32


# ---------------------------------------------------------------- the 8-bit cache

def e4m3_values():
    """Value of every code (NaN codes as NaN)."""
    v = np.zeros(256)
    for c in range(256):
        e, m = c >> 3 & 15, c & 7
        x = m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10)
        v[c] = math.nan if c & 127 == 127 else -x if c & 128 else x
    return v


VALUES = e4m3_values()


def round_e4m3(x):
    """Nearest e4m3 value of finite |x| <= 448 + half a step, ties to the even code."""
    x = np.asarray(x, np.float64)
    a = np.abs(x)
    step = 2.0 ** (np.floor(np.log2(np.maximum(a, 2.0 ** -6))) - 3)
    return np.sign(x) * np.minimum(np.rint(a / step) * step, 448.0)


def exponent(amax):
    """The least e >= -64 with amax <= 448 * 2^e."""
    e = -64
    if amax > 0:
        m, x = math.frexp(amax)
        e = max(e, x - 9 if m <= 0.875 else x - 8)
    return e


def store(values, scales, rows, table, portions, page):
    """values [pages][heads][page][dim] (of the codes, without scale) and scales [pages][heads], changed in place; rows [tokens][heads][dim]; portions = (start, count,
    slot, position) lists."""
    pages, heads = scales.shape
    for st, n, slot, p0 in portions:
        if n < 1 or p0 < 0 or not 0 <= slot < len(table) or st < 0 or st + n > len(rows):
            continue
        for block in range(p0 // page, (p0 + n - 1) // page + 1):
            if block >= table.shape[1] or not 0 <= table[slot, block] < pages:
                continue
            p = table[slot, block]
            lo, hi = max(p0, block * page), min(p0 + n, (block + 1) * page)
            for h in range(heads):
                x = rows[st + lo - p0:st + hi - p0, h].astype(np.float64)
                x = np.where(np.isnan(x), 0.0, x)
                fin = np.where(np.isinf(x), 0.0, np.abs(x))
                e = exponent(fin.max())
                r = lo - block * page
                if r:
                    old = exponent(scales[p, h] * 448.0)
                    e = max(e, old)
                    if e > old:
                        values[p, h, :r] = round_e4m3(values[p, h, :r] * 2.0 ** (old - e))
                scales[p, h] = 2.0 ** e
                y = np.clip(x * 2.0 ** -e, -448.0, 448.0)
                values[p, h, r:hi - block * page] = round_e4m3(y)


def attend(q, kv, ks, vv, vs, table, portions, page, scale, window=0, keep_first=0, chunk=0, softcap=0.0, sink=None, slopes=None, gate=None, half=F16, split=False):
    """q [tokens][Hq][dim]; kv, vv values of the codes [pages][heads][page][dim] -> out [tokens][Hq][dim] (NaN where no sequence has a row) and a bound of what the
    kernel's arithmetic may add to it before the last rounding.

    Bound: a score is a sum over dim in steps of 16 products.  The tensor core aligns a step's products and the running sum to the largest of the 17 and may cut each off at its
    2^-23: per step 2^-23 of the running sum and 17 times that of the largest product.  Then factors (four roundings); queries and weights
    enter as fp16, a tile's largest query at 2^15, a row's largest weight at 2^10 or more (2^-11 of a weight or 2^-25 2^-10 of the largest; 2^-22 as pairs).  A score's error d moves a weight by e^d; the numerator's sum and the denominator's add
    a rounding per 16 keys and per share."""
    T, Hq, D = q.shape
    pages, heads = ks.shape
    group = Hq // heads
    out, tol = np.full(q.shape, math.nan), np.zeros(q.shape)
    for st, n, slot, p0 in portions:
        if n < 1 or p0 < 0 or st < 0 or st + n > T:
            continue
        for i in range(n):
            pos = p0 + i
            lo = max(0, pos - window + 1) if window else 0
            if chunk:
                lo = max(lo, pos // chunk * chunk)
            keys = np.array([j for j in range(pos + 1) if (j >= lo or j < keep_first)], np.int64)
            if not 0 <= slot < len(table):
                keys = keys[:0]
            keys = keys[(keys // page) < table.shape[1]] if len(keys) else keys
            ids = table[slot, keys // page] if len(keys) else keys
            good = (ids >= 0) & (ids < pages)
            keys, ids = keys[good], ids[good]
            for h in range(Hq):
                g = h // group
                if not len(keys):
                    out[st + i, h] = 0.0
                    continue
                k = kv[ids, g, keys % page] * ks[ids, g][:, None]
                v = vv[ids, g, keys % page] * vs[ids, g][:, None]
                x = q[st + i, h]
                s = k @ x * scale
                mag = np.abs(k) @ np.abs(x) * abs(scale)
                dq = (2.0 ** -22 if split else 0.0) * mag + 2.0 ** -40 * np.abs(q[st:st + n]).max() * np.abs(k).sum(1) * abs(scale)
                ds = dq + ((D / 16 * (2 if split else 1) + 6) * mag + D / 16 * (2 if split else 1) * 17 * (np.abs(k) * np.abs(x)).max(1) * abs(scale)) * 2.0 ** -23
                if softcap:
                    s = softcap * np.tanh(s / softcap)
                    ds = ds + 8 * F32 * np.abs(s)
                if slopes is not None:
                    s = s - slopes[h] * (pos - keys)
                    ds = ds + 4 * F32 * (np.abs(s) + abs(slopes[h]) * (pos - keys))
                m = s.max() if sink is None else max(s.max(), sink[h])
                ds = ds + 6 * F32 * (np.abs(s - m) + np.abs(s)) + 2.0 ** -21  # exponents and their differences, exp2f
                w = np.exp(s - m)
                den = w.sum() + (0.0 if sink is None else math.exp(sink[h] - m))
                p = w / den
                o = p @ v
                adds = (len(keys) / 16 * (2 if split else 1) + 80) * 2.0 ** -23
                spread = p @ np.abs(v)
                cut = len(keys) / 16 * (2 if split else 1) * 17 * 2.0 ** -23 * (p[:, None] * np.abs(v)).max(0)  # as for the scores
                t = (p * ds) @ np.abs(v) + (p @ ds) * np.abs(o) + ((2.0 ** -22 if split else half) + adds) * spread + adds * np.abs(o) + cut
                # weights whose fp16 (or whose remainder's) is subnormal: half a step is 2^-25, the largest weight (times the largest value scale beside it, in whose units a
                # prompt's tile has its values) stands at 2^10 at least
                t = t + 2.0 ** -35 * np.abs(vv[ids, g, keys % page]).sum(0) * np.max(vs[ids, g]) * np.max(w) / den
                # codes in units of a scale that is 2^15 times their own or more fall under fp16's smallest step
                if np.max(vs[ids, g]) > 2.0 ** 15 * np.min(vs[ids, g]):
                    t = t + 2.0 ** -25 * np.max(vs[ids, g])
                # an exponential under 2^-126 may come out as zero: it multiplies sums of the values by weights of 2^15 at most, and den >= 1
                t = t + 2.0 ** -111 * np.abs(v).sum(0)
                if gate is not None:
                    f = 1.0 / (1.0 + np.exp(-gate[st + i, h]))
                    o, t = o * f, t * f + 4 * F32 * np.abs(o)
                out[st + i, h], tol[st + i, h] = o, t
    return out, tol

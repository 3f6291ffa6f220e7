"""Operators that serving many continuations of one long text rests on, each in its plain form and as calls of calm_b200.seqops.

  kind "rotate"   rows of query or key heads turned by their positions: pairs of neighbouring channels or of the two halves, a part of the head, frequencies
                  rescaled for long contexts
  kind "store"    a step's keys and values into a paged cache in 16 bits, the keys (and the step's queries beside them) rotated on the way
  kind "attend"   attention of a step's tokens over such a cache, where groups of sequences share the pages of a long prefix: beams, samples of one prompt,
                  questions about one document

The rotation.  Pair i of dims / 2 pairs turns by position * f_i, f_i = base^(-2 i / dims) before it is rescaled:
  linear       f_i / factor
  base         the base becomes base * factor^(dims / (dims - 2))
  wavelength   w = length f_i / 2 pi waves per original context: f_i / factor below `low`, f_i above `high`, a blend that is linear in w between
  ramp         the same by the pair's number, between the pairs that turn `fast` and `slow` times in the original context; cos and sin times 0.1 ln(factor) + 1

The cache.  A pool [pages][heads][page][dim] of keys and one of values; sequence s finds position p in page table[s][p // page], row p % page."""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

_DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_SCALINGS = {
    "none": None,
    "linear": {"kind": "linear", "factor": 4.0},
    "base": {"kind": "base", "factor": 8.0},
    "wavelength": {"kind": "wavelength", "factor": 8.0, "length": 8192, "low": 1.0, "high": 4.0},
    "ramp": {"kind": "ramp", "factor": 16.0, "length": 4096, "fast": 32.0, "slow": 1.0},
}


# --------------------------------------------------------------------------- the cases

def _rotate(name, seqs, new, before, heads, dim, dims, pairs, scaling, dtype, gap=0):
    return {"name": name, "kind": "rotate", "seqs": seqs, "new": new, "before": before, "heads": heads, "dim": dim, "dims": dims, "pairs": pairs, "scaling": scaling, "dtype": dtype,
            "gap": gap}


def _store(name, seqs, new, before, q_heads, heads, dim, dims, page, pairs, scaling, dtype, cache):
    return {"name": name, "kind": "store", "seqs": seqs, "new": new, "before": before, "q_heads": q_heads, "heads": heads, "dim": dim, "dims": dims, "page": page, "pairs": pairs,
            "scaling": scaling, "dtype": dtype, "cache": cache}


def _attend(name, groups, each, alone, shared, before, new, heads, kv_heads, dim, page, dtype, window=0, softcap=0.0, sink=False):
    return {"name": name, "kind": "attend", "groups": groups, "each": each, "alone": alone, "shared": shared, "before": before, "new": new, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "page": page, "dtype": dtype, "window": window, "softcap": softcap, "sink": sink}


def listed():
    return [
        # one decoded token's queries, a tail of a fused projection: the latency of a call
        _rotate("rotate 1x1", 1, 1, 4000, 32, 128, 128, "halves", "none", "bf16", gap=2048),
        # three prompts behind far positions, a quarter of the head turned in neighbouring pairs, 14 heads of an odd width
        _rotate("rotate 3x1100 far fp32", 3, 1100, 900000, 14, 80, 20, "neighbours", "ramp", "fp32"),
        # a whole batch of prompts, queries and keys of a 32-head model side by side
        _rotate("rotate 8x2048", 8, 2048, 0, 40, 128, 128, "halves", "wavelength", "bf16"),
        # one user's decoded token: queries turned, key and value stored
        _store("store 1x1", 1, 1, 4000, 32, 8, 128, 128, 16, "halves", "none", "bf16", "bf16"),
        # a full batch of decoded tokens in the runtime's fp32 rows, half of the head turned
        _store("store 64x1 fp32", 64, 1, 1500, 14, 2, 64, 32, 16, "neighbours", "linear", "fp32", "fp16"),
        # five prompts of different lengths
        _store("store 5x3000", 5, 3000, 7, 32, 8, 128, 128, 16, "halves", "wavelength", "bf16", "bf16"),
        # one user's request with four beams behind a prompt of 4000 tokens: the latency of a step
        _attend("attend 1x4 of 4000", 1, 4, 0, 4000, 40, 1, 32, 8, 128, 16, "bf16"),
        # eight such requests with eight beams each, the head layout of a 0.5B model
        _attend("attend 8x8 of 3000 fp16", 8, 8, 0, 3000, 60, 1, 14, 2, 64, 16, "fp16"),
        # 64 conversations behind one long system prompt
        _attend("attend 64 of 16000", 1, 64, 0, 16000, 1000, 1, 32, 8, 128, 16, "bf16"),
        # drafts of five tokens checked at once, three texts with four samples each and six others, a window, soft-capped scores and a sink, pages of an odd size
        _attend("attend drafts windowed", 3, 4, 6, 5000, 300, 5, 24, 4, 128, 24, "bf16", window=2048, softcap=30.0, sink=True),
        # a batch that shares nothing
        _attend("attend 32 alone", 0, 0, 32, 5000, 1000, 1, 32, 8, 128, 16, "bf16"),
        # questions of up to 300 tokens behind a document of 12000
        _attend("attend 16x300 of 12000", 1, 16, 0, 12000, 0, 300, 32, 8, 128, 16, "bf16"),
    ]


def _log(rng, a, b):
    return int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))


def _turn(rng, dim):
    pairs, scaling = rng.choice(["halves", "halves", "neighbours"]), rng.choice(["none", "linear", "base", "wavelength", "ramp"])
    return rng.choice([dim, dim, dim // 2, 4 * rng.randint(1, dim // 4)]), pairs, scaling


def draw(rng):
    kind = rng.choice(["rotate", "rotate", "store", "store", "attend", "attend", "attend", "attend"])
    if kind == "rotate":
        seqs, dim = _log(rng, 1, 64), rng.choice([64, 80, 96, 128, 128, 192, 256])
        heads = _log(rng, 1, 64)
        new = rng.choice([1, rng.randint(2, 9), _log(rng, 10, max(11, 80000000 // (seqs * heads * dim)))])
        dims, pairs, scaling = _turn(rng, dim)
        c = _rotate(None, seqs, min(new, 20000), rng.choice([0, _log(rng, 1, 1000000)]), heads, dim, dims, pairs, scaling, rng.choice(["fp32", "bf16", "bf16", "fp16"]),
                    gap=rng.choice([0, 0, 2 * rng.randint(1, 500), rng.randint(1, 999)]))
    elif kind == "store":
        seqs, dim, heads, group = _log(rng, 1, 64), rng.choice([64, 80, 128, 128, 256]), rng.choice([1, 2, 3, 4, 8]), rng.choice([1, 2, 4, 4, 7])
        new = rng.choice([1, 1, rng.randint(2, 9), _log(rng, 10, max(11, 15000 * 8 * 128 // (seqs * heads * dim)))])
        dims, pairs, scaling = _turn(rng, dim)
        c = _store(None, seqs, min(new, 4000), rng.choice([0, _log(rng, 1, 3000)]), heads * group, heads, dim, dims, rng.choice([1, 8, 16, 16, 24, 64]), pairs, scaling,
                   rng.choice(["fp32", "bf16", "fp16"]), rng.choice(["bf16", "bf16", "fp16"]))
    else:
        kv_heads, group, dim = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 4, 4, 7, 8]), rng.choice([64, 128, 128, 128, 80, 256])
        groups, each, alone = rng.choice([0, 1, 1, 1, _log(rng, 2, 8)]), _log(rng, 2, 64), rng.choice([0, 0, _log(rng, 1, 16)])
        each = min(each, 64 // max(1, groups))
        if not groups:
            each, alone = 0, _log(rng, 1, 48)
        seqs = groups * each + alone
        new = rng.choice([1, 1, 1, rng.randint(2, 9), _log(rng, 16, max(17, 4000 // seqs))])
        reach = 12000 if new < 16 else 6000
        c = _attend(None, groups, each, alone, rng.choice([0, _log(rng, 16, reach), _log(rng, 1000, reach)]), rng.choice([0, _log(rng, 1, 1000)]), new, kv_heads * group, kv_heads, dim,
                    rng.choice([8, 16, 16, 16, 24, 64, 5]), rng.choice(["bf16", "bf16", "fp16"]), window=rng.choice([0, 0, 0, _log(rng, 3, 3000)]),
                    softcap=rng.choice([0.0, 0.0, 0.0, 30.0]), sink=rng.random() < 0.25)
    del c["name"]
    return c


# --------------------------------------------------------------------------- inputs

def _ragged(i):
    """Sequences of one batch differ in length."""
    return 1.0 - 0.75 * ((i * 0.6180339887) % 1.0)


def _batch(c):
    """(new tokens, positions before, positions shared) of every sequence and the groups (first sequence, sequences, positions shared) on the host."""
    if c["kind"] != "attend":
        f = [_ragged(i) for i in range(c["seqs"])]
        return [max(1, round(c["new"] * x)) if c["new"] >= 16 else c["new"] for x in f], [round(c["before"] * x) for x in f], [0] * c["seqs"], []
    counts, before, shared, groups = [], [], [], []
    for g in range(c["groups"]):
        groups.append((len(counts), c["each"], round(c["shared"] * _ragged(g))))
        shared += [groups[-1][2]] * c["each"]
        counts += [c["new"]] * c["each"]
        before += [groups[-1][2]] * c["each"]
    for i in range(c["alone"]):
        counts.append(c["new"]), shared.append(0), before.append(round(c["shared"] * _ragged(i)))
    for i in range(len(counts)):
        before[i] += round(c["before"] * _ragged(i))
        counts[i] = max(1, round(counts[i] * _ragged(i))) if c["new"] >= 16 else counts[i]
    return counts, before, shared, groups


def _frequencies(dims, scaling, base=10000.0):
    """Step of every pair in 64 bits, and the factor on cos and sin."""
    s = _SCALINGS[scaling]
    if s and s["kind"] == "base" and dims > 2:
        base *= s["factor"] ** (dims / (dims - 2))
    i = np.arange(dims // 2, dtype=np.float64)
    f, gain = base ** (-2.0 * i / dims), 1.0
    if s and s["kind"] == "linear":
        f = f / s["factor"]
    elif s and s["kind"] == "wavelength":
        w = s["length"] * f / (2.0 * math.pi)
        blend = np.clip((w - s["low"]) / (s["high"] - s["low"]), 0.0, 1.0)
        f = (1.0 - blend) * f / s["factor"] + blend * f
    elif s and s["kind"] == "ramp":
        at = [dims * math.log(s["length"] / (2.0 * math.pi * t)) / (2.0 * math.log(base)) for t in (s["fast"], s["slow"])]
        lo, hi = max(math.floor(at[0]), 0), min(math.ceil(at[1]), dims - 1)
        blend = np.clip((i - lo) / max(hi - lo, 0.001), 0.0, 1.0)
        f, gain = f / s["factor"] * blend + f * (1.0 - blend), 0.1 * math.log(s["factor"]) + 1.0
    return f, gain


def _rows(n, heads, dim, t, g, gap=0):
    """Rows of heads as a part of a wider projection, which tokens differ in size in."""
    x = torch.randn(n, heads * dim + gap, generator=g, device="cuda") * torch.exp(0.5 * torch.randn(n, 1, generator=g, device="cuda"))
    return x.to(t)[:, gap:].unflatten(1, (heads, dim))


def _inputs(case, seed):
    g, c, dev = torch.Generator(device="cuda").manual_seed(seed), case, "cuda"
    host = np.random.default_rng(seed)
    counts, before, shared, groups = _batch(c)
    n, seqs, t = sum(counts), len(counts), _DTYPES[c["dtype"]]
    st = {"case": c, "counts": counts, "before": before, "groups": groups, "shared": shared}
    st["seq"] = torch.tensor(np.repeat(np.arange(seqs), counts), device=dev)
    st["pos"] = torch.tensor(np.concatenate([np.arange(b, b + k) for b, k in zip(before, counts)]), device=dev)
    st["row"] = torch.tensor(np.concatenate([np.arange(k) for k in counts]), device=dev)  # place of a token among its sequence's new ones
    if c["kind"] != "attend":
        f, st["gain"] = _frequencies(c["dims"], c["scaling"])
        st["freq"] = torch.tensor(f, device=dev)
    if c["kind"] == "rotate":
        st["x"] = _rows(n, c["heads"], c["dim"], t, g, c["gap"])
        return st
    page, kv = c["page"], c["heads"] if c["kind"] == "store" else c["kv_heads"]
    pages = [-(-(b + k) // page) for b, k in zip(before, counts)]
    full = [s // page for s in shared]                       # pages that a group holds once
    first = {f0: s for f0, _, s in groups}
    total = sum(p - f for p, f in zip(pages, full)) + sum(s // page for s in first.values())
    where, at = host.permutation(total + 3), 0
    table, parts = np.zeros((seqs, max(pages)), np.int64), []
    lead = 0
    for i in range(seqs):
        if i in first or not shared[i]:
            lead = i
        keep = full[i] if i != lead else 0
        table[i, :keep] = table[lead, :keep]
        table[i, keep:pages[i]], at = where[at:at + pages[i] - keep], at + pages[i] - keep
        if i != lead and shared[i] % page:                   # a page in part filled with the prefix is every sequence's own
            parts.append((table[lead, full[i]], table[i, full[i]]))
    st["table"] = torch.tensor(table.astype(np.int32), device=dev)
    shape, cache = (total + 3, kv, page, c["dim"]), _DTYPES[c["cache"] if c["kind"] == "store" else c["dtype"]]
    for name in "kv":
        pool = torch.empty(shape, dtype=cache, device=dev)
        gain = torch.exp(0.3 * torch.randn(kv, 1, c["dim"], generator=g, device=dev))
        for p in range(0, total + 3, 8192):
            pool[p:p + 8192] = torch.randn(min(8192, total + 3 - p), *shape[1:], generator=g, device=dev) * gain
        if parts:
            src, dst = (torch.tensor(x, device=dev) for x in zip(*parts))
            pool[dst] = pool[src]
        st[name + "c"] = pool
    if c["kind"] == "store":
        both = _rows(n, c["q_heads"] + 2 * kv, c["dim"], t, g)
        st["q"], st["k"], st["v"] = both[:, :c["q_heads"]], both[:, c["q_heads"]:c["q_heads"] + kv], both[:, c["q_heads"] + kv:]
    else:
        st["q"] = (torch.randn(n, c["heads"], c["dim"], generator=g, device=dev) * 1.2).to(t)
        st["sink"] = torch.randn(c["heads"], generator=g, device=dev) if c["sink"] else None
    return st


def prepare(case, seed):
    st = _inputs(case, seed)
    if own:  # what a serving program keeps beside its buffers: the step's description, the model's rotation, the pools' layout
        from calm_b200 import seqops

        c = case
        st["batch"] = seqops.Batch(range(len(st["counts"])), st["counts"], st["before"], shared=st["groups"])
        if c["kind"] != "attend":
            st["rotation"] = seqops.Rotation(c["dims"], base=10000.0, pairs=c["pairs"], scaling=_SCALINGS[c["scaling"]])
        if c["kind"] != "rotate":
            st["cache"] = seqops.Cache16(st["kc"], st["vc"])
    return st


# --------------------------------------------------------------------------- one pass

def _plain_rotate(x, pos, freq, gain, dims, pairs):
    angle = pos.double()[:, None] * freq
    cos, sin = (torch.cos(angle) * gain).float()[:, None], (torch.sin(angle) * gain).float()[:, None]
    y = x.float()
    turned, rest = y[..., :dims], y[..., dims:]
    if pairs == "halves":
        a, b = turned[..., :dims // 2], turned[..., dims // 2:]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    else:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    return torch.cat([turned, rest], -1)


def _plain_attend(st):
    c, table = st["case"], st["table"].long()
    seqs, page, dim, kv = table.shape[0], c["page"], c["dim"], c["kv_heads"]
    group, keys, most = c["heads"] // kv, table.shape[1] * page, max(st["counts"])

    def rows(pool):  # [seqs][kv heads][keys][dim]
        return pool[table].transpose(1, 2).reshape(seqs, kv, keys, dim).float()

    q = torch.zeros(seqs, most, c["heads"], dim, device=table.device)
    q[st["seq"], st["row"]] = st["q"].float()
    at = torch.full((seqs, most), -1, dtype=torch.int64, device=table.device)
    at[st["seq"], st["row"]] = st["pos"]
    key = torch.arange(keys, device=table.device)
    seen = key <= at[:, :, None]
    if c["window"]:
        seen &= key > at[:, :, None] - c["window"]
    q = q.view(seqs, most, kv, group, dim).permute(0, 2, 3, 1, 4).reshape(seqs, kv, group * most, dim)
    s = torch.matmul(q, rows(st["kc"]).transpose(2, 3)) * dim ** -0.5
    if c["softcap"]:
        s = c["softcap"] * torch.tanh(s / c["softcap"])
    s = s.view(seqs, kv, group, most, keys).masked_fill_(~seen[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    if st["sink"] is not None:
        sink = st["sink"].view(1, kv, group, 1, 1)
        top = torch.maximum(top, sink)
    top = torch.where(top == -math.inf, 0.0, top)
    p = s.sub_(top).exp_()
    below = p.sum(-1, keepdim=True)
    if st["sink"] is not None:
        below = below + torch.exp(sink - top)
    o = torch.matmul(p.view(seqs, kv, group * most, keys), rows(st["vc"])).view(seqs, kv, group, most, dim) / below
    o = o.permute(0, 3, 1, 2, 4).reshape(seqs, most, c["heads"], dim)
    return o[st["seq"], st["row"]].to(st["q"].dtype)


def run(st):
    c = st["case"]
    if c["kind"] == "rotate":
        if own:
            from calm_b200 import seqops

            return seqops.rotate(st["x"], st["batch"], st["rotation"])
        return _plain_rotate(st["x"], st["pos"], st["freq"], st["gain"], c["dims"], c["pairs"]).to(st["x"].dtype)
    if c["kind"] == "store":
        if own:
            q = st["cache"].store(st["k"], st["v"], st["table"], st["batch"], rotation=st["rotation"], q=st["q"])
        else:
            turn = (st["pos"], st["freq"], st["gain"], c["dims"], c["pairs"])
            q = _plain_rotate(st["q"], *turn).to(st["q"].dtype)
            page, off = st["table"].long()[st["seq"], st["pos"] // c["page"]], st["pos"] % c["page"]
            st["kc"][page, :, off] = _plain_rotate(st["k"], *turn).to(st["kc"].dtype)
            st["vc"][page, :, off] = st["v"].to(st["vc"].dtype)
        return {"q": q, "k": st["kc"], "v": st["vc"]}
    if own:
        return st["cache"].attend(st["q"], st["table"], st["batch"], scale=c["dim"] ** -0.5, window=c["window"], softcap=c["softcap"], sink=st["sink"])
    return _plain_attend(st)


# --------------------------------------------------------------------------- what a pass cannot do without

def _pairs(lo, hi, counts, before, window):
    """(query, key) pairs over the keys lo .. hi - 1 of sequences that bring `counts` tokens behind `before`, and the keys that any of them sees."""
    pairs, least, most = 0, hi, lo
    for k, b in zip(counts, before):
        pos = np.arange(b, b + k)
        low = np.maximum(lo, pos - window + 1) if window else np.full(k, lo)
        top = np.minimum(hi, pos + 1)
        pairs += int(np.maximum(0, top - low).sum())
        if int(low.min()) < int(top.max()):
            least, most = min(least, int(low.min())), max(most, int(top.max()))
    return pairs, max(0, most - least)


def work(case):
    c = case
    size = 4 if c["dtype"] == "fp32" else 2
    counts, before, shared, groups = _batch(c)
    n = sum(counts)
    if c["kind"] == "rotate":
        return {"bytes": 2 * n * c["heads"] * c["dim"] * size, "flops": 3.0 * n * c["heads"] * c["dims"]}
    if c["kind"] == "store":
        return {"bytes": n * c["dim"] * (2 * c["q_heads"] * size + 2 * c["heads"] * (size + 2)), "flops": 3.0 * n * (c["q_heads"] + c["heads"]) * c["dims"]}
    pairs = keys = 0
    for f, m, s in groups:
        p, k = _pairs(0, s, counts[f:f + m], before[f:f + m], c["window"])
        pairs, keys = pairs + p, keys + k
    for i in range(len(counts)):
        p, k = _pairs(shared[i], before[i] + counts[i], counts[i:i + 1], before[i:i + 1], c["window"])
        pairs, keys = pairs + p, keys + k
    return {"bytes": 2 * keys * c["kv_heads"] * c["dim"] * size + 2 * n * c["heads"] * c["dim"] * size, "flops": 4.0 * pairs * c["heads"] * c["dim"]}


# --------------------------------------------------------------------------- the definitions in 64 bits

def _exact_rotate(x, pos, case):
    """Pairs as complex numbers times e^(i angle)."""
    f, gain = _frequencies(case["dims"], case["scaling"])
    x, d = x.double(), case["dims"]
    half = x[..., :d].unflatten(-1, (2, d // 2)).transpose(-1, -2) if case["pairs"] == "halves" else x[..., :d].unflatten(-1, (d // 2, 2))
    angle = torch.tensor(pos.cpu().numpy().astype(np.float64)[:, None] * f, device=x.device)[:, None]
    z = torch.view_as_real(torch.complex(half[..., 0], half[..., 1]) * torch.polar(torch.full_like(angle, gain), angle))
    out = x.clone()
    out[..., :d] = (z.transpose(-1, -2) if case["pairs"] == "halves" else z).flatten(-2)
    return out


def exact(case, seed):
    c, st = case, _inputs(case, seed)
    if c["kind"] == "rotate":
        return _exact_rotate(st["x"], st["pos"], c)
    if c["kind"] == "store":
        k, v = st["kc"].double(), st["vc"].double()
        rows, at = _exact_rotate(st["k"], st["pos"], c), 0
        table = st["table"].tolist()
        for i, (n, b) in enumerate(zip(st["counts"], st["before"])):
            for block in range(b // c["page"], (b + n - 1) // c["page"] + 1):
                lo, hi = max(b, block * c["page"]), min(b + n, (block + 1) * c["page"])
                for pool, x in ((k, rows), (v, st["v"].double())):
                    pool[table[i][block], :, lo - block * c["page"]:hi - block * c["page"]] = x[at + lo - b:at + hi - b].transpose(0, 1)
            at += n
        return {"q": _exact_rotate(st["q"], st["pos"], c), "k": k, "v": v}
    out, at = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda"), 0
    group = c["heads"] // c["kv_heads"]
    for i, (n, b) in enumerate(zip(st["counts"], st["before"])):
        pages = st["table"][i, :-(-(n + b) // c["page"])].long()
        k, v = (st[name][pages].double().permute(1, 0, 2, 3).reshape(c["kv_heads"], -1, c["dim"])[:, :n + b] for name in ("kc", "vc"))
        dist = torch.arange(b, b + n, device="cuda")[:, None] - torch.arange(n + b, device="cuda")[None, :]
        hidden = (dist < 0) | (dist >= c["window"]) if c["window"] else dist < 0
        for h in range(c["heads"]):
            s = st["q"][at:at + n, h].double() @ k[h // group].T / math.sqrt(c["dim"])
            if c["softcap"]:
                s = c["softcap"] * torch.tanh(s / c["softcap"])
            s[hidden] = -math.inf
            if st["sink"] is not None:
                s = torch.cat([s, st["sink"][h].double().expand(n, 1)], 1)
            out[at:at + n, h] = torch.softmax(s, 1)[:, :n + b] @ v[h // group]
        at += n
    return out

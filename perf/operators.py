"""Operators that serving a layer-list model to many continuations of the same text rests on, each in its plain form and as calls of calm_b200.seqops.

  kind "beam"    the n best continuations of every group of beams: log-softmax over the vocabulary, the beams' running scores added, the highest of
                 all beams x tokens in order (ties: the lower beam, then the lower token)
  kind "copy"    pages of a paged cache and per-slot recurrent states copied inside their pools: forks of sequences, pages moved together
  kind "store"   new key and value rows into a cache held in 8 bits (e4m3 codes, a power of two as scale for every page and head)
  kind "attend"  attention of new tokens over such a cache: single tokens, short portions and prompts, grouped-query heads, windows

The 8-bit cache.  A pool holds codes [pages][heads][page][dim] and scales [pages][heads]; sequence s finds position p in page table[s][p // page], row
p % page.  Storing rows into a page raises the page's scale to the least power of two 2^e with max|row| <= 448 * 2^e (e >= -64) where it is not that high
already; the codes of the page's earlier rows are rounded to the raised scale.  A page whose first row is stored starts anew.  Value = code * scale."""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

_DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_LEAST = -64  # exponent of the smallest scale


# --------------------------------------------------------------------------- the cases

def _beam(name, groups, beams, vocab, n, dtype, first=False, masked=0.0):
    return {"name": name, "kind": "beam", "groups": groups, "beams": beams, "vocab": vocab, "n": n, "dtype": dtype, "first": first, "masked": masked}


def _copy(name, caches, page, width, pages, moves, filled, states, state, slots, forks, dtype="fp32"):
    return {"name": name, "kind": "copy", "caches": caches, "page": page, "width": width, "pages": pages, "moves": moves, "filled": filled, "states": states, "state": state,
            "slots": slots, "forks": forks, "dtype": dtype}


def _store(name, seqs, new, before, heads, dim, page, dtype):
    return {"name": name, "kind": "store", "seqs": seqs, "new": new, "before": before, "heads": heads, "dim": dim, "page": page, "dtype": dtype}


def _attend(name, seqs, new, before, heads, kv_heads, dim, page, dtype, window=0, keep_first=0, softcap=0.0, sink=False):
    return {"name": name, "kind": "attend", "seqs": seqs, "new": new, "before": before, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page, "dtype": dtype,
            "window": window, "keep_first": keep_first, "softcap": softcap, "sink": sink}


def listed():
    return [
        # one user's request with four beams, a 32000-token vocabulary: the latency of a step
        _beam("beam 1x4 of 32000", 1, 4, 32000, 8, "fp32"),
        # a few requests with three beams each, logits in 16 bits, rows that start at odd addresses, half of the vocabulary masked by a grammar
        _beam("beam 5x3 of 50257 bf16", 5, 3, 50257, 6, "bf16", masked=0.5),
        # a full batch: 32 requests of eight beams over the largest vocabulary of this repository's shapes
        _beam("beam 32x8 of 128256", 32, 8, 128256, 16, "fp32"),
        # a group of four beams forks three times: a page in part filled per cache, two recurrent states
        _copy("fork 3 of two blocks", 4, 16, 256, 96, 3, 7, 2, 131072, 8, 3),
        # 32 requests lose half of their beams at once: 96 forks, caches of 512-wide rows and states of 16 heads of 128 x 128
        _copy("fork 96 of four blocks", 4, 16, 512, 512, 96, 9, 4, 262144, 208, 96),
        # a cache's live pages move together before the pool is made smaller
        _copy("move 1500 pages", 8, 16, 512, 3600, 1500, 16, 0, 0, 0, 0),
        # one decoded token for each of 32 sequences
        _store("store 32x1", 32, 1, 1500, 8, 128, 16, "bf16"),
        # three prompts of different lengths
        _store("store 3x2100", 3, 2100, 0, 8, 128, 16, "fp32"),
        # one user far into a conversation
        _attend("attend 1x1 of 4000", 1, 1, 4000, 32, 8, 128, 16, "bf16"),
        # a full batch of conversations of different lengths
        _attend("attend 64x1 of 8000", 64, 1, 8000, 32, 8, 128, 16, "bf16"),
        # drafts of five tokens checked at once under a window that keeps the first positions, the head layout of a 0.5B model
        _attend("attend 8x5 of 3000 windowed", 8, 5, 3000, 14, 2, 64, 16, "fp32", window=1024, keep_first=64),
        # a question of 1500 tokens behind a document of 700, twice
        _attend("attend 2x1500 of 700", 2, 1500, 700, 16, 4, 128, 16, "bf16"),
    ]


def _log(rng, a, b):
    return int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))


def draw(rng):
    kind = rng.choice(["beam", "beam", "copy", "store", "attend", "attend", "attend"])
    if kind == "beam":
        beams = rng.choice([1, 2, 3, 4, 5, 6, 8, 12, 16])
        groups = _log(rng, 1, 256 // beams)
        vocab = _log(rng, 500, min(160000, 32800000 // (groups * beams)))
        c = _beam(None, groups, beams, vocab, min(rng.choice([beams, 2 * beams]), vocab), rng.choice(["fp32", "fp32", "bf16", "fp16"]), first=rng.random() < 0.2,
                  masked=rng.choice([0.0, 0.0, 0.5, 0.9]))
    elif kind == "copy":
        page, width, caches = rng.choice([8, 16, 16, 32]), 4 * _log(rng, 10, 256), rng.randint(1, 10)
        moves = _log(rng, 1, max(1, min(2000, 200000000 // (page * width * caches * 4))))
        states, forks = rng.randint(0, 6), _log(rng, 1, 64)
        c = _copy(None, caches, page, width, 2 * moves + rng.randint(1, 50), moves, rng.randint(1, page), states, 4 * _log(rng, 64, 65536) if states else 0, 2 * forks + 3 if states else 0,
                  forks if states else 0, rng.choice(["fp32", "fp32", "bf16"]))
    elif kind == "store":
        seqs = _log(rng, 1, 64)
        new = rng.choice([1, 1, rng.randint(2, 9), _log(rng, 10, max(11, 6000 // seqs))])
        c = _store(None, seqs, new, rng.choice([0, _log(rng, 1, 2000)]), rng.choice([1, 2, 3, 4, 8]), rng.choice([64, 80, 128, 256]), rng.choice([8, 16, 16, 32, 64]),
                   rng.choice(["fp32", "bf16", "fp16"]))
    else:
        seqs = _log(rng, 1, 64)
        kv_heads, group, dim = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 4, 4, 7, 8]), rng.choice([64, 128, 128, 256])
        new = rng.choice([1, 1, 1, rng.randint(2, 9), _log(rng, 16, max(17, 1200 // seqs))])
        before = rng.choice([0, _log(rng, 1, max(2, 160000 // seqs) if new < 16 else 1000)])
        before = min(before, 12000)
        window = rng.choice([0, 0, _log(rng, 3, 2000)])
        c = _attend(None, seqs, new, before, kv_heads * group, kv_heads, dim, rng.choice([8, 16, 16, 32, 64]), rng.choice(["bf16", "bf16", "fp16", "fp32"]), window=window,
                    keep_first=rng.choice([0, rng.randint(1, 70)]) if window else 0, softcap=rng.choice([0.0, 0.0, 0.0, 30.0]), sink=rng.random() < 0.25)
    del c["name"]
    return c


# --------------------------------------------------------------------------- inputs

def _spread(c, i):
    """New tokens and earlier positions of sequence i: lengths of one batch differ."""
    f = 1.0 - 0.75 * ((i * 0.6180339887) % 1.0)
    return (max(1, round(c["new"] * f)) if c["new"] >= 16 else c["new"]), round(c["before"] * f)


def _batch(c):
    """(counts, positions before, pages of each sequence) on the host."""
    counts, before = zip(*[_spread(c, i) for i in range(c["seqs"])])
    return list(counts), list(before), [-(-(n + b) // c["page"]) for n, b in zip(counts, before)]


def _pow2(e):
    return torch.ldexp(torch.ones((), device=e.device), e)


def _exponent(amax):
    """The least e >= -64 with amax <= 448 * 2^e (448 = 0.875 * 2^9)."""
    m, x = torch.frexp(amax)
    e = torch.where(m <= 0.875, x - 9, x - 8)
    return torch.where(amax > 0, e, torch.full_like(e, _LEAST)).clamp_min(_LEAST)


def _pool(shape, g):
    """A filled pool: blocks of normal rows whose channels have different sizes, as codes (uint8) and scales."""
    pages, heads, page, dim = shape
    gain = torch.exp(0.5 * torch.randn(heads, 1, dim, generator=g, device="cuda"))
    codes, scales = torch.empty(shape, dtype=torch.uint8, device="cuda"), torch.empty(pages, heads, device="cuda")
    for p in range(0, pages, 4096):
        x = torch.randn(min(4096, pages - p), heads, page, dim, generator=g, device="cuda") * gain
        e = _exponent(x.abs().amax((2, 3)))
        scales[p:p + 4096] = _pow2(e)
        codes[p:p + 4096] = (x * _pow2(-e)[:, :, None, None]).to(torch.float8_e4m3fn).view(torch.uint8)
    return codes, scales


def _inputs(case, seed):
    g, c, dev = torch.Generator(device="cuda").manual_seed(seed), case, "cuda"
    host = np.random.default_rng(seed)
    st = {"case": c}
    if c["kind"] == "beam":
        x = torch.randn(c["groups"], c["beams"], c["vocab"], generator=g, device=dev) * 2.5
        if c["masked"]:
            x[torch.rand(c["vocab"], generator=g, device=dev).expand_as(x) < c["masked"]] = -math.inf
        st["logits"] = x.to(_DTYPES[c["dtype"]])
        st["scores"] = -20.0 - 1.5 * torch.rand(c["groups"], c["beams"], generator=g, device=dev)
        if c["first"]:  # the first step: all beams hold the prompt, one of them counts
            st["scores"][:, 1:] = -math.inf
        return st
    if c["kind"] == "copy":
        t = _DTYPES[c["dtype"]]
        st["pages"] = [torch.randn(c["pages"], c["page"], c["width"], generator=g, device=dev).to(t) for _ in range(c["caches"])]
        st["states"] = [torch.randn(c["slots"], c["state"], generator=g, device=dev) for _ in range(c["states"])]
        where = host.permutation(c["pages"])
        st["src"], st["dst"] = where[:c["moves"]].tolist(), where[c["moves"]:2 * c["moves"]].tolist()
        st["rows"] = [c["filled"]] * c["moves"] if c["filled"] < c["page"] else None
        where = host.permutation(c["slots"])
        st["sfrom"], st["sto"] = where[:c["forks"]].tolist(), where[c["forks"]:2 * c["forks"]].tolist()
        st["lists"] = [torch.tensor(st[k], dtype=torch.int64, device=dev) for k in ("src", "dst", "sfrom", "sto")]
        return st
    counts, before, pages = _batch(c)
    heads = c["heads"] if c["kind"] == "store" else c["kv_heads"]
    total, n = sum(pages), sum(counts)
    st["kc"], st["ks"] = _pool((total + 3, heads, c["page"], c["dim"]), g)
    st["vc"], st["vs"] = _pool((total + 3, heads, c["page"], c["dim"]), g)
    where, at = host.permutation(total + 3)[:total], 0
    table = np.zeros((c["seqs"], max(pages)), np.int32)
    for i, k in enumerate(pages):
        table[i, :k], at = where[at:at + k], at + k
    st["table"], st["counts"], st["before"] = torch.tensor(table, device=dev), counts, before
    seq = np.repeat(np.arange(c["seqs"]), counts)
    pos = np.concatenate([np.arange(b, b + k) for b, k in zip(before, counts)])
    st["seq"], st["pos"] = torch.tensor(seq, device=dev), torch.tensor(pos, device=dev)
    t = _DTYPES[c["dtype"]]
    if c["kind"] == "store":
        # the rows come as parts of one projection, as a model computes them
        both = (torch.randn(n, 2 * heads * c["dim"], generator=g, device=dev) * torch.exp(0.7 * torch.randn(n, 1, generator=g, device=dev))).to(t)
        st["k"], st["v"] = both[:, :heads * c["dim"]].view(n, heads, c["dim"]), both[:, heads * c["dim"]:].view(n, heads, c["dim"])
        st["touched"] = torch.tensor(np.unique(table[seq, pos // c["page"]]).astype(np.int64), device=dev)
    else:
        st["q"] = (torch.randn(n, c["heads"], c["dim"], generator=g, device=dev) * 1.2).to(t)
        st["sink"] = torch.randn(c["heads"], generator=g, device=dev) if c["sink"] else None
        st["row"] = torch.tensor(np.concatenate([np.arange(k) for k in counts]), device=dev)  # place of a token among its sequence's new ones
    return st


def prepare(case, seed):
    st = _inputs(case, seed)
    if own:  # what a serving program keeps beside its buffers: the pools' layout, the step's description
        from calm_b200 import seqops

        if case["kind"] == "copy":
            st["pool"] = seqops.UnitPool(st["pages"], st["states"])
        elif case["kind"] in ("store", "attend"):
            st["cache"] = seqops.Cache8(st["kc"], st["ks"], st["vc"], st["vs"])
            st["batch"] = seqops.Batch(range(case["seqs"]), st["counts"], st["before"])
    return st


# --------------------------------------------------------------------------- one pass

def _plain_beam(logits, scores, n):
    groups, beams, vocab = logits.shape
    x = logits.double()
    top = x.amax(-1, keepdim=True)
    lse = top + torch.log(torch.exp(x - top).sum(-1, keepdim=True))
    total = (scores.double()[:, :, None] + (x - lse)).nan_to_num(nan=-math.inf).view(groups, beams * vocab)
    best, at = torch.sort(total, dim=1, descending=True, stable=True)
    best, at = best[:, :n], at[:, :n]
    none = best == -math.inf
    return torch.where(none, -1, at % vocab).int(), torch.where(none, -1, at // vocab).int(), best.float()


def _plain_copy(st):
    src, dst, sfrom, sto = st["lists"]
    rows = st["case"]["filled"]
    for t in st["pages"]:
        t[dst, :rows] = t[src, :rows]
    for t in st["states"]:
        t[sto] = t[sfrom]


def _plain_store(codes, scales, rows, page, off, touched):
    """Rows [n][heads][dim] into rows `off` of the pages `page`."""
    pages, heads = scales.shape
    x = rows.float()
    x = torch.where(x.isnan(), 0.0, x)
    need = torch.where(x.isinf(), 0.0, x).abs().amax(-1)  # [n][heads]
    amax = torch.zeros_like(scales).scatter_reduce_(0, page[:, None].expand(-1, heads), need, "amax")
    first = torch.full((pages,), codes.shape[2], dtype=off.dtype, device=off.device).scatter_reduce_(0, page, off, "amin")
    e_new, e_old = _exponent(amax[touched]), _exponent(scales[touched] * 448.0)
    e = torch.where(first[touched, None] == 0, e_new, torch.maximum(e_new, e_old))
    kept = codes[touched].view(torch.float8_e4m3fn).float() * _pow2(e_old - e)[:, :, None, None]
    early = torch.arange(codes.shape[2], device=off.device)[None, :] < first[touched, None]
    codes[touched] = torch.where(early[:, None, :, None], kept.clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8), codes[touched])
    scales[touched] = _pow2(e)
    y = (x / scales[page][:, :, None]).clamp(-448, 448)
    codes[page, :, off] = y.to(torch.float8_e4m3fn).view(torch.uint8)


def _plain_attend(st):
    c, table = st["case"], st["table"].long()
    seqs, page, dim, kv = c["seqs"], c["page"], c["dim"], c["kv_heads"]
    group, keys, most = c["heads"] // kv, table.shape[1] * page, max(st["counts"])

    def rows(codes, scales):  # [seqs][kv heads][keys][dim]
        x = codes[table].view(torch.float8_e4m3fn).float() * scales[table][:, :, :, None, None]
        return x.transpose(1, 2).reshape(seqs, kv, keys, dim)

    k, v = rows(st["kc"], st["ks"]), rows(st["vc"], st["vs"])
    q = torch.zeros(seqs, most, c["heads"], dim, device=table.device)
    q[st["seq"], st["row"]] = st["q"].float()
    at = torch.full((seqs, most), -1, dtype=torch.int64, device=table.device)
    at[st["seq"], st["row"]] = st["pos"]
    key = torch.arange(keys, device=table.device)
    seen = key <= at[:, :, None]
    if c["window"]:
        seen &= (key > at[:, :, None] - c["window"]) | (key < c["keep_first"])
    q = q.view(seqs, most, kv, group, dim).permute(0, 2, 3, 1, 4).reshape(seqs, kv, group * most, dim)
    s = torch.matmul(q, k.transpose(2, 3)) * dim ** -0.5
    if c["softcap"]:
        s = c["softcap"] * torch.tanh(s / c["softcap"])
    s = s.view(seqs, kv, group, most, keys).masked_fill(~seen[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    if st["sink"] is not None:
        sink = st["sink"].view(1, kv, group, 1, 1)
        top = torch.maximum(top, sink)
    top = torch.where(top == -math.inf, 0.0, top)
    p = torch.exp(s - top)
    below = p.sum(-1, keepdim=True)
    if st["sink"] is not None:
        below = below + torch.exp(sink - top)
    o = torch.matmul(p.view(seqs, kv, group * most, keys), v).view(seqs, kv, group, most, dim) / below
    o = o.permute(0, 3, 1, 2, 4).reshape(seqs, most, c["heads"], dim)
    return o[st["seq"], st["row"]].to(st["q"].dtype)


def run(st):
    c = st["case"]
    if c["kind"] == "beam":
        if own:
            from calm_b200 import seqops

            tokens, parents, scores = seqops.beam_select(st["logits"], st["scores"], c["n"])
        else:
            tokens, parents, scores = _plain_beam(st["logits"], st["scores"], c["n"])
        return {"tokens": tokens, "parents": parents, "scores": scores}
    if c["kind"] == "copy":
        if own:
            st["pool"].copy(pages=(st["src"], st["dst"], st["rows"]), slots=(st["sfrom"], st["sto"]))
        else:
            _plain_copy(st)
        return {"pages": st["pages"], "states": st["states"]}
    if c["kind"] == "store":
        if own:
            st["cache"].store(st["k"], st["v"], st["table"], st["batch"])
        else:
            page, off = st["table"].long()[st["seq"], st["pos"] // c["page"]], st["pos"] % c["page"]
            _plain_store(st["kc"], st["ks"], st["k"], page, off, st["touched"])
            _plain_store(st["vc"], st["vs"], st["v"], page, off, st["touched"])
        return {"k": st["kc"].view(torch.float8_e4m3fn), "k_scale": st["ks"], "v": st["vc"].view(torch.float8_e4m3fn), "v_scale": st["vs"]}
    if own:
        return st["cache"].attend(st["q"], st["table"], st["batch"], scale=c["dim"] ** -0.5, window=c["window"], keep_first=c["keep_first"], softcap=c["softcap"], sink=st["sink"])
    return _plain_attend(st)


# --------------------------------------------------------------------------- what a pass cannot do without

def work(case):
    c = case
    size = 4 if c["dtype"] == "fp32" else 2
    if c["kind"] == "beam":
        rows = c["groups"] * (1 if c["first"] else c["beams"])
        return {"bytes": rows * c["vocab"] * size + c["groups"] * (4 * c["beams"] + 12 * c["n"]), "flops": 4.0 * rows * c["vocab"]}
    if c["kind"] == "copy":
        return {"bytes": 2 * (c["moves"] * c["caches"] * c["filled"] * c["width"] * size + c["forks"] * c["states"] * c["state"] * 4), "flops": 0}
    counts, before, _ = _batch(c)
    n = sum(counts)
    if c["kind"] == "store":
        rows = n * c["heads"] * c["dim"]
        blocks = sum(-(-(b % c["page"] + k) // c["page"]) for b, k in zip(before, counts))
        return {"bytes": 2 * (rows * (size + 1) + blocks * c["heads"] * 8), "flops": 4.0 * rows}
    pairs = read = 0
    for k, b in zip(counts, before):
        pos = np.arange(b, b + k)
        seen = pos + 1
        read_here = b + k
        if c["window"]:
            low = np.maximum(0, pos - c["window"] + 1)
            seen = pos - low + 1 + np.minimum(c["keep_first"], low)
            read_here = b + k - int(low[0]) + min(c["keep_first"], int(low[0]))
        pairs, read = pairs + int(seen.sum()), read + read_here
    return {"bytes": 2 * read * c["kv_heads"] * c["dim"] + 2 * n * c["heads"] * c["dim"] * size, "flops": 4.0 * pairs * c["heads"] * c["dim"]}


# --------------------------------------------------------------------------- the definitions in 64 bits

def _exact_code(x):
    """Nearest e4m3 value (ties to the even code) of |x| <= 448, in 64 bits."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -6))) - 3)
    return torch.round(x / step) * step


def _exact_store(codes, scales, rows, table, counts, before, page):
    value, scale = codes.view(torch.float8_e4m3fn).float().double(), scales.double()
    rows, at = rows.double(), 0
    table = table.tolist()
    for i, (k, b) in enumerate(zip(counts, before)):
        for block in range(b // page, (b + k - 1) // page + 1):
            lo, hi = max(b, block * page), min(b + k, (block + 1) * page)
            p, x = table[i][block], rows[at + lo - b:at + hi - b].transpose(0, 1)
            need = torch.exp2(torch.ceil(torch.log2(x.abs().amax((1, 2)).clamp_min(448.0 * 2.0 ** _LEAST) / 448.0)))
            if lo > block * page:
                need = torch.maximum(need, scale[p])
                value[p, :, :lo - block * page] = _exact_code(value[p, :, :lo - block * page] * (scale[p] / need)[:, None, None])
            scale[p] = need
            value[p, :, lo - block * page:hi - block * page] = _exact_code(x / need[:, None, None])
        at += k
    return value, scale


def exact(case, seed):
    c = case
    if c["kind"] == "copy":
        return None
    st = _inputs(case, seed)
    if c["kind"] == "beam":
        tokens, parents, scores = [], [], []
        for g in range(c["groups"]):
            log_p = torch.log_softmax(st["logits"][g].double(), -1) + st["scores"][g].double()[:, None]
            log_p = torch.where(torch.isnan(log_p), -math.inf, log_p).cpu().numpy().reshape(-1)
            near = np.argpartition(-log_p, min(4 * c["n"], log_p.size - 1))[:4 * c["n"]]
            order = near[np.lexsort((near, -log_p[near]))][:c["n"]]
            good = log_p[order] > -math.inf
            tokens.append(np.where(good, order % c["vocab"], -1)), parents.append(np.where(good, order // c["vocab"], -1)), scores.append(log_p[order])
        return {"tokens": torch.tensor(np.stack(tokens), dtype=torch.int32), "parents": torch.tensor(np.stack(parents), dtype=torch.int32), "scores": torch.tensor(np.stack(scores))}
    if c["kind"] == "store":
        k, ks = _exact_store(st["kc"], st["ks"], st["k"], st["table"], st["counts"], st["before"], c["page"])
        v, vs = _exact_store(st["vc"], st["vs"], st["v"], st["table"], st["counts"], st["before"], c["page"])
        return {"k": k, "k_scale": ks, "v": v, "v_scale": vs}
    out, at = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda"), 0
    group = c["heads"] // c["kv_heads"]
    for i, (n, b) in enumerate(zip(st["counts"], st["before"])):
        own_pages = st["table"][i, :-(-(n + b) // c["page"])].long()

        def rows(codes, scales):
            x = codes[own_pages].view(torch.float8_e4m3fn).float().double() * scales[own_pages].double()[:, :, None, None]
            return x.permute(1, 0, 2, 3).reshape(c["kv_heads"], -1, c["dim"])[:, :n + b]

        k, v = rows(st["kc"], st["ks"]), rows(st["vc"], st["vs"])
        dist = torch.arange(b, b + n, device="cuda")[:, None] - torch.arange(n + b, device="cuda")[None, :]
        hidden = dist < 0
        if c["window"]:
            hidden |= (dist >= c["window"]) & (torch.arange(n + b, device="cuda")[None, :] >= c["keep_first"])
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

"""Rotary positions, the paged cache in 16 bits and attention over prefixes that sequences share against their plain 64-bit statements (cache16_plain.py), at the sizes and values where they
can go wrong."""
import math
import os
import sys

import numpy as np
import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import cache16_plain as plain  # noqa: E402

pytestmark = pytest.mark.gpu

from calm_b200 import seqops  # noqa: E402

DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SCALINGS = [None, {"kind": "linear", "factor": 4.0}, {"kind": "base", "factor": 8.0}, {"kind": "wavelength", "factor": 8.0, "length": 512, "low": 1.0, "high": 4.0},
            {"kind": "ramp", "factor": 16.0, "length": 4096, "fast": 32.0, "slow": 1.0}]


def as64(t):
    return t.detach().float().cpu().numpy().astype(np.float64)


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def least(dtype):  # half of the type's smallest step
    return torch.finfo(dtype).tiny * torch.finfo(dtype).eps / 2


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def near(got, want, tol, dtype, where=None):
    """got (a tensor) is want to within tol and one rounding to dtype."""
    got, bound = as64(got), plain.rounded(want, tol, half_step(dtype), least(dtype))
    most = torch.finfo(dtype).max
    over = np.abs(want) + bound > most  # may round to an infinity
    ok = (np.abs(got - want) <= bound) | (np.isnan(want) & np.isnan(got)) | (got == want) | (over & np.isinf(got) & (np.sign(got) == np.sign(want)))
    if where is not None:
        ok |= ~where
    assert ok.all(), (np.argwhere(~ok)[:5], got[~ok][:5], want[~ok][:5], bound[~ok][:5])


def positions_of(counts, before):
    return np.concatenate([np.arange(b, b + n) for n, b in zip(counts, before)]) if len(counts) else np.zeros(0, np.int64)


# ---------------------------------------------------------------- rotation

def check_rotate(x, counts, before, rot, **kw):
    n = sum(counts)
    want, tol = plain.rotate(as64(x)[:n], positions_of(counts, before), rot.frequencies, rot.gain, rot.pairs)
    got = seqops.rotate(x, seqops.Batch(range(len(counts)), counts, before), rot, **kw)
    assert got.dtype == x.dtype and got.shape == x.shape
    near(got[:n], want, tol, x.dtype)
    assert torch.equal(got[:n, :, rot.dims:], as_was(x, n)[:n, :, rot.dims:])
    return got


def as_was(x, n):
    return x


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("pairs", ["halves", "neighbours"])
@pytest.mark.parametrize("heads,dim,dims,counts,before", [
    (32, 128, 128, [1], [4000]), (1, 2, 2, [1, 3], [0, 7]), (3, 64, 32, [5, 1, 2], [0, 100, 31]), (14, 80, 20, [130, 77], [3, 900000]), (2, 256, 256, [700], [0]), (7, 96, 12, [33], [5]),
    (40, 128, 128, [513, 1, 0, 64], [0, 9, 5, 8191]), (1, 1024, 1024, [9], [2 ** 31 - 10]), (5, 6, 4, [300], [12]), (65, 192, 96, [3], [1]), (3, 1022, 6, [2, 5], [8, 0]), (2, 770, 770, [3], [50])])
def test_rotated_rows(heads, dim, dims, counts, before, pairs, dtype):
    x = torch.randn(sum(counts), heads, dim, generator=gen(dim + heads), device="cuda").to(DT[dtype])
    check_rotate(x, counts, before, seqops.Rotation(dims, 10000.0, pairs))


@pytest.mark.parametrize("scaling", SCALINGS, ids=lambda s: s["kind"] if s else "none")
def test_rotation_of_far_positions_and_scalings(scaling):
    for pairs in ("halves", "neighbours"):
        x = torch.randn(24, 3, 128, generator=gen(1), device="cuda")
        check_rotate(x, [8, 8, 8], [0, 1000003, 2 ** 31 - 9], seqops.Rotation(128, 500000.0, pairs, scaling))
    check_rotate(x, [24], [77], seqops.Rotation(64, frequencies=-np.linspace(0.0, 3.0, 32)))


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("gap", [0, 2, 7, 8, 1])
@pytest.mark.parametrize("pairs", ["halves", "neighbours"])
def test_rotation_of_parts_of_a_projection_and_in_place(pairs, gap, dtype):
    wide = torch.randn(50, 4 * 64 + gap, generator=gen(gap), device="cuda").to(DT[dtype])
    x = wide[:, gap:].unflatten(1, (4, 64))
    rot, counts, before = seqops.Rotation(48, pairs=pairs), [20, 30], [3, 40]
    got = check_rotate(x, counts, before, rot)
    batch = seqops.Batch(range(2), counts, before)
    out = torch.full((53, 4, 64), 7.0, device="cuda", dtype=DT[dtype])  # rows behind the last sequence stay
    assert seqops.rotate(x, batch, rot, out=out) is out and torch.equal(out[:50], got) and (out[50:] == 7.0).all()
    longer = torch.cat([wide, wide[:5]])[:, gap:].unflatten(1, (4, 64))
    more = seqops.rotate(longer, batch, rot)
    assert torch.equal(more[:50], got) and (more[50:] == 0).all()
    kept = wide[:, :gap].clone()
    assert seqops.rotate(x, batch, rot, out=x).data_ptr() == x.data_ptr() and torch.equal(x, got) and torch.equal(wide[:, :gap], kept)
    heads_first = torch.randn(4, 50, 64, generator=gen(9), device="cuda").to(DT[dtype]).transpose(0, 1)
    check_rotate(heads_first, counts, before, rot)


def test_rotation_of_what_is_not_finite():
    x = torch.randn(6, 2, 32, generator=gen(2), device="cuda")
    x[0, 0, 3], x[1, 1, 20], x[2, 0, 31] = math.inf, math.nan, -math.inf
    got = seqops.rotate(x, seqops.Batch([0], [6], [1]), seqops.Rotation(16))
    want, tol = plain.rotate(as64(x), np.arange(1, 7), *(lambda r: (r.frequencies, r.gain, r.pairs))(seqops.Rotation(16)))
    near(got, want, tol, torch.float32)


def test_rotation_of_bad_descriptions_on_the_device():
    x = torch.randn(8, 2, 32, generator=gen(3), device="cuda")
    batch, rot, out = seqops.Batch([0, 1, 2, 3], [2, 2, 2, 2], [0, 5, 9, 1]), seqops.Rotation(32), torch.full((8, 2, 32), 7.0, device="cuda")
    batch.data[0, 1], batch.data[3, 2], batch.data[1, 3] = 7, -1, -5  # rows past the end, a negative position, a negative count
    seqops.rotate(x, batch, rot, out=out)
    want, tol = plain.rotate(as64(x)[:2], np.arange(2), rot.frequencies, rot.gain, rot.pairs)
    near(out[:2], want, tol, torch.float32)
    assert (out[2:] == 7.0).all()


# ---------------------------------------------------------------- storing

def check_store(pages, heads, page, dim, dtype, cache_dtype, counts, before, rot, q_heads, seed=0, wide=True):
    rng, n, need = np.random.default_rng(seed), sum(counts), [-(-(b + c) // page) for b, c in zip(before, counts)]
    table = np.full((len(counts) + 1, max(need) + 1), -1, np.int32)
    where, at = rng.permutation(pages), 0
    for i, k in enumerate(need):
        table[i, :k], at = where[at:at + k], at + k
    cache = seqops.Cache16(*(torch.randn(pages, heads, page, dim, generator=gen(seed + i), device="cuda").to(cache_dtype) for i in (1, 2)))
    k0, v0 = as64(cache.k), as64(cache.v)
    both = torch.randn(n, (q_heads + 2 * heads) * dim, generator=gen(seed + 3), device="cuda").to(dtype)
    q, k, v = (x.unflatten(1, (-1, dim)) for x in both.split([q_heads * dim, heads * dim, heads * dim], 1))
    slots = list(rng.permutation(len(counts)))
    batch, tab = seqops.Batch(slots, counts, before), torch.tensor(table[np.argsort(slots)] if False else table, device="cuda")
    pos = positions_of(counts, before)
    turn = (lambda x: plain.rotate(as64(x), pos, rot.frequencies, rot.gain, rot.pairs)) if rot else (lambda x: (as64(x), np.zeros(x.shape)))
    tab_np = np.full_like(table, -1)
    for i, s in enumerate(slots):
        tab_np[s] = table[i]
    tab = torch.tensor(tab_np, device="cuda")
    got = cache.store(k, v, tab, batch, rotation=rot, q=q if rot else None)
    wk, tk = k0.copy(), np.zeros(k0.shape)
    wv, touched, at = v0.copy(), np.zeros(k0.shape, bool), 0
    yk, ek = turn(k)
    for i, (c, b) in enumerate(zip(counts, before)):
        for j in range(c):
            p = tab_np[slots[i], (b + j) // page]
            wk[p, :, (b + j) % page], tk[p, :, (b + j) % page], wv[p, :, (b + j) % page] = yk[at + j], ek[at + j], as64(v)[at + j]
            touched[p, :, (b + j) % page] = True
        at += c
    near(cache.k, wk, tk, cache_dtype)
    near(cache.v, wv, np.zeros(wv.shape), cache_dtype)
    assert np.array_equal(as64(cache.k)[~touched], k0[~touched]) and np.array_equal(as64(cache.v)[~touched], v0[~touched])
    if rot:
        near(got, *turn(q), dtype)
    else:
        assert got is None


@pytest.mark.parametrize("dtype,cache_dtype", [("fp32", "bf16"), ("fp32", "fp16"), ("bf16", "bf16"), ("fp16", "bf16"), ("bf16", "fp16")])
@pytest.mark.parametrize("page,dim,heads,q_heads,dims,pairs", [(16, 128, 8, 32, 128, "halves"), (16, 64, 2, 14, 32, "neighbours"), (1, 16, 3, 3, 2, "halves"), (24, 80, 1, 7, 20, "neighbours"), (64, 256, 1, 1, 256, "halves"),
                                                         (5, 48, 2, 4, 20, "halves"), (16, 128, 2, 2, 0, "halves")])
def test_stored_rows(page, dim, heads, q_heads, dims, pairs, dtype, cache_dtype):
    rot = seqops.Rotation(dims, pairs=pairs, scaling=SCALINGS[3]) if dims else None
    check_store(220, heads, page, dim, DT[dtype], DT[cache_dtype], [1, 37, 0, 5], [100, 0, 3, page - 1], rot, q_heads)
    check_store(220, heads, page, dim, DT[dtype], DT[cache_dtype], [1], [0], rot, q_heads)


def test_stored_rows_of_prompts():
    check_store(400, 8, 16, 128, torch.bfloat16, torch.bfloat16, [1500, 700, 1, 999], [0, 33, 800, 7], seqops.Rotation(128, 500000.0), 32)


def test_stored_values_at_the_edges():
    """What is past float16's range becomes an infinity, NaNs and infinities stay what they are."""
    cache = seqops.Cache16.empty(2, 1, 4, 16, torch.float16)
    v = torch.zeros(4, 1, 16, device="cuda")
    v[0, 0, :6] = torch.tensor([65519.0, 65520.0, -1e30, math.inf, math.nan, 1e-9])
    assert cache.store(v, v, torch.tensor([[1]], dtype=torch.int32, device="cuda"), seqops.Batch([0], [4], [0])) is None
    assert torch.equal(cache.k.nan_to_num(nan=-1.0), cache.v.nan_to_num(nan=-1.0))
    assert torch.equal(cache.v[1, 0].nan_to_num(nan=-1.0), v[:, 0].half().nan_to_num(nan=-1.0)) and (cache.v[0] == 0).all()


def test_stored_rows_of_what_is_not_there_are_left_out():
    cache, rot = seqops.Cache16.empty(4, 2, 4, 32), seqops.Rotation(32)
    table = torch.tensor([[0, 9], [-1, 1], [2, 3]], dtype=torch.int32, device="cuda")
    batch = seqops.Batch([0, 1, 2, 3, 4], [6, 6, 3, 1, 2], [0, 0, 6, 0, 0])
    k, q = torch.randn(18, 2, 32, generator=gen(4), device="cuda").bfloat16(), torch.randn(18, 4, 32, generator=gen(5), device="cuda").bfloat16()
    want = seqops.rotate(k, batch, rot)
    got = cache.store(k, k, table, batch, rotation=rot, q=q)  # a page past the pool, one below it, positions past the table's, slots that it does not have
    assert torch.equal(got, seqops.rotate(q, batch, rot))
    filled = torch.zeros(4, 4, dtype=torch.bool)
    for page, row, token in [(0, r, r) for r in range(4)] + [(1, r, 10 + r) for r in range(2)] + [(3, 2 + r, 12 + r) for r in range(2)]:
        filled[page, row] = True
        assert torch.equal(cache.k[page, :, row], want[token]) and torch.equal(cache.v[page, :, row], k[token])
    assert (cache.k.transpose(1, 2)[~filled.cuda()] == 0).all() and (cache.v.transpose(1, 2)[~filled.cuda()] == 0).all()


def test_queries_turned_in_place():
    cache, rot = seqops.Cache16.empty(8, 2, 8, 64, torch.float16), seqops.Rotation(24, pairs="neighbours")
    x = torch.randn(9, 8, 64, generator=gen(6), device="cuda").half()
    q, k, v = x[:, :4], x[:, 4:6], x[:, 6:]
    batch, table = seqops.Batch([0], [9], [3]), torch.arange(8, dtype=torch.int32, device="cuda")[None]
    want, kept = seqops.rotate(q, batch, rot), x[:, 4:].clone()
    assert cache.store(k, v, table, batch, rotation=rot, q=q, q_out=q) is q
    assert torch.equal(q, want) and torch.equal(x[:, 4:], kept)


# ---------------------------------------------------------------- attention

def make(counts, before, groups, kv_heads, group, dim, page, dtype, seed=0, spare=3, gap=0):
    """A filled cache, its table, queries and the batch; sequences of a group hold the prefix's full pages in common."""
    rng, n = np.random.default_rng(seed), len(counts)
    share = np.zeros(n, int)
    for f, m, p in groups:
        share[f:f + m] = p
    need = [-(-(b + c) // page) for b, c in zip(before, counts)]
    total = sum(need) + spare
    slots = rng.permutation(n + 2)[:n]
    table = np.full((n + 2, max(need + [1]) + 1), -1, np.int32)
    where, at = rng.permutation(total), 0
    first = {b: f for f, m, _ in groups for b in range(f, f + m)}
    k, v = (torch.randn(total, kv_heads, page, dim, generator=gen(seed + i), device="cuda").to(dtype) for i in (1, 2))
    for i in range(n):
        f = first.get(i, i)
        keep = share[i] // page if f != i else 0
        table[slots[i], :keep] = table[slots[f], :keep]
        table[slots[i], keep:need[i]], at = where[at:at + need[i] - keep], at + need[i] - keep
        if f != i and share[i] % page:
            for x in (k, v):
                x[table[slots[i], keep]] = x[table[slots[f], keep]]
    T = sum(counts)
    wide = (torch.randn(T, kv_heads * group * dim + gap, generator=gen(seed + 3), device="cuda") * 1.3).to(dtype)
    q = wide[:, gap:].unflatten(1, (kv_heads * group, dim))
    return seqops.Cache16(k, v), table, q, seqops.Batch(slots.tolist(), list(counts), list(before), shared=groups), slots


def check_attend(cache, table, q, batch, slots, counts, before, groups, got=None, **opt):
    dev = torch.tensor(table, device="cuda")
    scale = opt.pop("scale", q.shape[2] ** -0.5)
    got = cache.attend(q, dev, batch, scale=scale, **opt) if got is None else got
    start = np.concatenate([[0], np.cumsum(counts)])[:-1]
    portions = list(zip(start.tolist(), counts, [int(s) for s in slots], before))
    if opt.get("sink") is not None:
        opt["sink"] = as64(opt["sink"])
    opt.pop("out", None)
    want, tol = plain.attend(as64(q), as64(cache.k), as64(cache.v), table, portions, groups, cache.page, scale, half=half_step(q.dtype), **opt)
    rows = ~np.isnan(want).all((1, 2))
    near(got[:len(want)], want, tol, q.dtype, np.broadcast_to(rows[:, None, None], want.shape) if not rows.all() else None)
    return got


def attention(counts, before, groups, kv_heads, group, dim, page, dtype, seed=0, gap=0, **opt):
    made = make(counts, before, groups, kv_heads, group, dim, page, DT[dtype], seed, gap=gap)
    if opt.pop("sinks", False):
        opt["sink"] = torch.randn(kv_heads * group, generator=gen(77), device="cuda")
    return check_attend(*made, counts, before, groups, **opt)


LAYOUTS = [(16, 128, 2, 4), (16, 64, 2, 7), (8, 256, 1, 8), (13, 80, 1, 1), (1, 16, 2, 3), (64, 48, 1, 20), (24, 128, 1, 33), (5, 64, 3, 2), (32, 112, 2, 4)]


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("page,dim,kv_heads,group", LAYOUTS)
def test_attention_that_shares_nothing(page, dim, kv_heads, group, dtype):
    attention([1], [0], [], kv_heads, group, dim, page, dtype)
    attention([1, 1, 3, 0, 1], [17, 300, 41, 5, 64], [], kv_heads, group, dim, page, dtype, gap=3)
    attention([40, 1, 70], [5, 0, 100], [], kv_heads, group, dim, page, dtype, seed=5)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("page,dim,kv_heads,group", LAYOUTS)
def test_attention_over_shared_prefixes(page, dim, kv_heads, group, dtype):
    attention([1, 1, 1, 1], [200, 207, 240, 201], [(0, 4, 200)], kv_heads, group, dim, page, dtype)                  # beams
    attention([1, 2, 1, 3, 1, 1], [90, 64, 63, 70, 5, 130], [(0, 1, 64), (2, 2, 61), (5, 1, 130)], kv_heads, group, dim, page, dtype, seed=3)  # groups of one, none, all of it shared
    attention([1] * 40, [350 + 3 * i for i in range(40)], [(0, 33, 350), (33, 7, 0)], kv_heads, group, dim, page, dtype, seed=8)  # many rows a group; nothing shared
    attention([9, 30, 1, 17], [130, 128, 200, 131], [(0, 4, 128)], kv_heads, group, dim, page, dtype, seed=9, gap=8)  # portions


@pytest.mark.parametrize("opt", [dict(window=7), dict(window=40), dict(window=250), dict(softcap=2.0), dict(sinks=True), dict(window=33, softcap=5.0, sinks=True), dict(scale=1.7), dict(scale=0.0)],
                         ids=lambda o: "-".join(o))
@pytest.mark.parametrize("dim", [64, 128, 80])
def test_attention_options(opt, dim):
    attention([1, 1, 5, 1], [200, 230, 210, 300], [(0, 3, 200)], 2, 4, dim, 16, "bf16", **opt)
    attention([60] * 5 + [3], [300, 301, 333, 300, 350, 90], [(0, 5, 300)], 2, 4, dim, 16, "bf16", seed=4, **opt)
    attention([300, 1, 140], [100, 90, 77], [(0, 2, 90)], 1, 3, dim, 16, "fp16", seed=5, **opt)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("page,dim,kv_heads,group,counts,before,groups", [
    (16, 128, 2, 4, [1] * 64, [1500 + 7 * i for i in range(64)], [(0, 64, 1500)]),             # a tile of 256 rows over one prefix
    (16, 64, 2, 8, [1] * 40, [900 + i for i in range(40)], [(0, 20, 900), (20, 20, 513)]),
    (24, 128, 1, 4, [5] * 50, [1003 + (3 * i) % 50 for i in range(50)], [(0, 50, 1001)]),
    (8, 96, 1, 2, [2] * 90, [640] * 90, [(0, 90, 640)]),
    (16, 128, 1, 4, [300, 1, 80, 513], [700, 700, 731, 0], [(0, 3, 700)]),                      # questions of different lengths behind a document
    (64, 64, 2, 2, [700, 350], [130, 1], []),
    (16, 128, 4, 1, [260, 260, 257], [512, 513, 600], [(0, 3, 512)]),
])
def test_attention_of_many_rows(page, dim, kv_heads, group, counts, before, groups, dtype):
    attention(counts, before, groups, kv_heads, group, dim, page, dtype)


def way_of(cache, table, q, batch):
    """The way that Cache16.attend's call takes."""
    import ctypes as C

    c = cache._with(torch.tensor(table, device="cuda"), batch)
    r = seqops._rows("q", q, 0, q.shape[1], cache.dim, batch.tokens)
    a = seqops._Attend16(r, r, q.shape[1], 1.0, 0, 0.0, None, batch.most_keys, batch._row_tiles(q.shape[1] // cache.heads), None, 0)
    return seqops._load().calm_b200_seq_attend16_way(C.byref(c), C.byref(batch.c), None if batch.shared is None else C.byref(batch.shared), C.byref(a))


@pytest.mark.parametrize("way,page,dim,kv_heads,group,counts,before,groups", [
    (0, 16, 128, 8, 4, [1] * 70, [200] * 70, []), (4, 16, 128, 2, 4, [1, 1], [1200, 1210], [(0, 2, 1200)]), (8, 16, 64, 4, 4, [1] * 9, [1000 * (i % 3) for i in range(9)], []),
    (1, 16, 128, 8, 4, [1] * 48, [6000 + i for i in range(48)], [(0, 48, 6000)]), (9, 8, 64, 2, 8, [1] * 50, [12000 + 40 * (i % 9) for i in range(48)] + [5000, 13], [(0, 24, 12000), (24, 24, 9001)]),
    (2, 16, 128, 37, 1, [256, 100, 3, 200], [0, 100, 600, 40], []), (10, 16, 128, 2, 4, [300, 1, 170, 90], [1500, 1500, 1500, 1600], [(0, 4, 1500)]), (10, 24, 80, 1, 4, [900], [0], [])])
def test_every_way(way, page, dim, kv_heads, group, counts, before, groups):
    made = make(counts, before, groups, kv_heads, group, dim, page, torch.bfloat16, 3)
    assert way_of(*made[:4]) == way
    check_attend(*made, counts, before, groups, sink=torch.randn(kv_heads * group, generator=gen(5), device="cuda"))


@pytest.mark.parametrize("way,group,counts,before,groups", [(1, 4, [1] * 700, [1200 + i % 40 for i in range(700)], [(0, 330, 1200), (330, 370, 1190)]), (0, 1, [1] * 400, [20 + i % 7 for i in range(400)], [(0, 400, 16)])])
def test_groups_of_more_sequences_than_a_block_has_threads(way, group, counts, before, groups):
    made = make(counts, before, groups, 2, group, 64, 16, torch.bfloat16, 21)
    check_attend(*made, counts, before, groups)
    assert way_of(*made[:4]) & 3 == way


def test_one_prompt_among_single_tokens():
    """As many blocks as the rows have tiles, not as many as if every sequence were as long as the longest."""
    for groups in ([], [(0, 30, 64)]):
        attention([1] * 40 + [1100] + [0] * 3 + [1] * 20, [64 + 9 * i for i in range(64)], groups, 2, 4, 64, 16, "bf16", seed=23)
        attention([1300, 0, 2], [0, 5, 100], [], 3, 2, 128, 8, "fp16", seed=24)


@pytest.mark.parametrize("opt", [dict(), dict(window=150), dict(window=40, softcap=4.0, sinks=True)], ids=lambda o: "-".join(o))
@pytest.mark.parametrize("dim,kv_heads,group,page,dtype", [(128, 8, 4, 16, "bf16"), (64, 4, 1, 8, "fp16"), (80, 3, 12, 24, "bf16"), (128, 2, 33, 16, "bf16")])
def test_single_tokens_go_apart_from_prompts(dim, kv_heads, group, page, dtype, opt):
    """Both kernels at once, with prefixes that single tokens, prompts and both share, and the same after counts have changed between the two kinds."""
    counts, before = [1] * 30 + [300] + [2] * 3 + [0, 1, 171] + [1] * 5, [300 + 7 * i for i in range(42)]
    for groups in ([], [(0, 20, 290), (28, 4, 490), (38, 3, 0)]):
        made = make(counts, before, groups, kv_heads, group, dim, page, DT[dtype], 31)
        sink = dict(sink=torch.randn(kv_heads * group, generator=gen(5), device="cuda")) if "sinks" in opt else {}
        more = dict({k: x for k, x in opt.items() if k != "sinks"}, **sink)
        check_attend(*made, counts, before, groups, **more)
        cache, table, q, batch, slots = made
        now = [300, 1] + counts[2:30] + [1] + counts[31:36] + [1] + counts[37:]  # (not more rows than there were)
        start = np.concatenate([[0], np.cumsum(now)])[:-1]
        if groups:
            continue  # (their sequences' pages are not long enough)
        room = seqops.Batch(slots.tolist(), counts, before)
        room.data[1].copy_(torch.tensor(now, dtype=torch.int32)), room.data[0].copy_(torch.tensor(start, dtype=torch.int32))
        check_attend(cache, table, q, room, slots, now, before, groups, got=cache.attend(q, torch.tensor(table, device="cuda"), room, scale=dim ** -0.5, **more), **more)


def test_apart_when_the_rule_says_so():
    import ctypes as C

    for counts, before, groups, apart in (([1] * 63 + [2048], [2000] * 63 + [0], [], True), ([300] * 16, [500] * 16, [], False), ([1] * 20 + [900] * 2, [1500] * 22, [(0, 22, 1500)], True)):
        batch = seqops.Batch(list(range(len(counts))), counts, before, shared=groups)
        cache = seqops.Cache16.empty(2, 8, 16, 128)
        q = torch.empty(batch.tokens, 32, 128, dtype=torch.bfloat16, device="cuda")
        c, r = cache._with(torch.zeros(len(counts), 300, dtype=torch.int32, device="cuda"), batch), seqops._rows("q", q, 0, 32, 128, batch.tokens)
        a = seqops._Attend16(r, r, 32, 1.0, 0, 0.0, None, batch.most_keys, 0, None, 0)
        a.row_tiles, a.few = batch._split(4)
        way = seqops._load().calm_b200_seq_attend16_way(C.byref(c), C.byref(batch.c), None if batch.shared is None else C.byref(batch.shared), C.byref(a))
        assert way & 3 == 2 and bool(way & 16) == apart


@pytest.mark.parametrize("counts,before,groups", [([1, 1, 2], [300, 310, 305], [(0, 2, 300)]), ([90] * 5, [300] * 5, [(0, 4, 288)]), ([400], [0], [])])
def test_scales_below_zero(counts, before, groups):
    attention(counts, before, groups, 2, 4, 128, 16, "bf16", seed=25, scale=-0.11)
    attention(counts, before, groups, 2, 4, 64, 16, "fp16", seed=26, scale=-0.11, softcap=3.0)


def test_groups_and_sequences_without_tokens():
    attention([0, 0, 1, 0, 40], [700, 700, 30, 9, 5], [(0, 2, 640), (3, 1, 9)], 2, 4, 128, 16, "bf16")
    attention([0, 0, 300], [700, 700, 30], [(0, 2, 640)], 2, 4, 128, 16, "bf16")
    made = make([0, 0], [700, 700], [(0, 2, 640)], 2, 4, 128, 16, torch.bfloat16)
    assert made[0].attend(made[2], torch.tensor(made[1], device="cuda"), made[3], scale=1.0).shape == (0, 8, 128)


def test_sequences_that_have_grown_since_the_call_was_captured():
    """Positions and counts past what the split of the work was planned for."""
    for counts, before, groups, more in (([1] * 6, [100] * 6, [(0, 4, 64)], 1800), ([1], [50], [], 3000), ([200, 100], [100, 64], [(0, 2, 64)], 700), ([1] * 40, [64] * 40, [(0, 40, 48)], 900)):
        now = [b + more for b in before]
        cache, table, q, batch, slots = make(counts, now, groups, 2, 4, 128, 16, torch.bfloat16, 5)
        small = seqops.Batch([int(s) for s in slots], counts, before, shared=groups)
        small.data[3] += more
        check_attend(cache, table, q, small, slots, counts, now, groups, got=cache.attend(q, torch.tensor(table, device="cuda"), small, scale=128 ** -0.5))


def test_attention_of_few_tokens_over_many_keys():
    attention([1], [40000], [], 2, 4, 128, 16, "bf16")
    attention([1, 1], [30000, 30010], [(0, 2, 30000)], 1, 8, 64, 16, "fp16")
    attention([1] * 150, [20 * i for i in range(150)], [], 2, 2, 64, 16, "bf16")  # shares that are folded through memory, some without keys


def test_attention_where_one_key_takes_all_and_scores_grow():
    for groups in ([], [(0, 3, 400)]):
        counts, before = [1, 200, 4], [500, 400, 450]
        cache, table, q, batch, slots = make(counts, before, groups, 1, 4, 128, 16, torch.bfloat16, 11)
        page, row = table[slots[0], 20], 3
        cache.k[page, 0, row] = 20 * q[0, 1]
        check_attend(cache, table, q, batch, slots, counts, before, groups)
        for i in range(26):  # every page's keys point further along the queries than the last one's
            cache.k[table[slots[1], i], 0] = q[5, 0] * (0.2 * i)
        check_attend(cache, table, q, batch, slots, counts, before, groups)


@pytest.mark.parametrize("dim", [64, 128, 48])
@pytest.mark.parametrize("tokens", [1, 70])
def test_what_is_behind_a_sequence_does_not_reach_it(tokens, dim):
    """Pages hold NaN and infinities behind their sequences' last tokens, before their windows and where no table points."""
    for groups in ([], [(0, 3, 300)], [(0, 3, 289)]):
        counts, before = [tokens, tokens, 1, tokens], [300, 311, 320, 45]
        cache, table, q, batch, slots = make(counts, before, groups, 2, 4, dim, 16, torch.bfloat16, 2)
        seen = torch.zeros(cache.pages, 16, dtype=torch.bool)
        for window in (0, 50):
            seen[:] = False
            for i, (n, b) in enumerate(zip(counts, before)):
                for p in range(max(0, b - window + 1) if window else 0, b + n):
                    s = slots[groups[0][0]] if groups and i < 3 and p < groups[0][2] else slots[i]
                    seen[table[s, p // 16], p % 16] = True
            hidden = (~seen.cuda())[:, None, :, None].expand(cache.k.shape)
            for k, v in ((math.nan, math.nan), (math.inf, -math.inf)):
                cache.k[hidden], cache.v[hidden] = k, v
                got = check_attend(cache, table, q, batch, slots, counts, before, groups, window=window)
                assert got.isfinite().all()
            cache.k[hidden], cache.v[hidden] = 1.0, 1.0


def test_one_sequences_numbers_do_not_reach_another():
    """Four beams in one tile: NaN and infinities among one's own keys and values stay with it."""
    counts, before, groups = [1, 1, 1, 1], [100, 110, 105, 120], [(0, 4, 96)]
    cache, table, q, batch, slots = make(counts, before, groups, 2, 4, 128, 16, torch.bfloat16, 2)
    page = table[slots[1], 6]
    cache.v[page, 0, 3, 5], cache.v[page, 1, 2, 9], cache.k[page, 1, 4, 0] = math.nan, math.inf, math.nan
    got = check_attend(cache, table, q, batch, slots, counts, before, groups)
    assert got[[0, 2, 3]].isfinite().all() and got[1, 0:4, 5].isnan().all() and got[1, 0:4, :5].isfinite().all() and got[1, 4:].isnan().all()
    cache.k[page, 1, 4, 0] = 0.0
    got = check_attend(cache, table, q, batch, slots, counts, before, groups)
    assert (got[1, 4:, 9] == math.inf).all() and got[1, 4:, 10:].isfinite().all() and got[[0, 2, 3]].isfinite().all()
    # the prefix is everybody's
    cache.v[table[slots[0], 2], 0, 1, 7] = -math.inf
    got = check_attend(cache, table, q, batch, slots, counts, before, groups)
    assert (got[:, :4, 7] == -math.inf).all() and got[:, :4, 6].isfinite().all()


def test_keys_that_are_not_there():
    """Tables that name pages outside the pool, positions past the table, slots that it does not have, tokens that see nothing."""
    counts, before, groups = [1, 2, 1, 1, 3], [70, 64, 90, 33, 10], [(0, 3, 60)]
    for hole in (-1, 1000):
        cache, table, q, batch, slots = make(counts, before, groups, 2, 3, 64, 16, torch.bfloat16, 6)
        table[slots[0], 1], table[slots[2], 4], table[slots[3], :] = hole, hole, hole
        got = check_attend(cache, table, q, batch, slots, counts, before, groups)
        assert (got[4] == 0).all()  # slot without a page: nothing is seen
        sink = torch.zeros(6, device="cuda")
        check_attend(cache, table, q, batch, slots, counts, before, groups, sink=sink)
    short = np.ascontiguousarray(table[:, :4])
    check_attend(cache, short, q, batch, slots, counts, before, groups)
    got = check_attend(cache, table[:2], q, batch, [s if s < 2 else 99 for s in slots], counts, before, [g for g in groups])
    assert got.isfinite().all()


@pytest.mark.parametrize("tokens", [1, 400])
def test_positions_far_behind_the_table(tokens):
    """A position near 2^31 over a table of few pages: keys that are not there are not walked."""
    counts, before = [tokens, tokens], [2 ** 31 - 500, 2 ** 31 - 500]
    cache, q = seqops.Cache16.empty(8, 1, 16, 64), torch.randn(2 * tokens, 4, 64, generator=gen(1), device="cuda").bfloat16()
    cache.v.copy_(torch.randn(cache.v.shape, generator=gen(2), device="cuda"))
    table = torch.arange(8, dtype=torch.int32, device="cuda").view(2, 4)
    want = cache.v[:4].float().mean((0, 2))[0]
    for groups in ([], [(0, 2, 64)]):
        batch = seqops.Batch([0, 1], counts, before, shared=groups)
        got = cache.attend(q, table, batch, scale=0.1).float()  # keys of zeros: the mean of the values
        assert ((got[0, 0] - want).abs() <= 2.0 ** -8 * (want.abs() + cache.v[:4].float().abs().mean((0, 2))[0]) + 1e-6).all()
        assert (cache.attend(q, table, batch, scale=0.1, window=100) == 0).all()  # a window that holds none


def test_bad_descriptions_on_the_device():
    counts, before, groups = [1, 1, 1, 1, 1], [70, 64, 90, 33, 80], [(0, 3, 60), (3, 2, 30)]
    cache, table, q, batch, slots = make(counts, before, groups, 2, 4, 128, 16, torch.bfloat16, 6)
    dev, out = torch.tensor(table, device="cuda"), torch.full_like(q, 7.0)
    good = cache.attend(q, dev, batch, scale=0.1)
    for name, row, col, value in (("data", 0, 1, 50), ("data", 1, 1, -3), ("data", 3, 1, -1), ("data", 3, 1, 2 ** 31 - 1), ("data", 1, 1, 2 ** 31 - 1)):
        was = batch.data[row, col].item()
        batch.data[row, col] = value
        out.fill_(7.0)
        cache.attend(q, dev, batch, scale=0.1, out=out)
        torch.cuda.synchronize()
        assert (out[1] == 7.0).all() and torch.equal(out[3:], good[3:])
        batch.data[row, col] = was
    for row, col, value in ((0, 0, -1), (0, 0, 5), (1, 0, 0), (1, 0, 6), (1, 0, 2 ** 31 - 1), (2, 0, -5)):
        was = batch.groups[row, col].item()
        batch.groups[row, col] = value
        cache.attend(q, dev, batch, scale=0.1, out=out)
        torch.cuda.synchronize()
        assert torch.equal(out[3:], good[3:])
        batch.groups[row, col] = was
    assert torch.equal(cache.attend(q, dev, batch, scale=0.1), good)


@pytest.mark.parametrize("counts,before,groups", [([1, 1, 1], [20, 300, 310], [(1, 2, 300)]), ([1] * 40, [500] * 40, [(0, 40, 490)]), ([200, 90], [64, 64], [(0, 2, 64)])])
def test_sinks_that_are_infinite(counts, before, groups):
    cache, table, q, batch, slots = make(counts, before, groups, 2, 2, 128, 16, torch.bfloat16, 4)
    sink = torch.tensor([-math.inf, 0.5, math.inf, -3.0], device="cuda")
    got = check_attend(cache, table, q, batch, slots, counts, before, groups, sink=sink)
    assert (got[:, 2] == 0).all()
    without = cache.attend(q, torch.tensor(table, device="cuda"), batch, scale=128 ** -0.5)
    assert torch.equal(got[:, 0], without[:, 0])


def test_rows_behind_the_batch_stay():
    counts, before, groups = [1, 3], [50, 50], [(0, 2, 48)]
    cache, table, q, batch, slots = make(counts, before, groups, 2, 2, 64, 16, torch.float16, 4)
    dev, want = torch.tensor(table, device="cuda"), cache.attend(q, torch.tensor(table, device="cuda"), batch, scale=0.1)
    longer = torch.cat([q, q])
    got = cache.attend(longer, dev, batch, scale=0.1)
    assert torch.equal(got[:4], want) and (got[4:] == 0).all()
    out = torch.full((9, 6, 64), 7.0, device="cuda", dtype=torch.float16)
    assert cache.attend(longer, dev, batch, scale=0.1, out=out[:, 1:5]).data_ptr() == out[:, 1:5].data_ptr()
    assert torch.equal(out[:4, 1:5], want) and (out[4:] == 7).all() and (out[:, 0] == 7).all() and (out[:, 5] == 7).all()


def test_refusals_of_tensors():
    cache, table, q, batch, slots = make([1, 1], [50, 50], [(0, 2, 48)], 2, 2, 64, 16, torch.float16, 4)
    dev, rot = torch.tensor(table, device="cuda"), seqops.Rotation(64)
    k = q[:, :2]
    for call, words in ((lambda: cache.attend(q.float(), dev, batch, scale=1.0), "type"), (lambda: cache.attend(q.bfloat16(), dev, batch, scale=1.0), "type"), (lambda: cache.attend(q[:, :3], dev, batch, scale=1.0), "query heads"),
                        (lambda: cache.attend(q[..., :32], dev, batch, scale=1.0), "must be"), (lambda: cache.attend(q[:1], dev, batch, scale=1.0), "rows"), (lambda: cache.attend(q, dev.long(), batch, scale=1.0), "table"),
                        (lambda: cache.attend(q, dev, batch, scale=1.0, window=2 ** 31), "32 bits"), (lambda: cache.attend(q, dev, batch, scale=1.0, window=-1), "range"),
                        (lambda: cache.attend(q, dev, batch, scale=1.0, sink=torch.zeros(3, device="cuda")), "sink"), (lambda: cache.attend(q, dev, batch, scale=1.0, out=q[:1]), "rows"),
                        (lambda: cache.store(k, k.float(), dev, batch), "values"), (lambda: cache.store(q, k, dev, batch), "must be"), (lambda: cache.store(k, k, dev, batch, q=q), "rotation"),
                        (lambda: cache.store(k, k, dev, batch, rotation=rot, q_out=q), "without q"), (lambda: cache.store(k, k, dev, batch, rotation=5), "Rotation"),
                        (lambda: cache.store(k, k, dev, batch, rotation=seqops.Rotation(66)), "channels"), (lambda: seqops.rotate(q, batch, seqops.Rotation(66)), "channels"),
                        (lambda: seqops.rotate(q[..., ::2], batch, rot), "contiguous"), (lambda: seqops.rotate(q[:1], batch, rot), "rows"), (lambda: seqops.rotate(q, batch, rot, out=q.float()), "type"),
                        (lambda: seqops.Cache16(cache.k, cache.v.bfloat16()), "one shape and type"), (lambda: seqops.Cache16(cache.k.float(), cache.v.float()), "bfloat16"), (lambda: seqops.Cache16.empty(2, 1, 4, 24), "multiple of 16")):
        with pytest.raises(ValueError, match=words):
            call()
    torch.cuda.synchronize()


def test_streams_and_replay():
    """Calls on another stream than their tensors' and two captured calls in one graph, replayed at other positions over other prefixes: neither lives off the other's workspace."""
    counts, before, groups = [1] * 48, [640 + i for i in range(48)], [(0, 24, 640), (24, 20, 512)]
    cache, table, q, batch, slots = make(counts, before, groups, 2, 4, 128, 16, torch.bfloat16, 12)
    dev = torch.tensor(table, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = cache.attend(q, dev, batch, scale=128 ** -0.5)
    side.synchronize()
    check_attend(cache, table, q, batch, slots, counts, before, groups, got=got)
    small = make([1, 1, 2], [90, 100, 95], [(0, 2, 90)], 1, 2, 64, 16, torch.float16, 13)
    rot = seqops.Rotation(64)
    x = torch.randn(4, 4, 64, generator=gen(3), device="cuda").half()
    dev2 = torch.tensor(small[1], device="cuda")
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        a = cache.attend(q, dev, batch, scale=128 ** -0.5)
        turned = small[0].store(x[:, 2:3], x[:, 3:], dev2, small[3], rotation=rot, q=x[:, :2])
        b = small[0].attend(turned, dev2, small[3], scale=0.125)
    for shift in (0, 5, 2):
        now = [p - shift for p in before]
        batch.data[3].copy_(torch.tensor(now, dtype=torch.int32))
        other = [(0, 24, 640 - 3 * shift), (24, 20, 512 - 16 * shift)]
        batch.groups[2].copy_(torch.tensor([g[2] for g in other], dtype=torch.int32))
        x.copy_(torch.randn(x.shape, generator=gen(shift), device="cuda"))
        q.copy_(torch.randn(q.shape, generator=gen(shift + 50), device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        check_attend(cache, table, q, batch, slots, counts, now, other, got=a)
        pos = np.array([90, 100, 95, 96])
        near(turned, *plain.rotate(as64(x[:, :2]), pos, rot.frequencies, rot.gain, rot.pairs), torch.float16)
        check_attend(small[0], small[1], turned, small[3], small[4], [1, 1, 2], [90, 100, 95], [(0, 2, 90)], got=b, scale=0.125)


def test_the_same_call_gives_the_same_bits():
    made = make([1] * 64, [1500 + i for i in range(64)], [(0, 64, 1500)], 2, 4, 128, 16, torch.bfloat16, 12)
    dev = torch.tensor(made[1], device="cuda")
    first = made[0].attend(made[2], dev, made[3], scale=0.09)
    for _ in range(5):
        assert torch.equal(made[0].attend(made[2], dev, made[3], scale=0.09), first)


def test_prompt_and_beams_as_they_are_used():
    """A prompt stored in two portions and read, forked into five sequences that share its full pages, then steps in which each goes its own way, against attention over all rows kept in 64 bits."""
    heads, kv, dim, page, prompt, beams = 8, 2, 64, 16, 150, 5
    rot, scale = seqops.Rotation(dim, 10000.0, "halves"), dim ** -0.5
    cache = seqops.Cache16.empty(64, kv, page, dim, torch.float16)
    table = torch.full((beams, 16), -1, dtype=torch.int32, device="cuda")
    table[0, :10] = torch.arange(10, dtype=torch.int32)
    g, kept = gen(21), [[] for _ in range(beams)]  # (turned key, value) rows of every sequence as the cache has them

    def step(slots, counts, before, shared):
        n = sum(counts)
        x = torch.randn(n, heads + 2 * kv, dim, generator=g, device="cuda")
        q, k, v = x[:, :heads].half(), x[:, heads:heads + kv].half(), x[:, heads + kv:].half()
        batch = seqops.Batch(slots, counts, before, shared=shared)
        turned = cache.store(k, v, table, batch, rotation=rot, q=q)
        out = cache.attend(turned, table, batch, scale=scale)
        pos = positions_of(counts, before)
        near(turned, *plain.rotate(as64(q), pos, rot.frequencies, rot.gain, rot.pairs), torch.float16)
        tab, at = table.cpu().numpy(), 0
        keys = as64(cache.k)
        for s, c, b in zip(slots, counts, before):
            for j in range(c):
                kept[s].append((keys[tab[s, (b + j) // page], :, (b + j) % page], as64(v)[at + j]))
            ks, vs = (np.stack([r[i] for r in kept[s]]) for i in (0, 1))
            ids = np.arange(-(-len(ks) // page))
            pool = [np.zeros((len(ids), kv, page, dim)) for _ in range(2)]
            for p in range(len(ks)):
                pool[0][p // page, :, p % page], pool[1][p // page, :, p % page] = ks[p], vs[p]
            want, tol = plain.attend(as64(turned)[at:at + c], *pool, ids[None], [(0, c, 0, b)], [], page, scale, half=half_step(torch.float16))
            near(out[at:at + c], want, tol, torch.float16)
            at += c

    step([0], [100], [0], [])
    step([0], [prompt - 100], [100], [])
    for s in range(1, beams):  # full pages in common, the one in part filled copied
        table[s, :9] = table[0, :9]
        table[s, 9] = 9 + s
        kept[s] = list(kept[0])
    seqops.UnitPool(cache.buffers()).copy(pages=([9] * (beams - 1), list(range(10, 9 + beams))))
    for t in range(12):
        if (prompt + t) % page == 0:
            table[:, (prompt + t) // page] = torch.arange(30, 30 + beams, dtype=torch.int32)
        step(list(range(beams)), [1] * beams, [prompt + t] * beams, [(0, beams, prompt - prompt % page)])
    step([2, 0, 4], [3, 1, 2], [prompt + 12] * 3, [(0, 2, 144)])

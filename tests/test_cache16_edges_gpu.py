"""Rotary positions, the paged cache in 16 bits and attention over shared prefixes at the edges of what their calls allow: the longest sequences, batches that change between replays, values and
scores at the ends of their types' ranges."""
import ctypes as C
import math
import os
import sys

import numpy as np
import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import cache16_plain as plain  # noqa: E402
from test_cache16_gpu import as64, check_attend, gen, make, near  # noqa: E402

pytestmark = pytest.mark.gpu

from calm_b200 import seqops  # noqa: E402


def test_a_sequence_of_as_many_tokens_as_an_int_holds():
    """Blocks of 21 tokens: the last one's threads count past 2^31.  (One row stands for all of them, the table has the first 32 positions.)"""
    cache, rot, n = seqops.Cache16.empty(4, 1, 16, 48, torch.float16), seqops.Rotation(48), 2 ** 31 - 1
    k, v = (torch.randn(1, 1, 48, generator=gen(i), device="cuda").half() for i in (1, 2))
    table = torch.tensor([[2, 0]], dtype=torch.int32, device="cuda")
    cache.store(k.expand(n, 1, 48), v.expand(n, 1, 48), table, seqops.Batch([0], [n], [0]), rotation=rot)
    pos = np.arange(32)
    want, tol = plain.rotate(np.broadcast_to(as64(k), (32, 1, 48)), pos, rot.frequencies, rot.gain, rot.pairs)
    near(torch.cat([cache.k[2, 0], cache.k[0, 0]])[:, None], want, tol, torch.float16)
    assert torch.equal(cache.v[[2, 0], 0], v.expand(2, 16, 48)) and (cache.k[[1, 3]] == 0).all() and (cache.v[[1, 3]] == 0).all()


# ---------------------------------------------------------------- attention

def way_of(cache, table, q, batch, **opt):
    """The way that Cache16.attend's call takes, as it describes the call (calm_b200_seq_attend16_way)."""
    c, rows = cache._with(torch.tensor(table, device="cuda"), batch), seqops._rows("q", q, 0, q.shape[1], cache.dim, batch.tokens)
    a = seqops._Attend16(rows, rows, q.shape[1], opt.get("scale", cache.dim ** -0.5), opt.get("window", 0), opt.get("softcap", 0.0), None, batch.most_keys, 0, None, 0)
    a.row_tiles, a.few = batch._split(q.shape[1] // cache.heads)
    shared = batch._shared_by(rows.rows)
    return seqops._load().calm_b200_seq_attend16_way(C.byref(c), C.byref(batch.c), None if shared is None else C.byref(shared), C.byref(a))


@pytest.mark.parametrize("way,kv_heads,page,counts,now,before,groups", [
    (4, 2, 16, [5, 1, 1, 1, 5], [5, 5, 1, 1, 1], [600, 610, 620, 605, 30], [(0, 2, 600), (2, 2, 590)]),                     # shares folded by clusters; as many rows as there were
    (4, 2, 16, [4, 1, 1], [4, 4, 4], [900, 903, 901], [(0, 3, 900)]),                                                      # more rows, which q has
    (8, 8, 16, [5, 1, 1, 1] * 4, [5, 5, 5, 1] * 4, [2600 + 7 * i for i in range(16)], [(4 * i, 4, 2600) for i in range(4)]),  # folded through memory
    (0, 16, 12, [6, 1, 1, 1] * 12, [6] * 48, [100 + 7 * i for i in range(48)], [(4 * i, 4, 96) for i in range(12)]),         # not split
    (1, 8, 16, [6] + [1] * 31 + [2], [6] * 32 + [1], [5000 + i for i in range(32)] + [900], [(0, 32, 5000)]),                 # the prefix as tiles of all of a group's rows: more tiles
    (9, 4, 16, [6] + [1] * 31 + [2], [6] * 32 + [1], [5000 + 40 * i for i in range(32)] + [900], [(0, 32, 5000)]),            # own keys folded
])
def test_groups_whose_counts_grow_between_replays(way, kv_heads, page, counts, now, before, groups):
    """Counts up to the longest one that was described, written after the call was captured: no row of a group is lost."""
    cache, table, q, _, slots = make(now, before, groups, kv_heads, 4, 64, page, torch.bfloat16, 41)
    batch, dev, out = seqops.Batch(slots.tolist(), counts, before, shared=groups), torch.tensor(table, device="cuda"), torch.empty_like(q)
    assert way_of(cache, table, q, batch) == way
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        cache.attend(q, dev, batch, scale=0.125, out=out)
    for c in (now, counts):
        batch.data[0].copy_(torch.tensor(np.concatenate([[0], np.cumsum(c)])[:-1], dtype=torch.int32))
        batch.data[1].copy_(torch.tensor(c, dtype=torch.int32))
        out.fill_(7.0)
        graph.replay()
        check_attend(cache, table, q, batch, slots, c, before, groups, got=out, scale=0.125)
        assert (out[sum(c):] == 7.0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim,group", [(64, 4), (128, 4), (128, 9), (256, 2)])
def test_opposite_infinities_are_no_number(dim, group, dtype):
    """Infinities of both signs in one channel of keys that some row sees only in part: NaN for the rows that see both, an infinity for those that see one, wherever the others' masks fall."""
    counts, before, groups = [1, 3, 1], [100, 100, 20], [(0, 2, 96)]
    cache, table, q, batch, slots = make(counts, before, groups, 1, group, dim, 16, dtype, 51)

    def at(seq, pos):
        s = slots[0] if seq < 2 and pos < 96 else slots[seq]
        return int(table[s, pos // 16]), 0, pos % 16

    cache.k[at(1, 100)] = cache.k[at(1, 99)]  # one key twice: one weight
    cache.v[at(1, 99)][3], cache.v[at(1, 100)][3] = math.inf, -math.inf
    cache.v[at(1, 98)][5], cache.v[at(1, 102)][5] = -math.inf, math.inf  # the last token sees both
    cache.v[at(2, 18)][7], cache.v[at(2, 19)][7], cache.v[at(2, 17)][8] = math.inf, -math.inf, -math.inf
    cache.v[at(2, 3)][9], cache.v[at(2, 4)][9] = math.nan, math.inf
    assert way_of(cache, table, q, batch) & 3 == 0
    got = check_attend(cache, table, q, batch, slots, counts, before, groups)
    assert got[1:4, :, 3].isnan().all() and (got[1:3, :, 5] == -math.inf).all() and got[3, :, 5].isnan().all()
    assert got[4, :, 7].isnan().all() and (got[4, :, 8] == -math.inf).all() and got[4, :, 9].isnan().all() and got[0].isfinite().all()


def capped_attention(q, k, v, p0, scale, softcap, half):
    """One sequence's rows q [n][heads][dim] at positions p0 .. over k, v [positions][kv heads][dim] in 64 bits, and what the kernels' arithmetic may be off by before the last rounding.

    Bound: as plain.attend's, but for the cap, which may change a score s by 12 2^-24 of |s|: a rational form of u = s / cap within 2^-24, its numerator and denominator within 1.5 2^-24 each, a
    reciprocal within 2 2^-24, three products within 2^-24 each, u itself within 3 2^-24, of which no more than as much reaches the score."""
    n, heads, dim = q.shape
    group, keys = heads // k.shape[1], p0 + n
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    seen = np.arange(keys)[None] <= p0 + np.arange(n)[:, None]
    for h in range(heads):
        x, kk, vv = q[:, h], k[:keys, h // group], v[:keys, h // group]
        s = x @ kk.T * scale
        mag, big = np.abs(x) @ np.abs(kk).T * abs(scale), np.abs(kk).max(1)[None] * np.abs(x).max(1)[:, None] * abs(scale)
        ds = ((dim / 16 + 6) * mag + dim / 16 * 17 * big) * 2.0 ** -23
        s = softcap * np.tanh(s / softcap)
        s = np.where(seen, s, -math.inf)
        m = s.max(1, keepdims=True)
        ds = np.where(seen, ds + 12 * plain.F32 * np.abs(s) + 6 * plain.F32 * (np.abs(s - m) + np.abs(s)) + 2.0 ** -21, 0.0)
        p = np.where(seen, np.exp(s - m), 0.0)
        p /= p.sum(1, keepdims=True)
        o, adds = p @ vv, (keys / 16 + 200) * 2.0 ** -23
        ds = np.where(seen, ds, 0.0)
        cut = keys / 16 * 17 * 2.0 ** -23 * p.max(1)[:, None] * np.abs(vv).max(0)
        out[:, h] = o
        tol[:, h] = (p * ds) @ np.abs(vv) + (p * ds).sum(1)[:, None] * np.abs(o) + (half + adds) * (p @ np.abs(vv)) + adds * np.abs(o) + cut + 2.0 ** -35 * seen @ np.abs(vv)
    return out, tol


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("softcap", [0.5, 30.0, 1e4, 1e6, 1e8, 1e20, 3e38])
@pytest.mark.parametrize("way,dim,kv,group,counts,before", [(4, 128, 2, 3, [2], [700]), (0, 64, 8, 3, [1, 4, 1], [400, 333, 90]), (2, 128, 8, 4, [300], [200]), (2, 64, 8, 4, [500, 530], [0, 70])])
def test_soft_caps_of_any_size(way, dim, kv, group, counts, before, softcap, dtype):
    """Scores of a deviation of 3, some far past a small cap: a large cap leaves them as they are."""
    cache, table, q, batch, slots = make(counts, before, [], kv, group, dim, 16, dtype, 61)
    q *= 3.0 / 1.3
    assert way_of(cache, table, q, batch, softcap=softcap) & ~8 == way
    got = cache.attend(q, torch.tensor(table, device="cuda"), batch, scale=dim ** -0.5, softcap=softcap)
    at = 0
    for i, (n, b) in enumerate(zip(counts, before)):
        ids = table[slots[i], :-(-(n + b) // 16)]
        k, v = (as64(x)[ids].transpose(0, 2, 1, 3).reshape(-1, kv, dim) for x in (cache.k, cache.v))
        want, tol = capped_attention(as64(q)[at:at + n], k, v, b, dim ** -0.5, softcap, torch.finfo(dtype).eps / 2)
        near(got[at:at + n], want, tol, dtype)
        at += n


def test_numbers_and_caches_that_mean_nothing_are_refused():
    cache, table, q, batch, _ = make([1, 1], [50, 50], [(0, 2, 48)], 2, 2, 64, 16, torch.float16, 4)
    dev = torch.tensor(table, device="cuda")
    for kw in (dict(scale="1"), dict(scale=None), dict(scale=math.nan), dict(scale=-math.inf), dict(scale=10 ** 400), dict(scale=3e38), dict(scale=1.0, softcap=1e-50), dict(scale=1.0, softcap="2"), dict(scale=1.0, softcap=1e39)):
        with pytest.raises(ValueError, match="scale|softcap|range"):
            cache.attend(q, dev, batch, **kw)
    assert torch.equal(cache.attend(q, dev, batch, scale=np.float32(0.125), softcap=np.float64(2.0)), cache.attend(q, dev, batch, scale=0.125, softcap=2))
    for shape in ((2, 0, 16, 64), (2, 2, 0, 64)):
        with pytest.raises(ValueError, match="a cache of"):
            seqops.Cache16.empty(*shape)


@pytest.mark.parametrize("strides", [(2, 1, 1), (1, 1, 1), (0, 1, 1), (0, 64, 1), (64, 0, 1)])
@pytest.mark.parametrize("rows", [3, 5])
def test_rows_that_overlap(strides, rows):
    """Windows on one line of numbers, rows that stand for many: results are tensors of their own."""
    line = torch.randn(2000, generator=gen(71), device="cuda").half()
    x, batch, rot = line.as_strided((rows, 2, 64), strides), seqops.Batch([0], [3], [5]), seqops.Rotation(64)
    apart = x.clone(memory_format=torch.contiguous_format)
    assert torch.equal(seqops.rotate(x, batch, rot), seqops.rotate(apart, batch, rot))
    caches = [seqops.Cache16(*(torch.randn(2, 1, 16, 64, generator=gen(i), device="cuda").half() for i in (1, 2))) for _ in range(2)]
    table = torch.tensor([[1]], dtype=torch.int32, device="cuda")
    turned = [c.store(y[:, :1], y[:, 1:], table, batch, rotation=rot, q=y) for c, y in zip(caches, (x, apart))]
    assert torch.equal(*turned) and torch.equal(caches[0].k, caches[1].k) and torch.equal(caches[0].v, caches[1].v)
    assert torch.equal(*(c.attend(y, table, batch, scale=0.125) for c, y in zip(caches, (x, apart))))


def test_results_whose_rows_overlap_are_refused():
    line, batch, rot = torch.zeros(4000, device="cuda").half(), seqops.Batch([0], [3], [5]), seqops.Rotation(64)
    cache, table = seqops.Cache16.empty(2, 1, 16, 64, torch.float16), torch.tensor([[1]], dtype=torch.int32, device="cuda")
    q = torch.randn(3, 2, 64, generator=gen(5), device="cuda").half()
    for strides in ((2, 1, 1), (0, 64, 1), (64, 0, 1), (64, 64, 1), (63, 256, 1), (256, 63, 1)):
        out = line.as_strided((3, 2, 64), strides)
        for call in (lambda: seqops.rotate(q, batch, rot, out=out), lambda: cache.store(q[:, :1], q[:, 1:], table, batch, rotation=rot, q=q, q_out=out), lambda: cache.attend(q, table, batch, scale=1.0, out=out)):
            with pytest.raises(ValueError, match="overlap"):
                call()
    assert (line == 0).all()
    for strides in ((128, 64, 1), (64, 192, 1), (70, 500, 1), (700, 64, 1)):
        out = line.as_strided((3, 2, 64), strides)
        assert torch.equal(seqops.rotate(q, batch, rot, out=out), seqops.rotate(q, batch, rot))
    one, single = line.as_strided((1, 1, 64), (0, 0, 1)), seqops.Batch([0], [1], [5])
    assert torch.equal(seqops.rotate(q[:1, :1], single, rot, out=one), seqops.rotate(q[:1, :1], single, rot))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim,group", [(64, 4), (128, 12), (256, 2)])
def test_infinities_of_little_weight_are_infinities(dim, group, dtype):
    """Keys whose softmax weight is far under what 16 bits hold, in a chunk that not every row sees whole."""
    counts, before = [1, 2], [90, 75]
    cache, table, q, batch, slots = make(counts, before, [], 1, group, dim, 16, dtype, 81)
    q[:] = q[:, :1].abs()  # rows alike
    at = int(table[slots[1], 70 // 16]), 0, 70 % 16
    cache.k[at] = -60.0 * dim ** 0.5 / dim  # scores of about -60
    cache.v[at][2], cache.v[at][4] = math.inf, -math.inf
    got = check_attend(cache, table, q, batch, slots, counts, before, [])
    assert (got[1:, :, 2] == math.inf).all() and (got[1:, :, 4] == -math.inf).all() and got[0].isfinite().all() and got[1:, :, 5:].isfinite().all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("way,counts,before,groups,kv_heads,group,dim,page,opt", [
    (2, [600], [0], [], 8, 4, 128, 16, {}),                                                             # a prompt
    (10, [700, 100], [40, 300], [], 4, 4, 64, 16, {}),                                                  # tasks cut by their keys
    (10, [900], [700], [], 2, 4, 80, 24, dict(window=150)),
    (2, [300], [200], [], 8, 4, 128, 16, dict(window=90)),
    (2, [30] * 40, [100] * 40, [], 8, 4, 128, 8, {}),                                                   # up to 128 rows: two groups of warps on every other tile
    (18, [1] * 63 + [600], [500] * 63 + [0], [], 8, 4, 128, 16, dict(softcap=30.0)),                    # single tokens apart
    (10, [300, 1, 170, 90], [1500] * 4, [(0, 4, 1500)], 2, 4, 128, 16, dict(window=1000)),              # tasks over a shared prefix
    (9, [1] * 48, [6000 + 5 * i for i in range(48)], [(0, 48, 6000)], 8, 4, 128, 16, dict(window=5000)),  # the prefix as tiles of a group's rows, which see different parts of it
    (9, [3] * 24, [6000 + 9 * i for i in range(24)], [(0, 24, 6000)], 8, 2, 64, 16, dict(window=5500)),
])
def test_values_that_are_not_finite_reach_the_rows_that_see_them(way, counts, before, groups, kv_heads, group, dim, page, opt, dtype):
    """Of tokens and sequences whose rows share a tile of 128 rows or more, those that do not see a key have nothing of its value."""
    made = make(counts, before, groups, kv_heads, group, dim, page, dtype, 91)
    cache, table, q, batch, slots = made
    assert way_of(cache, table, q, batch, **opt) == way
    rng, shared = np.random.default_rng(5), {f: p for f, _, p in groups}
    for i, (n, b) in enumerate(zip(counts, before)):  # the first rows' windows' edges, the new tokens themselves
        own = b + rng.integers(0, n, 3)
        edge = b - opt["window"] + rng.integers(2, 40, 3) if "window" in opt else own
        for j, pos in enumerate((own[0], own[1], edge[0], edge[1])):
            if pos < 0 or (i % 5 and n < 20):
                continue
            at = int(table[slots[i], pos // page]), j % kv_heads, int(pos % page)
            cache.v[at][(3 * j + i) % dim] = (math.nan, math.inf, -math.inf, math.nan)[(i + j) % 4]
    if "window" in opt:  # a prefix's values, which some rows' windows have left behind
        for f, p in shared.items():
            for j, pos in enumerate(before[f] - opt["window"] + np.array([3, 9, 30, 61, 62])):
                cache.v[int(table[slots[f], pos // page]), j % kv_heads, int(pos % page)][5 * j] = (math.inf, math.nan, -math.inf)[j % 3]
    got = check_attend(*made, counts, before, groups, **opt)
    assert 0 < (~got.isfinite()).sum() < got.numel() // 8


def test_values_that_are_not_finite_beside_pages_that_are_not_there():
    counts, before = [500, 300], [100, 0]
    made = make(counts, before, [], 8, 4, 64, 8, torch.bfloat16, 92)
    cache, table, q, batch, slots = made
    table[slots[0], 3], table[slots[0], 40], table[slots[1], 0] = -1, 10 ** 6, -1
    for pos, x in ((9, math.nan), (17, math.inf), (333, -math.inf), (560, math.nan)):
        cache.v[int(table[slots[0], pos // 8]), 2, pos % 8, pos % 64] = x
    assert way_of(cache, table, q, batch) & 3 == 2
    got = check_attend(*made, counts, before, [])
    assert got[:, 4:8].isfinite().all() and got[500:].isfinite().all() and (got[500:508] == 0).all()


@pytest.mark.parametrize("opt", [dict(), dict(window=150), dict(window=40, softcap=4.0)], ids=lambda o: "-".join(o))
@pytest.mark.parametrize("dim,kv_heads,group,page", [(128, 4, 4, 16), (64, 4, 1, 8), (80, 2, 12, 24), (128, 2, 33, 16)])
def test_single_tokens_beside_prompts(dim, kv_heads, group, page, opt):
    """Every layout really goes apart (units of one CTA and of several), and still does what it should after counts and positions have changed, between the two kinds too."""
    counts = [1] * 100 + [130] + [2] * 3 + [0, 1, 90] + [1] * 5
    before = [100 + 7 * (i % 30) for i in range(len(counts))]
    now = counts[:10] + [130, 2, 0] + counts[13:100] + [1] + counts[101:106] + [2] + counts[107:]  # (not more rows than there were)
    assert sum(now) <= sum(counts)
    later = [b + 45 for b in before]
    for groups in ([], [(0, 90, 90), (98, 4, 100)]):
        most = [max(a, b) for a, b in zip(counts, now)]
        cache, table, full, _, slots = make(most, later, groups, kv_heads, group, dim, page, torch.bfloat16, 31)
        q = full[:sum(counts)]
        batch, dev = seqops.Batch(slots.tolist(), counts, before, shared=groups), torch.tensor(table, device="cuda")
        assert way_of(cache, table, q, batch, **opt) & 19 == 18
        out = torch.empty_like(q)
        for c, at in ((counts, before), (now, later)):
            batch.data[0].copy_(torch.tensor(np.concatenate([[0], np.cumsum(c)])[:-1], dtype=torch.int32))
            batch.data[1].copy_(torch.tensor(c, dtype=torch.int32))
            batch.data[3].copy_(torch.tensor(at, dtype=torch.int32))
            out.fill_(7.0)
            cache.attend(q, dev, batch, scale=dim ** -0.5, out=out, **opt)
            check_attend(cache, table, q, batch, slots, c, at, groups, got=out, **opt)
            assert (out[sum(c):] == 7.0).all()

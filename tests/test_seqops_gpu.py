"""The operators on callers' memory against their plain 64-bit statements (seqops_plain.py), at the sizes and values where they can go wrong."""
import math
import os
import sys

import numpy as np
import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import seqops_plain as plain  # noqa: E402

pytestmark = pytest.mark.gpu

from calm_b200 import seqops  # noqa: E402

DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def as64(t):
    return t.detach().float().cpu().numpy().astype(np.float64)


# ---------------------------------------------------------------- beams

def check_beam(logits, scores, n, got=None):
    tok, par, best = got or seqops.beam_select(logits, scores, n)
    rt, rp, rb = plain.beam_select(as64(logits), as64(scores), n)
    tok, par, best = tok.cpu().numpy(), par.cpu().numpy(), as64(best)
    assert np.array_equal(tok, rt) and np.array_equal(par, rp), (tok, rt, par, rp)
    there = rt >= 0
    assert np.array_equal(best[~there], np.full((~there).sum(), -math.inf))
    off = np.abs(best[there] - rb[there])
    assert (off <= plain.F32 * np.abs(rb[there]) + plain.log_sum_bound(logits.shape[2])).all(), off.max()


@pytest.mark.parametrize("groups,beams,vocab,n,dtype", [
    (1, 1, 1, 1, "fp32"), (1, 1, 1, 5, "bf16"), (1, 1, 17, 20, "fp32"), (2, 3, 257, 6, "fp32"), (1, 4, 4096, 8, "fp32"), (1, 4, 4097, 8, "fp16"), (3, 5, 4099, 10, "bf16"),
    (1, 1, 50257, 64, "fp32"), (1, 64, 700, 64, "fp32"), (7, 16, 1000, 16, "fp16"), (2, 2, 131072, 3, "bf16"), (40, 8, 9001, 16, "fp32"), (300, 1, 33, 2, "fp32"),
    (150, 3, 40001, 10, "fp16"), (4, 64, 20000, 64, "fp32"), (1, 1, 3000000, 3, "bf16")])
def test_beams_of_random_logits(groups, beams, vocab, n, dtype):
    g = torch.Generator(device="cuda").manual_seed(vocab + n)
    logits = (torch.randn(groups, beams, vocab, generator=g, device="cuda") * 3).to(DT[dtype])
    scores = -30 * torch.rand(groups, beams, generator=g, device="cuda") / max(beams, 4)
    check_beam(logits, scores, n)


@pytest.mark.parametrize("order", ["equal", "rising", "falling", "late", "two values"])
@pytest.mark.parametrize("n", [1, 8, 64])
def test_beams_of_ordered_rows(order, n):
    V = 70001
    i = torch.arange(V, dtype=torch.float32, device="cuda")
    row = {"equal": torch.zeros_like(i), "rising": i * 1e-3, "falling": -i * 1e-3, "late": torch.where(i > V - 100, 5.0, i * 1e-5), "two values": torch.where(i % 2 == 1, 1.0, -1.0)}[order]
    logits = torch.stack([row, row - 1.0]).expand(2, 2, V)
    check_beam(logits, torch.tensor([[-1.0, -1.25], [-3.0, -2.5]], device="cuda"), n)


def test_beams_of_the_longest_rows():
    V = 1 << 21  # (2^27 candidates a group)
    row = torch.randperm(V, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").float() / (1 << 18)
    scores = torch.full((1, 64), -100.0, device="cuda")  # only beam 5 counts: no other beam's best reaches its 64th
    scores[0, 5] = -1.0
    tok, par, best = seqops.beam_select(row.expand(1, 64, V), scores, 64)
    top = torch.argsort(row, descending=True)[:64]
    assert torch.equal(tok[0].long(), top) and (par == 5).all()
    want = row[top].double() - torch.logsumexp(row.double(), 0) - 1.0
    off = (best[0].double() - want).abs()
    assert (off <= plain.F32 * want.abs() + plain.log_sum_bound(V)).all(), off.max()


def test_beams_with_rows_that_leave_nothing_and_special_values():
    V, inf, nan = 9000, math.inf, math.nan
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(8, 3, V, generator=g, device="cuda")
    x[0, 1] = -inf                      # a row whose mask leaves nothing
    x[1] = -inf                         # a group without any
    x[2, :, 5:] = -inf                  # fewer candidates than asked for
    x[3, 0, 4000] = inf                 # one token takes all of a row's probability, two share another's
    x[3, 1, 17], x[3, 1, 8999] = inf, inf
    x[4, :, ::3] = nan                  # NaNs are masked
    x[5, 2, 1], x[5, 2, 0] = 0.0, -0.0  # one value
    x[6] = torch.finfo(torch.float32).min
    x[6, 0, 8000] = -1e30
    s = torch.full((8, 3), -2.0, device="cuda")
    s[5, :2], s[7] = -inf, torch.tensor([nan, -inf, -1.0])
    x[5, 2, 2:] = -8.0
    for n in (1, 7, 20):
        check_beam(x, s, n)
    x[7, :2] = nan  # rows of beams that are not there are not looked at
    check_beam(x, s, 6)


def test_beams_whose_score_is_not_finite_are_not_there():
    x = torch.randn(2, 4, 500, generator=torch.Generator(device="cuda").manual_seed(6), device="cuda")
    s = torch.tensor([[-1.0, math.inf, math.nan, -2.0], [math.inf, math.inf, -math.inf, math.nan]], device="cuda")
    check_beam(x, torch.where(s.isfinite(), s, -math.inf), 12, seqops.beam_select(x, s, 12))


def test_beams_strides_streams_outputs_and_replay():
    g = torch.Generator(device="cuda").manual_seed(5)
    wide = torch.randn(3, 4, 1111, generator=g, device="cuda", dtype=torch.float32).bfloat16()
    view = wide[:, 1:3, 5:1006]  # rows that start at odd addresses
    s = torch.randn(3, 2, generator=g, device="cuda")
    check_beam(view, s, 9)
    side = torch.cuda.Stream()
    out = (torch.empty(3, 9, dtype=torch.int32, device="cuda"), torch.empty(3, 9, dtype=torch.int32, device="cuda"), torch.empty(3, 9, device="cuda"))
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = seqops.beam_select(view, s, 9, out=out)
    side.synchronize()
    assert got[0] is out[0]
    check_beam(view, s, 9, got)
    # two captured calls in one graph, replayed on other inputs: neither lives off the other's workspace
    x, y = torch.zeros(2, 3, 5000, device="cuda"), torch.zeros(1, 1, 300, device="cuda")
    sx, sy = torch.zeros(2, 3, device="cuda"), torch.zeros(1, 1, device="cuda")
    seqops.beam_select(x, sx, 6)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a, b = seqops.beam_select(x, sx, 6), seqops.beam_select(y, sy, 4)
    for seed in (1, 2):
        g.manual_seed(seed)
        x.copy_(torch.randn(x.shape, generator=g, device="cuda")), y.copy_(torch.randn(y.shape, generator=g, device="cuda")), sx.copy_(torch.randn(2, 3, generator=g, device="cuda"))
        graph.replay()
        check_beam(x, sx, 6, a), check_beam(y, sy, 4, b)


# ---------------------------------------------------------------- copies

@pytest.mark.parametrize("width,dtype,rows", [(256, "fp32", None), (7, "bf16", 3), (5, "fp32", 1), (64, "fp16", 0), (1, "bf16", None)])
def test_copies_of_pages_and_slots(width, dtype, rows):
    rng = np.random.default_rng(width)
    pages = [torch.randn(50, 8, w, device="cuda").to(DT[dtype]) for w in (width, 2 * width)]
    states = [torch.randn(20, 3, width, device="cuda"), torch.randn(20, device="cuda")]
    where, sw = rng.permutation(50), rng.permutation(20)
    src, dst, sf, st = where[:20].tolist(), where[20:40].tolist(), sw[:9].tolist(), sw[9:18].tolist()
    take = None if rows is None else [min(8, rows + i % 2) for i in range(20)]
    want_p, want_s = [t.clone() for t in pages], [t.clone() for t in states]
    for w in want_p:
        for i, (a, b) in enumerate(zip(src, dst)):
            k = 8 if take is None else take[i]
            w[b, :k] = w[a, :k]
    for w in want_s:
        for a, b in zip(sf, st):
            w[b] = w[a]
    seqops.UnitPool(pages, states).copy(pages=(src, dst, take), slots=(sf, st))
    assert all(torch.equal(a, b) for a, b in zip(pages + states, want_p + want_s))


def test_copies_of_many_pools_and_pairs_and_into_another_pool():
    rng = np.random.default_rng(1)
    pools = [torch.randn(3000, 2, 3 + i % 5, device="cuda") for i in range(70)]
    where = rng.permutation(3000)
    src, dst = where[:1400].tolist(), where[1400:2800].tolist()
    want = [t.clone() for t in pools]
    for w in want:
        w[dst] = w[src]
    seqops.UnitPool(pools).copy(pages=(src, dst))
    assert all(torch.equal(a, b) for a, b in zip(pools, want))
    # into a smaller pool, where a page may be read by several copies and numbers overlap
    small = [torch.zeros(4, 2, 3 + i % 5, device="cuda") for i in range(70)]
    seqops.UnitPool(pools, into=seqops.UnitPool(small)).copy(pages=([0, 2999, 0, 1], [0, 1, 2, 3]))
    assert all(torch.equal(b, a[[0, 2999, 0, 1]]) for a, b in zip(pools, small))


def test_a_captured_copy_holds_its_lists():
    t = torch.arange(40, dtype=torch.float32, device="cuda").view(10, 2, 2).clone()
    pool = seqops.UnitPool([t])
    pool.copy(pages=([0], [9]))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pool.copy(pages=([1, 2], [5, 6], [1, 2]))
    t.normal_()
    want = t.clone()
    want[5, :1], want[6] = want[1, :1], want[2]
    graph.replay()
    assert torch.equal(t, want)


# ---------------------------------------------------------------- the 8-bit cache

class Cached:
    """A cache with random content and a page table in random order."""

    def __init__(self, slots, table_pages, heads, page, dim, seed, spread=3.0):
        rng = np.random.default_rng(seed)
        self.page, self.heads, self.dim = page, heads, dim
        n = slots * table_pages + 2
        self.table = rng.permutation(n)[:slots * table_pages].reshape(slots, table_pages).astype(np.int32)
        codes = rng.integers(0, 256, (2, n, heads, page, dim), dtype=np.uint8)
        codes[codes & 127 == 127] ^= 1
        scales = 2.0 ** rng.integers(-3, 4, (2, n, heads)) / 64.0
        self.codes, self.scales, self.dtable = torch.tensor(codes, device="cuda"), torch.tensor(scales, dtype=torch.float32, device="cuda"), torch.tensor(self.table, device="cuda")
        self.cache = seqops.Cache8(self.codes[0], self.scales[0], self.codes[1], self.scales[1])

    def values(self):
        return plain.VALUES[self.codes.cpu().numpy()], as64(self.scales)


def portions_of(batch):
    d = batch.data.cpu().numpy()
    return [tuple(int(x) for x in d[:, i]) for i in range(d.shape[1])]


def check_store(c, k, v, batch):
    values, scales = c.values()
    for i, rows in enumerate((k, v)):
        plain.store(values[i], scales[i], as64(rows), c.table, portions_of(batch), c.page)
    c.cache.store(k, v, c.dtable, batch)
    got, gs = c.values()
    assert np.array_equal(gs, scales)
    assert np.array_equal(got, values)  # the definition leaves no room: every rounding is given


@pytest.mark.parametrize("page,dim,heads,dtype", [(16, 128, 2, "bf16"), (16, 64, 3, "fp32"), (8, 80, 1, "fp16"), (1, 16, 2, "fp32"), (64, 256, 1, "bf16"), (13, 48, 2, "bf16")])
def test_stored_rows(page, dim, heads, dtype):
    c = Cached(5, -(-150 // page), heads, page, dim, page + dim)
    g = torch.Generator(device="cuda").manual_seed(7)
    before = [0, 3, 15, 0, 40]
    for counts in ([1, 1, 1, 0, 1], [2, 14, 17, 100, 33], [1, 2, 1, 1, 5]):  # scales grow in pages that hold rows already
        n = sum(counts)
        both = (torch.randn(n + 2, 2 * heads * dim, generator=g, device="cuda") * torch.exp(2 * torch.randn(n + 2, 1, generator=g, device="cuda"))).to(DT[dtype])
        k, v = both[:, :heads * dim].view(-1, heads, dim), both[:, heads * dim:].view(-1, heads, dim)
        check_store(c, k, v, seqops.Batch([4, 0, 2, 3, 1], counts, before))
        before = [b + n for b, n in zip(before, counts)]


def test_stored_values_at_the_edges():
    c = Cached(1, 8, 1, 4, 16, 3)
    rows = torch.zeros(20, 1, 16, device="cuda")
    inf = math.inf
    edges = [448.0, 449.0, 448.0 * 2 ** -64, 1e-30, 3e38, 2.0 ** -126, 1.0, 464.0, 240.0, 17.0, 18.0, 19.0, 0.0, -0.0, 1e-45]
    for i, e in enumerate(edges):
        rows[i, 0] = torch.linspace(-e, e, 16) if i % 2 else e
    rows[15, 0, :4] = torch.tensor([inf, -inf, math.nan, 1.0])
    rows[16, 0] = inf
    rows[17, 0] = math.nan
    check_store(c, rows, -rows, seqops.Batch([0], [20], [0]))
    for i in range(20):  # one by one: rising and falling sizes inside a page
        check_store(c, rows[i:i + 1] * (1 + i % 3), rows[i:i + 1], seqops.Batch([0], [1], [i]))


def test_stored_rows_of_what_is_not_there_are_left_out():
    c = Cached(3, 4, 2, 8, 32, 11)
    c.table[1, 2], c.table[2, 0], c.table[0, 1] = -1, 99, 2 ** 31 - 1
    c.dtable.copy_(torch.tensor(c.table))
    rows = torch.randn(60, 2, 32, device="cuda")
    b = seqops.Batch([0, 1, 2], [20, 20, 20], [0, 6, 20])  # the last two pass the table's end
    check_store(c, rows, rows * 2, b)
    b.data[2, 0], b.data[2, 1], b.data[3, 2] = 3, -1, -5  # slots and a position that are not there
    check_store(c, rows, rows * 3, b)
    b = seqops.Batch([0, 1, 2], [20, 20, 20], [0, 0, 0])
    b.data[1, 2], b.data[0, 0], b.data[3, 1] = 21, -1, 2 ** 31 - 10  # rows behind the array's end and before its start, a position past 31 bits
    check_store(c, rows, rows * 4, b)


def check_attend(c, q, batch, out=None, rows=None, **opt):
    values, scales = c.values()
    split = q.dtype == torch.float32
    kw = {k: (as64(v) if isinstance(v, torch.Tensor) else v) for k, v in opt.items()}
    ref, tol = plain.attend(as64(q), values[0], scales[0], values[1], scales[1], c.table, portions_of(batch), c.page, split=split, **kw)
    before = None if out is None else out.clone()
    o = c.cache.attend(q, c.dtable, batch, out=out, **opt)
    got = as64(o)
    mine = ~np.isnan(ref)
    off = np.abs(got - ref)[mine] - (tol[mine] + plain.half_step(o.dtype) * (np.abs(ref[mine]) + tol[mine]) + (2.0 ** -24 if o.dtype == torch.float16 else 0.0))
    assert np.isfinite(got[mine]).all() and (off <= 0).all(), (off.max(), np.abs(got - ref)[mine].max())
    if (~mine).any():
        assert np.array_equal(got[~mine], np.zeros((~mine).sum()) if before is None else as64(before)[~mine])
    return o


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("page,dim,kv_heads,group", [(16, 128, 2, 4), (16, 64, 2, 7), (8, 256, 1, 8), (13, 80, 1, 1), (1, 16, 2, 3), (64, 48, 1, 20), (16, 128, 1, 33)])
def test_attention_of_tokens_and_portions(page, dim, kv_heads, group, dtype):
    c = Cached(5, -(-200 // page), kv_heads, page, dim, page + dim + group)
    g = torch.Generator(device="cuda").manual_seed(group)
    for counts, before in (([1, 1, 1, 1, 1], [0, 1, 31, 32, 150]), ([1, 5, 0, 40, 3], [199, 3, 7, 60, 0])):
        q = torch.randn(sum(counts), kv_heads * group, dim, generator=g, device="cuda").to(DT[dtype])
        check_attend(c, q, seqops.Batch([1, 3, 0, 2, 4], counts, before), scale=dim ** -0.5)


@pytest.mark.parametrize("opt", [dict(window=7), dict(window=40, keep_first=5), dict(window=3, keep_first=70), dict(chunk=32), dict(chunk=50, window=20, keep_first=2), dict(softcap=2.0),
                                 dict(sink=True), dict(slopes=True), dict(gate=True), dict(window=33, softcap=5.0, sink=True, slopes=True, gate=True)])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_attention_options(opt, dtype):
    c = Cached(4, 13, 2, 16, 64, 5)
    g = torch.Generator(device="cuda").manual_seed(9)
    counts, before = [1, 6, 50, 1], [130, 20, 0, 0]
    q = torch.randn(sum(counts), 6, 64, generator=g, device="cuda").to(DT[dtype])
    opt = dict(opt)
    for name in ("sink", "slopes"):
        if opt.get(name):
            opt[name] = torch.randn(6, generator=g, device="cuda").abs() * (2.0 if name == "sink" else 0.05)
    if opt.get("gate"):
        opt["gate"] = torch.randn(sum(counts), 6, 1, generator=g, device="cuda").expand(-1, -1, 64) if "window" in opt else torch.randn(sum(counts), 6, 64, generator=g, device="cuda")
    check_attend(c, q, seqops.Batch([3, 1, 0, 2], counts, before), scale=0.2, **opt)


@pytest.mark.parametrize("dtype", ["bf16", "fp32", "fp16"])
@pytest.mark.parametrize("page,dim,opt", [(16, 128, {}), (16, 64, {}), (13, 128, dict(window=70, keep_first=5)), (64, 64, dict(chunk=50)), (8, 128, dict(window=3, keep_first=90, sink=True, gate=True))])
def test_attention_of_prompts(page, dim, opt, dtype):
    """Rows enough for the tensor cores' tiles of 128: several sequences of different lengths, one token and none among them, tiles that end inside a token's heads."""
    c = Cached(5, -(-330 // page), 16, page, dim, page + dim)
    c.table[2, 3] = -1  # positions that are not there
    c.dtable.copy_(torch.tensor(c.table))
    g = torch.Generator(device="cuda").manual_seed(page)
    counts, before = [100, 37, 1, 0, 77], [0, 50, 300, 5, 130]
    q = torch.randn(sum(counts), 48, dim, generator=g, device="cuda").to(DT[dtype])
    opt = dict(opt)
    if opt.get("sink"):
        opt["sink"] = torch.randn(48, generator=g, device="cuda") * 3
    if opt.get("gate"):
        opt["gate"] = torch.randn(sum(counts), 48, dim, generator=g, device="cuda")
    check_attend(c, q, seqops.Batch([1, 2, 4, 0, 3], counts, before), scale=0.7 * dim ** -0.5, **opt)


def test_prompt_rows_whose_scores_grow():
    """Keys that grow along the sequence: references move in every tile and the sums are rescaled.  (Single tokens beside it make the batch one for the tensor cores' tiles.)"""
    c = Cached(8, 30, 2, 16, 128, 3)
    for i in range(30):
        c.scales[0, c.table[0, i]] = 2.0 ** (i / 2 - 14)
    q = torch.randn(137, 32, 128, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    check_attend(c, q.bfloat16(), seqops.Batch(list(range(8)), [130] + 7 * [1], [340] + 7 * [40]), scale=0.1)
    check_attend(c, q, seqops.Batch(list(range(8)), [130] + 7 * [1], 8 * [0]), scale=0.1)


def test_attention_of_one_token_over_many_keys():
    """Shares of the keys: single sequences whose keys many CTAs divide, lengths around their borders."""
    c = Cached(2, 200, 1, 16, 128, 21)
    for before in (0, 127, 128, 129, 1000, 3199):
        q = torch.randn(1, 4, 128, device="cuda", generator=torch.Generator(device="cuda").manual_seed(before)).bfloat16()
        check_attend(c, q, seqops.Batch([1], [1], [before]), scale=0.08)
        check_attend(c, q.float(), seqops.Batch([0], [1], [before]), scale=0.08, sink=torch.tensor([0.0, 3.0, -2.0, 90.0], device="cuda"))


def test_attention_where_one_key_takes_all():
    c = Cached(1, 20, 1, 16, 64, 2)
    q = torch.zeros(4, 2, 64, device="cuda").bfloat16()
    q[:] = 30.0 * torch.randn(4, 2, 64, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).bfloat16()
    check_attend(c, q, seqops.Batch([0], [4], [300]), scale=1.0)
    check_attend(c, q * 2.0 ** -60, seqops.Batch([0], [4], [300]), scale=1.0)
    check_attend(c, q * 2.0 ** 60, seqops.Batch([0], [4], [300]), scale=2.0 ** -60)


def test_attention_over_scales_far_apart():
    """Pages whose value scales differ by far more than fp16's range, pages of zeros."""
    c = Cached(1, 10, 1, 8, 64, 4)
    for i in range(10):
        c.scales[1, c.table[0, i]] = 2.0 ** (-64 if i % 3 == 0 else 20 * (i % 5) - 30)
    c.codes[1, c.table[0, 3]] = 0
    q = torch.randn(2, 2, 64, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    check_attend(c, q, seqops.Batch([0], [2], [78]), scale=0.3)
    check_attend(c, q.bfloat16(), seqops.Batch([0], [2], [70]), scale=0.3)


def test_attention_does_not_see_what_is_not_there():
    c = Cached(4, 6, 2, 8, 32, 8)
    bad = torch.full_like(c.codes[:, 0], 0x7F)  # NaN codes in pages and rows that no token sees
    c.codes[:, c.table[0, 5]] = bad
    c.codes[0, c.table[1, 2], :, 3:], c.codes[1, c.table[1, 2], :, 3:] = 0x7F, 0xFF
    c.scales[:, c.table[0, 5]] = math.nan
    c.table[2, 1], c.table[3, 0], c.table[3, 1] = -7, 26, 2 ** 31 - 1
    c.dtable.copy_(torch.tensor(c.table))
    q = torch.randn(16, 4, 32, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2))
    out = torch.full((16, 4, 32), 7.0, device="cuda")
    b = seqops.Batch([0, 1, 2, 3], [3, 1, 5, 4], [20, 18, 10, 0])
    check_attend(c, q, b, out=out, scale=0.2)  # the last sequence sees nothing: zeros; rows 13 .. stay
    assert (out[9:13] == 0).all() and (out[13:] == 7).all()
    check_attend(c, q, seqops.Batch([0, 2, 1], [3, 5, 1], [37, 44, 9]), scale=0.2, window=30)  # past the table's end
    b.data[2, 0], b.data[0, 1], b.data[3, 2] = 9, 16, -1
    check_attend(c, q, b, out=torch.full((16, 4, 32), 5.0, device="cuda"), scale=0.2)


@pytest.mark.parametrize("tokens", [1, 800])
@pytest.mark.parametrize("page", [8, 1])
def test_positions_far_behind_the_table(tokens, page):
    """Device arrays may hold any position: what lies behind the table is neither walked over nor stored, what is in it is still seen."""
    c = Cached(2, 32 // page, 2, page, 64, 10)  # 32 positions a slot
    one = torch.randn(1, 16, 64, device="cuda", generator=torch.Generator(device="cuda").manual_seed(4)).bfloat16()
    q, rows = one.expand(2 * tokens, 16, 64).contiguous(), torch.ones(2 * tokens, 2, 64, device="cuda")
    want = c.cache.attend(torch.cat([one, one]), c.dtable, seqops.Batch([0, 1], [1, 1], [31, 31]), 0.2).float()
    codes, scales = c.values()
    top = float((np.nan_to_num(np.abs(codes[1])).max((2, 3)) * scales[1]).max())
    # each of the two is off by half a bf16 step and by its weights' fp16 rounding, in numerator and denominator
    bound = 2 * (plain.BF16 * want.abs() + 2 * plain.F16 * top)
    b = seqops.Batch([0, 1], [tokens, tokens], [20, 20])
    for far in (2 ** 31 - 1 - tokens, 2 ** 30):
        b.data[3] = far
        before = [x.clone() for x in c.cache.buffers()]
        c.cache.store(rows, rows, c.dtable, b)
        assert all(torch.equal(x, y) for x, y in zip(before, c.cache.buffers()))
        got = c.cache.attend(q, c.dtable, b, 0.2).float().view(2, tokens, 16, 64)
        assert ((got - want[:, None]).abs() <= bound[:, None]).all()
        assert (c.cache.attend(q, c.dtable, b, 0.2, window=16) == 0).all()


def test_a_later_tokens_codes_reach_no_earlier_one():
    c = Cached(1, 8, 1, 8, 64, 9)
    q = torch.randn(8, 4, 64, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3)).bfloat16()
    b = seqops.Batch([0], [8], [40])
    first = c.cache.attend(q, c.dtable, b, scale=0.2)
    c.codes[0, c.table[0, 5], :, 4:], c.codes[1, c.table[0, 5], :, 4:] = 0x7E, 0xFE
    second = c.cache.attend(q, c.dtable, b, scale=0.2)
    assert torch.equal(first[:4], second[:4]) and not torch.equal(first[4:], second[4:])


def test_attention_strides_streams_and_replay():
    c = Cached(3, 30, 2, 16, 128, 12)
    g = torch.Generator(device="cuda").manual_seed(4)
    wide = torch.randn(3, 3 * 8 * 128, generator=g, device="cuda").bfloat16()
    q = wide[:, 8 * 128:2 * 8 * 128].view(3, 8, 128)
    big = torch.zeros(3, 10, 136, device="cuda", dtype=torch.bfloat16)
    b = seqops.Batch([2, 0, 1], [1, 1, 1], [100, 470, 0])
    check_attend(c, q, b, out=big[:, 1:9, 3:131], scale=0.1)
    assert (big[:, 0] == 0).all() and (big[:, 9] == 0).all() and (big[:, :, :3] == 0).all()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        o = c.cache.attend(q, c.dtable, b, scale=0.1)
    side.synchronize()
    assert torch.equal(o, big[:, 1:9, 3:131])
    # a decode step captured once: positions, rows and queries are data
    k, v, q = torch.zeros(3, 2, 128, device="cuda"), torch.zeros(3, 2, 128, device="cuda"), torch.zeros(3, 8, 128, device="cuda")
    b = seqops.Batch([0, 1, 2], [1, 1, 1], [50, 60, 470])
    b.data[3] = 1  # (the split was planned for 471 keys)

    def step():
        c.cache.store(k, v, c.dtable, b)
        return c.cache.attend(q, c.dtable, b, scale=0.1)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = step()
        o2 = c.cache.attend(q, c.dtable, b, scale=0.1)
    for pos in ([15, 16, 17], [16, 17, 18], [400, 3, 471]):
        k.copy_(torch.randn(k.shape, generator=g, device="cuda")), v.copy_(torch.randn(v.shape, generator=g, device="cuda")), q.copy_(torch.randn(q.shape, generator=g, device="cuda"))
        b.data[3] = torch.tensor(pos, dtype=torch.int32)
        graph.replay()
        got = o.clone()
        assert torch.equal(o, o2)
        values, scales = c.values()
        ref, tol = plain.attend(as64(q), values[0], scales[0], values[1], scales[1], c.table, portions_of(b), 16, 0.1, split=True)
        assert (np.abs(as64(got) - ref) <= tol + plain.F32 * np.abs(ref)).all()


def test_store_and_attention_as_they_are_used():
    """Prompt, decoded tokens, a fork by page copies, decoding on in both: against attention over the rows as they were, within what 8 bits lose."""
    heads, dim, page = 2, 64, 8
    cache = seqops.Cache8.empty(40, heads, page, dim)
    pool = seqops.UnitPool(cache.buffers())
    table = torch.zeros(2, 16, dtype=torch.int32, device="cuda")
    table[0, :8] = torch.arange(8)
    g = torch.Generator(device="cuda").manual_seed(6)
    rows = torch.randn(2, 60, 3, heads, dim, generator=g, device="cuda")
    rows[1, :29] = rows[0, :29]  # the second sequence continues the first's 29 tokens
    cache.store(rows[0, :20, 0], rows[0, :20, 1], table, seqops.Batch([0], [20], [0]))
    for p in range(20, 29):
        cache.store(rows[0, p:p + 1, 0], rows[0, p:p + 1, 1], table, seqops.Batch([0], [1], [p]))
    table[1, :3] = table[0, :3]            # full pages are shared
    table[1, 3:8] = torch.arange(20, 25)   # the one in part filled is copied
    pool.copy(pages=([3], [20]))
    for p in range(29, 60):
        b = seqops.Batch([0, 1], [1, 1], [p, p])
        cache.store(rows[:, p, 0], rows[:, p, 1], table, b)
        o = cache.attend(rows[:, p, 2], table, b, scale=dim ** -0.5)
        for s in range(2):
            k, v = as64(rows[s, :p + 1, 0]), as64(rows[s, :p + 1, 1])
            for h in range(heads):
                x = k[:, h] @ as64(rows[s, p, 2, h]) * dim ** -0.5
                w = np.exp(x - x.max())
                want = w @ v[:, h] / w.sum()
                # a code is off by 2^-4 of its value at most: scores by 2^-4 sum |q k|, values by 2^-4, typically a quarter of the random sums of these
                ds = 2.0 ** -4 * np.sqrt(((k[:, h] * as64(rows[s, p, 2, h])) ** 2).sum(1).max()) * dim ** -0.5
                assert np.abs(as64(o[s, h]) - want).max() <= 4 * (2.0 ** -4 + ds) * np.abs(v[:, h]).max()


def check_rows_beside(c, q, odd, batch, opt, heads, near=None):
    """Attention of all of q, then the rows that are not odd against the definition, which works on each by itself: their reference and their bound come from queries without the odd
    ones.  heads: the key heads looked at."""
    o = c.cache.attend(q, c.dtable, batch, **opt)
    group = q.shape[1] // c.heads
    clean = q.masked_fill(odd[:, :, None], 0.0)
    values, scales = c.values()
    for h in heads:
        mine = slice(h * group, (h + 1) * group)
        kw = {k: (as64(v)[mine] if isinstance(v, torch.Tensor) else v) for k, v in opt.items()}
        ref, tol = plain.attend(as64(clean[:, mine]), values[0][:, h:h + 1], scales[0][:, h:h + 1], values[1][:, h:h + 1], scales[1][:, h:h + 1], c.table, portions_of(batch), c.page,
                                split=q.dtype == torch.float32, **kw)
        got, there = as64(o[:, mine]), ~odd[:, mine].cpu().numpy()
        if near is not None:
            there &= near(h)[:, None]
        bound = tol + plain.half_step(o.dtype) * (np.abs(ref) + tol) + (2.0 ** -24 if o.dtype == torch.float16 else 0.0)
        assert there.any() and np.isfinite(got[there]).all() and (np.abs(got - ref)[there] <= bound[there]).all(), (h, np.abs(got - ref)[there].max())
    return o


ODD = {"inf": math.inf, "nan": math.nan, "2^40": 2.0 ** 40, "2^-30 2^100": 2.0 ** 100}


@pytest.mark.parametrize("odd", list(ODD))
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("dim,opt", [(128, {}), (64, {}), (256, dict(softcap=4.0)), (80, dict(slopes=True))])
def test_odd_queries_beside_ordinary_ones(dim, opt, dtype, odd):
    """One element of one head's query is infinite, no number, or far above what the others hold: the other heads and tokens keep their values (tiles of eight and of sixteen rows)."""
    if dtype == "fp16" and "2^" in odd:
        pytest.skip("not a value of the type")
    g = torch.Generator(device="cuda").manual_seed(dim)
    for seqs, tokens in ((3, 1), (30, 5)):
        c = Cached(seqs, 6, 2, 16, dim, dim + seqs)
        q = torch.randn(seqs * tokens, 12, dim, generator=g, device="cuda").to(DT[dtype])
        if "2^-30" in odd:
            q = q * 2.0 ** -30
        at = torch.zeros(q.shape[:2], dtype=torch.bool, device="cuda")
        for token, head in ((0, 7), (seqs * tokens - 1, 11)):
            q[token, head, 5], at[token, head] = ODD[odd] * (-1) ** token, True
        kw = dict(scale=0.2 * (2.0 ** 30 if "2^-30" in odd else 1.0), **opt)
        if "slopes" in opt:
            kw["slopes"] = torch.rand(12, generator=g, device="cuda") * 0.1
        check_rows_beside(c, q, at, seqops.Batch(range(seqs), [tokens] * seqs, [60 + i % 30 for i in range(seqs)]), kw, [1])


@pytest.mark.parametrize("odd", list(ODD))
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("dim", [64, 128])
def test_odd_queries_in_a_prompt(dim, dtype, odd):
    """The same in the tensor cores' tiles of 128: a later token's query reaches neither earlier tokens nor other heads."""
    if dtype == "fp16" and "2^" in odd:
        pytest.skip("not a value of the type")
    c = Cached(5, 21, 16, 16, dim, dim)
    g = torch.Generator(device="cuda").manual_seed(dim + 1)
    counts, before = [100, 37, 1, 0, 77], [0, 50, 300, 5, 130]
    q = torch.randn(sum(counts), 48, dim, generator=g, device="cuda").to(DT[dtype])
    if "2^-30" in odd:
        q = q * 2.0 ** -30
    at = torch.zeros(q.shape[:2], dtype=torch.bool, device="cuda")
    for token, head in ((60, 7), (99, 6), (120, 47), (214, 8)):
        q[token, head, 3], at[token, head] = ODD[odd], True
    check_rows_beside(c, q, at, seqops.Batch([1, 2, 4, 0, 3], counts, before), dict(scale=0.7 * dim ** -0.5 * (2.0 ** 30 if "2^-30" in odd else 1.0)), [2, 15])


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("far", [14, 18, 40, 110])
def test_values_that_a_prompts_rows_do_not_see(dim, far, dtype):
    """Pages whose value scale is 2^far times the others', ahead of some rows and behind the window of others that share their tiles of keys: those rows' results know nothing of it."""
    c = Cached(5, 21, 16, 16, dim, dim + far)
    for slot in (0, 1):
        c.scales[1, c.table[slot, 3]] *= 2.0 ** far
    g = torch.Generator(device="cuda").manual_seed(far)
    counts, before = [100, 100, 1, 1, 77], [0, 0, 300, 5, 130]
    q = torch.randn(sum(counts), 48, dim, generator=g, device="cuda").to(DT[dtype])
    none = torch.zeros(q.shape[:2], dtype=torch.bool, device="cuda")
    batch = seqops.Batch([0, 1, 2, 3, 4], counts, before)
    check_rows_beside(c, q, none, batch, dict(scale=dim ** -0.5), [0, 7], near=lambda h: np.arange(sum(counts)) % 100 < 48)
    pos = np.concatenate([b + np.arange(n) for n, b in zip(counts, before)])
    check_rows_beside(c, q, none, batch, dict(scale=dim ** -0.5, window=10), [0, 7], near=lambda h: (pos < 48) | (pos >= 64 + 9))
    check_rows_beside(c, q, none, batch, dict(scale=dim ** -0.5), [0, 7])  # and those that see it, within what their own bound says


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("far", [17, 60])
def test_small_values_that_take_a_prompts_weights(dim, far, dtype):
    """Keys with small values score far above keys with large ones: the result is the small values' mean, as if the others were not there (their weights are e^-100 2^far at most)."""
    c = Cached(5, 21, 16, 16, dim, dim + far)
    g = torch.Generator(device="cuda").manual_seed(far)
    counts, before = [100, 37, 1, 0, 77], [0, 50, 300, 5, 130]
    batch = seqops.Batch([1, 2, 4, 0, 3], counts, before)
    q = (1.0 + 0.05 * torch.rand(sum(counts), 48, dim, generator=g, device="cuda")).to(DT[dtype])
    c.codes[0], c.scales[0] = 0x38, 1.0  # keys of ones (1.0 is code 0x38)
    seen = c.table.copy()
    for slot in range(5):
        for block in range(1, 21, 3):
            p = c.table[slot, block]
            c.codes[0, p], c.scales[1, p] = 0xB8, c.scales[1, p] * 2.0 ** far  # minus ones
            seen[slot, block] = -1
    o = as64(c.cache.attend(q, c.dtable, batch, scale=100.0 / dim))
    values, scales = c.values()
    for h in (0, 9):
        mine = slice(3 * h, 3 * h + 3)
        ref, tol = plain.attend(as64(q[:, mine]), *[x[:, h:h + 1] for x in (values[0], scales[0], values[1], scales[1])], seen, portions_of(batch), c.page, 100.0 / dim, split=dtype == "fp32")
        rest = 2.0 ** (far - 2 * 100 / math.log(2)) * 448.0 * 330
        bound = tol + plain.half_step(DT[dtype]) * (np.abs(ref) + tol) + rest
        assert (np.abs(o[:, mine] - ref) <= bound).all(), np.abs(o[:, mine] - ref).max()


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("seqs,tokens,before", [(2, 1, 20), (1, 1, 300), (150, 1, 300), (5, 60, 200)])
def test_sinks_that_are_infinite(seqs, tokens, before, dtype):
    """exp(-inf) = 0 adds nothing, also where a token sees nothing; exp(+inf) takes everything.  (One share, a cluster's, shares through memory, a prompt's tiles.)"""
    c = Cached(seqs, 23, 16, 16, 128, seqs)
    c.table[0] = -1
    c.dtable.copy_(torch.tensor(c.table))
    q = torch.randn(seqs * tokens, 48, 128, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2)).to(DT[dtype])
    b = seqops.Batch(range(seqs), [tokens] * seqs, [before] * seqs)
    sink = torch.zeros(48, device="cuda")
    sink[::3], sink[1::3] = -math.inf, math.inf
    got, free = c.cache.attend(q, c.dtable, b, 0.1, sink=sink), c.cache.attend(q, c.dtable, b, 0.1)
    assert (got[:tokens] == 0).all() and (got[:, 1::3] == 0).all() and (free[:tokens] == 0).all()
    # the same weights over the same denominator: a rounding each where the factor 1 is applied, and the output's own
    off = (got[:, ::3].double() - free[:, ::3].double()).abs()
    assert (off <= (2 * plain.half_step(DT[dtype]) + 4 * plain.F32) * free[:, ::3].double().abs()).all()


def test_beams_of_no_groups():
    tok, par, best = seqops.beam_select(torch.zeros(0, 3, 50, device="cuda"), torch.zeros(0, 3, device="cuda"), 4)
    assert tok.shape == par.shape == best.shape == (0, 4)


def test_tokens_of_one_beam_come_in_their_logits_order():
    """Logits whose difference is lost beside the row's maximum, or beside the beam's score, in 64 bits: n = 1, 2, ... continuations are prefixes of one order, in and across slices."""
    V = 20000
    x = torch.full((1, 3, V), -50.0, device="cuda")
    x[0, 0, 7] = 5.0
    low = torch.tensor([3, 19000, 9000, 4, 12000, 18999], device="cuda")
    x[0, 0, low] = torch.arange(1, 7, device="cuda") * 1e-20
    x[0, 1:, :8] = torch.arange(8, device="cuda") * 2.0 ** -24 - 0.25  # (fp32 holds the steps, a score of -2^40 beside them does not)
    s = torch.tensor([[-1.0, -2.0 ** 40, -2.0 ** 40]], device="cuda")
    want = [7] + low.flip(0).tolist()
    for n in range(1, 8):
        tok, par, _ = seqops.beam_select(x, s, n)
        assert tok[0].tolist() == want[:n] and (par == 0).all(), (n, tok)
    s[0, 0] = -math.inf
    for n in range(1, 17):
        tok, par, _ = seqops.beam_select(x, s, n)
        assert tok[0].tolist() == (2 * list(range(7, -1, -1)))[:n] and par[0].tolist() == (8 * [1] + 8 * [2])[:n], (n, tok, par)


@pytest.mark.parametrize("vocab", [97, 32000, 128256])
def test_beams_that_lie_just_apart(vocab):
    """Two beams with the same logits in different places, their scores further apart than the two log-sums' bounds: every candidate of the higher beam comes before the other's same one."""
    g = torch.Generator(device="cuda").manual_seed(vocab)
    row = torch.randn(vocab, generator=g, device="cuda") * 3
    row[:8] = 20.0 + torch.arange(8, device="cuda")
    for seed in range(8):
        g.manual_seed(seed)
        place = [torch.randperm(vocab, generator=g, device="cuda") for _ in range(2)]
        x = torch.stack([row[p] for p in place])[None]
        apart = 2.02 * (2.0 ** -22 + (25 + math.ceil(vocab / 4096)) * 2.0 ** -24)  # what is documented, and a little
        for high in (0, 1):
            s = torch.zeros(1, 2, device="cuda")
            s[0, 1 - high] = -apart
            tok, par, _ = seqops.beam_select(x, s, 16)
            assert par[0].tolist() == [high, 1 - high] * 8
            assert [int(place[p][t]) for t, p in zip(tok[0].tolist(), par[0].tolist())] == [i for i in range(7, -1, -1) for _ in range(2)]


def test_pages_of_an_8_bit_cache_are_copied_whole():
    """Their second axis is heads, not tokens: a copy of a page's first rows is refused, alone and beside a wide cache, and nothing is copied then."""
    c = Cached(1, 6, 3, 8, 32, 5)
    wide = torch.randn(8, 8, 4, device="cuda")
    for pool in (seqops.UnitPool(c.cache.buffers()), seqops.UnitPool([wide] + c.cache.buffers())):
        before = [x.clone() for x in (wide, c.codes, c.scales)]
        with pytest.raises(ValueError, match="rows"):
            pool.copy(pages=([0], [1], [3]))
        assert all(torch.equal(x, y) for x, y in zip(before, (wide, c.codes, c.scales)))
        pool.copy(pages=([0, 2], [1, 3]))
        for t in (*c.codes, *c.scales):
            assert torch.equal(t[0], t[1]) and torch.equal(t[2], t[3])
    assert torch.equal(wide[0], wide[1]) and torch.equal(wide[2], wide[3])
    assert all(x.shape[0] == 0 for x in seqops.Cache8.empty(0, 3, 8, 32).buffers())


def test_whole_numbers_that_pass_32_bits_are_refused():
    c = Cached(1, 4, 1, 16, 64, 5)
    q, b = torch.zeros(1, 2, 64, device="cuda"), seqops.Batch([0], [1], [30])
    for name in ("window", "keep_first", "chunk"):
        for v in (2 ** 32 + 5, -1, 1.5):
            with pytest.raises(ValueError, match=name):
                c.cache.attend(q, c.dtable, b, 0.1, **{name: v})
    x, s = torch.zeros(1, 2, 8, device="cuda"), torch.zeros(1, 2, device="cuda")
    for n in (2 ** 32 + 3, 0, 65, -1, 2.5):
        for groups in (1, 0):
            with pytest.raises(ValueError, match="n"):
                seqops.beam_select(x[:groups], s[:groups], n)
    with pytest.raises(ValueError, match="vocabulary"):
        seqops.beam_select(torch.empty(1, 1, 2 ** 32 + 5, dtype=torch.bfloat16, device="cuda"), s[:, :1].contiguous(), 2)


def test_8_bit_pages_of_other_shapes_are_refused_as_a_destination():
    a, b = seqops.Cache8.empty(4, 2, 16, 64), seqops.Cache8.empty(4, 2, 64, 16)  # as many bytes a page
    with pytest.raises(ValueError, match="shape"):
        seqops.UnitPool(a.buffers(), into=seqops.UnitPool(b.buffers()))

"""Branches, resized caches, beams and 8-bit caches of the layer-list runtime, over every family's kinds of cache and state."""
import math
import os
import sys

import numpy as np
import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import bovinex_plain  # noqa: E402
import seqops_plain  # noqa: E402

pytestmark = pytest.mark.gpu

from calm_b200 import bovinex, fasulix, seqbench, seqlib, serving, sopepel, tabisun, vimulorn, zazilix  # noqa: E402

SIZE = dict(width=64, ff=64, blocks=2, heads=4, dim=16, kv_heads=2, kv_rank=32, q_rank=24, window=24, vocab=97)
FAMILIES = {"vimulorn": vimulorn, "bovinex": bovinex, "zazilix": zazilix, "sopepel": sopepel, "fasulix": fasulix, "tabisun": tabisun}


def family(name):
    cfg = getattr(seqbench, name + "_config")(SIZE)
    return FAMILIES[name], cfg, FAMILIES[name].random_tensors(cfg, 3)


def build(name, dtype="float32", **kw):
    mod, cfg, t = family(name)
    return mod.from_tensors(cfg, t, dtype, **{"max_tokens": 600, "max_seqs": 8, "page": 4, **kw})


def text(n, seed):
    return [int(x) for x in np.random.default_rng(seed).integers(0, SIZE["vocab"], n)]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name", list(FAMILIES))
def test_branches_go_on_as_sequences_of_their_own(name, dtype):
    """A prompt, three branches of it, different tokens in each: bit for bit what three sequences give that ran the prompt themselves."""
    for P in (1, 7, 8, 33):
        with build(name, dtype) as a, build(name, dtype) as b:
            prompt = text(P, P)
            s = a.open()
            a.step([s], [prompt], [P - 1])
            sa = [s] + a.fork(s, 2)
            sb = [b.open() for _ in range(3)]
            for x in sb:
                b.step([x], [prompt], [P - 1])
            for i in range(6):
                t = [[x] for x in text(3, 10 * P + i)]
                assert np.array_equal(a.step(sa, t, [0, 1, 2]), b.step(sb, t, [0, 1, 2])), (P, i)
            # two of them end, one goes on three times
            sa = a.branch(sa, [1, 1, 1])
            for i in range(5):
                t = [[x] for x in text(3, 20 * P + i)]
                got = a.step(sa, t, [0, 1, 2])
                assert np.array_equal(got[0], b.step([sb[1], sb[0], sb[2]], t, [0, 1, 2])[0])
            assert [a.length(x) for x in sa] == [P + 11] * 3
            for x in sa:
                a.close_seq(x)
            assert a.free_pages() == 150 + 8


@pytest.mark.parametrize("cache_bits", [32, 8])
@pytest.mark.parametrize("name", ["bovinex", "zazilix", "fasulix", "tabisun"])
def test_a_walk_of_branches_ends_and_resizes(name, cache_bits):
    """Random branches, ends, steps and resizes; a twin without any of them runs every surviving text in the same portions."""
    if cache_bits == 8 and name == "fasulix":
        with pytest.raises(ValueError, match="8 bits"):
            build(name, cache_bits=8)
        return
    rng = np.random.default_rng(1)
    with build(name, cache_bits=cache_bits) as m:
        live = {}  # slot -> portions fed
        for step in range(60):
            what = rng.integers(0, 6)
            if not live or (what == 0 and len(live) < 8):
                s = m.open()
                live[s] = [text(int(rng.integers(1, 12)), step)]
                m.step([s], live[s], [])
            elif what == 1 and len(live) > 1:
                s = int(rng.choice(list(live)))
                m.close_seq(s)
                del live[s]
            elif what in (2, 3):
                src = [int(x) for x in rng.permutation(list(live))[:int(rng.integers(1, len(live) + 1))]]
                room = 8 - len(live) + len(src)
                parents = [int(x) for x in rng.integers(0, len(src), int(rng.integers(1, room + 1)))]
                out = m.branch(src, parents)
                kept = {o: live[src[p]] for o, p in zip(out, parents)}
                assert len(set(out)) == len(out) and all(src[p] in out for p in parents)
                for s in src:
                    del live[s]
                assert not set(live) & set(out)
                live.update({o: list(t) for o, t in kept.items()})
            elif what == 4 and step % 3 == 0:
                held = sum(-(-sum(map(len, t)) // 4) for t in live.values())
                m.resize(int(rng.integers(4 * held + 40, 900)))
            else:
                s = [int(x) for x in rng.permutation(list(live))[:3]]
                t = [text(int(rng.integers(1, 6)), 100 * step + i) for i in range(len(s))]
                m.step(s, t, [])
                for x, y in zip(s, t):
                    live[x] = live[x] + [y]
            assert all(m.length(s) == sum(map(len, t)) for s, t in live.items())
        with build(name, cache_bits=cache_bits) as twin:
            for s, portions in live.items():
                x = twin.open()
                for p in portions:
                    twin.step([x], [p], [])
                got, want = m.step([s], [[5]], [0]), twin.step([x], [[5]], [0])
                assert np.abs(got - want).max() <= 2e-5 * np.abs(want).max(), (s, np.abs(got - want).max())
                twin.close_seq(x)
        for s in live:
            m.close_seq(s)
        assert m.free_pages() == -(-m.desc.max_tokens // 4) + 8


def test_refused_branches_and_sizes_change_nothing():
    with build("bovinex", max_tokens=40, max_seqs=4) as m:
        a, b = m.open(), m.open()
        m.step([a, b], [text(30, 1), text(13, 2)], [])
        pages = m.free_pages()  # 14 in all, 8 + 4 held
        assert pages == 2
        for slots, parents in (([a, a], [0, 1]), ([3], [0]), ([9], [0]), ([-1], [0]), ([a], [1]), ([a], [-1]), ([], [])):
            with pytest.raises(seqlib.SeqError, match="bad branch"):
                m.branch(slots, parents)
        with pytest.raises(seqlib.SeqError, match="slot"):
            m.branch([a, b], [0, 0, 0, 1, 1])
        for n in (0, -5):
            with pytest.raises(seqlib.SeqError, match="positive"):
                m.resize(n)
        m.open()
        with pytest.raises(seqlib.SeqError, match="slot"):
            m.branch([a], [0, 0, 0])
        m.close_seq(2)
        m.step([b], [text(7, 3)], [])  # 20 tokens: full pages
        assert m.free_pages() == 1
        assert m.branch([a, b], [0, 0, 1, 1]) == [a, 2, b, 3]  # a's page in part filled takes the last page, b's pages are shared
        assert m.free_pages() == 0 and [m.length(x) for x in (a, 2, b, 3)] == [30, 30, 20, 20]
        m.branch([2], [])
        with pytest.raises(seqlib.SeqError, match="pool"):
            m.step([b, 3], [[1], [2]], [])
        with pytest.raises(seqlib.SeqError, match="tokens"):
            m.resize(4)
        with build("bovinex", max_tokens=40, max_seqs=4) as twin:
            x = twin.open()
            twin.step([x], [text(30, 1)], [])
            assert np.array_equal(m.step([a], [[7]], [0]), twin.step([x], [[7]], [0]))
        assert m.branch([a, b, 3], []) == [] and m.free_pages() == 14


def test_more_branches_than_slots_and_pools_past_an_operators_range_are_refused():
    with build("bovinex", max_tokens=40, max_seqs=4, cache_bits=8) as m:
        a = m.open()
        m.step([a], [text(20, 1)], [])
        with pytest.raises(seqlib.SeqError, match="slot"):
            m.branch([a], [0] * 1000)
        with pytest.raises(seqlib.SeqError, match="bad branch"):
            m.branch([a] * 1000, [0])
        with pytest.raises(seqlib.SeqError):  # more rows than the operators over 8-bit caches take
            m.resize(2 ** 31 - 200)
        with build("bovinex", max_tokens=40, max_seqs=4, cache_bits=8) as twin:
            x = twin.open()
            twin.step([x], [text(20, 1)], [])
            assert np.array_equal(m.step([a], [[7]], [0]), twin.step([x], [[7]], [0]))


def test_a_pool_made_smaller_gives_memory_back():
    with build("bovinex", max_tokens=400000, page=16) as m:
        s = m.open()
        m.step([s], [text(50, 1)], [])
        before = torch.cuda.mem_get_info()[0]
        m.resize(1000)
        assert torch.cuda.mem_get_info()[0] - before > 0.9 * 4 * 399000 * 2 * SIZE["kv_heads"] * SIZE["dim"] * 2  # two layers' keys and values
        with pytest.raises(seqlib.SeqError, match="memory"):
            m.resize(2 ** 30)
        m.step([s], [text(900, 2)], [])
        assert m.length(s) == 950


def log_p(cfg, t, texts):
    out = bovinex_plain.forward(cfg, t, texts)[-1]
    return out - out.max() - math.log(np.exp(out - out.max()).sum())


def test_beam_search_of_a_model():
    """The scheduler on the device against a search with the plain model."""
    _, cfg, t = family("bovinex")
    t64 = {k: v.float().numpy().astype(np.float64) for k, v in t.items()}
    prompts, K, new = [text(9, 1), text(5, 2)], 3, 5
    with build("bovinex") as m:
        s = serving.Scheduler(m)
        reqs = [serving.Request(str(i), p, new, beams=K) for i, p in enumerate(prompts)]
        for r in reqs:
            s.add(r)
        out = s.run()
        for r in reqs:
            live = [(0.0, [])]
            for _ in range(new):
                cand = [(sc + lp, tx + [k]) for sc, tx in live for k, lp in enumerate(log_p(cfg, t64, r.prompt + tx))]
                live = sorted(cand, key=lambda c: -c[0])[:K]
            assert [h[1] for h in r.hyps] == [x for _, x in live] and out[r.rid] == live[0][1]
            assert np.allclose([h[0] * new for h in r.hyps], [x for x, _ in live], atol=2e-3)  # five logits, each within 2e-5 of rows whose spread is under 20
        assert m.free_pages() == 150 + 8
    # all beams at once: the best of every continuation of two tokens
    with build("bovinex") as m:
        r = serving.Request("a", prompts[0], 1, beams=8)
        s = serving.Scheduler(m)
        s.add(r)
        s.run()
        lp = log_p(cfg, t64, prompts[0])
        assert [h[1][0] for h in r.hyps] == np.argsort(-lp, kind="stable")[:8].tolist()


def test_beams_of_the_last_step():
    with build("tabisun") as m:
        s = m.open()
        m.step([s], [text(6, 1)], [1, 3, 5])
        x = m.step([s], [text(6, 2)], [0, 2, 4, 5])
        tok, par, best = m.beams(np.array([[-1.0, -2.0], [-0.5, -np.inf]], np.float32), 5)
        rt, rp, rb = seqops_plain.beam_select(x.reshape(2, 2, -1).astype(np.float64), np.array([[-1.0, -2.0], [-0.5, -np.inf]]), 5)
        assert np.array_equal(tok, rt) and np.array_equal(par, rp) and np.abs(best - rb).max() <= 1e-5
        tok, par, _ = m.beams(np.zeros((1, 1), np.float32), 3, row0=3)
        assert tok[0].tolist() == np.argsort(-x[3], kind="stable")[:3].tolist() and (par == 0).all()
        for args in ((np.zeros((1, 5), np.float32), 3), (np.zeros((1, 1), np.float32), 3, 4), (np.zeros((1, 1), np.float32), 0), (np.zeros((1, 1), np.float32), 65), (np.zeros((1, 1), np.float32), 3, -1)):
            with pytest.raises(seqlib.SeqError):
                m.beams(*args)


# ---------------------------------------------------------------- 8-bit caches

def attention8(portions, page):
    """bovinex_plain.attention_mixer over a cache in 8 bits: the text comes in portions, each stored before its queries look."""

    def mixer(h, W, mx, eps):
        T, H, G, D = h.shape[0], mx["heads"], mx["kv_heads"], mx["dim"]
        q = bovinex_plain.rms_norm(h @ W["q"].T + W["q.b"], W["q.norm"], eps, False).reshape(T, H, D)
        k = bovinex_plain.rms_norm(h @ W["k"].T + W["k.b"], W["k.norm"], eps, False).reshape(T, G, D)
        v = (h @ W["v"].T + W["v.b"]).reshape(T, G, D)
        if mx.get("rot"):
            q, k = bovinex_plain.rotate(q, np.arange(T), mx["rot"]), bovinex_plain.rotate(k, np.arange(T), mx["rot"])
        mask = mx.get("mask") or {}
        pages = -(-T // page)
        table = np.arange(pages)[None]
        codes, scales = np.zeros((2, pages, G, page, D)), np.zeros((2, pages, G))
        out, at = np.zeros((T, H, D)), 0
        for n in portions:
            for c, s, rows in ((codes[0], scales[0], k), (codes[1], scales[1], v)):
                seqops_plain.store(c, s, rows[at:at + n], table, [(0, n, 0, at)], page)
            out[at:at + n] = seqops_plain.attend(q[at:at + n], codes[0], scales[0], codes[1], scales[1], table, [(0, n, 0, at)], page, mx["scale"], mask.get("size", 0), mask.get("keep_first", 0))[0]
            at += n
        return (out.reshape(T, H * D) * bovinex_plain.sigmoid(h @ W["g"].T)) @ W["o"].T

    return mixer


@pytest.mark.parametrize("portions", [[45], [20, 1, 1, 1, 1, 1, 3, 17], [1] * 45])
@pytest.mark.parametrize("dtype,tol", [("float32", 2e-5), ("bfloat16", 8e-2)])
def test_a_model_over_an_8_bit_cache(portions, dtype, tol, monkeypatch):
    """Logits against the plain model with the same roundings.  float32: what is left is the model's own tolerance.  bfloat16: keys and values that differ by 2^-8 round to the neighbouring code
    now and then (one in 2^4 of them by a step of 2^-3), twice the mode's own tolerance."""
    _, cfg, t = family("bovinex")
    t64 = {k: v.float().numpy().astype(np.float64) for k, v in t.items()}
    toks = text(45, 8)
    monkeypatch.setattr(bovinex_plain, "attention_mixer", attention8(portions, 4))
    ref = bovinex_plain.forward(cfg, t64, toks)
    with build("bovinex", dtype, cache_bits=8) as m:
        s, rows, at = m.open(), [], 0
        for n in portions:
            rows.append(m.step([s], [toks[at:at + n]], list(range(n))))
            at += n
        d = np.concatenate(rows) - ref
    d, r = d - d.mean(-1, keepdims=True), ref - ref.mean(-1, keepdims=True)
    assert float(np.sqrt((d * d).mean(-1)).max() / np.sqrt((r * r).mean())) < tol


@pytest.mark.parametrize("name", ["bovinex", "zazilix", "sopepel", "tabisun"])
def test_8_bit_caches_stay_near_the_wide_ones(name):
    """Every family that has such layers (distance slopes, an added one, blocks of positions, gates of all kinds, soft caps): prompts and decode steps within what 8 bits lose,
    and far from it nowhere.  e4m3 keeps a value within 2^-4, a quarter of that in the mean: logits of six layers within 2^-3 of their spread."""
    for dtype in ("float32", "bfloat16"):
        with build(name, dtype) as a, build(name, dtype, cache_bits=8) as b:
            sa, sb = [a.open() for _ in range(3)], [b.open() for _ in range(3)]
            prompts = [text(n, n) for n in (40, 3, 17)]
            ends = [39, 42, 59]
            pairs = [(a.step(sa, prompts, ends), b.step(sb, prompts, ends))]
            for i in range(20):
                t = [[x] for x in text(3, i)]
                pairs.append((a.step(sa, t, [0, 1, 2]), b.step(sb, t, [0, 1, 2])))
            x, y = np.concatenate([p for p, _ in pairs]), np.concatenate([q for _, q in pairs])
            d, r = y - x, x - x.mean(-1, keepdims=True)
            assert 0 < np.sqrt((d * d).mean()) <= 2.0 ** -3 * np.sqrt((r * r).mean())


def test_captured_steps_and_eager_ones_agree_over_an_8_bit_cache(monkeypatch):
    def run():
        with build("sopepel", "bfloat16", cache_bits=8, max_tokens=4000) as m:
            s = [m.open() for _ in range(2)]
            m.step(s, [text(700, 1), text(3, 2)], [])
            return np.concatenate([m.step(s, [[x] for x in text(2, i)], [0, 1]) for i in range(12)])

    first = run()
    monkeypatch.setenv("CALM_B200_SEQ_GRAPH", "0")
    assert np.array_equal(first, run())


def test_the_command_line_searches_beams_over_an_8_bit_cache(tmp_path):
    import json
    import subprocess

    from calm_b200 import container, registry

    mod, cfg, t = family("bovinex")
    (tmp_path / "config.json").write_text(json.dumps(cfg))
    container.write_tensors(str(tmp_path / "model.safetensors"), t)
    args = ["--tokens", "5,17,3", "--tokens", "8,9,10,11", "-n", "6", "--beams", "3", "--eos", "2"]
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    for bits in ("32", "8"):
        r = subprocess.run([sys.executable, "-m", "calm_b200.serving", str(tmp_path), *args, "--cache-bits", bits], cwd=root, capture_output=True, text=True, timeout=300)
        assert r.returncode == 0, r.stderr
        got = [[int(x) for x in line.split(",")] for line in r.stdout.split()]
        with registry.load_model(str(tmp_path), max_tokens=200, max_seqs=6, cache_bits=int(bits)) as m:
            assert got == serving.generate(m, [[5, 17, 3], [8, 9, 10, 11]], 6, beams=3, eos=2) and all(1 <= len(x) <= 6 for x in got)

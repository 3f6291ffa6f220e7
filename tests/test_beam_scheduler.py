"""Beam search of the scheduler against a search written out in full, over a model that is a function of the text; mixed batches, slots and pages.  No GPU."""
import math

import numpy as np
import pytest

from calm_b200 import serving


class Desc:
    def __init__(self, page, max_seqs):
        self.page, self.max_seqs, self.max_positions = page, max_seqs, 0


class TextModel:
    """Logits of a text are drawn from it; slots, pages and branches are checked as the runtime counts them."""

    def __init__(self, vocab=13, page=4, max_seqs=12, pages=60):
        self.vocab, self.desc = vocab, Desc(page, max_seqs)
        self.texts, self.pages, self.free, self.steps, self.least = {}, {}, pages, 0, pages
        self.refs = {}

    def free_pages(self):
        return self.free

    def _take(self):
        assert self.free > 0, "page pool exhausted"
        self.free -= 1
        self.least = min(self.least, self.free)
        p = object()
        self.refs[p] = 1
        return p

    def _leave(self, slot):
        for p in self.pages.pop(slot):
            self.refs[p] -= 1
            self.free += self.refs[p] == 0
        del self.texts[slot]

    def open(self):
        slot = min(set(range(self.desc.max_seqs)) - set(self.texts))
        self.texts[slot], self.pages[slot] = [], []
        return slot

    def close_seq(self, slot):
        self._leave(slot)

    def logits_of(self, text):
        return np.random.default_rng(abs(hash(tuple(text))) % 2 ** 32).normal(0, 2, self.vocab).astype(np.float32)

    def step(self, slots, token_lists, want, fetch=True):
        assert len(set(slots)) == len(slots)
        self.steps += 1
        rows = []
        for s, t in zip(slots, token_lists):
            for x in t:
                self.texts[s].append(x)
                if len(self.texts[s]) > len(self.pages[s]) * self.desc.page:
                    self.pages[s].append(self._take())
                rows.append(self.logits_of(self.texts[s]))
        self.last = np.stack([rows[i] for i in want])
        return self.last.copy() if fetch else None

    def argmax(self, n):
        return self.last[:n].argmax(1)

    def beams(self, scores, n, row0=0):
        G, K = scores.shape
        x = self.last[row0:row0 + G * K].astype(np.float64).reshape(G, K, -1)
        d = scores[:, :, None] + x - np.log(np.exp(x).sum(-1, keepdims=True))
        order = np.argsort(-d.reshape(G, -1), kind="stable", axis=1)[:, :n]
        pad = n - order.shape[1]
        best = np.take_along_axis(d.reshape(G, -1), order, 1).astype(np.float32)
        tok, par = (order % self.vocab).astype(np.int32), (order // self.vocab).astype(np.int32)
        return tuple(np.pad(a, ((0, 0), (0, pad)), constant_values=c) for a, c in ((tok, -1), (par, -1), (best, -math.inf)))

    def branch(self, slots, parents):
        kids = [parents.count(i) for i in range(len(slots))]
        for s, k in zip(slots, kids):
            if not k:
                self._leave(s)
        out, kept = [], set()
        for p in parents:
            s = slots[p]
            if p in kept:
                s = self.open()
                self.texts[s], self.pages[s] = list(self.texts[slots[p]]), list(self.pages[slots[p]])
                for q in self.pages[s]:
                    self.refs[q] += 1
                if len(self.texts[s]) % self.desc.page:
                    self.refs[self.pages[s][-1]] -= 1
                    self.pages[s][-1] = self._take()
            kept.add(p)
            out.append(s)
        return out


def search(model, prompt, K, max_new, eos, lp):
    """Beam search written out: every continuation of every beam, sorted."""
    live, hyps = [(0.0, [])], []
    for length in range(1, max_new + 1):
        cand = []
        for b, (score, text) in enumerate(live):
            x = model.logits_of(prompt + text).astype(np.float64)
            lse = math.log(np.exp(x).sum())
            cand += [(np.float32(score) + (x[t] - lse), b, t) for t in range(model.vocab)]
        cand.sort(key=lambda c: (-c[0], c[1], c[2]))
        new = []
        for rank, (score, b, t) in enumerate(cand[:K if eos is None else 2 * K]):
            text = live[b][1] + [t]
            if len(new) == K:
                break
            if t == eos:
                if rank < K:
                    hyps.append((np.float32(score) / len(text) ** lp, text))
            else:
                new.append((np.float32(score), text))
        hyps = sorted(hyps, key=lambda h: -h[0])[:K]
        if not new:
            break
        if length == max_new:
            hyps += [(s / length ** lp, t) for s, t in new]
            break
        if len(hyps) == K and new[0][0] / length ** lp <= hyps[-1][0]:
            break
        live = new
    return sorted(hyps, key=lambda h: -h[0])[:K]


@pytest.mark.parametrize("K,max_new,eos,lp", [(2, 1, None, 1.0), (3, 6, None, 1.0), (4, 9, 2, 1.0), (2, 12, 0, 0.0), (5, 7, 5, 2.0), (2, 3, 1, -1.0)])
def test_beams_are_those_of_the_full_search(K, max_new, eos, lp):
    for seed in range(4):
        m = TextModel()
        prompt = [seed, 3, 7, 1, seed][:2 + seed]
        s = serving.Scheduler(m)
        r = serving.Request("a", prompt, max_new, eos=eos, beams=K, length_penalty=lp)
        s.add(r)
        out = s.run()
        want = search(m, prompt, K, max_new, eos, lp)
        assert out["a"] == want[0][1] and [t for _, t in r.hyps] == [t for _, t in want]
        assert np.allclose([h for h, _ in r.hyps], [h for h, _ in want], rtol=1e-6)
        assert not m.texts and m.free == 60


def test_requests_of_all_kinds_in_one_batch():
    m = TextModel(max_seqs=9, pages=40)
    s = serving.Scheduler(m)
    asked = [("g0", 1, 5, None), ("b3", 3, 6, None), ("c3", 3, 6, None), ("b2", 2, 4, 2), ("g1", 1, 3, 4), ("b4", 4, 5, 1), ("d4", 4, 8, None)]
    for i, (rid, K, n, eos) in enumerate(asked):
        s.add(serving.Request(rid, [i, 2, 9][:1 + i % 3], n, eos=eos, beams=K))
    out = s.run()
    assert set(out) == {a[0] for a in asked} and not m.texts and m.free == 40
    for i, (rid, K, n, eos) in enumerate(asked):
        prompt, text = [i, 2, 9][:1 + i % 3], []
        if K == 1:
            while len(text) < n and (not text or text[-1] != eos):
                text.append(int(m.logits_of(prompt + text).argmax()))
            assert out[rid] == text
        else:
            assert out[rid] == search(m, prompt, K, n, eos, 1.0)[0][1]


def test_pages_asked_for_are_enough():
    """The pages that admission counts cover what beams hold at worst: a pool of exactly that size never runs dry."""
    for P, n, K, page in ((7, 9, 4, 4), (8, 8, 3, 4), (1, 13, 5, 2), (16, 1, 2, 8)):
        m = TextModel(page=page, max_seqs=K, pages=1000)
        s = serving.Scheduler(m)
        r = serving.Request("a", list(range(P)), n, beams=K)
        m.free = m.least = s._pages_for(r)
        s.add(r)
        s.run()
        assert m.free == s._pages_for(r)


def test_refused_requests():
    s = serving.Scheduler(TextModel(max_seqs=4))
    for kw in (dict(beams=0), dict(beams=65), dict(beams=33, eos=1), dict(beams=2, temperature=0.5), dict(beams=5)):
        with pytest.raises(ValueError):
            s.add(serving.Request("a", [1], 3, **kw))


def test_sampled_batches_hand_the_steps_own_logits_on():
    """Without beams every row is a request's: the array goes to the sampler as the step gave it, not a copy of a vocabulary a request; beside beams the rows are the requests'."""

    class Sampled(serving.Scheduler):
        def _sample(self, reqs, n, logits):
            seen.append((len(reqs), n, logits is m.given[-1] if logits is not None else None, None if logits is None else np.array(logits)))
            return [int(r.argmax()) for r in logits]

    class Keeping(TextModel):
        given = None

        def step(self, *a, **kw):
            out = super().step(*a, **kw)
            self.given = (self.given or []) + [out]
            return out

    m, seen = Keeping(), []
    s = Sampled(m)
    for i in range(3):
        s.add(serving.Request(str(i), [i, 4], 3, temperature=0.7))
    s.run()
    assert len(seen) == 3 and all(x[:3] == (3, 3, True) for x in seen)
    m, seen = Keeping(), []
    s = Sampled(m)
    s.add(serving.Request("b", [5], 3, beams=2))
    s.add(serving.Request("a", [7, 4], 3, temperature=0.7))
    s.run()
    assert [x[:3] for x in seen] == [(1, 1, False)] * 3
    assert np.array_equal(seen[0][3][0], m.logits_of([7, 4])) and np.array_equal(seen[1][3][0], m.given[1][-1])


def test_the_command_line_refuses_a_number_of_beams_that_is_none(capsys):
    """Before a model of no tokens and no slots is prepared, which ends the process."""
    for beams in ("0", "-2"):
        with pytest.raises(SystemExit) as e:
            serving.main(["nowhere", "--tokens", "1,2", "--beams", beams])
        assert e.value.code == 2 and "--beams" in capsys.readouterr().err

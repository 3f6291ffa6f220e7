"""Serving loop of the layer-list runtime: a scheduler that forms batches, steps them through the model's step function,
samples, and gives finished sequences' pages and slots back.

Batching policy (static batches): waiting requests are admitted together, as many as slots and pages allow; the batch's
prompts run as one packed step, then the batch decodes one token per live request per step; requests leave as they
finish and the next batch is admitted when the batch is empty.  Sampling: greedy on the device; temperature / min-p
through the library's device sampler (the calm sampler kernels, lib.sample_logits) with its xorshift* generator.

Beam search (Request.beams > 1): the prompt runs once, then a step feeds one token for each live beam; the best continuations of all beams are picked on the
device (model.beams) and the beams' sequences branch (model.branch: full cache pages are shared, one launch copies what is still written).  A continuation that
ends in `eos` and is among the first `beams` becomes a hypothesis, scored by its log-probability over (its tokens)^length_penalty; a request leaves when its beams
have reached max_new tokens, or when it has `beams` hypotheses and no live beam scores above the least of them.

Command line:  python -m calm_b200.serving MODEL_DIR --tokens 5,17,3 [--tokens ...] -n 32 [-t 0.8 --minp 0.05 --seed 1] [--beams 4 --eos 2 --length-penalty 1.0] [--cache-bits 8]"""
from __future__ import annotations

import argparse
import sys
from dataclasses import dataclass, field
from typing import Dict, List, Optional, Tuple

import numpy as np


@dataclass
class Request:
    rid: str
    prompt: List[int]
    max_new: int
    temperature: float = 0.0
    minp: float = 0.05
    eos: Optional[int] = None
    out: List[int] = field(default_factory=list)
    slot: int = -1
    done: bool = False
    beams: int = 1
    length_penalty: float = 1.0
    hyps: List[Tuple[float, List[int]]] = field(default_factory=list)  # beam search: finished continuations, best first
    live: List[Tuple[int, float, List[int]]] = field(default_factory=list)  # (slot, log-probability, tokens) of each live beam

    def picks(self) -> int:
        """Continuations asked for in a step: any number of the first `beams` may end, and `beams` are to go on."""
        return self.beams if self.eos is None else 2 * self.beams


class Scheduler:
    def __init__(self, model, max_batch: int = 32, seed: int = 1):
        self.model, self.max_batch = model, max_batch
        self.waiting: List[Request] = []
        self.batch: List[Request] = []
        self.rng_state = seed or 1
        self.page = model.desc.page

    def add(self, req: Request) -> None:
        if not req.prompt:
            raise ValueError("empty prompt")
        limit = int(getattr(getattr(self.model, "desc", None), "max_positions", 0) or 0)
        if limit and len(req.prompt) + req.max_new - 1 > limit:  # the last generated token is never fed back
            raise ValueError(f"request {req.rid}: {len(req.prompt)} prompt tokens + {req.max_new} new ones pass the model's {limit} positions")
        if req.beams < 1 or (req.beams > 1 and (req.temperature != 0.0 or req.picks() > 64)):
            raise ValueError(f"request {req.rid}: 1 to 64 beams (32 with an end token), without a temperature")
        if req.beams > self._slots():
            raise ValueError(f"request {req.rid}: {req.beams} beams, the model has {self._slots()} sequence slots")
        self.waiting.append(req)

    def _slots(self) -> int:
        return int(getattr(getattr(self.model, "desc", None), "max_seqs", 0) or 1 << 30)

    def _pages_for(self, r: Request) -> int:
        total, shared = -(-(len(r.prompt) + r.max_new) // self.page), len(r.prompt) // self.page if r.beams > 1 else 0
        return shared + r.beams * (total - shared)

    def _admit(self) -> None:
        budget, slots = self.model.free_pages(), self._slots()
        while self.waiting and len(self.batch) < self.max_batch and self.waiting[0].beams <= slots:
            need = self._pages_for(self.waiting[0])
            if need > budget:
                if not self.batch:
                    raise RuntimeError(f"request {self.waiting[0].rid} needs {need} pages, the pool has {budget}")
                break
            r = self.waiting.pop(0)
            r.slot = self.model.open()
            budget, slots = budget - need, slots - r.beams
            if r.beams > 1:
                r.live = [(r.slot, 0.0, [])]
            self.batch.append(r)

    def _sample(self, reqs: List[Request], n: int, logits: Optional[np.ndarray]) -> List[int]:
        if logits is None:
            return [int(t) for t in self.model.argmax(n)]
        from . import build as cbuild
        from . import lib

        cbuild.build(target="engine")  # the device sampler lives in the calm engine's library: built on first use
        out = []
        for r, row in zip(reqs, logits):
            tok, self.rng_state = lib.sample_logits(row, r.temperature, r.minp, self.rng_state)
            out.append(int(tok))
        return out

    def _advance(self, live: List[Request]) -> None:
        """One step: the prompt of a request that has not started, the last token of every sequence of the others."""
        rows, slots, token_lists, ends, at = [], [], [], [], 0  # rows: (first row, how many) of each request's logits
        for r in live:
            seqs = [(b[0], b[2]) for b in r.live] if r.beams > 1 else [(r.slot, r.out)]
            rows.append((len(slots), len(seqs)))
            for slot, text in seqs:
                t = [text[-1]] if text else r.prompt
                at += len(t)
                slots.append(slot), token_lists.append(t), ends.append(at - 1)
        single, beams = [i for i, r in enumerate(live) if r.beams == 1], [i for i, r in enumerate(live) if r.beams > 1]
        greedy = all(live[i].temperature == 0.0 for i in single)
        logits = self.model.step(slots, token_lists, ends, fetch=not greedy)
        if single:
            took = [rows[i][0] for i in single]
            if logits is None:
                every = self._sample([], len(slots), None)
                toks = [every[k] for k in took]
            else:
                toks = self._sample([live[i] for i in single], len(took), logits[took] if beams else logits)  # (a choice of rows is a copy of them)
            for i, tok in zip(single, toks):
                r = live[i]
                r.out.append(tok)
                if len(r.out) >= r.max_new or (r.eos is not None and tok == r.eos):
                    r.done = True
                    self.model.close_seq(r.slot)
        if beams:
            self._branch([live[i] for i in beams], [rows[i] for i in beams])

    def _branch(self, reqs: List[Request], rows: List[Tuple[int, int]]) -> None:
        """Picks the continuations of every request's beams and lets their sequences branch, all in one go."""
        picked, i = [], 0
        while i < len(reqs):  # requests side by side with as many beams and picks: one call
            j, n = i, reqs[i].picks()
            while j < len(reqs) and rows[j] == (rows[i][0] + (j - i) * rows[i][1], rows[i][1]) and reqs[j].picks() == n:
                j += 1
            scores = np.array([[b[1] for b in r.live] for r in reqs[i:j]], np.float32)
            tok, par, best = self.model.beams(scores, n, rows[i][0])
            picked += [list(zip(tok[k].tolist(), par[k].tolist(), best[k].tolist())) for k in range(j - i)]
            i = j
        slots, parents, grown = [], [], []
        for r, picks in zip(reqs, picked):
            new = []
            for rank, (tok, par, score) in enumerate(picks):
                if tok < 0 or len(new) == r.beams:
                    break
                text = r.live[par][2] + [tok]
                if r.eos is not None and tok == r.eos:
                    if rank < r.beams:
                        self._finish(r, score, text)
                else:
                    new.append((par, score, text))
            length = len(r.live[0][2]) + 1
            if new and length >= r.max_new:
                for _, score, text in new:
                    self._finish(r, score, text)
                new = []
            elif new and len(r.hyps) == r.beams and new[0][1] / length ** r.length_penalty <= r.hyps[-1][0]:
                new = []
            base = len(slots)
            slots += [b[0] for b in r.live]
            parents += [base + par for par, _, _ in new]
            grown.append(new)
        took = self.model.branch(slots, parents)  # sequences without a continuation are closed
        for r, new in zip(reqs, grown):
            r.live = [(slot, score, text) for slot, (_, score, text) in zip(took, new)]
            took = took[len(new):]
            if not new:
                r.done, r.out = True, r.hyps[0][1] if r.hyps else []

    @staticmethod
    def _finish(r: Request, score: float, text: List[int]) -> None:
        r.hyps.append((score / len(text) ** r.length_penalty, text))
        r.hyps.sort(key=lambda h: -h[0])
        del r.hyps[r.beams:]

    def run(self) -> Dict[str, List[int]]:
        """Serve everything that was added; returns rid -> generated tokens."""
        finished: Dict[str, List[int]] = {}
        while self.waiting or self.batch:
            if not self.batch:
                self._admit()
            self._advance(self.batch)
            for r in self.batch:
                if r.done:
                    finished[r.rid] = r.out
            self.batch = [r for r in self.batch if not r.done]
        return finished


def generate(model, prompts: List[List[int]], max_new: int, temperature: float = 0.0, minp: float = 0.05, seed: int = 1, max_batch: int = 32,
             beams: int = 1, eos: Optional[int] = None, length_penalty: float = 1.0):
    s = Scheduler(model, max_batch=max_batch, seed=seed)
    for i, p in enumerate(prompts):
        s.add(Request(str(i), list(p), max_new, temperature, minp, eos, beams=beams, length_penalty=length_penalty))
    done = s.run()
    return [done[str(i)] for i in range(len(prompts))]


def main(argv=None) -> int:
    ap = argparse.ArgumentParser(description="generate token ids with a layer-list model")
    ap.add_argument("model")
    ap.add_argument("--tokens", action="append", required=True, help="a prompt as comma-separated token ids (repeatable)")
    ap.add_argument("-n", type=int, default=32, help="tokens to generate per prompt")
    ap.add_argument("-t", "--temperature", type=float, default=0.0)
    ap.add_argument("--minp", type=float, default=0.05)
    ap.add_argument("--seed", type=int, default=1)
    ap.add_argument("--dtype", default="bfloat16", choices=["bfloat16", "float32"])
    ap.add_argument("--beams", type=int, default=1, help="beam search with this many beams")
    ap.add_argument("--eos", type=int, default=None, help="token that ends a continuation")
    ap.add_argument("--length-penalty", type=float, default=1.0, help="exponent of a hypothesis's length in its score")
    ap.add_argument("--cache-bits", type=int, default=32, choices=[8, 32], help="8: grouped-query layers cache keys and values in 8 bits")
    a = ap.parse_args(argv)
    if a.beams < 1:
        ap.error("--beams must be at least 1")
    from . import registry

    prompts = [[int(x) for x in p.split(",")] for p in a.tokens]
    total = a.beams * sum(len(p) + a.n for p in prompts)
    more = {"cache_bits": a.cache_bits} if a.cache_bits != 32 else {}
    with registry.load_model(a.model, dtype=a.dtype, max_tokens=total, max_seqs=a.beams * len(prompts), **more) as model:
        for p, out in zip(prompts, generate(model, prompts, a.n, a.temperature, a.minp, a.seed, len(prompts), a.beams, a.eos, a.length_penalty)):
            print(",".join(map(str, out)))
    return 0


if __name__ == "__main__":
    sys.exit(main())

"""Generation with drafted tokens (crates/glassbox-core/src/spec.rs:79-240): a cheap guess at a request's next tokens, one step of the model over all of
them, and what the model would have written itself is kept (``Engine.verify_step``). The text that comes out is the model's: greedy requests get
the tokens that they would get one by one, requests with a temperature tokens of the same distribution, both from logits that a step of several rows may round
otherwise than a step of one (in bfloat16 nearly equal ones may fall the other way).

Two sources of drafts, as there: ``PromptLookup`` takes what followed earlier where the text's last tokens occurred before (of several such places a
tree), ``DraftModel`` lets a smaller model of the same vocabulary write ahead (a chain, with the distributions it was drawn from).
"""
from __future__ import annotations

from collections import deque
from dataclasses import dataclass, field
from typing import Deque, Dict, List, Optional, Sequence, Tuple

import numpy as np
import torch

from .. import kernels
from ..cache.manager import OutOfPages
from ..sampling.sampler import Sampler, SamplerConfig
from .engine import Engine, StepEntry
from .scheduler import LENGTH, STOP


_DRAFTS, _COINS = 1, 2
_M64, _STEP = (1 << 64) - 1, 0x9E3779B97F4A7C15


def _mix(x: int) -> int:
    """The output function of SplitMix64 (Steele, Lea and Flood, Fast splittable pseudorandom number generators, 2014) behind a step of its state."""
    x = (x + _STEP) & _M64
    x = ((x ^ x >> 30) * 0xBF58476D1CE4E5B9) & _M64
    x = ((x ^ x >> 27) * 0x94D049BB133111EB) & _M64
    return x ^ x >> 31


def _numbers(what: int, seeds: Sequence[int], at: int, count: int) -> np.ndarray:
    """``count`` random numbers in [0, 1) for one use, by a request whose text has ``at`` tokens: a stream for each use, seeds and place, of a generator that is
    not the one that requests draw their tokens with. Rejection holds only where what was drafted, the coins that take it and what is drawn in its place are
    independent, also where all seeds are equal."""
    state = _mix(what)
    for s in (*seeds, at):
        state = _mix(state ^ (int(s) & _M64))
    return np.array([_mix(state + i * _STEP) >> 40 for i in range(count)], dtype=np.float32) / np.float32(1 << 24)


def _fits(engine: Engine, text: Sequence[int]) -> bool:
    """Whether there are pages for all of a text and one to grow into. One that found too few waits for them, or it would be read over and over."""
    for g, group in enumerate(engine.cache.groups):
        held = len(text) if group.reach is None else min(len(text), group.reach + engine.max_batch_tokens)
        if engine.cache.free_pages(g) < engine.cache.pages_needed(held, g) + 1:
            return False
    return True


class PromptLookup:
    """Drafts from the text itself: where its last ``match`` tokens (or fewer, down to one) occurred before, what followed there, up to ``tokens`` of
    them, for up to ``branches`` such places, the latest first. Places that go on alike share the tokens that are alike."""

    def __init__(self, tokens: int = 8, match: int = 3, branches: int = 3):
        if tokens < 1 or match < 1 or branches < 1:
            raise ValueError("a lookup needs at least one token, one token to match and one branch")
        self.tokens, self.match, self.branches = int(tokens), int(match), int(branches)

    def propose(self, text: Sequence[int], room: int) -> Tuple[List[int], List[int]]:
        """(tokens, parents) of a tree whose first token is the text's last one, with at most ``room`` drafts."""
        x = np.asarray(text, dtype=np.int64)
        tokens, parents, children = [int(x[-1])], [-1], {}
        places: List[int] = []
        for m in range(min(self.match, len(x) - 1), 0, -1):
            windows = np.lib.stride_tricks.sliding_window_view(x[:-1], m)
            ends = np.nonzero((windows == x[-m:]).all(axis=1))[0] + m          # what followed begins here
            places += [int(e) for e in ends[::-1] if int(e) not in places]
            if len(places) >= self.branches:
                break
        for place in places[:self.branches]:
            at = 0
            for t in x[place:place + self.tokens].tolist():
                if (at, t) not in children:
                    if len(tokens) > room:
                        break
                    children[(at, t)] = len(tokens)
                    tokens.append(t)
                    parents.append(at)
                at = children[(at, t)]
        return tokens, parents

    def drop(self, rid) -> None:
        pass


class DraftModel:
    """Drafts from a smaller model: ``tokens`` of them, written one after another by ``engine`` (an ``Engine`` of a model with the same vocabulary, used for
    nothing else meanwhile), greedily for greedy requests, else drawn at the request's temperature by random numbers that are none of the request's own: they
    follow from ``seed``, the request's seed and its text's length, so a run with the same seeds drafts the same."""

    def __init__(self, engine: Engine, tokens: int = 4, seed: int = 0):
        if tokens < 1:
            raise ValueError("a drafting model needs to write at least one token")
        self.engine, self.tokens, self.seed = engine, int(tokens), int(seed)

    def propose_all(self, rids: Sequence[object], texts: Sequence[Sequence[int]], rooms: Sequence[int], temperatures: Sequence[float],
                    seeds: Sequence[int]):
        """For each request ``(tokens, parents)`` as ``PromptLookup.propose``, and of all rows the logits that their children were drawn from. ``seeds`` of the
        requests."""
        engine = self.engine
        counts = [max(0, min(self.tokens, room, engine.max_position - len(text))) for room, text in zip(rooms, texts)]
        for j, (rid, text) in enumerate(zip(rids, texts)):
            if counts[j] and not self._catch_up(rid, text):
                counts[j] = 0
            elif len(text) >= engine.max_position:       # (a text that its context does not hold)
                self.drop(rid)
        firsts = np.concatenate([[0], np.cumsum([c + 1 for c in counts])])
        logits = torch.zeros(int(firsts[-1]), engine.config.vocab_size, device=engine.device)
        drafts = [[int(text[-1])] for text in texts]
        heat = torch.tensor(temperatures, dtype=torch.float32)
        numbers = [_numbers(_DRAFTS, (self.seed, seed), len(text), c) for seed, text, c in zip(seeds, texts, counts)]
        for i in range(max(counts, default=0)):
            every = [j for j, c in enumerate(counts) if c > i]
            for a in range(0, len(every), engine.max_batch_tokens):
                live = every[a:a + engine.max_batch_tokens]
                rows = None
                while live and rows is None:
                    try:
                        rows = engine.step([StepEntry(rids[j], [drafts[j][-1]], [0]) for j in live])
                    except OutOfPages:                   # the last one's pages are for the others; what it has drafted stands
                        j = live.pop()
                        counts[j] = i
                        self.drop(rids[j])
                if rows is None:
                    continue
                logits.index_copy_(0, torch.tensor([int(firsts[j]) + i for j in live], device=engine.device), rows)
                picked = torch.empty(len(live), dtype=torch.int32, device=engine.device)
                draws = torch.tensor([float(numbers[j][i]) for j in live], dtype=torch.float32).to(engine.device)
                kernels.sample(rows, picked, heat[live].to(engine.device), draws)
                for j, t in zip(live, picked.tolist()):
                    drafts[j].append(t)
        done = [int(f) + k for f, d in zip(firsts, drafts) for k in range(len(d))]
        if len(done) < len(logits):
            logits = logits[torch.tensor(done, device=engine.device)]
        return [(d, list(range(-1, len(d) - 1))) for d in drafts], logits

    def _catch_up(self, rid, text: Sequence[int]) -> bool:
        """The request's cache holds all of the text but its last token. What was drafted and not kept is taken back; where that cannot be (a state has taken it in,
        a window has given back the pages before it) the text is read anew. False: there are no pages or no slot for it now, and it holds none."""
        try:
            if self.engine.cache.has(rid) or _fits(self.engine, text):
                self._read(rid, text)
                return True
        except OutOfPages:
            self.drop(rid)
        return False

    def _read(self, rid, text: Sequence[int]) -> None:
        engine = self.engine
        if not engine.cache.has(rid):
            engine.add_request(rid, list(text))
        held = engine.cache.tokens(rid)[:engine.length(rid)]
        same = limit = min(len(held), len(text) - 1)
        if limit:
            differ = np.nonzero(np.asarray(held[:limit]) != np.asarray(text[:limit]))[0]
            same = int(differ[0]) if len(differ) else limit
        if same < len(held) and not self._take_back(rid, same):
            engine.free_request(rid)
            engine.add_request(rid, list(text))
        for a in range(engine.length(rid), len(text) - 1, engine.max_batch_tokens):
            engine.step([StepEntry(rid, list(text[a:min(a + engine.max_batch_tokens, len(text) - 1)]))])

    def _take_back(self, rid, length: int) -> bool:
        if self.engine.device_cache.has_state:
            return False
        try:
            self.engine.cache.truncate(rid, length)
        except ValueError:                               # (of pages that are gone, before anything changes)
            return False
        return True

    def drop(self, rid) -> None:
        if self.engine.cache.has(rid):
            self.engine.free_request(rid)


@dataclass
class _Text:
    rid: object
    index: int
    tokens: List[int]
    prompt: int
    sampler: Sampler
    order: int = 0
    reason: Optional[str] = None
    waits: bool = False      # it had to make room once
    draws: List[float] = field(default_factory=list)     # random numbers ahead of the generator: one for each token that is next to be drawn


@dataclass
class DraftCounts:
    """How drafts fared in a run of ``generate``."""
    steps: int = 0           # steps of the model, of one request each
    drafted: int = 0
    accepted: int = 0


def generate(engine: Engine, prompts: Sequence[Sequence[int]], max_tokens: int, drafts, config: SamplerConfig, stop: Sequence[int] = (),
             max_seqs: Optional[int] = None) -> Tuple[List[List[int]], List[str], DraftCounts]:
    """Generate after each prompt with ``drafts`` (a ``PromptLookup`` or ``DraftModel``); request i samples with seed ``config.seed + i``. Returns the new tokens and
    why each request ended, in the order given, and how the drafts fared. Prompts are read one by one, all running requests go through the model in one
    step. When pages run out drafts go first, then the request that was admitted last waits and is read again; one that does not fit by itself ends by its
    length, or raises ``OutOfPages`` where other requests of the engine hold slots or pages."""
    if config.needs_host:
        raise ValueError("drafted generation is greedy or at a temperature: top_k, top_p, min_p and repetition_penalty are not built for it")
    if not engine.model.takes_trees:
        raise ValueError(f"{engine.config.architecture} takes no drafted trees: {engine.model.why_no_trees()}")
    most = min(max_seqs or engine.max_requests, engine.max_requests, engine.max_batch_tokens)      # requests that run at once
    if isinstance(drafts, DraftModel):
        if drafts.engine is engine:
            raise ValueError("a model cannot draft for itself")
        if drafts.engine.config.vocab_size != engine.config.vocab_size:
            raise ValueError(f"the drafting model knows {drafts.engine.config.vocab_size} tokens, the model {engine.config.vocab_size}")
        if drafts.engine.max_requests < min(len(prompts), most):
            raise ValueError(f"the drafting model's engine holds {drafts.engine.max_requests} requests, fewer than run at once")
    limit = engine.max_position
    generate.runs += 1
    texts = [_Text(("drafted", generate.runs, i), i, [int(t) for t in p], len(p), Sampler(SamplerConfig(temperature=config.temperature, seed=config.seed + i)))
             for i, p in enumerate(prompts)]
    counts = DraftCounts()
    waiting: Deque[_Text] = deque(texts)
    running: List[_Text] = []

    def leave(t: _Text, reason: Optional[str]) -> None:
        t.reason = reason
        if engine.cache.has(t.rid):
            engine.free_request(t.rid)
        drafts.drop(t.rid)

    def others() -> bool:
        """Whether requests that are not of this run hold slots and pages: what does not fit may fit without them."""
        mine = {t.rid for t in texts}
        return any(rid not in mine for rid in engine.cache.request_ids())

    def read(t: _Text) -> None:
        """All of a text but its last token into the cache."""
        engine.add_request(t.rid, t.tokens)
        for a in range(engine.length(t.rid), len(t.tokens) - 1, engine.max_batch_tokens):
            engine.step([StepEntry(t.rid, t.tokens[a:min(a + engine.max_batch_tokens, len(t.tokens) - 1)])])

    def propose(room: int):
        rooms = [max(0, min(room, max_tokens - (len(t.tokens) - t.prompt) - 1, limit - len(t.tokens))) for t in running]
        if isinstance(drafts, DraftModel) and max(rooms) > 0:
            trees, logits = drafts.propose_all([t.rid for t in running], [t.tokens for t in running], rooms, [config.temperature] * len(running),
                                               [t.sampler.config.seed for t in running])
            # (without drafts there is nothing that came from a distribution)
            return trees, None if config.greedy or all(len(tokens) == 1 for tokens, _ in trees) else logits
        return [drafts.propose(t.tokens, r) if r and isinstance(drafts, PromptLookup) else ([t.tokens[-1]], [-1]) for t, r in zip(running, rooms)], None

    def numbers(trees) -> Optional[np.ndarray]:
        """The requests' random numbers: a row's second one is that of the token behind it, counted from the text's end, so that what is drawn
        does not depend on what was drafted; the first ones, coins for drafts with a distribution, are of a generator of their own."""
        if config.greedy:
            return None
        parts = []
        for t, (_, parents) in zip(running, trees):
            depth = []
            for p in parents:
                depth.append(depth[p] + 1 if depth else 0)
            while len(t.draws) <= max(depth):
                t.draws.append(t.sampler.rng.next_f32())
            coins = _numbers(_COINS, (t.sampler.config.seed,), len(t.tokens), len(parents))
            parts.append(np.stack([coins, np.array([t.draws[d] for d in depth], np.float32)], axis=1))
        return np.concatenate(parts)

    try:
        while waiting or running:
            while waiting and len(running) < most:
                t = waiting[0]
                if max_tokens <= len(t.tokens) - t.prompt or len(t.tokens) > limit:
                    waiting.popleft()
                    leave(t, LENGTH)
                    continue
                if running and t.waits and not _fits(engine, t.tokens):
                    break
                try:
                    read(t)
                except OutOfPages:
                    t.waits = True
                    if not running and others():
                        raise
                    leave(t, LENGTH if not running else None)      # alone it is too long for the cache
                    if running:
                        break
                    waiting.popleft()
                    continue
                waiting.popleft()
                running.append(t)
            if not running:
                continue
            room = engine.max_batch_tokens // len(running) - 1
            trees, logits = propose(min(room, kernels.TREE_MAX_ROWS - 1))
            kept = None
            while kept is None:
                entries = [StepEntry(t.rid, tokens, parents=parents) for t, (tokens, parents) in zip(running, trees)]
                try:
                    kept = engine.verify_step(entries, [config.temperature] * len(running), numbers(trees), logits)
                except OutOfPages:
                    if any(len(tokens) > 1 for tokens, _ in trees):
                        trees, logits = [([t.tokens[-1]], [-1]) for t in running], None
                        continue
                    t = running.pop()
                    if not running:
                        crowded = others()
                        leave(t, LENGTH)
                        if crowded:
                            raise
                        break
                    leave(t, None)
                    t.waits = True
                    waiting.appendleft(t)
                    trees = trees[:-1]
            if kept is None:
                continue
            done = []
            for t, k, (tokens, _) in zip(running, kept, trees):
                if k.next_token < 0:
                    raise ValueError(f"prompt {t.index}: the model's logits are no distribution")
                counts.steps += 1
                counts.drafted += len(tokens) - 1
                counts.accepted += len(k.tokens)
                for token in k.tokens + [k.next_token]:
                    if t.draws:
                        t.draws.pop(0)
                    if token in stop:
                        done.append((t, STOP))
                        break
                    t.tokens.append(token)
                    if len(t.tokens) - t.prompt >= max_tokens or len(t.tokens) >= limit:
                        done.append((t, LENGTH))
                        break
            for t, reason in done:
                running.remove(t)
                leave(t, reason)
        engine.check()
    finally:
        for t in running + list(waiting):
            leave(t, t.reason)
    return [t.tokens[t.prompt:] for t in texts], [t.reason for t in texts], counts


generate.runs = 0

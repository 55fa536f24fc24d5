"""Stand-ins for engines, on the CPU: the real cache bookkeeping, logits from a function of the text."""
from types import SimpleNamespace

import numpy as np
import torch

import tree_plain as plain
from glassbox_b200.cache.manager import CacheManager, GroupSpec, OutOfPages
from glassbox_b200.engine.engine import Kept


class FakeEngine:
    """``logits_of(text)`` gives the logits behind a text. With ``state`` the text is what the request was fed since its slot was new, which ``truncate``
    does not take back."""

    def __init__(self, vocab, logits_of, pages=64, page_size=4, max_position=64, budget=32, max_requests=8, window=None, state=False):
        self.config = SimpleNamespace(vocab_size=vocab, architecture="fake", max_position=max_position)
        self.model = SimpleNamespace(takes_trees=True)
        self.cache = CacheManager([GroupSpec(pages, page_size, window=window)], max_requests, has_state=state)
        self.device_cache = SimpleNamespace(has_state=state)
        self.device, self.page_size, self.max_position, self.max_batch_tokens, self.max_requests = "cpu", page_size, max_position, budget, max_requests
        self.logits_of, self.state, self.fed, self.log = logits_of, state, {}, []

    def add_request(self, rid, prompt=()):
        self.fed[rid] = []
        return self.cache.add_request(rid, prompt)

    def free_request(self, rid):
        self.cache.free_request(rid)

    def length(self, rid):
        return self.cache.length(rid)

    def check(self):
        self.cache.check_invariants()

    def _reserve(self, entries):
        n = sum(len(e.tokens) for e in entries)
        if not 0 < n <= self.max_batch_tokens:
            raise ValueError(f"a step of {n} tokens, max_batch_tokens {self.max_batch_tokens}")
        for e in entries:
            if self.length(e.request) + len(e.tokens) > self.max_position:
                raise ValueError("beyond max_position")
        done = []
        try:
            for e in entries:
                self.cache.reserve(e.request, len(e.tokens))
                done.append(e.request)
        except OutOfPages:
            for rid in done:
                self.cache.truncate(rid, self.length(rid))
            raise
        self.log.append([(e.request, len(e.tokens)) for e in entries])

    def _before(self, rid):
        return self.fed[rid] if self.state else self.cache.tokens(rid)[:self.length(rid)]

    def step(self, entries):
        self._reserve(entries)
        rows = []
        for e in entries:
            before = list(self._before(e.request))
            rows += [self.logits_of(before + list(e.tokens[:w + 1])) for w in e.want]
            self.cache.commit(e.request, e.tokens)
            self.fed[e.request] += list(e.tokens)
        return torch.tensor(np.array(rows, dtype=np.float32).reshape(len(rows), self.config.vocab_size))

    def verify_step(self, entries, temperatures, uniform, draft_logits):
        n = sum(len(e.tokens) for e in entries)
        if draft_logits is not None and tuple(draft_logits.shape) != (n, self.config.vocab_size):
            raise ValueError(f"draft_logits must be [{n}, {self.config.vocab_size}]")
        assert uniform is None or uniform.shape == (n, 2)
        self._reserve(entries)
        out, at = [], 0
        for e, t in zip(entries, temperatures):
            before, texts, k = self._before(e.request), [], len(e.tokens)
            for i, p in enumerate(e.parents):
                texts.append((texts[p] if i else list(before)) + [e.tokens[i]])
            logits = np.array([self.logits_of(x) for x in texts], dtype=np.float32)
            u = np.zeros((k, 2), np.float32) if uniform is None else uniform[at:at + k]
            kept, token = plain.verify(logits, e.tokens, list(e.parents), u, t, None if draft_logits is None else draft_logits[at:at + k].numpy())
            out.append(Kept(kept, [e.tokens[r] for r in kept[1:]], token))
            self.cache.commit(e.request, [e.tokens[r] for r in kept])
            self.cache.truncate(e.request, self.length(e.request))
            at += k
        return out


def sample(logits, out, temperature, uniform):
    """``kernels.sample`` on the CPU."""
    for i, (x, t, u) in enumerate(zip(logits.numpy(), temperature.tolist(), uniform.tolist())):
        out[i] = plain.draw(plain.softmax(x, t), u) if t > 0 else int(x.argmax())

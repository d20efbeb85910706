"""A batch of users from end to end: one prompt for all of them, pages of the cache handed out on the GPU, attention that reads
the prompt once for the whole batch, and the next tokens sampled with each user's own settings - every operator through the C ABI.

``Batch`` decodes for several users with the synthetic decoder of ``Speculator``. ``python -m nebula_b200.serve`` lets users ask
different things after one prompt, some of them longer than others, and says how many pages that took; every user's text is the
one that the user alone would have got.
"""
from __future__ import annotations

import argparse
import ctypes as C
from dataclasses import dataclass, field

import numpy as np

from . import lib as L
from .speculate import F32, Speculator, check_settings


@dataclass
class User:
    """What a user asks for, and the tokens that are there: those to be read before the first is chosen, then those chosen."""

    waiting: list
    uniforms: object  # an iterator of numbers in [0, 1)
    settings: tuple = (0.0, 0, 1.0, 0.0)  # temperature, top_k, top_p, min_p
    text: list = field(default_factory=list)
    drawn: float | None = None  # the number for the next token, until that is there


class Batch(Speculator):
    """``users`` places, at most 64. ``capacity``: tokens of the longest sequence; ``pages``: pages of the pool, by default enough
    for all places. The other sizes are Speculator's."""

    def __init__(self, users=8, capacity=512, page=64, pages=None, **size):
        super().__init__(capacity=capacity, nodes=users, page=page, **size)
        self.users, self.page = users, page
        table_pages = -(-capacity // page)
        self.capacity = table_pages * page
        pages = users * table_pages if pages is None else pages
        layer_bytes = pages * page * self.kv_heads * self.head_dim * 2
        self.k, self.v = L.Device(nbytes=self.layers * layer_bytes), L.Device(nbytes=self.layers * layer_bytes)
        self.table = L.Device(np.zeros((users, table_pages), np.int32))
        self.lengths = L.Device(np.full(users, -1, np.int32))
        self.held, self.free = L.Device(np.zeros(users, np.int32)), L.Device(np.arange(pages, dtype=np.int32))
        self.cache = L.KvCache(self.k.p, self.v.p, self.table.p, self.lengths.p, layer_bytes, self.layers, pages, page, table_pages,
                               self.kv_heads, self.head_dim, held=self.held.p)
        self.free_count = L.Device(np.array([pages], np.int32))
        self.pool = L.PagePool(self.table.p, self.held.p, self.free.p, self.free_count.p, pages, page, table_pages)
        i = lambda n: L.Device(np.zeros(n, np.int32))  # noqa: E731
        f = lambda n: L.Device(np.zeros(n, np.float32))  # noqa: E731
        self.counts, self.taken, self.freed, self.shared = i(users), i(users), i(users), i(1)
        self.path, self.accepted, self.sampled = i(users), i(users), i(users)
        self.temperature, self.top_k, self.top_p, self.min_p, self.uniforms = f(users), i(users), f(users), f(users), f(users)
        self.shared_ws = L.shared_attention_workspace(users, 1, self.q_heads, self.kv_heads, self.head_dim)
        self.prompt_pages, self.places = np.zeros(0, np.int32), [None] * users

    def forward(self, *_) -> None:
        raise NotImplementedError("one sequence's: a batch reads with read_prompt, join and step")

    prefill = forward

    def read_prompt(self, tokens) -> list:
        """The prompt's whole pages are read once, for all users that come. Returns the tokens after them: each user's first."""
        if any(self.places) or len(self.prompt_pages):
            raise ValueError("the prompt comes first, once")
        whole = len(tokens) // self.page * self.page
        if whole + 1 > self.capacity or not all(0 <= int(t) < self.vocab for t in tokens):
            raise ValueError("a prompt that fits the cache, of the vocabulary's tokens")
        self._put(self.lengths, [0] + [-1] * (self.users - 1), np.int32)
        try:
            for at in range(whole):
                self._reserve([1] + [0] * (self.users - 1))
                self._forward([int(tokens[at])] + [0] * (self.users - 1))
                self._commit()
        except RuntimeError:  # no page of what there is may stay behind
            self._put(self.lengths, [-1] * self.users, np.int32)
            L.call("pages_release", C.byref(self.pool), self.freed.p, self.lengths.p, 0, self.users)
            raise
        n = whole // self.page
        self.prompt_pages = self.table.get()[0, :n].copy()
        self._put(self.held, [0] * self.users, np.int32)  # the prompt's pages are no one user's
        self._put(self.lengths, [-1] * self.users, np.int32)
        self._put(self.shared, [whole], np.int32)
        return [int(t) for t in tokens[whole:]]

    def join(self, user: User) -> int:
        """A user takes a free place, with the prompt's pages in its row of the table. Returns the place."""
        if not user.waiting or not all(0 <= int(t) < self.vocab for t in user.waiting):
            raise ValueError("a user begins with at least one token of the vocabulary")
        if not isinstance(user.settings, (tuple, list)) or len(user.settings) != 4:
            raise ValueError("settings are temperature, top_k, top_p and min_p")
        check_settings(*user.settings)
        if None not in self.places:
            raise ValueError("no free place")
        at, n = self.places.index(None), len(self.prompt_pages)
        self.places[at] = user
        if n:
            row = np.ascontiguousarray(self.prompt_pages, np.int32)
            L.call("write", self.table.p + 4 * at * self.cache.table_pages, row.ctypes.data, row.nbytes)
        for buf, value in ((self.held, n), (self.lengths, n * self.page)):
            one = np.array([value], np.int32)
            L.call("write", buf.p + 4 * at, one.ctypes.data, 4)
        return at

    def leave(self, at: int) -> User:
        """The user's pages go back to the pool, but for the prompt's."""
        if not isinstance(at, (int, np.integer)) or not 0 <= at < self.users or self.places[at] is None:
            raise ValueError(f"place {at} has no user")
        user, self.places[at] = self.places[at], None
        one = np.array([-1], np.int32)
        L.call("write", self.lengths.p + 4 * at, one.ctypes.data, 4)
        L.call("pages_release", C.byref(self.pool), self.freed.p, self.lengths.p, len(self.prompt_pages), self.users)
        return user

    def _reserve(self, counts) -> None:
        self._put(self.counts, counts, np.int32)
        L.call("pages_reserve", C.byref(self.pool), None, self.taken.p, self.lengths.p, self.counts.p, self.users, 1)
        if none := [at for at, (c, t) in enumerate(zip(counts, self.taken.get())) if c and t < 0]:
            raise RuntimeError(f"places {none}: the pool has no pages left, or the sequence is as long as the table")

    def _forward(self, tokens) -> None:
        self.layers_of(tokens, lambda layer: L.call(
            "shared_attention", self.attended.p, self.q.p, C.byref(self.cache), layer, self.shared.p, None, self.head_dim ** -0.5, self.users,
            1, self.q_heads, self.shared_ws.p), None, self.users)

    def _commit(self) -> None:
        L.call("cache_commit", C.byref(self.cache), self.lengths.p, self.path.p, self.accepted.p, self.users, 1)

    def step(self) -> None:
        """Every user reads a token that waits, or gets the next one of its text. Where a row is refused the step raises, names the
        places and keeps nothing: without those users it can be made again."""
        users = self.places
        last = [u is not None and len(u.waiting) <= 1 for u in users]  # a token is chosen after what the user reads
        for at, (user, chosen) in enumerate(zip(users, last)):
            if chosen and user.drawn is None:
                user.drawn = next(user.uniforms, None)
            if chosen and (user.drawn is None or user.drawn != user.drawn):
                raise ValueError(f"place {at} has no number in [0, 1) for its next token")
        self._reserve([int(u is not None) for u in users])
        self._forward([0 if u is None else u.waiting[0] if u.waiting else u.text[-1] for u in users])
        L.call("matmul", self.logits.p, self.head.p, F32, self.vocab, self.hidden, self.x.p, self.users)
        asked = [u.settings if u is not None else (0.0, 0, 1.0, 0.0) for u in users]
        for buf, values, kind in zip((self.temperature, self.top_k, self.top_p, self.min_p), zip(*asked), (np.float32, np.int32, np.float32, np.float32)):
            self._put(buf, values, kind)
        self._put(self.uniforms, [u.drawn if chosen else 0.0 for u, chosen in zip(users, last)], np.float32)
        L.call("sample", self.sampled.p, self.logits.p, self.uniforms.p, self.temperature.p, self.top_k.p, self.top_p.p, self.min_p.p, 1,
               self.users, self.vocab)
        tokens = self.sampled.get()
        if none := [at for at, (chosen, token) in enumerate(zip(last, tokens)) if chosen and token < 0]:
            raise RuntimeError(f"the model gave no distribution for places {none}")
        self._commit()
        for user, chosen, token in zip(users, last, tokens):
            if user is None:
                continue
            user.waiting = user.waiting[1:]
            if chosen:
                user.text.append(int(token))
                user.drawn = None

    def pages_in_use(self) -> int:
        return self.cache.pages - int(self.free_count.get()[0])


def uniforms(seed):
    rng = np.random.default_rng(seed)
    while True:
        yield float(np.float32(rng.random() * (1 - 2.0 ** -24)))


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--users", type=int, default=6)
    ap.add_argument("--prompt", type=int, default=150, help="tokens of the prompt")
    ap.add_argument("--count", type=int, default=12, help="tokens of each text")
    a = ap.parse_args()
    rng = np.random.default_rng(0)
    prompt = [int(t) for t in rng.integers(0, 1024, a.prompt)]
    questions = [[int(t) for t in rng.integers(0, 1024, 1 + n % 5)] for n in range(a.users)]
    settings = [(0.0, 0, 1.0, 0.0), (0.8, 40, 0.95, 0.0), (1.0, 0, 0.9, 0.0), (0.7, 0, 1.0, 0.05)]
    size = dict(page=16, capacity=a.prompt + 8 + a.count)

    def users(batch):
        rest = batch.read_prompt(prompt)
        return [User(rest + q, uniforms(n), settings[n % len(settings)]) for n, q in enumerate(questions)]

    batch = Batch(a.users, **size)
    everyone = users(batch)
    for user in everyone:
        batch.join(user)
    used = 0
    while min(len(u.text) for u in everyone) < a.count:
        batch.step()
        used = max(used, batch.pages_in_use())
        for at, user in enumerate(batch.places):
            if user is not None and len(user.text) == a.count:
                batch.leave(at)
    for n in range(a.users):
        alone = Batch(1, **size)
        user = users(alone)[n]
        alone.join(user)
        while len(user.text) < a.count:
            alone.step()
        if user.text != everyone[n].text:
            raise SystemExit(f"user {n} got another text")
    own = sum(-(-(len(prompt) + len(q) + a.count) // 16) for q in questions)
    print(f"{a.users} users, {a.count} tokens each: {used} pages in use at most, {own} without a shared prompt; every text as alone")


if __name__ == "__main__":
    main()

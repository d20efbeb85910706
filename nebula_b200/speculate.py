"""A verify step from end to end: drafted tokens through attention over a paged cache and the routed MoE, then their
acceptance and the commit of the accepted ones - every operator through the C ABI, every buffer allocated once.

``Speculator`` is a small decoder of synthetic weights (queries, keys and values in one projection, tree attention, the
512-expert MoE layer, an output projection). ``python -m nebula_b200.speculate`` decodes greedily one token at a time,
then the same text with drafted trees, and says how many steps each took; the texts are equal, because a draft is only
kept where the target would have chosen it.
"""
from __future__ import annotations

import argparse
import ctypes as C

import numpy as np

from . import lib as L

Q4_K, F32 = 12, 0


def tree_masks(parents) -> np.ndarray:
    """One 64-bit mask per node: the node and its ancestors (parent -1: none)."""
    masks = np.zeros(len(parents), np.uint64)
    for i, p in enumerate(parents):
        masks[i] = (masks[p] if i and p >= 0 else np.uint64(0)) | np.uint64(1 << i)
    return masks


def depths(parents) -> np.ndarray:
    """The nodes' distances from the root: their positions after the committed tokens."""
    d = np.zeros(len(parents), np.int32)
    for i, p in enumerate(parents):
        d[i] = d[p] + 1 if i and p >= 0 else 0
    return d


def check_settings(temperature, top_k, top_p, min_p) -> None:
    """What sampling takes: the entry points refuse the rows of other settings. (As the 32-bit numbers that they are there.)"""
    try:
        with np.errstate(over="ignore"):
            t, p, m = (np.float32(x) for x in (temperature, top_p, min_p))
        sound = 0 <= t < np.inf and p == p and m == m and -(1 << 31) <= top_k < 1 << 31 and top_k == int(top_k)
    except (TypeError, ValueError, OverflowError):
        sound = False
    if not sound:
        raise ValueError(f"temperature {temperature}, top_k {top_k}, top_p {top_p}, min_p {min_p}")


class Speculator:
    """One sequence. ``nodes``: the largest tree (the last token and its drafts), at most 64. ``capacity``: tokens that the
    cache has room for, drafts of the last step included; ``committed``: those it holds."""

    def __init__(self, layers=2, vocab=1024, capacity=512, nodes=9, q_heads=24, kv_heads=2, head_dim=256, rotary=64, page=64,
                 hidden=2048, ffn=512, seed=1):
        self.layers, self.vocab, self.nodes, self.hidden, self.ffn = layers, vocab, nodes, hidden, ffn
        self.q_heads, self.kv_heads, self.head_dim, self.rotary = q_heads, kv_heads, head_dim, rotary
        self.width = (q_heads + 2 * kv_heads) * head_dim
        w = lambda k, rows, cols, std, typ=F32: L.synth_weights(typ, rows, cols, seed * 100 + k, std)  # noqa: E731
        self.embed, self.head = w(1, vocab, hidden, 1.0), w(2, vocab, hidden, 0.05)
        self.weights = []
        for i in range(layers):
            k = 10 * (i + 1)
            self.weights.append(dict(
                qkv=w(k, self.width, hidden, 0.02), out=w(k + 1, hidden, q_heads * head_dim, 0.02),
                gate=w(k + 2, 512 * ffn, hidden, 0.02, Q4_K), up=w(k + 3, 512 * ffn, hidden, 0.02, Q4_K),
                down=w(k + 4, 512 * hidden, ffn, 0.02, Q4_K), router=w(k + 5, 512, hidden, 0.02),
                sg=w(k + 6, ffn, hidden, 0.02, Q4_K), su=w(k + 7, ffn, hidden, 0.02, Q4_K),
                sd=w(k + 8, hidden, ffn, 0.02, Q4_K), sr=w(k + 9, 1, hidden, 0.02)))
        ones = np.ones(head_dim, np.float32)
        self.q_weight, self.k_weight = L.Device(ones), L.Device(ones)

        # the cache: one page table for all layers, pages in any order
        pages = -(-(capacity + nodes) // page)
        self.capacity, self.committed = pages * page, 0
        layer_bytes = pages * page * kv_heads * head_dim * 2
        self.k, self.v = L.Device(nbytes=layers * layer_bytes), L.Device(nbytes=layers * layer_bytes)
        self.table = L.Device(np.random.default_rng(seed).permutation(pages).astype(np.int32))
        self.lengths = L.Device(np.zeros(1, np.int32))
        self.cache = L.KvCache(self.k.p, self.v.p, self.table.p, self.lengths.p, layer_bytes, layers, pages, page, pages, kv_heads,
                               head_dim)
        self.rope = L.Device.empty((self.capacity, rotary // 2, 2), np.float32)
        L.call("rope_table", self.rope.p, self.capacity, rotary, 1e6)

        f = lambda *shape: L.Device.empty(shape, np.float32)  # noqa: E731
        i = lambda *shape: L.Device.empty(shape, np.int32)  # noqa: E731
        self.x, self.y, self.qkv = f(nodes, hidden), f(nodes, hidden), f(nodes, self.width)
        self.q, self.attended, self.logits = f(nodes, q_heads, head_dim), f(nodes, q_heads, head_dim), f(nodes, vocab)
        self.masks, self.offsets = L.Device.empty(nodes, np.uint64), i(nodes)
        self.draft, self.parents, self.uniforms = i(nodes), i(nodes), f(nodes)
        self.path, self.accepted, self.next = i(nodes), i(1), i(1)
        self.temperature, self.top_k, self.top_p, self.min_p = f(1), i(1), f(1), f(1)
        self.ids, self.route = i(nodes, 10), f(nodes, 10)
        self.moe_ws = L.workspace(nodes, hidden, ffn)
        self.attention_ws = L.attention_workspace(1, nodes, q_heads, kv_heads, head_dim)
        self.verify_ws = L.verify_workspace(1, nodes, vocab)

    def _put(self, buf, values, dtype):
        values = np.ascontiguousarray(values, dtype)
        L.call("write", buf.p, values.ctypes.data, values.nbytes)

    def _check(self, tokens, parents) -> None:
        """The buffers hold ``nodes`` rows and the embedding ``vocab``: nothing outside them may reach an entry point."""
        t = len(tokens)
        if not 1 <= t <= self.nodes or len(parents) != t:
            raise ValueError(f"{t} tokens and {len(parents)} parents: one parent each, at most {self.nodes}")
        if not all(0 <= int(x) < self.vocab for x in tokens):
            raise ValueError(f"a token outside the vocabulary of {self.vocab}")
        if not all(-1 <= int(p) < i for i, p in enumerate(parents) if i):
            raise ValueError("a node's parent comes before it")
        if self.committed + t > self.capacity:
            raise ValueError(f"{self.committed} tokens committed, {t} more: the cache holds {self.capacity}")

    def forward(self, tokens, parents) -> None:
        """The nodes through every layer; their keys and values follow the committed ones in the cache."""
        self._check(tokens, parents)
        t, d = len(tokens), self.head_dim
        self._put(self.masks, tree_masks(parents), np.uint64)
        self._put(self.offsets, depths(parents), np.int32)
        self.layers_of(tokens, lambda layer: L.call(
            "tree_attention", self.attended.p, self.q.p, C.byref(self.cache), layer, self.masks.p, d ** -0.5, 1, t, self.q_heads,
            self.attention_ws.p), self.offsets.p, 1)

    def layers_of(self, tokens, attend, offsets, seqs) -> None:
        """The tokens' rows through every layer; ``attend(layer)`` is the attention."""
        t, d = len(tokens), self.head_dim
        for n, token in enumerate(tokens):
            L.call("gather", self.x.p + 4 * n * self.hidden, self.embed.p, F32, self.hidden, int(token))
        for layer, w in enumerate(self.weights):
            L.call("matmul", self.qkv.p, w["qkv"].p, F32, self.width, self.hidden, self.x.p, t)
            k = self.qkv.p + 4 * self.q_heads * d
            L.call("qk_norm_rope", self.q.p, C.byref(self.cache), layer, self.qkv.p, self.width, k, self.width,
                   k + 4 * self.kv_heads * d, self.width, self.q_weight.p, self.k_weight.p, 1e-6, self.rope.p, self.capacity,
                   self.rotary, offsets, seqs, t // seqs, self.q_heads)
            attend(layer)
            L.call("matmul", self.y.p, w["out"].p, F32, self.hidden, self.q_heads * d, self.attended.p, t)
            L.call("binary", self.x.p, self.x.p, self.y.p, t * self.hidden, 0)
            L.call("moe_layer", self.y.p, self.ids.p, self.route.p, self.x.p, t, w["router"].p, None, w["gate"].p, Q4_K, w["up"].p, Q4_K,
                   w["down"].p, Q4_K, w["sg"].p, Q4_K, w["su"].p, Q4_K, w["sd"].p, Q4_K, w["sr"].p, self.hidden, self.ffn,
                   self.moe_ws.p)
            L.call("binary", self.x.p, self.x.p, self.y.p, t * self.hidden, 0)

    def prefill(self, tokens) -> None:
        """Tokens that are given: all of them are kept."""
        if self.committed + len(tokens) > self.capacity:
            raise ValueError(f"{self.committed} tokens committed, {len(tokens)} more: the cache holds {self.capacity}")
        if not all(0 <= int(x) < self.vocab for x in tokens):
            raise ValueError(f"a token outside the vocabulary of {self.vocab}")
        for at in range(0, len(tokens), self.nodes):
            part = tokens[at : at + self.nodes]
            self.forward(part, range(-1, len(part) - 1))
            self._put(self.path, range(len(part)), np.int32)
            self._put(self.accepted, [len(part) - 1], np.int32)
            L.call("cache_commit", C.byref(self.cache), self.lengths.p, self.path.p, self.accepted.p, 1, len(part))
            self.committed += len(part)

    def step(self, tokens, parents, uniforms=None, temperature=0.0, top_k=0, top_p=1.0, min_p=0.0):
        """``tokens[0]`` is the last token chosen, the others are drafts. Returns the accepted nodes (the root first) and
        the token after them; the accepted nodes' keys and values stay in the cache. ``top_k``, ``top_p`` and ``min_p`` truncate
        the target's distribution first (0, 1 and 0: not at all)."""
        t = len(tokens)
        self._check(tokens, parents)
        uniforms = np.zeros(t) if uniforms is None else np.asarray(uniforms, np.float64)
        if uniforms.shape != (t,) or not ((uniforms >= 0) & (uniforms < 1)).all():
            raise ValueError(f"{t} uniforms in [0, 1)")
        truncates = top_k > 0 or top_p < 1 or min_p > 0
        check_settings(temperature if truncates else 0.0, top_k, top_p, min_p)
        self.forward(tokens, parents)
        L.call("matmul", self.logits.p, self.head.p, F32, self.vocab, self.hidden, self.x.p, t)
        if truncates:
            temperature = float(np.float32(temperature))  # one temperature for what is kept and what is accepted
            for buf, value, kind in ((self.temperature, temperature, np.float32), (self.top_k, top_k, np.int32), (self.top_p, top_p, np.float32),
                                     (self.min_p, min_p, np.float32)):
                self._put(buf, [value], kind)
            L.call("truncate_logits", self.logits.p, self.logits.p, self.temperature.p, self.top_k.p, self.top_p.p, self.min_p.p, t, t, self.vocab)
        self._put(self.draft, tokens, np.int32)
        self._put(self.parents, list(parents), np.int32)
        self._put(self.uniforms, np.minimum(uniforms, 1 - 2.0 ** -24), np.float32)  # none is rounded to 1
        L.call("verify_tree", self.path.p, self.accepted.p, self.next.p, self.logits.p, self.draft.p, self.parents.p, None,
               self.uniforms.p, temperature, 1, t, self.vocab, self.verify_ws.p)
        L.call("cache_commit", C.byref(self.cache), self.lengths.p, self.path.p, self.accepted.p, 1, t)
        accepted = int(self.accepted.get()[0])
        if accepted < 0:
            raise RuntimeError("the target gave no distribution")
        self.committed += accepted + 1
        return [int(n) for n in self.path.get()[: accepted + 1]], int(self.next.get()[0])


def greedy(model, prompt, count):
    """``count`` tokens after the prompt, one at a time."""
    model.prefill(prompt[:-1])
    out, last = [], prompt[-1]
    for _ in range(count):
        _, last = model.step([last], [-1])
        out.append(last)
    return out


def speculative(model, prompt, count, drafter):
    """The same with drafts: ``drafter(chosen)`` gives the drafted tokens and their parents (node 0 is the last chosen
    token). Returns the tokens and the number of steps."""
    model.prefill(prompt[:-1])
    out, last, steps = [], prompt[-1], 0
    while len(out) < count:
        drafts, parents = drafter(out)
        tokens = [last, *drafts]
        path, last = model.step(tokens, [-1, *parents])
        out += [tokens[n] for n in path[1:]] + [last]
        steps += 1
    return out[:count], steps


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--layers", type=int, default=2)
    ap.add_argument("--count", type=int, default=24, help="tokens to decode")
    ap.add_argument("--right", type=float, default=0.7, help="how often a draft is the target's choice")
    a = ap.parse_args()
    rng = np.random.default_rng(0)
    prompt = [int(t) for t in rng.integers(0, 1024, 20)]
    size = dict(layers=a.layers, capacity=len(prompt) + a.count)
    plain = greedy(Speculator(**size), prompt, a.count)

    def drafter(chosen):  # a stand-in for a draft model: often right; two candidates for each of three positions
        drafts, parents, at = [], [], 0
        for i in range(3):
            right = plain[len(chosen) + i] if len(chosen) + i < a.count and rng.random() < a.right else int(rng.integers(1024))
            drafts += [int(rng.integers(1024)), right]
            parents += [at, at]
            at = len(drafts)
        return drafts, parents

    text, steps = speculative(Speculator(**size), prompt, a.count, drafter)
    if text != plain:
        raise SystemExit("the texts differ")
    print(f"{a.count} tokens: {a.count} steps one at a time, {steps} steps with drafted trees, the same text")


if __name__ == "__main__":
    main()

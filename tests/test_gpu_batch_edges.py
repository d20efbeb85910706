"""Operators for a batch of users on a B200, at the edges of what their header allows and next to each other."""
import ctypes as C
import threading

import numpy as np
import pytest

from conftest import assert_parity
from oracle import batch as B
from oracle import speculate as S
from test_gpu_sample import L, check, peaked  # noqa: F401  (L is a fixture)
from test_gpu_shared_attention import SharedCache, attend_shared, scores_off
from test_gpu_speculate import attend, expected, random_tree

pytestmark = pytest.mark.gpu


# ---- sampling --------------------------------------------------------------


@pytest.mark.parametrize("least", [np.nextafter(np.float32(1), np.float32(2)), 1.5, np.inf])
def test_min_p_above_one_leaves_the_first_of_equals(L, least):  # noqa: F811
    """No probability is more than the largest, so nothing stays but the token that is always kept."""
    rng = np.random.default_rng(21)
    x = np.round(rng.normal(size=(8, 5003)) * 4) / 4
    for r, n in enumerate((1, 2, 40, 300, 1500, 5003, 7, 600)):
        x[r, rng.choice(5003, n, replace=False)] = 9.0
    u = np.array([0.0, 0.9, 0.99, 0.3, 0.7, 0.999, 0.5, 0.6])
    for k, p in ((0, 1.0), (50, 1.0), (400, 1.0), (2000, 1.0), (5002, 0.9), (0, 0.9), (0, 0.0), (1, 1.0)):
        check(L, x, u, [1.0] * 8, [k] * 8, [p] * 8, [least] * 8)


@pytest.mark.parametrize("zeros,small", [(1500, 1500), (300, 500), (1200, 40), (40, 1200)])
def test_keys_of_zero_and_of_the_numbers_next_to_it(L, zeros, small):  # noqa: F811
    """Borders among logits just below 0 (multiples of 2^-149) with zeros above them, where the range of keys that is left ends between the two:
    the largest logit's mantissa is all ones, so that bins of keys begin there."""
    rng = np.random.default_rng(1)
    row = np.full(20000, -300.0, np.float32)
    below = -(rng.integers(1, 100000, small).astype(np.uint32).view(np.float32))
    some = np.concatenate([rng.uniform(0.3, 0.99, 3999), [np.float32(0.99999994)], np.zeros(zeros), below]).astype(np.float32)
    row[: len(some)] = rng.permutation(some)
    k = 4000 + zeros + small // 2
    w = np.sort(np.exp((row.astype(np.float64) - row.max()) / 60))[::-1]
    p = float((np.cumsum(w)[k - 1] - w[k - 1] / 2) / w.sum())  # as many as k, with a temperature of 60
    x, u = np.tile(row, (4, 1)), rng.random(4)
    check(L, x, u, [1.0, 60.0, 60.0, 60.0], [k, k, 0, 15000], [1.0, 1.0, p, p])


def test_threads_that_sample_different_vocabularies(L):  # noqa: F811
    """Entry points are called by several host threads; what one call asks of the kernel is not another's."""
    rng = np.random.default_rng(22)
    work = []
    for vocab, rows in ((1000, 2), (360445, 1), (131072, 1), (50001, 3)):
        x, u = peaked(rng, rows, vocab).astype(np.float32), rng.random(rows).astype(np.float32)
        work.append((x, u, L.Device(x), L.Device(u), L.Device(np.zeros(rows, np.int32)), L.Device(np.full(rows, 40, np.int32)), L.Device(x)))
    failed = []

    def go(n):
        x, u, dx, du, token, k, out = work[n]
        try:
            for _ in range(1500):
                L.call("sample", token.p, dx.p, du.p, None, k.p, None, None, 1, *x.shape)
                L.call("truncate_logits", out.p, dx.p, None, k.p, None, None, 1, *x.shape)
        except Exception as e:  # (an assertion in a thread would be lost)
            failed.append((n, e))

    threads = [threading.Thread(target=go, args=(n,)) for n in range(len(work))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed
    for x, u, _, _, token, _, out in work:
        got, cut = token.get(), out.get()
        for r in range(len(x)):
            assert got[r] == B.sample(x[r], u[r], top_k=40)[0]
            assert sorted(np.flatnonzero(cut[r] > -np.inf)) == sorted(int(b) for b in B.kept(x[r], top_k=40)[0])


def test_one_graph_of_different_vocabularies(L):  # noqa: F811
    rng = np.random.default_rng(23)
    work = []
    for vocab in (360445, 1000, 131072):
        x, u = peaked(rng, 2, vocab).astype(np.float32), rng.random(2).astype(np.float32)
        work.append((x, u, L.Device(x), L.Device(u), L.Device(np.zeros(2, np.int32)), L.Device(np.full(2, 0.7, np.float32))))
    g = C.c_void_p()
    L.call("graph_begin", C.byref(g))
    for x, _, dx, du, token, t in work:
        L.call("sample", token.p, dx.p, du.p, t.p, None, None, None, 1, *x.shape)
    L.call("graph_end", g)
    for _ in range(3):
        L.call("graph_launch", g)
    for x, u, _, _, token, _ in work:
        got = token.get()
        for r in range(2):
            assert got[r] == B.sample(x[r], u[r], temperature=float(np.float32(0.7)))[0]
    L.graph_destroy(g)


# ---- attention with a shared prefix ------------------------------------------


@pytest.mark.parametrize("hq,hkv,d", [(2, 2, 64), (8, 2, 64), (4, 2, 128), (32, 8, 128)])
@pytest.mark.parametrize("shared", [0, 128])
def test_scores_of_single_tokens_of_few_heads_are_not_stretched(L, hq, hkv, d, shared):  # noqa: F811
    """One key at score 0 and one at -64, both of the sequence's own: the second's share is e^-64 to within what the roundings on its way can do.
    The score is exact but for log2(e) as a float (2^-24 of 64); beside it ex2 (2^-22) and a dozen roundings (2^-24 each). With a
    prefix, its keys are at -512 and weigh nothing."""
    rng = np.random.default_rng(d)
    cache = SharedCache(L, rng, shared, [1, 1, 1], 1, hkv, d, 16)
    cache.k[:], cache.v[:] = 0.0, 0.0
    for s in range(3):
        if shared:
            cache.k[0, cache.rows(s, 0, shared), :, 0] = -64.0
        at = cache.rows(s, shared + 1, 1)
        cache.k[0, at, :, 0], cache.v[0, at] = -8.0, 1.0
    cache.upload()
    q = np.zeros((3, 1, hq, d), np.float32)
    q[..., 0] = 8.0
    got = attend_shared(L, cache, q, None, 1.0).astype(np.float64)
    ref = np.exp(-64.0) / (1 + np.exp(-64.0))
    assert np.abs(got / ref - 1).max() <= (64 + 4 + 12) * 2.0 ** -24


@pytest.mark.parametrize("hq,hkv,d,tokens", [(8, 2, 64, 1), (32, 8, 128, 1), (8, 2, 128, 3), (24, 2, 256, 5)])
def test_a_prefix_that_weighs_a_little_more_or_less(L, hq, hkv, d, tokens):  # noqa: F811
    """Maxima of a thousand that lie 2 apart between the prefix and a sequence's own keys: neither part may be lost, nor scaled by the
    other's. The bound is the first order's, as for scores of some hundreds."""
    rng = np.random.default_rng(31)
    cache = SharedCache(L, rng, 256, [40, 300], tokens, hkv, d, 64)
    for s, (far, near) in enumerate(((1000.0, 998.0), (1000.0, 1002.0))):
        if s == 0:
            cache.k[0, cache.rows(s, 0, 256), :, 0] = np.float16(far)
        n = cache.lengths[s] + tokens - 256
        cache.k[0, cache.rows(s, 256, n), :, 0] = np.float16(near)
    cache.upload()
    q = (0.1 * rng.normal(size=(2, tokens, hq, d))).astype(np.float32)
    q[..., 0] = 1.0
    got, ref = attend_shared(L, cache, q, None, 1.0), expected(cache, q, None, 1.0)
    told = 0
    for s, n in enumerate(cache.lengths):
        rows = cache.rows(s, 0, n + tokens)
        for t in range(tokens):
            for h in range(hq):
                k, v = (x[0, rows[: n + t + 1], h // (hq // hkv)].astype(np.float64) for x in (cache.k, cache.v))
                score = k @ q[s, t, h].astype(np.float64)
                w = np.exp(score - score.max())
                w /= w.sum()
                off = float(scores_off(q[s, t, h][None], k)[0])
                assert off < 0.05
                bound = 1.1 * off * (w @ np.abs(v - ref[s, t, h])) + 1e-5 * np.abs(ref[s, t, h]).max()
                assert (np.abs(got[s, t, h] - ref[s, t, h]) <= bound).all(), (s, t, h)
                lost = w[256:] if s == 0 else w[:256]  # the lighter part
                other = slice(0, 256) if s == 0 else slice(256, None)
                without = w[other] @ v[other] / w[other].sum()
                told += bool(lost.sum() > 0 and (np.abs(without - ref[s, t, h]) > bound).any())
    assert told == 2 * tokens * hq  # the inputs would show a part that is missing


# ---- pages that a sequence no longer has -------------------------------------


def prepared(L, cache, seqs, tokens, q_heads, rows, ones):  # noqa: F811
    """Keys and values of one step into the cache, without rotation; their normalised queries."""
    hkv, d = cache.kv_heads, cache.head_dim
    x = L.Device(np.ascontiguousarray(rows, np.float32))
    width = (q_heads + 2 * hkv) * d
    out = L.Device.empty((seqs * tokens, q_heads, d), np.float32)
    L.call("qk_norm_rope", out.p, C.byref(cache), 0, x.p, width, x.p + 4 * q_heads * d, width, x.p + 4 * (q_heads + hkv) * d, width, ones.p, ones.p,
           1e-6, None, 0, 0, None, seqs, tokens, q_heads)
    return out


class Paged:
    """A cache of one layer whose pages come from a pool."""

    def __init__(self, L, seqs, pages, table_pages, hkv=2, d=64, page=16):  # noqa: F811
        self.L, self.seqs, self.page, self.hkv, self.d, self.pages = L, seqs, page, hkv, d, pages
        self.k, self.v = (L.Device(np.full((pages * page, hkv, d), 0.5, np.float16)) for _ in range(2))
        self.table, self.held = L.Device(np.zeros((seqs, table_pages), np.int32)), L.Device(np.zeros(seqs, np.int32))
        self.free, self.count = L.Device(np.arange(pages, dtype=np.int32)), L.Device(np.array([pages], np.int32))
        self.lengths, self.taken, self.freed = (L.Device(np.zeros(seqs, np.int32)) for _ in range(3))
        self.pool = L.PagePool(self.table.p, self.held.p, self.free.p, self.count.p, pages, page, table_pages)
        self.cache = L.KvCache(k=self.k.p, v=self.v.p, page_table=self.table.p, lengths=self.lengths.p, layer_bytes=self.k.nbytes, layers=1, pages=pages,
                               page_tokens=page, table_pages=table_pages, kv_heads=hkv, head_dim=d, held=self.held.p)
        self.ones = L.Device(np.ones(d, np.float32))

    def reserve(self, counts, tokens):
        n = None if counts is None else self.L.Device(np.array(counts, np.int32))
        self.L.call("pages_reserve", C.byref(self.pool), None, self.taken.p, self.lengths.p, n.p if n else None, self.seqs, tokens)
        return list(self.taken.get())

    def release(self):
        self.L.call("pages_release", C.byref(self.pool), self.freed.p, self.lengths.p, 0, self.seqs)
        return list(self.freed.get())

    def rows(self, s, start, count):
        return S.positions_rows(self.table.get()[s], self.page, start, count)


def test_a_sequence_that_got_no_page_writes_into_no_other(L):  # noqa: F811
    """A pool of one page: sequence 0 has it, ends, and sequence 1 gets it. Sequence 0's row of the table still names the page when it
    begins anew and gets none: nothing of the step may reach sequence 1's keys, and sequence 0 waits."""
    rng = np.random.default_rng(41)
    p = Paged(L, 2, 1, 4)
    p.lengths.set(np.array([0, -1], np.int32))
    assert p.reserve([1, 0], 1) == [1, -1]
    p.lengths.set(np.array([-1, -1], np.int32))
    assert p.release() == [1, 0]
    p.lengths.set(np.array([-1, 0], np.int32))
    assert p.reserve([0, 5], 5) == [-1, 1]
    k, v = rng.normal(size=(2, 16, 2, 64)).astype(np.float16)
    p.k.set(k)
    p.v.set(v)
    p.lengths.set(np.array([0, 5], np.int32))
    assert p.reserve([1, 1], 1) == [-2, 0]
    q = prepared(L, p.cache, 2, 1, 4, rng.normal(size=(2, 8 * 64)), p.ones)
    now = p.k.get(), p.v.get()
    for a, b in zip(now, (k, v)):
        np.testing.assert_array_equal(np.delete(a, 5, 0), np.delete(b, 5, 0))
    out, shared = L.Device.empty((2, 4, 64), np.float32), L.Device(np.zeros(1, np.int32))
    for name, ws in (("tree", L.attention_workspace(2, 1, 4, 2, 64)), ("shared", L.shared_attention_workspace(2, 1, 4, 2, 64))):
        prefix = (shared.p,) if name == "shared" else ()
        L.call(name + "_attention", out.p, q.p, C.byref(p.cache), 0, *prefix, None, 0.125, 2, 1, 4, ws.p)
        got = out.get()
        assert np.isnan(got[0]).all()
        ref = S.attention(q.get()[1:], now[0][:6], now[1][:6], S.chain_masks(1), 0.125)
        assert_parity(got[1], ref[0])
    path, accepted = L.Device(np.zeros(2, np.int32)), L.Device(np.zeros(2, np.int32))
    L.call("cache_commit", C.byref(p.cache), p.lengths.p, path.p, accepted.p, 2, 1)
    assert list(p.lengths.get()) == [0, 6]


@pytest.mark.parametrize("hq,hkv,d,tokens", [(8, 2, 64, 1), (8, 2, 128, 1), (8, 2, 128, 4), (24, 2, 256, 1), (24, 2, 256, 7)])
def test_pages_held_bound_what_a_step_reaches(L, hq, hkv, d, tokens):  # noqa: F811
    """Sequences whose pages do not reach their last node are refused, whatever their row of the table says behind them."""
    rng = np.random.default_rng(42)
    lengths = [30, 32 - tokens, 33 - tokens, 100, 0, 70, 40]
    cache = SharedCache(L, rng, 0, lengths, tokens, hkv, d, 16)
    table = cache.table.copy()
    table[table == 1 << 30] = 0
    cache.dt.set(table)
    need = [-(-(n + tokens) // 16) for n in lengths]
    assert need[1] == 2 and need[2] == 3
    held = [need[0], 2, 2, need[3] - 1, 0, -(1 << 31), cache.table_pages + 1]
    cache.c.held_entries = 2  # without its flag in page_tokens: no address, and not looked at
    q = rng.normal(size=(7, tokens, hq, d)).astype(np.float32)
    assert_parity(attend(L, cache, q, None, 0.1), expected(cache, q, None, 0.1))
    cache.c.held = (keep := L.Device(np.array(held, np.int32))).p
    ref, good, bad = expected(cache, q, None, 0.1), [0, 1], [2, 3, 4, 5, 6]
    for got in (attend(L, cache, q, None, 0.1, calls=2), attend_shared(L, cache, q, None, 0.1, calls=2)):
        assert np.isnan(got[bad]).all()
        assert_parity(got[good], ref[good])
    path, accepted, out = L.Device(np.zeros((7, tokens), np.int32)), L.Device(np.zeros(7, np.int32)), L.Device(np.zeros(7, np.int32))
    L.call("cache_commit", C.byref(cache.c), out.p, path.p, accepted.p, 7, tokens)
    assert list(out.get()) == [n + (s in good) for s, n in enumerate(lengths)]
    before = cache.dk.get()
    width = (hq + 2 * hkv) * d
    ones = L.Device(np.ones(d, np.float32))
    prep = prepared(L, cache.c, 7, tokens, hq, rng.normal(size=(7 * tokens, width)), ones).get().reshape(7, tokens, hq, d)
    assert np.isnan(prep[bad]).all() and np.isfinite(prep[good]).all()
    changed = np.flatnonzero((before[0].view(np.uint16) != cache.dk.get()[0].view(np.uint16)).any(axis=(1, 2)))
    assert set(changed) <= {int(r) for s in good for r in cache.rows(s, lengths[s], tokens)}
    assert keep.get()[0] == held[0]


@pytest.mark.parametrize("pages", [6, 60])
def test_steps_of_users_with_drafts_of_different_number(L, pages):  # noqa: F811
    """Pages, preparation, attention of trees, truncation, acceptance, commit and the pages given back, step after step, from one graph's worth of
    calls without the host: a sequence sits out with a count of 0, has all of the step's nodes otherwise, waits where the pool has
    nothing left, and every sequence's committed keys and values are the ones that its accepted nodes had."""
    seqs, tokens, hq, hkv, d, vocab = 6, 5, 4, 2, 64, 97
    rng = np.random.default_rng(pages)
    p = Paged(L, seqs, pages, 8)
    want = [np.zeros((0, 2, hkv, d), np.float16) for _ in range(seqs)]
    shared, aws, vws = L.Device(np.zeros(1, np.int32)), L.shared_attention_workspace(seqs, tokens, hq, hkv, d), L.verify_workspace(seqs, tokens, vocab)
    out, weights = L.Device.empty((seqs, tokens, hq * d), np.float32), L.Device(rng.normal(size=(vocab, hq * d)).astype(np.float32))
    logits = L.Device.empty((seqs, tokens, vocab), np.float32)
    path, accepted, after = L.Device.empty((seqs, tokens), np.int32), L.Device.empty(seqs, np.int32), L.Device.empty(seqs, np.int32)
    lengths, refused, advanced = np.zeros(seqs, np.int32), 0, 0
    for step in range(24):
        ended = rng.random(seqs) < 0.15
        for s in np.flatnonzero(ended):
            want[s] = want[s][:0]
        p.lengths.set(np.where(ended, -1, lengths).astype(np.int32))
        p.release()
        lengths[ended] = 0
        p.lengths.set(lengths)
        counts = np.where(rng.random(seqs) < 0.25, 0, tokens)
        counts[lengths + tokens > 8 * 16] = 0
        taken = p.reserve(counts, tokens)
        sits = counts == 0
        parents = np.array([random_tree(rng, tokens) for _ in range(seqs)], np.int32)
        drafts, u = rng.integers(0, vocab, (seqs, tokens)).astype(np.int32), rng.random((seqs, tokens)).astype(np.float32)
        masks = L.Device(np.array([S.tree_masks(list(r)) for r in parents], np.uint64))
        q = prepared(L, p.cache, seqs, tokens, hq, rng.normal(size=(seqs * tokens, (hq + 2 * hkv) * d)), p.ones)
        stored = [np.stack([x.get()[p.rows(s, lengths[s], tokens)] for x in (p.k, p.v)], axis=1) if taken[s] >= 0 and not sits[s] else None for s in range(seqs)]
        L.call("shared_attention", out.p, q.p, C.byref(p.cache), 0, shared.p, masks.p, 0.125, seqs, tokens, hq, aws.p)
        L.call("matmul", logits.p, weights.p, 0, vocab, hq * d, out.p, seqs * tokens)
        t, k = L.Device(np.full(seqs, 0.9, np.float32)), L.Device(np.full(seqs, 20, np.int32))
        L.call("truncate_logits", logits.p, logits.p, t.p, k.p, None, None, tokens, seqs * tokens, vocab)
        dd, dp, du = L.Device(drafts), L.Device(parents), L.Device(u)
        L.call("verify_tree", path.p, accepted.p, after.p, logits.p, dd.p, dp.p, None, du.p, float(np.float32(0.9)), seqs, tokens, vocab, vws.p)
        took = accepted.get()
        took[sits] = -1  # (who sits out has no say, whether or not its last page has room)
        accepted.set(took)
        L.call("cache_commit", C.byref(p.cache), p.lengths.p, path.p, accepted.p, seqs, tokens)
        steps, now = path.get(), p.lengths.get()
        for s in range(seqs):
            if sits[s] or taken[s] < 0:
                refused += taken[s] == -2
                assert now[s] == lengths[s] and (sits[s] or (took[s] == -1 and after.get()[s] == -1))
                continue
            assert took[s] >= 0 and now[s] == lengths[s] + took[s] + 1
            want[s] = np.concatenate([want[s], stored[s][steps[s, : took[s] + 1]]])
            advanced += 1
        lengths = now.copy()
        keys, values = p.k.get(), p.v.get()
        for s in range(seqs):
            rows = p.rows(s, 0, lengths[s])
            np.testing.assert_array_equal(np.stack([keys[rows], values[rows]], axis=1), want[s], err_msg=f"step {step}, sequence {s}")
    assert advanced > 20 and (refused > 0) == (pages == 6)


# ---- users ---------------------------------------------------------------------


@pytest.fixture(scope="module")
def V(gpu_lib):
    from nebula_b200 import serve
    return serve


SIZE = dict(layers=1, page=16, capacity=64)


def alone(V, question, seed, settings, count):
    batch = V.Batch(1, **SIZE)
    user = V.User(batch.read_prompt([3, 4, 5]) + question, V.uniforms(seed), settings)
    batch.join(user)
    while len(user.text) < count:
        batch.step()
    return user.text[:count]


@pytest.mark.parametrize("place", [0, 1, 2])
def test_a_user_without_a_distribution_stops_no_other(V, place):
    """A refused row raises before anything is kept of the step; without that user the others get the texts they get alone."""
    from nebula_b200 import lib
    settings = [(0.8, 40, 0.95, 0.0), (1.0, 0, 0.9, 0.0), (0.7, 0, 1.0, 0.05)]
    texts = [alone(V, [7 + n], n, settings[n], 8) for n in range(3)]
    batch = V.Batch(3, **SIZE)
    rest = batch.read_prompt([3, 4, 5])
    nothing = np.full(batch.hidden, np.nan, np.float32)  # a token whose embedding is not a number
    lib.call("write", batch.embed.p + 4 * 1000 * batch.hidden, nothing.ctypes.data, nothing.nbytes)
    users = [V.User(rest + [7 + n], V.uniforms(n), settings[n]) for n in range(3)]
    users[place].waiting.append(1000)
    for user in users:
        batch.join(user)
    others = [n for n in range(3) if n != place]
    for _ in range(20):
        try:
            batch.step()
        except RuntimeError as e:
            assert str(place) in str(e)
            with pytest.raises(RuntimeError):
                batch.step()  # it stays so
            assert batch.leave(place) is users[place]
            break
    else:
        pytest.fail("the row was not refused")
    while min(len(users[n].text) for n in others) < 8:
        batch.step()
    for n in others:
        assert users[n].text[:8] == texts[n], n
    assert users[place].text == []


@pytest.mark.parametrize("numbers", [[0.5, 0.25], [0.5, 0.25, float("nan")]])
def test_a_user_without_uniforms_stops_no_other(V, numbers):
    """Numbers that end, or are none, take no number from the other users."""
    settings = (1.0, 0, 1.0, 0.0)
    texts = [alone(V, [7 + n], n, settings, 8) for n in range(3)]
    batch = V.Batch(3, **SIZE)
    rest = batch.read_prompt([3, 4, 5])
    users = [V.User(rest + [7 + n], V.uniforms(n), settings) for n in range(3)]
    users[1].uniforms = iter(numbers)
    for user in users:
        batch.join(user)
    with pytest.raises(ValueError, match="1"):
        for _ in range(20):
            batch.step()
    assert len(users[1].text) == 2
    batch.leave(1)
    while len(users[0].text) < 8:
        batch.step()
    assert [users[0].text[:8], users[2].text[:8]] == [texts[0], texts[2]]


BAD = [(-1.0, 0, 1.0, 0.0), (float("nan"), 0, 1.0, 0.0), (float("inf"), 0, 1.0, 0.0), (1e39, 0, 1.0, 0.0), (1.0, 0, float("nan"), 0.0),
       (1.0, 0, 1.0, float("nan")), (1.0, 1 << 31, 1.0, 0.0), (1.0, 0.5, 1.0, 0.0), (1.0, 0, 1.0), None]


def test_settings_that_no_row_can_have_are_refused(V):
    batch = V.Batch(2, **SIZE)
    for settings in BAD:
        with pytest.raises(ValueError):
            batch.join(V.User([1], V.uniforms(0), settings))
    assert batch.places == [None, None]
    user = V.User([1], V.uniforms(0), (0.5, -3, 1.5, -1.0))
    batch.join(user)
    batch.step()
    assert len(user.text) == 1


def test_places_that_no_one_has(V):
    batch = V.Batch(2, **SIZE)
    batch.join(V.User([1], V.uniforms(0)))
    for at in (-1, -2, 1, 2, 0.0, None):
        with pytest.raises(ValueError):
            batch.leave(at)
    batch.leave(0)
    with pytest.raises(ValueError):
        batch.leave(0)
    assert batch.pages_in_use() == 0


def test_a_prompt_that_the_pool_has_no_room_for(V):
    """Its pages go back, and the batch is as it was: a shorter prompt, and users, find all of the pool."""
    batch = V.Batch(2, **dict(SIZE, pages=2))
    for _ in range(3):
        with pytest.raises(RuntimeError):
            batch.read_prompt(list(range(63)))  # three whole pages
        assert batch.pages_in_use() == 0
    rest = batch.read_prompt(list(range(20)))
    assert batch.pages_in_use() == 1 and rest == [16, 17, 18, 19]
    full = V.User(rest + [7], V.uniforms(0))
    batch.join(full)
    while len(full.text) < 3:
        batch.step()
    batch.leave(0)
    assert batch.pages_in_use() == 1


def test_those_who_get_no_page_are_named(V):
    """Without them the others go on, and get the texts that they get alone."""
    texts = [alone(V, [7 + n], n, (0.8, 40, 0.95, 0.0), 40) for n in (0, 2)]
    batch = V.Batch(3, **dict(SIZE, pages=6))
    rest = batch.read_prompt([3, 4, 5])
    users = [V.User(rest + [7 + n], V.uniforms(n), (0.8, 40, 0.95, 0.0)) for n in range(3)]
    users[1].waiting *= 8  # 32 tokens to read
    for user in users:
        batch.join(user)
    with pytest.raises(RuntimeError, match=r"\[0, 1, 2\]"):
        for _ in range(64):
            batch.step()
    assert batch.pages_in_use() == 6
    batch.leave(1)
    while min(len(users[n].text) for n in (0, 2)) < 40:
        batch.step()
    assert [users[n].text[:40] for n in (0, 2)] == texts

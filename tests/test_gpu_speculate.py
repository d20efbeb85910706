"""The verify step's operators on a B200 against their 64-bit definitions (oracle/speculate.py): preparation of queries
and keys, tree attention over the paged cache, acceptance of drafted tokens, commit of the accepted ones."""
import ctypes as C

import numpy as np
import pytest

from conftest import assert_parity
from oracle import speculate as S

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def L(gpu_lib):
    from nebula_b200 import lib
    return lib


class Cache:
    """A paged cache with pages in random order; what no sequence may read is NaN."""

    def __init__(self, L, rng, lengths, tokens, hkv, d, page, layers=1, spare=2, room=0):
        self.lengths, self.tokens, self.hkv, self.d, self.page, self.layers = list(lengths), tokens, hkv, d, page, layers
        self.table_pages = -(-(max(lengths) + tokens + room) // page)
        self.pages = len(lengths) * self.table_pages + spare
        self.table = rng.permutation(self.pages)[: len(lengths) * self.table_pages].reshape(len(lengths), -1).astype(np.int32)
        shape = (layers, self.pages * page, hkv, d)
        self.k, self.v = np.full(shape, np.nan, np.float16), np.full(shape, np.nan, np.float16)
        for s, n in enumerate(lengths):
            rows = self.rows(s, 0, n + tokens)
            self.k[:, rows] = rng.normal(size=(layers, n + tokens, hkv, d))
            self.v[:, rows] = rng.normal(size=(layers, n + tokens, hkv, d))
            used = -(-(n + tokens) // page)
            self.table[s, used:] = 1 << 30  # entries past the end are never read

        self.dk, self.dv, self.dt = L.Device(self.k), L.Device(self.v), L.Device(self.table)
        self.dl = L.Device(np.array(lengths, np.int32))
        self.c = L.KvCache(self.dk.p, self.dv.p, self.dt.p, self.dl.p, self.k[0].nbytes, layers, self.pages, page,
                           self.table_pages, hkv, d)

    def rows(self, s, start, count):
        return S.positions_rows(self.table[s], self.page, start, count)

    def upload(self):
        self.dk.set(self.k)
        self.dv.set(self.v)


def random_tree(rng, tokens):
    return [-1] + [int(rng.integers(0, i)) for i in range(1, tokens)]


def attend(L, cache, q, masks, scale, layer=0, calls=1):
    seqs, tokens, hq, d = q.shape
    dq, out = L.Device(q.astype(np.float32)), L.Device(np.full(q.shape, 7.0, np.float32))
    dm = None if masks is None else L.Device(np.array(masks, np.uint64))
    ws = L.attention_workspace(seqs, tokens, hq, cache.hkv, d)
    got = []
    for _ in range(calls):
        L.call("tree_attention", out.p, dq.p, C.byref(cache.c), layer, dm.p if dm else None, scale, seqs, tokens, hq, ws.p)
        got.append(out.get())
    for other in got[1:]:
        np.testing.assert_array_equal(other, got[0])  # the same bits every time
    return got[0]


def expected(cache, q, masks, scale, layer=0):
    tokens = q.shape[1]
    out = []
    for s, n in enumerate(cache.lengths):
        rows = cache.rows(s, 0, n + tokens)
        out.append(S.attention(q[s], cache.k[layer, rows], cache.v[layer, rows],
                               S.chain_masks(tokens) if masks is None else masks[s], scale))
    return np.stack(out)


SHAPES = [  # hq, hkv, d, lengths, tokens, page, tree
    (24, 2, 256, [0], 1, 16, False),
    (24, 2, 256, [1], 1, 16, False),
    (24, 2, 256, [63], 1, 64, False),
    (24, 2, 256, [64], 17, 64, True),
    (24, 2, 256, [1000, 0, 47], 17, 32, True),
    (24, 2, 256, [2111], 17, 64, True),
    (24, 2, 256, [300], 64, 128, True),
    (8, 8, 128, [129, 5, 640, 31], 1, 16, False),
    (32, 8, 128, [77, 1500], 7, 256, True),
    (10, 2, 128, [333], 64, 32, False),
    (16, 4, 64, [15, 16, 17, 511], 5, 16, False),
    (6, 1, 64, [4000], 33, 64, True),
    (64, 1, 64, [97], 64, 16, True),
    (3, 3, 256, [90] * 9, 2, 16, False),
]


# The path's bar (conftest: rel-L2 1e-5, max-abs 1e-4 of the largest): F32 sums of up to a few thousand terms and
# operands that keep 22 bits are off by about 1e-6.
@pytest.mark.parametrize("hq,hkv,d,lengths,tokens,page,tree", SHAPES)
def test_attention(L, hq, hkv, d, lengths, tokens, page, tree):
    rng = np.random.default_rng(hq * 1000 + d + tokens + len(lengths))
    cache = Cache(L, rng, lengths, tokens, hkv, d, page)
    q = (1.5 * rng.normal(size=(len(lengths), tokens, hq, d))).astype(np.float32)
    masks = [S.tree_masks(random_tree(rng, tokens)) for _ in lengths] if tree else None
    got = attend(L, cache, q, masks, d ** -0.5, calls=2)
    assert_parity(got, expected(cache, q, masks, d ** -0.5))


@pytest.mark.parametrize("hq,hkv,d,tokens", [(16, 4, 64, 25), (16, 4, 64, 32), (32, 8, 128, 25), (8, 2, 128, 9), (24, 2, 256, 5),
                                             (24, 2, 256, 17), (8, 2, 256, 1)])
def test_attention_many_short_sequences(L, hq, hkv, d, tokens):
    """Several sequences to a CTA, one following the other while the last unit of the one before is still at work."""
    rng = np.random.default_rng(d * tokens)
    lengths = [int(n) for n in rng.integers(0, 700, 60)]
    cache = Cache(L, rng, lengths, tokens, hkv, d, 64)
    q = (1.5 * rng.normal(size=(len(lengths), tokens, hq, d))).astype(np.float32)
    got = attend(L, cache, q, None, d ** -0.5, calls=3)
    assert_parity(got, expected(cache, q, None, d ** -0.5))


@pytest.mark.parametrize("hq,hkv,d", [(4, 4, 64), (6, 2, 64), (4, 1, 128), (4, 2, 128), (32, 8, 128)])
@pytest.mark.parametrize("page", [16, 128])
def test_attention_single_tokens_of_few_heads(L, hq, hkv, d, page):
    """Lengths around the eight keys of a warp, the unit and the page; the token may see itself or not."""
    rng = np.random.default_rng(hq * d + page)
    lengths = [0, 1, 6, 7, 8, 9, 119, 120, 127, 128, 129, 255, 1001, 5000, 33000]
    cache = Cache(L, rng, lengths, 1, hkv, d, page)
    q = (1.5 * rng.normal(size=(len(lengths), 1, hq, d))).astype(np.float32)
    assert_parity(attend(L, cache, q, None, d ** -0.5, calls=3), expected(cache, q, None, d ** -0.5))
    masks = [[s % 2] for s in range(len(lengths))]
    ref = expected(cache, q, masks, d ** -0.5)
    for s in range(0, len(lengths), 2):  # what is not seen may be anything
        cache.k[0, cache.rows(s, lengths[s], 1)] = np.nan
        cache.v[0, cache.rows(s, lengths[s], 1), :, ::2] = np.inf
    cache.upload()
    got = attend(L, cache, q, masks, d ** -0.5, calls=2)
    assert_parity(got, ref)
    assert np.array_equal(got[0], np.zeros_like(got[0]))
    q[3, 0, hq - 1, 5] = np.nan
    again = attend(L, cache, q, masks, d ** -0.5)
    assert np.isnan(again[3, 0, hq - 1]).all()
    again[3, 0, hq - 1] = got[3, 0, hq - 1]
    np.testing.assert_array_equal(again, got)
    table = cache.table.copy()
    table[12, 1], table[14, 200] = cache.pages, -1
    cache.dt.set(table)
    now = np.array(lengths, np.int32)
    now[2], now[5] = -1, 1 << 20
    cache.dl.set(now)
    again, bad = attend(L, cache, q, masks, d ** -0.5), [2, 5, 12, 14]
    assert np.isnan(again[bad]).all()
    keep = [s for s in range(len(lengths)) if s not in bad and s != 3]
    assert_parity(again[keep], ref[keep])


@pytest.mark.parametrize("d", [64, 128, 256])
def test_attention_layers_and_large_scores(L, d):
    """The layer asked for is the one read; scores of some hundreds leave one key with all the weight."""
    rng = np.random.default_rng(d)
    cache = Cache(L, rng, [200, 513], 3, 2, d, 32, layers=3)
    q = rng.normal(size=(2, 3, 8, d)).astype(np.float32) * 10
    for layer in (2, 0):
        assert_parity(attend(L, cache, q, None, 1.0, layer), expected(cache, q, None, 1.0, layer))


@pytest.mark.parametrize("d,tokens", [(64, 9), (128, 20), (256, 17), (256, 1)])
def test_attention_empty_rows_are_zero(L, d, tokens):
    rng = np.random.default_rng(d + tokens)
    cache = Cache(L, rng, [0, 70], tokens, 2, d, 16)
    q = rng.normal(size=(2, tokens, 6, d)).astype(np.float32)
    masks = [[0] * tokens, [0] * tokens]
    got = attend(L, cache, q, masks, 0.1)
    assert np.array_equal(got[0], np.zeros_like(got[0]))  # nothing committed, nothing seen
    assert_parity(got[1], expected(cache, q, masks, 0.1)[1])
    masks[0] = [1 << i if i % 2 else 0 for i in range(tokens)]
    got = attend(L, cache, q, masks, 0.1)
    ref = expected(cache, q, masks, 0.1)
    assert np.array_equal(got[0, ::2], np.zeros_like(got[0, ::2]))
    if tokens > 1:
        assert_parity(got[0, 1::2], ref[0, 1::2])


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf, 65504.0])
def test_attention_unseen_nodes_have_no_effect(L, d, value):
    """A node's key and value may be anything: the rows that do not see it are as if it were not there."""
    rng = np.random.default_rng(3)
    cache = Cache(L, rng, [40, 0, 190], 6, 2, d, 32)
    q = rng.normal(size=(3, 6, 4, d)).astype(np.float32)
    masks = [S.tree_masks([-1, 0, 0, 1, 2, 3])] * 3
    clean = expected(cache, q, masks, 0.1)
    for s, n in enumerate(cache.lengths):
        row = cache.rows(s, n + 2, 1)  # node 2: seen by itself and node 4
        cache.k[0, row, :, ::3] = value
        cache.v[0, row, :, 1::2] = value
    cache.upload()
    got = attend(L, cache, q, masks, 0.1)
    blind = [0, 1, 3, 5]
    assert_parity(got[:, blind], clean[:, blind])
    if not np.isfinite(value):
        assert not np.isfinite(got[:, [2, 4]][..., 1::2]).any()


@pytest.mark.parametrize("value", [np.nan, np.inf])
def test_attention_seen_values_that_are_not_finite(L, value):
    """They reach the columns they are in, and no other."""
    rng = np.random.default_rng(8)
    cache = Cache(L, rng, [75], 4, 2, 128, 16)
    q = rng.normal(size=(1, 4, 4, 128)).astype(np.float32)
    clean = expected(cache, q, None, 0.1)
    cache.v[0, cache.rows(0, 75 + 1, 1), :, 5] = value
    cache.upload()
    got = attend(L, cache, q, None, 0.1)
    keep = np.arange(128) != 5
    assert_parity(got[..., keep], clean[..., keep])
    assert not np.isfinite(got[:, 1:, :, 5]).any()
    assert np.isfinite(got[:, 0]).all()


def test_attention_query_that_is_not_finite(L):
    rng = np.random.default_rng(9)
    cache = Cache(L, rng, [130], 5, 2, 64, 16)
    q = rng.normal(size=(1, 5, 4, 64)).astype(np.float32)
    clean = expected(cache, q, None, 0.1)
    q[0, 2, 1, 3] = np.nan
    got = attend(L, cache, q, None, 0.1)
    assert np.isnan(got[0, 2, 1]).all()
    got[0, 2, 1] = clean[0, 2, 1]
    assert_parity(got, clean)


def test_attention_bad_sequences_get_nan_rows(L):
    rng = np.random.default_rng(10)
    cache = Cache(L, rng, [100, 90, 80, 70], 3, 2, 128, 32)
    q = rng.normal(size=(4, 3, 4, 128)).astype(np.float32)
    ref = expected(cache, q, None, 0.1)
    table = cache.table.copy()
    table[1, 1] = cache.pages
    table[3, 0] = -1
    cache.dt.set(table)
    cache.dl.set(np.array([100, 90, 1 << 20, 70], np.int32))
    got = attend(L, cache, q, None, 0.1)
    assert np.isnan(got[1:]).all()
    assert_parity(got[0], ref[0])
    cache.dl.set(np.array([100, 90, -1, 70], np.int32))
    assert np.isnan(attend(L, cache, q, None, 0.1)[2]).all()


def test_attention_spread_of_magnitudes(L):
    """One key far above thousands of others that together weigh as much, and keys that come in rising order."""
    rng = np.random.default_rng(11)
    cache = Cache(L, rng, [6000, 900], 2, 1, 128, 64)
    q = np.ones((2, 2, 4, 128), np.float32)
    cache.k[:] = 0
    cache.k[0, cache.rows(0, 17, 1), 0, 0] = np.float16(9.0)  # exp(9) = 8103 of 14103
    for i in range(900):
        cache.k[0, cache.rows(1, i, 1), 0, 0] = np.float16(i / 8.0)
    cache.upload()
    assert_parity(attend(L, cache, q, None, 1.0), expected(cache, q, None, 1.0))


def test_attention_past_32_bit_offsets(L):
    """Pages that start more than 2^32 bytes into the pool."""
    rng = np.random.default_rng(12)
    page, d, hkv, tokens, n = 64, 256, 2, 3, 150
    pages = (5 << 30) // (page * hkv * d * 2)
    dk, dv = (L.Device(nbytes=pages * page * hkv * d * 2) for _ in range(2))
    table = np.array([[pages - 1, 3, pages // 2]], np.int32)
    k, v = (rng.normal(size=(n + tokens, hkv, d)).astype(np.float16) for _ in range(2))
    for pool, x in ((dk, k), (dv, v)):
        for i, p in enumerate(table[0]):
            part = np.ascontiguousarray(x[i * page : (i + 1) * page])
            L.call("write", pool.p + int(p) * page * hkv * d * 2, part.ctypes.data, part.nbytes)
    dt, dl = L.Device(table), L.Device(np.array([n], np.int32))
    c = L.KvCache(dk.p, dv.p, dt.p, dl.p, 0, 1, pages, page, 3, hkv, d)
    q = rng.normal(size=(tokens, 8, d)).astype(np.float32)
    dq, out = L.Device(q), L.Device.empty(q.shape, np.float32)
    ws = L.attention_workspace(1, tokens, 8, hkv, d)
    L.call("tree_attention", out.p, dq.p, C.byref(c), 0, None, 0.1, 1, tokens, 8, ws.p)
    assert_parity(out.get(), S.attention(q, k, v, S.chain_masks(tokens), 0.1))
    # and the store there
    kv = rng.normal(size=(tokens, (8 + 2 * hkv) * d)).astype(np.float32)
    x, w = L.Device(kv), L.Device(np.ones(d, np.float32))
    L.call("qk_norm_rope", out.p, C.byref(c), 0, x.p, kv.shape[1], x.p + 4 * 8 * d, kv.shape[1], x.p + 4 * (8 + hkv) * d,
           kv.shape[1], w.p, w.p, 1e-6, None, 0, 0, None, 1, tokens, 8)
    got = np.empty((tokens, hkv, d), np.float16)
    L.call("read", got.ctypes.data, dv.p + (int(table[0, 2]) * page + n - 2 * page) * hkv * d * 2, got.nbytes)
    np.testing.assert_array_equal(got, kv[:, (8 + hkv) * d :].reshape(tokens, hkv, d).astype(np.float16))


def test_attention_one_workspace_for_changing_batches(L):
    """Sized for the largest batch, used for smaller ones in between."""
    rng = np.random.default_rng(13)
    ws = L.attention_workspace(3, 17, 24, 2, 256)
    for lengths, tokens in (([700, 20, 3], 17), ([900], 1), ([65, 64], 5), ([2000, 0, 130], 17), ([0], 1)):
        cache = Cache(L, rng, lengths, tokens, 2, 256, 32)
        q = rng.normal(size=(len(lengths), tokens, 24, 256)).astype(np.float32)
        dq, out = L.Device(q), L.Device.empty(q.shape, np.float32)
        L.call("tree_attention", out.p, dq.p, C.byref(cache.c), 0, None, 0.0625, len(lengths), tokens, 24, ws.p)
        assert_parity(out.get(), expected(cache, q, None, 0.0625))


# ---- preparation -----------------------------------------------------------


@pytest.mark.parametrize("positions,rotary,base", [(1, 2, 10000.0), (300, 64, 1e6), (98304, 64, 1e7), (50, 256, 500.0)])
def test_rope_table(L, positions, rotary, base):
    out = L.Device.empty((positions, rotary // 2, 2), np.float32)
    L.call("rope_table", out.p, positions, rotary, base)
    # rounded once, plus what 64-bit pow leaves in an angle of up to 1e5 radians (about 1e5 * 2^-51)
    np.testing.assert_allclose(out.get(), S.rope_table(positions, rotary, base), rtol=0, atol=2.0 ** -25 + 2e-10)


# hq, hkv, d, rotary, lengths, tokens, page, offsets, one fused projection
PREP = [
    (24, 2, 256, 64, [0], 1, 16, False, True),
    (24, 2, 256, 64, [5000, 17], 17, 64, True, True),
    (10, 10, 128, 128, [31, 0, 200], 3, 16, False, False),
    (16, 4, 64, 64, [15], 33, 16, True, True),
    (5, 1, 64, 18, [3], 4, 32, False, False),
    (4, 2, 128, 0, [9, 9], 2, 16, False, True),
    (4, 2, 256, 254, [70], 5, 128, True, False),
]


@pytest.mark.parametrize("hq,hkv,d,rotary,lengths,tokens,page,tree,fused", PREP)
def test_preparation(L, hq, hkv, d, rotary, lengths, tokens, page, tree, fused):
    rng = np.random.default_rng(hq + d + rotary + tokens)
    cache = Cache(L, rng, lengths, tokens, hkv, d, page, layers=2)
    rows = len(lengths) * tokens
    width = [(hq + 2 * hkv) * d + 3 if fused else w * d for w in (hq, hkv, hkv)]  # odd rows when fused
    if fused:
        x = L.Device((3.0 * rng.normal(size=(rows, width[0]))).astype(np.float32))
        host = x.get()
        parts = [host[:, a * d : b * d].reshape(rows, -1, d) for a, b in ((0, hq), (hq, hq + hkv), (hq + hkv, hq + 2 * hkv))]
        ptrs = [x.p, x.p + 4 * hq * d, x.p + 4 * (hq + hkv) * d]
    else:
        bufs = [L.Device(rng.normal(size=(rows, w)).astype(np.float32)) for w in width]
        parts, ptrs = [b.get().reshape(rows, -1, d) for b in bufs], [b.p for b in bufs]
    qw, kw = (1 + 0.2 * rng.normal(size=(2, d))).astype(np.float32)
    depth = np.array([[bin(m).count("1") - 1 for m in S.tree_masks(random_tree(rng, tokens))] for _ in lengths], np.int32)
    offsets = depth if tree else np.tile(np.arange(tokens, dtype=np.int32), (len(lengths), 1))
    limit = max(lengths) + tokens
    rope, out = L.Device.empty((limit, max(rotary, 2) // 2, 2), np.float32), L.Device.empty((rows, hq, d), np.float32)
    L.call("rope_table", rope.p, limit, max(rotary, 2), 10000.0)
    dqw, dkw, doff = L.Device(qw), L.Device(kw), L.Device(offsets)
    L.call("qk_norm_rope", out.p, C.byref(cache.c), 1, ptrs[0], width[0], ptrs[1], width[1], ptrs[2], width[2], dqw.p, dkw.p, 1e-6,
           rope.p, limit, rotary, doff.p if tree else None, len(lengths), tokens, hq)
    turn = rope.get()[(np.array(lengths)[:, None] + offsets).ravel()]
    ref_q, ref_k = S.norm_rope(parts[0], qw, 1e-6, turn, rotary), S.norm_rope(parts[1], kw, 1e-6, turn, rotary)
    got = out.get()
    # F32: a sum of 256 squares (8 terms, then 5 shuffles: 13 roundings, halved by the root), rsqrt's 2 ulp, two products,
    # three operations of the rotation: below 16 * 2^-24, relative to the head's largest value
    bound = 16 * 2.0 ** -24 * np.abs(ref_q).max(axis=2, keepdims=True)
    assert np.all(np.abs(got - ref_q) <= bound)
    k, v = cache.dk.get(), cache.dv.get()
    changed = np.zeros(k.shape[1], bool)
    for s, n in enumerate(lengths):
        at = cache.rows(s, n, tokens)
        changed[at] = True
        r, rk = slice(s * tokens, (s + 1) * tokens), ref_k[s * tokens : (s + 1) * tokens]
        # half a unit of F16 (at least half of its smallest step), and the F32 error before it
        off = np.abs(k[1, at].astype(np.float64) - rk)
        assert np.all(off <= 2.0 ** -11 * np.abs(rk) * (1 + 2.0 ** -10) + 2.0 ** -25 + 16 * 2.0 ** -24 * np.abs(rk).max(axis=2, keepdims=True))
        np.testing.assert_array_equal(v[1, at], parts[2][r].astype(np.float16))
    # nothing else is written
    np.testing.assert_array_equal(k[0], cache.k[0])
    np.testing.assert_array_equal(k[1, ~changed], cache.k[1, ~changed])
    np.testing.assert_array_equal(v[1, ~changed], cache.v[1, ~changed])


def test_preparation_in_place_and_bad_rows(L):
    rng = np.random.default_rng(21)
    cache = Cache(L, rng, [10, 20, 30], 2, 1, 64, 16)
    x = rng.normal(size=(6, 4, 64)).astype(np.float32)
    kv = L.Device(rng.normal(size=(6, 64)).astype(np.float32))
    q, w, rope = L.Device(x), L.Device(np.ones(64, np.float32)), L.Device.empty((64, 32, 2), np.float32)
    L.call("rope_table", rope.p, 64, 64, 1e4)
    cache.dl.set(np.array([10, 10000, 30], np.int32))  # the second leaves no room
    off = L.Device(np.array([0, 1, 0, 1, 0, 40], np.int32))  # 30 + 40 is outside the table of 64
    L.call("qk_norm_rope", q.p, C.byref(cache.c), 0, q.p, 256, kv.p, 64, kv.p, 64, w.p, w.p, 1e-6, rope.p, 64, 64, off.p, 3, 2, 4)
    got = q.get()
    good, bad = [0, 1, 4], [2, 3, 5]
    ref = S.norm_rope(x[good], np.ones(64), 1e-6, rope.get()[[10, 11, 30]], 64)
    assert np.all(np.abs(got[good] - ref) <= 16 * 2.0 ** -24 * np.abs(ref).max(axis=2, keepdims=True))
    assert np.isnan(got[bad]).all()
    k = cache.dk.get()
    for s, n, node in ((1, 20, 0), (1, 20, 1), (2, 30, 1)):
        at = cache.rows(s, n + node, 1)
        np.testing.assert_array_equal(k[0, at], cache.k[0, at])


# ---- acceptance ------------------------------------------------------------


def verify(L, logits, draft, parents, probs, uniforms, temperature, calls=2):
    seqs, tokens, vocab = logits.shape
    bufs = [L.Device(np.ascontiguousarray(x)) for x in (logits.astype(np.float32), draft.astype(np.int32), parents.astype(np.int32),
                                                        uniforms.astype(np.float32))]
    dp = None if probs is None else L.Device(probs.astype(np.float32))
    path, acc, nxt = L.Device(np.full((seqs, tokens), 5, np.int32)), L.Device.empty(seqs, np.int32), L.Device.empty(seqs, np.int32)
    ws = L.verify_workspace(seqs, tokens, vocab)
    got = None
    for _ in range(calls):
        L.call("verify_tree", path.p, acc.p, nxt.p, bufs[0].p, bufs[1].p, bufs[2].p, dp.p if dp else None, bufs[3].p, temperature, seqs,
               tokens, vocab, ws.p)
        now = path.get(), acc.get(), nxt.get()
        assert got is None or all(np.array_equal(x, y) for x, y in zip(got, now))
        got = now
    return got


VERIFY = [  # seqs, tokens, vocab, temperature, tree, sampled
    (1, 1, 1, 1.0, False, False),
    (2, 1, 7, 0.7, False, False),
    (3, 5, 33, 1.0, True, False),
    (4, 17, 1000, 0.6, True, False),
    (5, 64, 257, 1.3, True, False),
    (6, 17, 4099, 0.0, True, False),
    (3, 8, 5001, 1.0, False, True),
    (2, 17, 131072, 0.8, True, False),
    (4, 6, 131071, 0.9, False, True),
    (2, 4, 300, 0.0, False, True),
]


@pytest.mark.parametrize("seqs,tokens,vocab,temperature,tree,sampled", VERIFY)
def test_acceptance(L, seqs, tokens, vocab, temperature, tree, sampled):
    rng = np.random.default_rng(tokens * 7 + vocab)
    logits = (2.5 * rng.normal(size=(seqs, tokens, vocab))).astype(np.float32)
    for s in range(seqs):
        for t in range(tokens):
            logits[s, t, rng.integers(0, vocab, 4)] += rng.uniform(4, 12, 4).astype(np.float32)
    if vocab > 30:
        logits[:, :, rng.integers(0, vocab, 5)] = -np.inf
    parents = np.array([random_tree(rng, tokens) if tree else list(range(-1, tokens - 1)) for _ in range(seqs)])
    draft, probs, uniforms = np.zeros((seqs, tokens), np.int64), None, np.zeros((seqs, tokens), np.float32)
    if sampled:
        probs = np.zeros((seqs, tokens, vocab), np.float32)
    for s in range(seqs):
        for c in range(1, tokens):
            p = int(parents[s, c])
            if sampled:
                probs[s, c] = S.target(logits[s, p] + 0.8 * rng.normal(size=vocab), max(temperature, 0.5))
                cdf = np.cumsum(probs[s, c].astype(np.float64))
                draft[s, c] = int((cdf <= rng.random() * cdf[-1]).sum())
            else:
                elder = [int(draft[s, e]) for e in range(1, c) if parents[s, e] == p]
                ranked = [int(t) for t in np.argsort(-logits[s, p])[:70] if int(t) not in elder]
                draft[s, c] = ranked[0 if rng.random() < 0.6 else min(1, len(ranked) - 1)] if ranked else 0
    want, ref = [], None
    for s in range(seqs):
        while True:  # uniforms at which no decision is closer than what 32-bit weights can be off by
            uniforms[s] = rng.random(tokens, dtype=np.float32)
            path, nxt, margin = S.verify(logits[s], draft[s], parents[s], None if probs is None else probs[s], uniforms[s], temperature)
            if margin > 1e-5:
                break
        want.append((path, nxt))
    path, accepted, nxt = verify(L, logits, draft, parents, probs, uniforms, temperature)
    for s, (p, n) in enumerate(want):
        assert list(path[s]) == p + [-1] * (tokens - len(p))
        assert accepted[s] == len(p) - 1
        assert nxt[s] == n


def test_acceptance_edges(L):
    """One row per sequence: what has no distribution, equal logits, uniforms of 0 and just below 1."""
    nan, inf = np.nan, np.inf
    rows = np.zeros((9, 1, 40), np.float32)
    rows[0, 0, 3] = nan
    rows[1, 0, 3] = inf
    rows[2, 0, :] = -inf
    rows[3, 0, :] = -inf
    rows[3, 0, 7] = -5.0  # all the mass on one token
    rows[4, 0, 0] = -inf  # the first token that has any, at uniform 0
    rows[6, 0, 5] = 3e38  # so far above that all others are nothing
    rows[7, 0, :] = -3e38
    rows[8, 0, 1] = -nan
    u = np.array([.5, .5, .5, .999, 0, 1 - 2.0 ** -24, .3, .5, .5], np.float32)[:, None]
    zero = np.zeros((9, 1), np.int32)
    path, accepted, nxt = verify(L, rows, zero, zero - 1, None, u, 1.0)
    assert list(nxt) == [-1, -1, -1, 7, 1, 39, 5, 20, -1]
    assert list(accepted) == [-1, -1, -1, 0, 0, 0, 0, 0, -1]
    assert list(path[:, 0]) == [-1, -1, -1, 0, 0, 0, 0, 0, -1]
    _, _, nxt = verify(L, rows, zero, zero - 1, None, u, 0.0)
    assert list(nxt) == [-1, -1, -1, 7, 1, 0, 5, 0, -1]  # the lowest of equals


def test_acceptance_malformed_trees(L):
    rng = np.random.default_rng(31)
    logits = rng.normal(size=(6, 4, 50)).astype(np.float32)
    logits[:, :, 2] = 30.0  # token 2 is all but certain
    draft = np.full((6, 4), 2)
    parents = np.array([[-1, 0, 1, 2], [-1, 0, 2, 1], [-1, 0, -2, 1], [-1, 0, 1, -1], [-1, 0, 1, 2], [-1, 0, 1, 2]])
    draft[4, 2] = 50
    logits[5, 1, 9] = np.nan
    path, accepted, nxt = verify(L, logits, draft, parents, None, np.full((6, 4), 0.5), 1.0)
    assert list(accepted) == [3, -1, -1, 2, -1, -1]
    assert list(nxt) == [2, -1, -1, 2, -1, -1]
    assert list(path[3]) == [0, 1, 2, -1]
    # two children are refused when drafts were drawn
    probs = np.full((1, 3, 50), 0.02, np.float32)
    for first in (2, 7):  # accepted first, or tried after a refusal
        _, accepted, nxt = verify(L, logits[:1, :3], np.array([[0, first, 2]]), np.array([[-1, 0, 0]]), probs, np.full((1, 3), 0.5), 1.0)
        assert nxt[0] == (2 if first == 2 else -1)


@pytest.mark.parametrize("tokens", [6, 64])
def test_acceptance_of_equal_siblings(L, tokens):
    """A star whose drafts repeat: a refused token leaves p once, and its equals are refused after it."""
    rng = np.random.default_rng(tokens)
    vocab = 9
    logits = rng.normal(size=(4, tokens, vocab)).astype(np.float32)
    parents = np.array([[-1] + [0] * (tokens - 1)] * 4)
    draft = rng.integers(0, 5, (4, tokens))
    want, uniforms = [], np.zeros((4, tokens), np.float32)
    for s in range(4):
        while True:
            uniforms[s] = rng.random(tokens, dtype=np.float32)
            uniforms[s, 1:] = 0.75 + uniforms[s, 1:] / 4  # most are refused
            p, n, margin = S.verify(logits[s], draft[s], parents[s], None, uniforms[s], 1.0)
            if margin > 1e-5:
                break
        want.append((len(p) - 1, n))
    _, accepted, nxt = verify(L, logits, draft, parents, None, uniforms, 1.0)
    assert list(zip(accepted, nxt)) == want


@pytest.mark.parametrize("sampled", [False, True])
def test_acceptance_far_from_zero(L, sampled):
    """Logits at which t is beyond 2^21; with this temperature t is the logit, so 32 bits hold it."""
    rng = np.random.default_rng(77)
    seqs, tokens, vocab, temperature = 3, 5, 5003, 1.4426950408889634
    logits = (rng.integers(-40, 1, (seqs, tokens, vocab)) / 4 + 2.0 ** 21).astype(np.float32)
    parents = np.array([list(range(-1, tokens - 1))] * seqs)
    draft = rng.integers(0, vocab, (seqs, tokens))
    probs = np.full((seqs, tokens, vocab), 1 / vocab, np.float32) if sampled else None
    want, uniforms = [], np.zeros((seqs, tokens), np.float32)
    for s in range(seqs):
        while True:
            uniforms[s] = rng.random(tokens, dtype=np.float32)
            p, n, margin = S.verify(logits[s], draft[s], parents[s], None if probs is None else probs[s], uniforms[s], temperature)
            if margin > 1e-5:
                break
        want.append((len(p) - 1, n))
    _, accepted, nxt = verify(L, logits, draft, parents, probs, uniforms, temperature)
    assert list(zip(accepted, nxt)) == want


@pytest.mark.parametrize("mask", [-np.inf, -1e9, -1e30, np.finfo(np.float32).min])
@pytest.mark.parametrize("sampled", [False, True])
def test_acceptance_of_masked_logits(L, mask, sampled):
    """Tokens taken out by very low logits: next to the others, in whole runs, and at nearly every place."""
    rng = np.random.default_rng(13)
    seqs, tokens, vocab = 3, 3, 9001
    logits = rng.normal(size=(seqs, tokens, vocab)).astype(np.float32)
    logits[0, :, ::2] = mask
    logits[1, :, 1000:8000] = mask
    logits[2] = mask
    logits[2, :, [5, 4500, 9000]] = 1.0
    parents = np.array([[-1, 0, 1]] * seqs)
    draft = np.array([[0, 3, 5], [0, 10, 2000], [0, 5, 9000]])
    probs = np.full((seqs, tokens, vocab), 1 / vocab, np.float32) if sampled else None
    want, uniforms = [], np.zeros((seqs, tokens), np.float32)
    for s in range(seqs):
        while True:
            uniforms[s] = rng.random(tokens, dtype=np.float32)
            p, n, margin = S.verify(logits[s], draft[s], parents[s], None if probs is None else probs[s], uniforms[s], 0.7)
            if margin > 1e-5:
                break
        want.append((len(p) - 1, n))
    _, accepted, nxt = verify(L, logits, draft, parents, probs, uniforms, 0.7)
    assert list(zip(accepted, nxt)) == want


def test_acceptance_of_the_targets_own_drafts(L):
    """Drafts drawn from the target itself are all accepted; a draft distribution that covers the target leaves the target."""
    vocab, tokens = 64, 5
    logits = np.zeros((1, tokens, vocab), np.float32)  # every weight is 1, every probability exactly 1/64
    probs = np.full((1, tokens, vocab), 1 / 64, np.float32)
    chain = np.arange(-1, tokens - 1)[None]
    path, accepted, nxt = verify(L, logits, np.arange(tokens)[None], chain, probs, np.full((1, tokens), 0.875), 1.0)
    assert accepted[0] == tokens - 1 and nxt[0] == 56
    probs[:] = 1.0
    path, accepted, nxt = verify(L, logits, np.arange(tokens)[None], chain, probs, np.full((1, tokens), 0.25), 1.0)
    assert accepted[0] == 0 and nxt[0] == 16


# ---- commit ----------------------------------------------------------------


@pytest.mark.parametrize("hkv,d,page,lengths,tokens,layers,in_place", [
    (2, 256, 64, [0], 1, 1, True), (2, 256, 64, [60, 0, 333], 17, 3, True), (8, 128, 16, [1, 2, 3, 4, 5], 32, 2, False),
    (1, 64, 16, [14], 64, 5, True)])
def test_commit(L, hkv, d, page, lengths, tokens, layers, in_place):
    rng = np.random.default_rng(tokens + layers)
    cache = Cache(L, rng, lengths, tokens, hkv, d, page, layers=layers)
    path, accepted = np.full((len(lengths), tokens), -1, np.int32), np.zeros(len(lengths), np.int32)
    k, v = cache.k.copy(), cache.v.copy()
    for s, n in enumerate(lengths):
        accepted[s] = rng.integers(0, tokens)
        path[s, : accepted[s] + 1] = [0, *sorted(1 + rng.permutation(tokens - 1)[: accepted[s]])]
        at = cache.rows(s, n, tokens)
        for pool in (k, v):
            pool[:, at[: accepted[s] + 1]] = pool[:, at[path[s, : accepted[s] + 1]]]
    out = cache.dl if in_place else L.Device.empty(len(lengths), np.int32)
    dpath, dacc = L.Device(path), L.Device(accepted)
    L.call("cache_commit", C.byref(cache.c), out.p, dpath.p, dacc.p, len(lengths), tokens)
    np.testing.assert_array_equal(out.get(), np.array(lengths) + accepted + 1)
    np.testing.assert_array_equal(cache.dk.get(), k)
    np.testing.assert_array_equal(cache.dv.get(), v)


def test_commit_leaves_bad_sequences(L):
    rng = np.random.default_rng(41)
    cache = Cache(L, rng, [10] * 7, 5, 2, 64, 16)
    cache.dl.set(np.array([10, 10, 10, 10, 10, -3, 10], np.int32))
    path = np.array([[0, 2, 4, -1, -1], [0, 3, 2, -1, -1], [0, 2, 9, -1, -1], [0, 1, 2, 3, 4], [0, 2, -1, -1, -1], [0, 2, 3, -1, -1],
                     [0, 1, 2, 3, 4]], np.int32)
    accepted = np.array([2, 2, 2, -1, 2, 2, 5], np.int32)
    k = cache.k.copy()
    at = cache.rows(0, 10, 5)
    k[0, at[:3]] = k[0, at[[0, 2, 4]]]
    dpath, dacc = L.Device(path), L.Device(accepted)
    L.call("cache_commit", C.byref(cache.c), cache.dl.p, dpath.p, dacc.p, 7, 5)
    assert list(cache.dl.get()) == [13, 10, 10, 10, 10, -3, 10]
    np.testing.assert_array_equal(cache.dk.get(), k)


# ---- together --------------------------------------------------------------


def test_step_in_a_graph(L):
    """The four operators record into a graph, and its replay does what the calls do."""
    rng = np.random.default_rng(51)
    lengths, tokens, hq, hkv, d, vocab = [50, 7], 6, 8, 2, 128, 900
    parents = np.array([random_tree(rng, tokens) for _ in lengths])
    masks = np.array([S.tree_masks(p) for p in parents], np.uint64)
    depth = np.array([[bin(int(m)).count("1") - 1 for m in ms] for ms in masks], np.int32)
    x = rng.normal(size=(len(lengths) * tokens, (hq + 2 * hkv) * d)).astype(np.float32)
    logits = (4 * rng.normal(size=(len(lengths), tokens, vocab))).astype(np.float32)
    draft = np.array([[logits[s, max(p, 0)].argmax() for p in ps] for s, ps in enumerate(parents)])
    results = []
    for graph in (False, True):
        cache = Cache(L, np.random.default_rng(52), lengths, tokens, hkv, d, 32, layers=2)
        dx, dw, rope = L.Device(x), L.Device(np.ones(d, np.float32)), L.Device.empty((128, d // 2, 2), np.float32)
        L.call("rope_table", rope.p, 128, d, 1e4)
        bufs = [L.Device(np.ascontiguousarray(b)) for b in (masks, depth, logits, draft.astype(np.int32), parents.astype(np.int32),
                                                            rng.random(parents.shape).astype(np.float32) * 0 + np.float32(0.5))]
        q, out = L.Device.empty((len(lengths) * tokens, hq, d), np.float32), L.Device.empty((len(lengths) * tokens, hq, d), np.float32)
        path, acc, nxt = L.Device.empty(parents.shape, np.int32), L.Device.empty(2, np.int32), L.Device.empty(2, np.int32)
        aws, vws = L.attention_workspace(2, tokens, hq, hkv, d), L.verify_workspace(2, tokens, vocab)
        g = C.c_void_p()
        if graph:
            L.call("graph_begin", C.byref(g))
        w = x.shape[1]
        for layer in range(2):
            L.call("qk_norm_rope", q.p, C.byref(cache.c), layer, dx.p, w, dx.p + 4 * hq * d, w, dx.p + 4 * (hq + hkv) * d, w, dw.p, dw.p,
                   1e-6, rope.p, 128, d, bufs[1].p, 2, tokens, hq)
            L.call("tree_attention", out.p, q.p, C.byref(cache.c), layer, bufs[0].p, d ** -0.5, 2, tokens, hq, aws.p)
        L.call("verify_tree", path.p, acc.p, nxt.p, bufs[2].p, bufs[3].p, bufs[4].p, None, bufs[5].p, 0.7, 2, tokens, vocab, vws.p)
        L.call("cache_commit", C.byref(cache.c), cache.dl.p, path.p, acc.p, 2, tokens)
        if graph:
            L.call("graph_end", g)
            L.call("graph_launch", g)
        results.append([b.get() for b in (out, path, acc, nxt, cache.dl, cache.dk, cache.dv)])
        if graph:
            L.graph_destroy(g)
    for a, b in zip(*results):
        np.testing.assert_array_equal(a, b)
    assert results[0][2].max() >= 1  # something was accepted

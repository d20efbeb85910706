"""Attention of sequences that share a prefix on a B200, against the 64-bit definition (oracle/speculate.py) of each sequence
on its own."""
import ctypes as C

import numpy as np
import pytest

from conftest import assert_parity
from oracle import speculate as S
from test_gpu_speculate import L, Cache, attend, expected, random_tree  # noqa: F401  (L is a fixture)

pytestmark = pytest.mark.gpu


class SharedCache(Cache):
    """The first pages are one sequence's for all; the others' entries for pages that are read once are not read at all."""

    def __init__(self, L, rng, shared, own, tokens, hkv, d, page, layers=1, hide=True, source=0):  # noqa: F811
        super().__init__(L, rng, [shared + n for n in own], tokens, hkv, d, page, layers)
        self.table[:, : shared // page] = self.table[source, : shared // page]
        upload = self.table.copy()
        once = shared // max(128, page) * max(128, page) // page
        if hide:
            upload[[s for s in range(len(own)) if s != source], :once] = -(1 << 30)
        self.dt.set(upload)
        self.shared, self.upload_table = L.Device(np.array([shared], np.int32)), upload


def attend_shared(L, cache, q, masks, scale, layer=0, calls=1, ws=None):  # noqa: F811
    seqs, tokens, hq, d = q.shape
    dq, out = L.Device(q.astype(np.float32)), L.Device(np.full((seqs * tokens * hq * d + 64,), 7.0, np.float32))
    dm = None if masks is None else L.Device(np.array(masks, np.uint64))
    ws = ws or L.shared_attention_workspace(seqs, tokens, hq, cache.hkv, d)
    got = []
    for _ in range(calls):
        L.call("shared_attention", out.p, dq.p, C.byref(cache.c), layer, cache.shared.p, dm.p if dm else None, scale, seqs, tokens, hq, ws.p)
        got.append(out.get())
    for other in got[1:]:
        np.testing.assert_array_equal(other, got[0])  # the same bits every time
    assert (got[0][-64:] == 7.0).all()
    return got[0][:-64].reshape(q.shape)


SHAPES = [  # hq, hkv, d, shared, own lengths, tokens, page, tree
    (24, 2, 256, 128, [0], 1, 16, False),
    (24, 2, 256, 208, [4, 9], 1, 16, False),
    (24, 2, 256, 1024, [0, 1, 127, 128, 129], 1, 64, False),
    (24, 2, 256, 2048, [300, 5, 1000], 17, 64, True),
    (24, 2, 256, 512, [33, 0, 700, 64, 65, 66, 90], 64, 256, True),
    (16, 8, 256, 640, [3, 500, 20], 5, 128, True),
    (3, 3, 256, 384, [90] * 9, 2, 16, False),
    (32, 8, 128, 4112, [77, 1500, 0, 3], 1, 16, False),
    (32, 8, 128, 256, [77, 1500], 7, 256, True),
    (10, 10, 128, 1264, [12, 333, 5], 33, 16, True),
    (8, 8, 128, 12800, [1] * 20, 1, 32, False),
    (16, 4, 64, 1504, [15, 16, 17, 511], 5, 32, False),
    (6, 1, 64, 4000, [100, 2], 33, 32, True),
    (64, 1, 64, 144, [97], 64, 16, True),
    (4, 4, 64, 20000, [0, 0], 1, 16, False),
    (24, 2, 256, 0, [100, 400], 3, 16, True),
    (8, 2, 128, 112, [300, 10], 4, 16, True),
    (8, 2, 128, 256, [300, 10], 4, 256, True),
]


# The bar of the attention without a prefix (conftest: rel-L2 1e-5, max-abs 1e-4 of the largest), for the same reasons.
@pytest.mark.parametrize("hq,hkv,d,shared,own,tokens,page,tree", SHAPES)
def test_attention(L, hq, hkv, d, shared, own, tokens, page, tree):  # noqa: F811
    rng = np.random.default_rng(hq * 1000 + d + tokens + shared)
    cache = SharedCache(L, rng, shared, own, tokens, hkv, d, page)
    q = (1.5 * rng.normal(size=(len(own), tokens, hq, d))).astype(np.float32)
    masks = [S.tree_masks(random_tree(rng, tokens)) for _ in own] if tree else None
    got = attend_shared(L, cache, q, masks, d ** -0.5, calls=3)
    assert_parity(got, expected(cache, q, masks, d ** -0.5))
    cache.dt.set(cache.table)
    assert_parity(got, attend(L, cache, q, masks, d ** -0.5))


@pytest.mark.parametrize("hq,hkv,d,tokens", [(16, 4, 64, 4), (32, 8, 128, 1), (8, 2, 128, 9), (24, 2, 256, 5), (24, 2, 256, 17), (8, 8, 256, 1)])
def test_attention_many_short_sequences(L, hq, hkv, d, tokens):  # noqa: F811
    """Several items to a CTA: the prefix's, then sequences of all lengths."""
    rng = np.random.default_rng(d * tokens)
    own = [int(n) for n in rng.integers(0, 500, 70)]
    cache = SharedCache(L, rng, 1360, own, tokens, hkv, d, 16)
    q = (1.5 * rng.normal(size=(len(own), tokens, hq, d))).astype(np.float32)
    masks = [S.tree_masks(random_tree(rng, tokens)) for _ in own]
    assert_parity(attend_shared(L, cache, q, masks, d ** -0.5, calls=3), expected(cache, q, masks, d ** -0.5))


@pytest.mark.parametrize("hq,hkv,d", [(4, 2, 64), (2, 2, 128), (2, 1, 256)])
def test_attention_the_most_sequences(L, hq, hkv, d):  # noqa: F811
    """1024 sequences, a few of them refused, the first among these."""
    rng = np.random.default_rng(d)
    own = [int(n) for n in rng.integers(0, 60, 1024)]
    cache = SharedCache(L, rng, 256, own, 2, hkv, d, 16, source=3)
    q = rng.normal(size=(1024, 2, hq, d)).astype(np.float32)
    now = np.array(cache.lengths, np.int32)
    bad = [0, 1, 2, 500, 1023]
    now[bad] = [-1, 255, 1 << 20, 0, -(1 << 31)]
    cache.dl.set(now)
    got, keep = attend_shared(L, cache, q, None, 0.1, calls=2), [s for s in range(1024) if s not in bad]
    assert np.isnan(got[bad]).all()
    assert_parity(got[keep], expected(cache, q, None, 0.1)[keep])


def test_attention_what_is_asked_for_as_shared(L):  # noqa: F811
    """Any number of positions: none, fewer than a unit, within a page, all of the shortest sequence; more refuses those that are shorter."""
    rng = np.random.default_rng(1)
    cache = SharedCache(L, rng, 512, [0, 40, 700], 3, 2, 128, 64, hide=False)
    q = rng.normal(size=(3, 3, 8, 128)).astype(np.float32)
    ref = expected(cache, q, None, 0.1)
    for n in (-5, 0, 1, 127, 128, 200, 256, 383, 511, 512):
        cache.shared.set(np.array([n], np.int32))
        assert_parity(attend_shared(L, cache, q, None, 0.1), ref)
    cache.table[0, : 1212 // 64] = cache.table[2, : 1212 // 64]
    cache.dt.set(cache.table)
    for n, refused in ((513, [0]), (553, [0, 1]), (1212, [0, 1]), (1213, [0, 1, 2]), (1 << 30, [0, 1, 2]), (2 ** 31 - 1, [0, 1, 2])):
        cache.shared.set(np.array([n], np.int32))
        got, keep = attend_shared(L, cache, q, None, 0.1), [s for s in range(3) if s not in refused]
        assert np.isnan(got[refused]).all()
        if keep:
            assert_parity(got[keep], ref[keep])


@pytest.mark.parametrize("d,tokens", [(64, 9), (128, 20), (256, 17), (256, 1)])
def test_attention_rows_that_see_no_node(L, d, tokens):  # noqa: F811
    rng = np.random.default_rng(d + tokens)
    cache = SharedCache(L, rng, 128, [0, 70], tokens, 2, d, 16)
    q = rng.normal(size=(2, tokens, 6, d)).astype(np.float32)
    masks = [[0] * tokens, [1 << i if i % 2 else 0 for i in range(tokens)]]
    assert_parity(attend_shared(L, cache, q, masks, 0.1), expected(cache, q, masks, 0.1))
    cache = SharedCache(L, rng, 0, [0, 70], tokens, 2, d, 16)
    got = attend_shared(L, cache, q, [[0] * tokens] * 2, 0.1)
    assert np.array_equal(got[0], np.zeros_like(got[0]))  # nothing committed, nothing seen
    assert_parity(got[1], expected(cache, q, [[0] * tokens] * 2, 0.1)[1])


@pytest.mark.parametrize("hq,d", [(4, 64), (4, 128), (4, 256), (24, 256)])
@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf, 65504.0])
def test_attention_unseen_nodes_have_no_effect(L, hq, d, value):  # noqa: F811
    rng = np.random.default_rng(3)
    cache = SharedCache(L, rng, 256, [40, 0, 190] * 5, 6, 2, d, 32)
    q = rng.normal(size=(15, 6, hq, d)).astype(np.float32)
    masks = [S.tree_masks([-1, 0, 0, 1, 2, 3])] * 15
    clean = expected(cache, q, masks, 0.1)
    for s, n in enumerate(cache.lengths):
        row = cache.rows(s, n + 2, 1)  # node 2: seen by itself and node 4
        cache.k[0, row, :, ::3] = value
        cache.v[0, row, :, 1::2] = value
    cache.upload()
    got = attend_shared(L, cache, q, masks, 0.1, calls=2) if value == 65504.0 else attend_shared(L, cache, q, masks, 0.1)
    blind = [0, 1, 3, 5]
    assert_parity(got[:, blind], clean[:, blind])
    if not np.isfinite(value):
        assert not np.isfinite(got[:, [2, 4]][..., 1::2]).any()


@pytest.mark.parametrize("value", [np.nan, np.inf])
@pytest.mark.parametrize("d", [128, 256])
def test_attention_values_that_are_not_finite(L, d, value):  # noqa: F811
    """A node's reach the columns they are in for the rows that see them, a shared position's all rows."""
    rng = np.random.default_rng(8)
    cache = SharedCache(L, rng, 384, [75] * 40, 4, 2, d, 16)
    q = rng.normal(size=(40, 4, 8, d)).astype(np.float32)
    clean = expected(cache, q, None, 0.1)
    keep = np.arange(d) != 5
    cache.v[0, cache.rows(1, 384 + 75 + 1, 1), :, 5] = value
    cache.upload()
    got = attend_shared(L, cache, q, None, 0.1)
    assert_parity(got[..., keep], clean[..., keep])
    assert not np.isfinite(got[1, 1:, :, 5]).any()
    got[1, 1:, :, 5] = clean[1, 1:, :, 5]
    assert_parity(got, clean)
    cache.v[0, cache.rows(0, 200, 1), :, 5] = value
    cache.upload()
    got = attend_shared(L, cache, q, None, 0.1)
    assert_parity(got[..., keep], clean[..., keep])
    assert not np.isfinite(got[..., 5]).any()


def test_attention_queries_that_are_not_finite(L):  # noqa: F811
    rng = np.random.default_rng(9)
    cache = SharedCache(L, rng, 256, [130, 3], 5, 2, 64, 16)
    q = rng.normal(size=(2, 5, 4, 64)).astype(np.float32)
    clean = expected(cache, q, None, 0.1)
    q[0, 2, 1, 3], q[1, 0, 0, 0] = np.nan, np.inf
    got = attend_shared(L, cache, q, None, 0.1)
    for at in ((0, 2, 1), (1, 0, 0)):
        assert np.isnan(got[at]).all()
        got[at] = clean[at]
    assert_parity(got, clean)


def test_attention_bad_pages(L):  # noqa: F811
    rng = np.random.default_rng(10)
    cache = SharedCache(L, rng, 256, [100, 90, 80, 70], 3, 2, 128, 32)
    q = rng.normal(size=(4, 3, 4, 128)).astype(np.float32)
    ref = expected(cache, q, None, 0.1)
    table = cache.upload_table.copy()
    table[1, 9], table[3, 8] = cache.pages, -1
    cache.dt.set(table)
    got = attend_shared(L, cache, q, None, 0.1)
    assert np.isnan(got[[1, 3]]).all()
    assert_parity(got[[0, 2]], ref[[0, 2]])
    table[0, 3] = cache.pages
    cache.dt.set(table)
    assert np.isnan(attend_shared(L, cache, q, None, 0.1)).all()


def scores_off(q, k):
    """How far a score may be off. Q keeps 22 bits (2^-23 of each value), and a sum on the tensor cores takes 2 d/16 steps, in
    each of which up to 2^-23 of the running sum is cut off; the running sum is at most the sum of the magnitudes."""
    most = np.abs(np.asarray(q, np.float64)) @ np.abs(np.asarray(k, np.float64)).T
    return (1 + q.shape[-1] / 8) * 2.0 ** -23 * most.max(axis=1)


@pytest.mark.parametrize("d", [64, 128, 256])
def test_attention_layers_and_large_scores(L, d):  # noqa: F811
    """Scores of some hundreds, where their rounding is what the weights are off by: scores that are off by e_j move
    sum(w_j v_j) by sum(w_j e_j (v_j - out)), to first order, so by max|e| sum(w_j |v_j - out|) at most. Beside it the path's bar."""
    rng = np.random.default_rng(d)
    cache = SharedCache(L, rng, 384, [200, 513], 3, 2, d, 32, layers=3)
    q = rng.normal(size=(2, 3, 8, d)).astype(np.float32) * 10
    for layer, scale in ((2, 1.0), (0, 1.0), (1, -0.5)):
        got, ref = attend_shared(L, cache, q, None, scale, layer), expected(cache, q, None, scale, layer)
        for s, n in enumerate(cache.lengths):
            rows = cache.rows(s, 0, n + 3)
            for t in range(3):
                for h in range(8):
                    k, v = (x[layer, rows[: n + t + 1], h // 4].astype(np.float64) for x in (cache.k, cache.v))
                    score = k @ q[s, t, h].astype(np.float64) * scale
                    w = np.exp(score - score.max())
                    spread = (w / w.sum()) @ np.abs(v - ref[s, t, h])
                    off = abs(scale) * float(scores_off(q[s, t, h][None], k)[0])
                    assert off < 0.05  # (the square of it is what the first order leaves out)
                    bound = 1.1 * off * spread + 1e-5 * np.abs(ref[s, t, h]).max()
                    assert (np.abs(got[s, t, h] - ref[s, t, h]) <= bound).all(), (layer, s, t, h)


def test_attention_one_workspace_for_changing_batches(L):  # noqa: F811
    """Sized for the largest batch, used for smaller ones in between."""
    rng = np.random.default_rng(13)
    ws = L.shared_attention_workspace(6, 17, 24, 2, 256)
    for shared, own, tokens in ((512, [700, 20, 3, 5, 6, 7], 17), (256, [900], 1), (128, [65, 64], 5), (0, [2000, 0, 130], 17), (1024, [0], 1)):
        cache = SharedCache(L, rng, shared, own, tokens, 2, 256, 32)
        q = rng.normal(size=(len(own), tokens, 24, 256)).astype(np.float32)
        assert_parity(attend_shared(L, cache, q, None, 0.0625, ws=ws), expected(cache, q, None, 0.0625))


def test_attention_captured_and_replayed(L):  # noqa: F811
    """Lengths and what is shared change between replays of one graph."""
    rng = np.random.default_rng(14)
    cache = SharedCache(L, rng, 640, [300, 17, 200], 4, 2, 128, 32, hide=False)
    q = rng.normal(size=(3, 4, 16, 128)).astype(np.float32)
    dq, out, ws = L.Device(q), L.Device.empty(q.shape, np.float32), L.shared_attention_workspace(3, 4, 16, 2, 128)
    args = (out.p, dq.p, C.byref(cache.c), 0, cache.shared.p, None, 0.1, 3, 4, 16, ws.p)
    L.call("shared_attention", *args)
    g = C.c_void_p()
    L.call("graph_begin", C.byref(g))
    L.call("shared_attention", *args)
    L.call("graph_end", g)
    for shared, lengths in ((640, [940, 657, 840]), (128, [500, 130, 640]), (0, [3, 0, 700]), (512, [512, 512, 513])):
        cache.shared.set(np.array([shared], np.int32))
        cache.dl.set(np.array(lengths, np.int32))
        cache.lengths = lengths
        L.call("graph_launch", g)
        assert_parity(out.get(), expected(cache, q, None, 0.1))
    L.graph_destroy(g)


@pytest.mark.parametrize("hq,hkv,d", [(4, 4, 64), (6, 2, 64), (16, 4, 64), (4, 1, 128), (4, 2, 128), (32, 8, 128)])
@pytest.mark.parametrize("page", [16, 256])
def test_attention_single_tokens_of_few_heads(L, hq, hkv, d, page):  # noqa: F811
    """The sequences' own keys without tensor cores: lengths around the eight keys of a warp, the unit and the page; tokens that see
    themselves or not, refused sequences, bad pages, infinite queries."""
    rng = np.random.default_rng(hq * d + page)
    own = [0, 1, 6, 7, 8, 9, 119, 120, 127, 128, 129, 255, 1001, 3000]
    cache = SharedCache(L, rng, 512, own, 1, hkv, d, page, layers=2)
    q = (1.5 * rng.normal(size=(len(own), 1, hq, d))).astype(np.float32)
    assert_parity(attend_shared(L, cache, q, None, d ** -0.5, layer=1, calls=3), expected(cache, q, None, d ** -0.5, layer=1))
    masks = [[s % 2] for s in range(len(own))]
    ref = expected(cache, q, masks, d ** -0.5)
    for s in range(0, len(own), 2):  # what is not seen may be anything
        at = cache.rows(s, cache.lengths[s], 1)
        cache.k[0, at] = np.nan
        cache.v[0, at, :, ::2] = np.inf
    cache.upload()
    got = attend_shared(L, cache, q, masks, d ** -0.5, calls=2)
    assert_parity(got, ref)
    q[3, 0, hq - 1, 5] = np.inf
    again = attend_shared(L, cache, q, masks, d ** -0.5)
    assert np.isnan(again[3, 0, hq - 1]).all()
    again[3, 0, hq - 1] = got[3, 0, hq - 1]
    np.testing.assert_array_equal(again, got)
    table = cache.upload_table.copy()
    table[12, 512 // page], table[13, 2048 // page] = cache.pages, -1
    cache.dt.set(table)
    now = np.array(cache.lengths, np.int32)
    now[2], now[5], now[6] = -1, 1 << 20, 511
    cache.dl.set(now)
    again, bad = attend_shared(L, cache, q, masks, d ** -0.5), [2, 5, 6, 12, 13]
    assert np.isnan(again[bad]).all()
    keep = [s for s in range(len(own)) if s not in bad and s != 3]
    assert_parity(again[keep], ref[keep])
    table[0, 0] = -5  # a page of the prefix
    cache.dt.set(table)
    assert np.isnan(attend_shared(L, cache, q, masks, d ** -0.5)).all()


def test_attention_single_tokens_of_few_heads_and_any_prefix(L):  # noqa: F811
    """No prefix, one that is less than a unit, longer than some sequences, changed between replays of a graph."""
    rng = np.random.default_rng(2)
    cache = SharedCache(L, rng, 1024, [300, 0, 17, 900], 1, 8, 128, 32, hide=False)
    q = rng.normal(size=(4, 1, 32, 128)).astype(np.float32)
    ref = expected(cache, q, None, 0.1)
    dq, out, ws = L.Device(q), L.Device.empty(q.shape, np.float32), L.shared_attention_workspace(4, 1, 32, 8, 128)
    g = C.c_void_p()
    L.call("graph_begin", C.byref(g))
    L.call("shared_attention", out.p, dq.p, C.byref(cache.c), 0, cache.shared.p, None, 0.1, 4, 1, 32, ws.p)
    L.call("graph_end", g)
    for n, refused in ((1024, []), (0, []), (-7, []), (100, []), (1000, []), (128, []), (1025, [1]), (1 << 30, [0, 1, 2, 3]), (1024, [])):
        cache.shared.set(np.array([n], np.int32))
        L.call("graph_launch", g)
        got, keep = out.get(), [s for s in range(4) if s not in refused]
        assert np.isnan(got[refused]).all()
        if keep:
            assert_parity(got[keep], ref[keep])
    L.graph_destroy(g)
    # a row of zeros where nothing is there to see
    cache = SharedCache(L, rng, 0, [0, 5], 1, 8, 128, 32)
    got = attend_shared(L, cache, q[:2], [[0], [1]], 0.1)
    assert np.array_equal(got[0], np.zeros_like(got[0]))
    assert_parity(got[1], expected(cache, q[:2], [[0], [1]], 0.1)[1])


def test_attention_spread_of_magnitudes(L):  # noqa: F811
    """Maxima that lie thousands apart between the prefix and a sequence's own keys, either way."""
    rng = np.random.default_rng(11)
    for hq, tokens in ((8, 1), (32, 3)):
        cache = SharedCache(L, rng, 256, [40, 300], tokens, 8, 128, 64)
        cache.k[0, cache.rows(0, 0, 256), :, 0] = np.float16(2000.0)
        cache.k[0, cache.rows(1, 300, 1), :, 1] = np.float16(30000.0)
        cache.upload()
        q = rng.normal(size=(2, tokens, hq, 128)).astype(np.float32)
        q[..., :2] = 1.0
        got, ref = attend_shared(L, cache, q, None, 1.0), expected(cache, q, None, 1.0)
        # scores of up to 30,000 are off by some 30,000 * 2^-20 = 0.03 (22 bits of Q, sums cut off), and so are the weights: next to
        # these far maxima all the weight lies on one key, or on 256 keys whose scores differ by their small values alone
        assert np.abs(got - ref).max() <= 0.1 * np.abs(ref).max()
        assert_parity(got[1], ref[1])


@pytest.mark.parametrize("hq,hkv,d,tokens", [(8, 2, 64, 1), (32, 8, 128, 1), (8, 2, 128, 5), (8, 2, 256, 3), (24, 2, 256, 17)])
def test_attention_rows_are_nan_while_the_error_word_is_set(L, hq, hkv, d, tokens):  # noqa: F811
    """A wait that ran out leaves its mark in the workspace: every row is NaN until the workspace is cleared."""
    rng = np.random.default_rng(d)
    cache = SharedCache(L, rng, 256, [40, 7], tokens, hkv, d, 32)
    q = rng.normal(size=(2, tokens, hq, d)).astype(np.float32)
    ws = L.shared_attention_workspace(2, tokens, hq, hkv, d)
    ref = expected(cache, q, None, 0.1)
    mark = np.array([4], np.int32)
    L.call("write", ws.p, mark.ctypes.data, 4)
    for _ in range(2):
        assert np.isnan(attend_shared(L, cache, q, None, 0.1, ws=ws)).all()
    L.call("zero", ws.p, ws.nbytes)
    assert_parity(attend_shared(L, cache, q, None, 0.1, ws=ws), ref)

"""The verify step's operators on a B200 where their arithmetic runs out of room. Against the 64-bit definitions
(oracle/speculate.py)."""
import ctypes as C

import numpy as np
import pytest

from conftest import assert_parity
from oracle import speculate as S
from test_gpu_speculate import L, Cache, attend, expected  # noqa: F401  (L is a fixture)

pytestmark = pytest.mark.gpu


MARK = 123456789  # in next before the call: no token


def accept(L, logits, draft, parents, probs, uniforms, temperature):  # noqa: F811
    seqs, tokens, vocab = logits.shape
    up = lambda x, t: L.Device(np.ascontiguousarray(x, t))  # noqa: E731
    bufs = [up(logits, np.float32), up(draft, np.int32), up(parents, np.int32), up(uniforms, np.float32)]
    dp = None if probs is None else up(probs, np.float32)
    path, acc, nxt = (up(np.full(n, MARK), np.int32) for n in ((seqs, tokens), seqs, seqs))
    ws = L.verify_workspace(seqs, tokens, vocab)
    L.call("verify_tree", path.p, acc.p, nxt.p, bufs[0].p, bufs[1].p, bufs[2].p, dp.p if dp else None, bufs[3].p, temperature, seqs,
           tokens, vocab, ws.p)
    return path.get(), acc.get(), nxt.get()


def check(L, logits, draft, parents, probs, uniforms, temperature):  # noqa: F811
    logits, uniforms = np.asarray(logits, np.float32), np.asarray(uniforms, np.float32)
    path, acc, nxt = accept(L, logits, np.asarray(draft), np.asarray(parents), probs, uniforms, temperature)
    for s in range(len(logits)):
        p, n, _ = S.verify(logits[s], draft[s], parents[s], None if probs is None else np.asarray(probs, np.float32)[s], uniforms[s],
                           temperature)
        assert list(path[s]) == p + [-1] * (len(parents[s]) - len(p)), s
        assert acc[s] == len(p) - 1
        assert nxt[s] == n, s


# ---- weights far below the row's largest -----------------------------------


def cliff(gap, vocab=9000, high=1000):
    """A row whose first logits are `gap` below its last ones."""
    row = np.full(vocab, -gap, np.float32)
    row[-high:] = 0.0
    return row


@pytest.mark.parametrize("drawn", [False, True])
@pytest.mark.parametrize("gap,temperature", [(60, 1.0), (100, 1.0), (10, 0.1), (140, 0.5), (420, 1.0), (5e5, 8e3)])
def test_uniform_of_zero_takes_the_first_token_with_any_mass(L, drawn, gap, temperature):  # noqa: F811
    """Chunks of the vocabulary up to 600 octaves below the largest weight; the row begins with tokens without any."""
    row = cliff(gap)
    row[:10] = -np.inf
    rows = np.stack([[row, row], [np.roll(row, 4500), row]])
    probs = np.full((2, 2, 9000), 1 / 9000) if drawn else None
    # the draft has no mass, or is refused at no uniform; then the next token is drawn at uniform 0
    check(L, rows, [[0, 3], [0, 20]], [[-1, 0]] * 2, probs, [[0, 0.5], [0, 1 - 2.0 ** -24]], temperature)


def test_uniform_of_zero_where_the_logits_are_large(L):  # noqa: F811
    """Logits at which t is beyond 2^22; with this temperature t is the logit, so 32 bits hold it."""
    row = cliff(150) + np.float32(2.0 ** 22)
    check(L, np.stack([[row], [np.roll(row, -500)]]), [[0]] * 2, [[-1]] * 2, None, [[0], [0]], 1.4426950408889634)


@pytest.mark.parametrize("drawn", [False, True])
def test_uniform_of_zero_accepts_a_draft_with_any_mass(L, drawn):  # noqa: F811
    rows = np.stack([[cliff(110)] * 3])
    probs = np.full((1, 3, 9000), 1 / 9000) if drawn else None
    check(L, rows, [[0, 17, 4321]], [[-1, 0, 1]], probs, [[0, 0, 0]], 1.0)


@pytest.mark.parametrize("drawn", [False, True])
def test_uniforms_among_tiny_weights(L, drawn):  # noqa: F811
    """Uniforms so small that the aim falls among weights of e^-100."""
    tiny = np.exp(-100.0)
    u = [np.float32(k * 2.0 ** -149) for k in range(1, 200)]
    # the aim in units of the tiny weight, away from where the token changes
    u = [x for x in u if 0.1 < float(x) * (1000 + 8000 * tiny) / tiny % 1 < 0.9 and float(x) * 1000 < 7990 * tiny][:40]
    assert len(u) > 20
    rows = np.stack([[cliff(100)]] * len(u))
    probs = np.full((len(u), 1, 9000), 1 / 9000) if drawn else None
    check(L, rows, [[0]] * len(u), [[-1]] * len(u), probs, [[x] for x in u], 1.0)


def test_what_a_drafts_distribution_leaves_may_be_tiny(L):  # noqa: F811
    """q is above p wherever p has visible mass: max(p - q, 0) has its mass on tokens of e^-100."""
    probs = np.zeros((2, 2, 9000), np.float32)
    probs[:, 1, 8000:] = 0.0011
    check(L, np.stack([[cliff(100)] * 2] * 2), [[0, 8003]] * 2, [[-1, 0]] * 2, probs, [[0.50007, 1 - 2.0 ** -24], [0, 1 - 2.0 ** -24]], 1.0)


# ---- what refused drafts leave ---------------------------------------------


LAST = 1 - 2.0 ** -24


@pytest.mark.parametrize("vocab", [40, 9000])
def test_the_last_token_left_is_accepted(L, vocab):  # noqa: F811
    """Two refused drafts hold all but 1e-14 of the mass: the third is the only token left and is taken at any uniform."""
    seqs, places = 16, [3, 5, vocab - 9]
    rows = np.full((seqs, 4, vocab), -np.inf, np.float32)
    for s in range(seqs):
        rows[s, :, places] = np.array([0.0, -15.5, -31.0 - 0.06 * s], np.float32)[:, None]
    check(L, rows, [[0, *places]] * seqs, [[-1, 0, 0, 0]] * seqs, None, np.full((seqs, 4), LAST), 1.0)


@pytest.mark.parametrize("first", [0.0, 0.25, LAST])
def test_a_chunk_whose_tokens_were_all_refused_is_not_drawn_from(L, first):  # noqa: F811
    seqs = 16
    rows = np.full((seqs, 3, 9000), -np.inf, np.float32)
    for s in range(seqs):
        rows[s, :, [3, 5, 8000]] = np.array([0.0, -22.0 - 0.1 * s, -15.5], np.float32)[:, None]
    check(L, rows, [[0, 3, 5]] * seqs, [[-1, 0, 0]] * seqs, None, [[first, LAST, LAST]] * seqs, 1.0)


def test_what_is_left_beside_a_refused_draft(L):  # noqa: F811
    """The refused draft holds all but 1e-10 of its chunk: the others of the chunk are drawn by their own weights."""
    seqs, vocab = 32, 9000
    rng = np.random.default_rng(3)
    rows = np.full((seqs, 2, vocab), -np.inf, np.float32)
    rows[:, :, 100:140] = -28.0 + rng.normal(size=(seqs, 1, 40))
    rows[:, :, 7] = 0.0
    rows[:, :, 8000] = -15.5
    u = np.full((seqs, 2), LAST, np.float32)
    draft = [[0, 7]] * seqs
    for s in range(seqs):  # an aim among the 40, and away from where the token changes
        while True:
            u[s, 0] = rng.random() * 1e-4
            _, n, _ = S.verify(rows[s], draft[s], [-1, 0], None, u[s], 1.0)
            p = S.target(rows[s, 0], 1.0)
            p[7] = 0.0
            run = np.cumsum(p)
            if 100 <= n < 140 and np.abs(run[99:140] - u[s, 0] * run[-1]).min() > 1e-5 * run[139]:
                break
    check(L, rows, draft, [[-1, 0]] * seqs, None, u, 1.0)


# ---- large scores ----------------------------------------------------------


@pytest.mark.parametrize("hq,hkv,d,tokens", [(4, 1, 64, 1), (4, 1, 64, 3), (16, 4, 64, 25), (32, 8, 128, 1), (8, 1, 128, 1),
                                             (32, 8, 128, 17), (24, 2, 256, 1), (24, 2, 256, 9), (24, 2, 256, 17)])
@pytest.mark.parametrize("size", [1e6, 1e8, 1e11])
@pytest.mark.parametrize("sign", [1, -1])
def test_attention_of_scores_far_beyond_a_unit(L, hq, hkv, d, tokens, size, sign):  # noqa: F811
    """One key of each sequence is far above the others (by a tenth of the scores' size): the row is its value."""
    rng = np.random.default_rng(d + tokens)
    lengths = [40, 300, 2500]
    cache = Cache(L, rng, lengths, tokens, hkv, d, 32)
    cache.k[:] = np.where(np.isnan(cache.k), cache.k, 0)
    for s, n in enumerate(lengths):
        rows = cache.rows(s, 0, n + tokens)
        cache.k[0, rows, :, 0] = rng.integers(900, 1000, (n + tokens, 1)) if sign > 0 else rng.integers(1300, 1400, (n + tokens, 1))
        cache.k[0, rows[n // 3], :, 0] = 1200
    cache.upload()
    q = np.zeros((len(lengths), tokens, hq, d), np.float32)
    q[..., 0] = sign * size / 1000 * (1 + rng.random(q.shape[:3]))
    got = attend(L, cache, q, None, 1.0)
    want = expected(cache, q, None, 1.0)
    assert np.isfinite(got).all()
    # all other weights are below 2^-1000 of the largest; P is 2^15 and V an F16
    np.testing.assert_array_equal(got, want.astype(np.float32))


# ---- values that are not finite --------------------------------------------


@pytest.mark.parametrize("hq,hkv,tokens", [(24, 2, 17), (16, 2, 33), (24, 2, 5)])
def test_attention_values_of_nodes_that_are_not_finite_in_every_sequence(L, hq, hkv, tokens):  # noqa: F811
    """Many short sequences to a CTA, or to a pair of CTAs of which one may be an item ahead: each finds its own nodes."""
    rng = np.random.default_rng(hq + tokens)
    lengths = [int(n) for n in rng.integers(0, 200, 150)]
    cache = Cache(L, rng, lengths, tokens, hkv, 256, 16)
    q = rng.normal(size=(len(lengths), tokens, hq, 256)).astype(np.float32)
    masks = [S.tree_masks([-1] + [int(rng.integers(0, i)) for i in range(1, tokens)]) for _ in lengths]
    clean = expected(cache, q, masks, 0.1)
    odd = np.zeros(clean.shape, bool)
    for s, n in enumerate(lengths):
        node, col = int(rng.integers(1, tokens)), int(rng.integers(256))
        cache.v[0, cache.rows(s, n + node, 1), s % hkv, col] = np.nan
        sees = [t for t in range(tokens) if masks[s][t] >> node & 1]
        odd[s, sees, s % hkv * (hq // hkv) : (s % hkv + 1) * (hq // hkv), col] = True
    cache.upload()
    got = attend(L, cache, q, masks, 0.1, calls=3)
    assert np.isnan(got[odd]).all()
    assert np.isfinite(got[~odd]).all()
    np.testing.assert_allclose(got[~odd], clean[~odd], rtol=0, atol=1e-4 * np.abs(clean).max())


@pytest.mark.parametrize("hq,hkv,d,tokens", [(4, 1, 64, 3), (16, 4, 64, 10), (8, 2, 128, 4), (4, 4, 128, 1), (24, 2, 256, 5), (24, 2, 256, 17)])
@pytest.mark.parametrize("value", [np.inf, -np.inf])
def test_attention_of_infinite_values_of_nodes(L, hq, hkv, d, tokens, value):  # noqa: F811
    """An infinity in a node's value is what the rows that see it have in its column, whatever the other keys are."""
    rng = np.random.default_rng(d + tokens)
    lengths = [0, 20, 77, 100, 126]
    cache = Cache(L, rng, lengths, tokens, hkv, d, 16)
    q = rng.normal(size=(len(lengths), tokens, hq, d)).astype(np.float32)
    for s, n in enumerate(lengths):
        cache.v[0, cache.rows(s, n + tokens // 2, 1), :, 5] = value
    cache.upload()
    got, want = attend(L, cache, q, None, 0.1), expected(cache, q, None, 0.1)
    odd = ~np.isfinite(want)
    assert odd.any()
    np.testing.assert_array_equal(got[odd], want[odd])
    np.testing.assert_allclose(got[~odd], want[~odd], rtol=0, atol=1e-4 * np.abs(want[~odd]).max())


# ---- after a wait that ran out ---------------------------------------------


@pytest.mark.parametrize("hq,hkv,d,tokens", [(8, 8, 128, 1), (16, 4, 64, 5), (32, 8, 128, 17), (24, 2, 256, 1), (24, 2, 256, 17)])
def test_attention_after_an_error_every_row_is_nan_until_the_workspace_is_cleared(L, hq, hkv, d, tokens):  # noqa: F811
    """The error word (the workspace's first) is written from the host, as a wait that ran out would leave it."""
    rng = np.random.default_rng(d + tokens)
    lengths = [20, 700]
    cache = Cache(L, rng, lengths, tokens, hkv, d, 32)
    q = rng.normal(size=(2, tokens, hq, d)).astype(np.float32)
    dq, out = L.Device(q), L.Device(np.zeros(q.shape, np.float32))
    ws = L.attention_workspace(2, tokens, hq, hkv, d)

    def call():
        L.call("tree_attention", out.p, dq.p, C.byref(cache.c), 0, None, 0.1, 2, tokens, hq, ws.p)
        return out.get()

    want = expected(cache, q, None, 0.1)
    assert_parity(call(), want)
    word = np.array([4], np.int32)
    L.call("write", ws.p, word.ctypes.data, 4)
    for _ in range(2):
        assert np.isnan(call()).all()
    L.call("zero", ws.p, ws.nbytes)
    assert_parity(call(), want)

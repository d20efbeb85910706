"""Sampling and truncation of logits on a B200 against their 64-bit definition (oracle/batch.py): the same tokens, the same
kept sets."""
import numpy as np
import pytest

from oracle import batch as B

pytestmark = pytest.mark.gpu

# Weights are whole multiples of 2^-44 of the largest, each off by half of one and 2^-46 of itself at most: n of them put a
# border n * 2^-44 off. Inputs whose border is nearer to a sum than that say nothing, and are asserted not to occur.
STEP = 2.0 ** -44


@pytest.fixture(scope="module")
def L(gpu_lib):
    from nebula_b200 import lib
    return lib


def device(L, values, dtype):
    return None if values is None else L.Device(np.asarray(values, dtype))


def ptr(x):
    return x.p if x is not None else None


def run(L, logits, uniforms, temperature=None, top_k=None, top_p=None, min_p=None, per=1, skip=0):
    """(tokens, truncated logits); `skip`: floats that the rows lie behind a multiple of 16 bytes."""
    logits = np.ascontiguousarray(logits, np.float32)
    rows, vocab = logits.shape
    x = L.Device(np.concatenate([np.full(skip, 5.0, np.float32), logits.ravel(), np.full(5, 7.0, np.float32)]))
    out = L.Device(np.full(logits.size + 8, 3.0, np.float32))
    token, u = L.Device(np.full(rows, -9, np.int32)), L.Device(np.asarray(uniforms, np.float32))
    s = [device(L, temperature, np.float32), device(L, top_k, np.int32), device(L, top_p, np.float32), device(L, min_p, np.float32)]
    at = x.p + 4 * skip
    L.call("sample", token.p, at, u.p, *map(ptr, s), per, rows, vocab)
    L.call("truncate_logits", out.p + 4, at, *map(ptr, s), per, rows, vocab)
    cut = out.get()
    assert (cut[:1] == 3.0).all() and (cut[1 + logits.size:] == 3.0).all()
    L.call("truncate_logits", at, at, *map(ptr, s), per, rows, vocab)  # in place
    both = x.get()
    assert (both[:skip] == 5.0).all() and (both[skip + logits.size:] == 7.0).all()
    np.testing.assert_array_equal(both[skip:skip + logits.size], cut[1:1 + logits.size])
    return token.get(), cut[1:1 + logits.size].reshape(rows, vocab)


def check(L, logits, uniforms, temperature=None, top_k=None, top_p=None, min_p=None, per=1, skip=0):
    tokens, cut = run(L, logits, uniforms, temperature, top_k, top_p, min_p, per, skip)
    f = lambda v, r, d: d if v is None else np.asarray(v, np.float32)[r // per].astype(np.float64)  # noqa: E731
    for r, row in enumerate(np.asarray(logits, np.float32)):
        settings = dict(temperature=float(f(temperature, r, 1.0)), top_k=0 if top_k is None else int(top_k[r // per]),
                        top_p=float(f(top_p, r, 1.0)), min_p=float(f(min_p, r, 0.0)))
        found = B.kept(row, **settings)
        if found is None:
            assert tokens[r] == -1 and np.isnan(cut[r]).all(), (r, settings)
            continue
        best, w, margin = found
        limit = len(row) * STEP
        assert margin > limit, (r, settings, "the inputs' own border")
        want = np.full(len(row), -np.inf, np.float32)
        want[best] = row[best]
        np.testing.assert_array_equal(cut[r], want, err_msg=f"row {r}: {settings}")
        token, margin = B.sample(row, np.float32(uniforms[r]), **settings)
        assert margin > limit or uniforms[r] in (0.0, 1.0)
        assert tokens[r] == token, (r, settings, uniforms[r])


SETTINGS = [(1.0, 0, 1.0, 0.0), (0.8, 40, 0.95, 0.0), (1.0, 0, 0.9, 0.0), (0.7, 0, 1.0, 0.05), (0.0, 7, 0.5, 0.5), (1.3, 200, 1.0, 0.1),
            (0.6, 1, 1.0, 0.0), (2.0, 0, 0.999, 0.0), (1.0, 1000, 0.5, 0.001), (1.0, 0, 0.0, 0.0), (0.05, 0, 0.9, 0.0),
            (30.0, 0, 0.7, 0.0), (1.0, 1 << 30, 1.5, -1.0), (1.0, -5, 0.3, 1.0)]


def peaked(rng, rows, vocab):
    x = 2 * rng.normal(size=(rows, vocab))
    for r in range(rows):
        x[r, rng.integers(0, vocab, 3)] += rng.uniform(4, 12, 3)
    return x


@pytest.mark.parametrize("vocab", [1, 2, 3, 5, 31, 127, 1000, 2045, 2046, 4097, 16381, 50001, 131072, 360445])
def test_vocabularies(L, vocab):
    rng = np.random.default_rng(vocab)
    n = len(SETTINGS) if vocab <= 50001 else 6
    t, k, p, m = zip(*SETTINGS[:n])
    check(L, peaked(rng, n, vocab), rng.random(n), t, k, p, m, skip=vocab % 4)


@pytest.mark.parametrize("skip", [0, 1, 2, 3])
def test_rows_that_start_anywhere(L, skip):
    rng = np.random.default_rng(skip)
    t, k, p, m = zip(*SETTINGS[:7])
    check(L, peaked(rng, 7, 5003), rng.random(7), t, k, p, m, skip=skip)


@pytest.mark.parametrize("steps", [1, 0.25, 0.03125])
def test_equal_logits(L, steps):
    """Heads with 16-bit outputs: many equals, of which the lowest indices are kept."""
    rng = np.random.default_rng(int(100 * steps))
    t, k, p, m = zip(*(SETTINGS + [(1.0, 333, 0.77, 0.0), (1.0, 5000, 0.6, 0.0)]))
    x = np.round(2 * rng.normal(size=(len(t), 30011)) / steps) * steps
    check(L, x, rng.random(len(t)), t, k, p, m)


def test_all_equal_and_signed_zeros(L):
    x = np.zeros((6, 9001), np.float32)
    x[1::2, ::2] = -0.0
    check(L, x, [0.0, 0.3, 0.5001, 0.77, 0.999, 0.1], top_k=[0, 0, 17, 17, 4000, 9000], top_p=[1.0, 0.5001, 1.0, 0.501, 0.33, 0.9])


def test_far_apart(L):
    """Masks of the type's lowest value, huge and tiny logits, temperatures at the ends."""
    rng = np.random.default_rng(3)
    low = np.finfo(np.float32).min
    x = peaked(rng, 8, 3001)
    x[0, ::2] = low
    x[1, :] = low
    x[1, 700] = 1.0
    x[2] = rng.normal(size=3001) * 1e30
    x[3] = rng.normal(size=3001) * 1e-30
    x[4] = -np.exp(rng.normal(size=3001) * 20)
    x[5, :2990] = -np.inf
    x[6] = low
    x[7] = 3e38 * rng.uniform(-1, 1, 3001)
    for t in (1.0, 0.2, 1e20, 1e-20, 1e-42, 3e38):
        check(L, x, rng.random(8), [t] * 8, [0, 0, 50, 0, 0, 40, 100, 0], [0.9, 0.5, 0.9, 0.8, 0.7, 0.95, 0.33, 1.0])
        check(L, x, rng.random(8), [t] * 8, [0, 2000, 0, 0, 0, 1, 0, 900], [1.0] * 8, [0.01, 0.0, 0.0, 0.5, 0.2, 0.0, 0.9, 0.0])


def test_narrow_around_zero_and_negative(L):
    rng = np.random.default_rng(4)
    x = np.stack([rng.normal(size=4099) * 1e-3, -np.abs(rng.normal(size=4099)), -5 - rng.random(4099), np.log(rng.dirichlet(np.full(4099, 0.3)) + 1e-30)])
    for k in (0, 3, 100, 2000, 4098, 4099):
        check(L, x, rng.random(4), None, [k] * 4, [0.4, 0.9, 0.99, 0.8])


def test_refused_rows(L):
    rng = np.random.default_rng(5)
    x = peaked(rng, 8, 2500)
    x[1, 7], x[2, 2499], x[3] = np.nan, np.inf, -np.inf
    check(L, x, rng.random(8), [1, 1, 1, 1, -1, np.nan, np.inf, 1], [3] * 8)
    check(L, x, rng.random(8), [0] * 8, [3] * 8)
    check(L, x, rng.random(8), None, None, [1, 1, 1, 1, np.nan, 0.5, 0.4, 0.3], [0, 0, 0, 0, 0, np.nan, 0.1, 0.2])
    tokens, _ = run(L, x, [np.nan] * 8)
    assert (tokens == -1).all()


def test_uniforms_at_the_ends(L):
    rng = np.random.default_rng(6)
    x = np.tile(rng.normal(size=(1, 6001)), (6, 1))
    tokens, cut = run(L, x, [0.0, -3.0, 1.0, np.inf, 0.99999994, -np.inf], top_k=[50] * 6)
    first, last = np.flatnonzero(cut[0] > -np.inf)[[0, -1]]
    assert list(tokens) == [first, first, last, last, last, first]


def test_settings_of_a_user_for_several_rows(L):
    rng = np.random.default_rng(7)
    check(L, peaked(rng, 14, 4001), rng.random(14), [0.0, 0.8, 1.0], [0, 5, 0], [1.0, 1.0, 0.8], None, per=5)


def test_many_rows(L):
    rng = np.random.default_rng(8)
    n = 700
    pick = [SETTINGS[i] for i in rng.integers(0, len(SETTINGS), n)]
    t, k, p, m = zip(*pick)
    check(L, peaked(rng, n, 8191), rng.random(n), t, k, p, m)


def test_the_tokens_follow_the_distribution(L):
    rng = np.random.default_rng(9)
    row, n = peaked(rng, 1, 300)[0], 20000
    u = (np.arange(n) + 0.5) / n  # every token as often as its probability says, to within one draw
    tokens, _ = run(L, np.tile(row, (n, 1)), u, [0.9] * n, [12] * n)
    best, w, _ = B.kept(np.float32(row), float(np.float32(0.9)), 12)
    counts = np.bincount(tokens, minlength=300)
    assert set(np.flatnonzero(counts)) <= set(int(b) for b in best)
    assert np.abs(counts[best] - w / w.sum() * n).max() <= 1.01


def test_captured_and_replayed(L):
    import ctypes as C
    rng = np.random.default_rng(10)
    x = peaked(rng, 3, 20011).astype(np.float32)
    d, out, token, u = L.Device(x), L.Device(x), L.Device(np.zeros(3, np.int32)), L.Device(np.zeros(3, np.float32))
    p, k = L.Device(np.full(3, 0.9, np.float32)), L.Device(np.full(3, 30, np.int32))
    call = lambda: (L.call("truncate_logits", out.p, d.p, None, k.p, None, None, 1, 3, 20011),  # noqa: E731
                    L.call("sample", token.p, out.p, u.p, None, None, p.p, None, 1, 3, 20011))
    call()
    g = C.c_void_p()
    L.call("graph_begin", C.byref(g))
    call()
    L.call("graph_end", g)
    for i in range(3):
        v = rng.random(3).astype(np.float32)
        x = peaked(rng, 3, 20011).astype(np.float32)
        d.set(x)
        u.set(v)
        L.call("graph_launch", g)
        got = token.get()
        for r in range(3):
            assert got[r] == B.sample(x[r], v[r], top_k=30, top_p=float(np.float32(0.9)))[0]
    L.graph_destroy(g)


def test_fewer_logits_than_asked_for(L):
    """top_k above the number of finite logits leaves them all, to top-p and min_p too."""
    rng = np.random.default_rng(11)
    x = np.full((6, 40000), -np.inf)
    for r, n in enumerate((1, 2, 100, 300, 2000, 9000)):
        x[r, rng.choice(40000, n, replace=False)] = rng.normal(size=n)
    for k in (3, 200, 257, 1000, 5000, 39999):
        check(L, x, rng.random(6), None, [k] * 6, [0.7] * 6)
        check(L, x, rng.random(6), None, [k] * 6, None, [0.2] * 6)
        check(L, x, rng.random(6), None, [k] * 6)


def test_two_graphs_at_once(L):
    """Calls share no memory but their arguments: graphs of both entry points replayed one after the other without a wait."""
    import ctypes as C
    rng = np.random.default_rng(12)
    graphs, bufs = [], []
    for n in range(2):
        x = peaked(rng, 9, 30000).astype(np.float32)
        u = rng.random(9).astype(np.float32)
        d, out, token, du = L.Device(x), L.Device(np.zeros_like(x)), L.Device(np.zeros(9, np.int32)), L.Device(u)
        p = L.Device(np.full(9, 0.9, np.float32))
        g = C.c_void_p()
        L.call("graph_begin", C.byref(g))
        L.call("truncate_logits", out.p, d.p, None, None, p.p, None, 1, 9, 30000)
        L.call("sample", token.p, d.p, du.p, None, None, p.p, None, 1, 9, 30000)
        L.call("graph_end", g)
        graphs.append(g)
        bufs.append((x, u, d, out, token, du, p))
    for _ in range(5):
        for g in graphs:
            L.call("graph_launch", g)
    for x, u, _, out, token, _, _ in bufs:
        cut, got = out.get(), token.get()
        for r in range(9):
            best, _, _ = B.kept(x[r], top_p=float(np.float32(0.9)))
            assert set(np.flatnonzero(cut[r] > -np.inf)) == set(int(b) for b in best)
            assert got[r] == B.sample(x[r], u[r], top_p=float(np.float32(0.9)))[0]
    for g in graphs:
        L.graph_destroy(g)


@pytest.mark.parametrize("rows,vocab", [(60, 4097), (6, 10001), (100, 12288), (6, 12288), (13, 40001), (9, 50001), (6, 20000), (6, 65537),
                                        (6, 24576), (6, 50001), (6, 200000)])
def test_clusters_of_any_size(L, rows, vocab):
    """Rows and lengths for which a row has 2, 5, 1, 6, 7, 9, 10, 11, 12, 13 and 14 CTAs: with borders that come out of a list, of more
    than a list, of min-p within what top-p keeps, and of top-k where it leaves all that is finite."""
    rng = np.random.default_rng(rows * vocab)
    x = peaked(rng, rows, vocab).astype(np.float32)
    chosen = [(1.0, 0, 0.9, 0.0), (1.0, 0, 0.9, 0.002), (3.0, 1000, 0.8, 0.0), (25.0, 0, 0.7, 0.0), (1.5, 2000, 0.9, 0.0), (1.0, 0, 0.98, 1e-4)]
    t, k, p, m = zip(*[chosen[r % 6] for r in range(rows)])
    for r in range(4, rows, 6):
        x[r, rng.permutation(vocab)[:-700]] = -np.inf
    check(L, x, rng.random(rows), t, k, p, m)


def test_min_p_within_a_nucleus_row_after_row(L):
    """More rows than clusters, of one kind, with a border that is found twice."""
    rng = np.random.default_rng(8)
    x = peaked(rng, 400, 8191)
    for least in (0.0005, 0.01):
        check(L, x, rng.random(400), [1.0] * 400, [0] * 400, [0.97] * 400, [least] * 400)


@pytest.mark.parametrize("steps", [1e-6, 0.25])
def test_top_p_of_as_many_as_a_list_holds(L, steps):
    """Where top-p goes through a list of top-k's logits, and through passes over the row: 1,024 of them, and one more; equals at the border."""
    rng = np.random.default_rng(9)
    k = [257, 1023, 1024, 1025, 700, 1024]
    x = np.round(2 * rng.normal(size=(6, 30011)) / steps) * steps
    check(L, x, rng.random(6), [1.0, 2.0, 1.0, 1.0, 0.7, 1e6], k, [0.9, 0.99, 0.5, 0.5, 1e-7, 0.999], [0.0, 0.0, 0.0, 0.0, 0.0, 0.0])

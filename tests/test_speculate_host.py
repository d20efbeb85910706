"""Refusals of the verify step's entry points: every bad argument returns cudaErrorInvalidValue before any launch (no
GPU needed; the pointers are never dereferenced)."""
import ctypes as C

import numpy as np
import pytest

from nebula_b200 import lib as L
from oracle import speculate as S

INVALID = 1
P16, P8, P4 = 1 << 20, (1 << 20) + 8, (1 << 20) + 4


def cache(**over):
    f = dict(k=P16, v=P16, page_table=P16, lengths=P16, layer_bytes=64 * 16 * 2 * 128 * 2, layers=3, pages=64, page_tokens=16,
             table_pages=8, kv_heads=2, head_dim=128)
    f.update(over)
    return C.byref(L.KvCache(**f))


BAD_CACHE = [dict(k=None), dict(v=None), dict(page_table=None), dict(lengths=None), dict(k=P8), dict(v=P4), dict(pages=0),
             dict(page_tokens=8), dict(page_tokens=48), dict(page_tokens=512), dict(table_pages=0), dict(kv_heads=0),
             dict(head_dim=96), dict(head_dim=512), dict(layers=0), dict(layer_bytes=64), dict(layer_bytes=(1 << 20) + 8),
             dict(pages=1 << 28), dict(table_pages=1 << 28)]


def attention(c, **over):
    f = dict(out=P16, q=P16, layer=0, tree=P16, scale=0.1, seqs=2, tokens=4, q_heads=8, ws=P16)
    f.update(over)
    return L.code("tree_attention", f["out"], f["q"], c, f["layer"], f["tree"], f["scale"], f["seqs"], f["tokens"], f["q_heads"],
                  f["ws"])


def prep(c, **over):
    f = dict(q_out=P16, layer=0, q=P16 + 64, qs=1536, k=P16, ks=1536, v=P16, vs=1536, qw=P16, kw=P16, eps=1e-6, rope=P16, rp=128,
             rotary=64, off=None, seqs=2, tokens=4, q_heads=8)
    f.update(over)
    return L.code("qk_norm_rope", f["q_out"], c, f["layer"], f["q"], f["qs"], f["k"], f["ks"], f["v"], f["vs"], f["qw"], f["kw"],
                  f["eps"], f["rope"], f["rp"], f["rotary"], f["off"], f["seqs"], f["tokens"], f["q_heads"])


def commit(c, **over):
    f = dict(out=P16, path=P16, accepted=P16, seqs=2, tokens=4)
    f.update(over)
    return L.code("cache_commit", c, f["out"], f["path"], f["accepted"], f["seqs"], f["tokens"])


def verify(**over):
    f = dict(path=P16, accepted=P16, next=P16, logits=P16, draft=P16, parents=P16, probs=None, uniforms=P16, temperature=1.0,
             seqs=2, tokens=4, vocab=1000, ws=P16)
    f.update(over)
    return L.code("verify_tree", *f.values())


@pytest.mark.parametrize("over", BAD_CACHE, ids=str)
def test_caches_are_refused(over):
    assert attention(cache(**over)) == INVALID
    assert prep(cache(**over)) == INVALID
    assert commit(cache(**over)) == INVALID


@pytest.mark.parametrize("over", [dict(seqs=0), dict(seqs=1025), dict(tokens=0), dict(tokens=65)], ids=str)
def test_batches_are_refused(over):
    assert attention(cache(), **over) == INVALID
    assert prep(cache(), **over) == INVALID
    assert commit(cache(), **over) == INVALID
    assert verify(**over) == INVALID


def test_attention_refuses():
    for over in (dict(out=None), dict(q=None), dict(ws=None), dict(layer=-1), dict(layer=3), dict(q_heads=0), dict(q_heads=1),
                 dict(q_heads=7), dict(q_heads=2048), dict(out=P8), dict(q=P4), dict(tree=P4), dict(ws=P8)):
        assert attention(cache(), **over) == INVALID, over
    assert attention(None) == INVALID
    n = C.c_size_t(0)
    for bad in ((0, 4, 8, 2, 128), (2, 65, 8, 2, 128), (2, 4, 7, 2, 128), (2, 4, 8, 0, 128), (2, 4, 8, 2, 80)):
        assert L.code("attention_workspace_bytes", *bad, C.byref(n)) == INVALID
    assert L.code("attention_workspace_bytes", 2, 4, 8, 2, 128, None) == INVALID
    assert L.code("attention_workspace_bytes", 2, 4, 8, 2, 128, C.byref(n)) == 0 and n.value > 0


def test_preparation_refuses():
    for over in (dict(q_out=None), dict(q=None), dict(k=None), dict(v=None), dict(qw=None), dict(kw=None), dict(eps=-1.0),
                 dict(eps=float("nan")), dict(rope=None), dict(rp=0), dict(rotary=63), dict(rotary=130), dict(rotary=-2),
                 dict(qs=1023), dict(ks=255), dict(vs=0), dict(q_heads=0), dict(q_out=P16 + 64), dict(layer=3), dict(rope=P4)):
        assert prep(cache(), **over) == INVALID, over
    for bad in ((None, 8, 64, 1e4), (P16, 0, 64, 1e4), (P16, 8, 63, 1e4), (P16, 8, 0, 1e4), (P16, 8, 258, 1e4), (P16, 8, 64, 0.0)):
        assert L.code("rope_table", *bad) == INVALID


def test_commit_refuses():
    for over in (dict(out=None), dict(path=None), dict(accepted=None)):
        assert commit(cache(), **over) == INVALID


def test_verify_refuses():
    for over in (dict(path=None), dict(accepted=None), dict(next=None), dict(logits=None), dict(draft=None), dict(parents=None),
                 dict(uniforms=None), dict(ws=None), dict(ws=P8), dict(temperature=-1.0), dict(temperature=float("nan")),
                 dict(temperature=1e-300), dict(temperature=float("inf")), dict(vocab=0), dict(vocab=(1 << 24) + 1)):
        assert verify(**over) == INVALID, over
    n = C.c_size_t(0)
    for bad in ((0, 4, 10), (2, 65, 10), (2, 4, 0)):
        assert L.code("verify_workspace_bytes", *bad, C.byref(n)) == INVALID


# ---- the definitions themselves -------------------------------------------


@pytest.mark.parametrize("given", [True, False])
def test_accepted_tokens_follow_the_target(given):
    """Over all uniforms the first new token has the target's distribution, whatever the drafts were."""
    rng = np.random.default_rng(5)
    logits = rng.normal(size=(4, 6))
    p = S.target(logits[0], 0.7)
    parents = [-1, 0, 0, 0] if given else [-1, 0, 1, 2]
    q = S.target(rng.normal(size=6), 1.0)
    counts, n = np.zeros(6), 20000
    for _ in range(n):
        draft = [0, *rng.permutation(6)[:3]] if given else [0, *rng.choice(6, size=3, p=q)]
        path, nxt, _ = S.verify(logits, draft, parents, None if given else [q] * 4, rng.random(4), 0.7)
        counts[draft[path[1]] if len(path) > 1 else nxt] += 1
    # five standard deviations of a count
    assert np.all(np.abs(counts / n - p) < 5 * np.sqrt(p * (1 - p) / n))


def test_tree_masks_are_the_ancestors():
    assert S.tree_masks([-1, 0, 0, 2, 1]) == [0b1, 0b11, 0b101, 0b1101, 0b10011]
    assert S.tree_masks([-1, 0, 1]) == S.chain_masks(3)

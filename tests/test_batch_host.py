"""The operators for a batch of users, without a GPU: refusals before any launch (the pointers are never dereferenced), and the
definitions that the GPU tests compare with."""
import ctypes as C

import numpy as np
import pytest

from nebula_b200 import lib as L
from oracle import batch as B

INVALID = 1
P4 = 1 << 20


def sample(**over):
    f = dict(token=P4, logits=P4, uniforms=P4, temperature=P4, top_k=P4, top_p=P4, min_p=P4, per=1, rows=4, vocab=1000)
    f.update(over)
    return L.code("sample", *f.values())


def truncate(**over):
    f = dict(out=P4, logits=P4, temperature=P4, top_k=P4, top_p=P4, min_p=P4, per=1, rows=4, vocab=1000)
    f.update(over)
    return L.code("truncate_logits", *f.values())


SIZES = [dict(rows=0), dict(rows=-1), dict(rows=(1 << 20) + 1), dict(vocab=0), dict(vocab=360446), dict(per=0), dict(per=-2)]


UNALIGNED = [dict(logits=P4 + 2), dict(temperature=P4 + 1), dict(top_k=P4 + 2), dict(top_p=P4 + 3), dict(min_p=P4 + 2)]


@pytest.mark.parametrize("over", [dict(token=None), dict(logits=None), dict(uniforms=None), dict(token=P4 + 2), dict(uniforms=P4 + 1), *UNALIGNED,
                                  *SIZES], ids=str)
def test_sample_refuses(over):
    assert sample(**over) == INVALID


@pytest.mark.parametrize("over", [dict(out=None), dict(logits=None), dict(out=P4 + 1), *UNALIGNED, dict(out=P4 + 4),
                                  dict(out=P4 + 4 * 4 * 1000 - 4), dict(out=P4 - 4 * 4 * 1000 + 4), *SIZES], ids=str)
def test_truncate_refuses(over):
    assert truncate(**over) == INVALID


def pool(**over):
    f = dict(page_table=P4, held=P4, free_pages=P4, free_count=P4, pages=100, page_tokens=16, table_pages=20)
    f.update(over)
    return C.byref(L.PagePool(**f))


def reserve(p, **over):
    f = dict(slots=P4, taken=P4 + 4096, lengths=P4, counts=P4, seqs=3, tokens=5)
    f.update(over)
    return L.code("pages_reserve", p, *f.values())


def release(p, **over):
    f = dict(freed=P4 + 4096, lengths=P4, shared=0, seqs=3)
    f.update(over)
    return L.code("pages_release", p, *f.values())


@pytest.mark.parametrize("over", [dict(page_table=None), dict(held=None), dict(free_pages=None), dict(free_count=None), dict(pages=0),
                                  dict(page_tokens=8), dict(page_tokens=20), dict(page_tokens=512), dict(table_pages=0),
                                  dict(pages=1 << 27), dict(table_pages=1 << 27), dict(page_table=P4 + 2), dict(held=P4 + 1),
                                  dict(free_pages=P4 + 2), dict(free_count=P4 + 3)], ids=str)
def test_pools_are_refused(over):
    assert reserve(pool(**over)) == INVALID
    assert release(pool(**over)) == INVALID


def test_pages_refuse():
    assert reserve(None) == INVALID and release(None) == INVALID
    for over in (dict(taken=None), dict(lengths=None), dict(seqs=0), dict(seqs=1025), dict(tokens=0), dict(seqs=1024, tokens=1 << 21),
                 dict(seqs=1, tokens=(1 << 30) + 1), dict(taken=P4 + 2), dict(slots=P4 + 1), dict(lengths=P4 + 2), dict(counts=P4 + 1),
                 dict(taken=P4, lengths=P4, counts=None), dict(taken=P4 + 64, lengths=P4, counts=P4 + 64)):
        assert reserve(pool(), **over) == INVALID, over
    for over in (dict(freed=P4, lengths=P4), dict(freed=P4 + 2), dict(freed=None), dict(lengths=None), dict(seqs=0), dict(seqs=1025), dict(shared=-1), dict(shared=21)):
        assert release(pool(), **over) == INVALID, over


def test_definition_of_what_is_kept():
    row = [1.0, 3.0, -np.inf, 3.0, 2.0]
    keep = lambda **s: sorted(int(i) for i in B.kept(row, **s)[0])  # noqa: E731
    assert keep() == [0, 1, 3, 4]
    assert keep(top_k=1) == [1] and keep(top_k=2) == [1, 3] and keep(top_k=9) == [0, 1, 3, 4]
    assert keep(temperature=0.0) == [1]
    assert keep(top_p=0.0) == [1] and keep(top_p=0.3) == [1] and keep(top_p=0.5) == [1, 3]  # each of the two has 0.399
    assert keep(min_p=0.3) == [1, 3, 4] and keep(min_p=1.0) == [1, 3] and keep(min_p=2.0) == [1]
    assert keep(top_k=2, top_p=0.6) == [1, 3] and keep(top_k=2, top_p=0.4) == [1]
    assert B.sample(row, 0.0)[0] == 0 and B.sample(row, 1.0)[0] == 4 and B.sample(row, 0.5, top_k=2)[0] == 3
    for bad in ([np.nan, 1.0], [np.inf, 1.0], [-np.inf]):
        assert B.kept(bad) is None and B.sample(bad, 0.5)[0] == -1
    assert B.sample(row, np.nan)[0] == -1 and B.kept(row, temperature=-1.0) is None and B.kept(row, top_p=np.nan) is None


def test_definition_of_pages():
    p = B.Pages([[9, 0, 0], [8, 7, 0]], [1, 2], [1, 2, 3], 16)
    taken, slots = p.reserve([16, 30], [2, 2], 2, 10)
    assert taken == [1, 0] and p.stack == [1, 2] and p.table[0][:2] == [9, 3]
    assert slots == [[48, 49], [7 * 16 + 14, 7 * 16 + 15]]
    assert p.release([5, -1], 0, 10) == [1, 2] and p.stack == [1, 2, 7, 8, 3] and p.held == [1, 0]
    assert p.reserve([-1, 0], [1, 3], 2, 10)[0] == [-1, -1]
    assert p.reserve([40, 0], [2, 2], 2, 10)[0] == [2, 1] and p.stack == [1, 2]
    assert p.reserve([40, 16], [2, 2], 2, 10)[0] == [0, 1]
    p.held[0] = 0
    assert p.reserve([40, 16], [2, 2], 2, 10)[0] == [-2, 0]


def cache(**over):
    f = dict(k=P4, v=P4, page_table=P4, lengths=P4, layer_bytes=64 * 16 * 2 * 128 * 2, layers=3, pages=64, page_tokens=16,
             table_pages=8, kv_heads=2, head_dim=128)
    f.update(over)
    return C.byref(L.KvCache(**f))


def attention(c, **over):
    f = dict(out=P4 + (1 << 24), q=P4, layer=0, shared=P4, tree=P4, scale=0.1, seqs=2, tokens=4, q_heads=8, ws=P4)
    f.update(over)
    return L.code("shared_attention", f["out"], f["q"], c, f["layer"], f["shared"], f["tree"], f["scale"], f["seqs"], f["tokens"], f["q_heads"],
                  f["ws"])


@pytest.mark.parametrize("over", [dict(k=None), dict(v=None), dict(page_table=None), dict(lengths=None), dict(k=P4 + 8), dict(pages=0),
                                  dict(page_tokens=8), dict(page_tokens=512), dict(table_pages=0), dict(kv_heads=0), dict(head_dim=96),
                                  dict(layers=0), dict(layer_bytes=64), dict(pages=1 << 28), dict(table_pages=1 << 28)], ids=str)
def test_shared_attention_refuses_caches(over):
    assert attention(cache(**over)) == INVALID


@pytest.mark.parametrize("over", [dict(out=None), dict(q=None), dict(shared=None), dict(ws=None), dict(layer=-1), dict(layer=3), dict(q_heads=0),
                                  dict(q_heads=7), dict(q_heads=2048), dict(out=P4 + 8), dict(q=P4 + 4), dict(tree=P4 + 4), dict(ws=P4 + 8),
                                  dict(out=P4), dict(out=P4 + 2 * 4 * 8 * 128 * 4 - 16), dict(out=P4, q=P4 + 16), dict(shared=P4 + 2),
                                  dict(seqs=0), dict(seqs=1025), dict(tokens=0), dict(tokens=65), dict(scale=float("inf")),
                                  dict(scale=float("nan")), dict(seqs=1024, tokens=64, q_heads=258)], ids=str)
def test_shared_attention_refuses(over):
    assert attention(cache(), **over) == INVALID


def test_shared_attention_workspace():
    n = C.c_size_t(0)
    for bad in ((0, 4, 8, 2, 128), (1025, 4, 8, 2, 128), (2, 65, 8, 2, 128), (2, 4, 7, 2, 128), (2, 4, 8, 0, 128), (2, 4, 8, 2, 80),
                (1024, 64, 512, 2, 128)):
        assert L.code("shared_attention_workspace_bytes", *bad, C.byref(n)) == INVALID
    assert L.code("shared_attention_workspace_bytes", 2, 4, 8, 2, 128, None) == INVALID
    assert L.code("shared_attention_workspace_bytes", 2, 4, 8, 2, 128, C.byref(n)) == 0 and n.value > 0
    assert L.code("shared_attention_workspace_bytes", 1024, 64, 256, 2, 256, C.byref(n)) == 0 and n.value > 1 << 34

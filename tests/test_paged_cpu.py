"""The cache in pages and trees of drafted tokens where no GPU is needed: every refusal of their C entry points
(they check their arguments before they ask for a context, so these calls launch nothing), and the oracle's own
properties."""
import ctypes
import os
import re
import subprocess

import numpy as np
import pytest

from oracle import paged as O
from tests.conftest import ROOT
from tests.test_integration_examples import NOTES, THERE, blocks, header_members, same_kind
from zwhisper_b200 import _lib

P = 1 << 20  # an aligned address that is never read: each call is refused before a launch
BIG = 1 << 62


def seqs(n_batch=2, n=3, n_past=5, past=None, count=None, first=None):
    return _lib.SeqsC(n_batch, n, n_past, past, count, first)


def rows(data=P, batch=3 * 4 * 64, token=4 * 64):
    return _lib.RowsC(data, batch, token)


def cache(**kw):
    d = dict(k=P, v=P, type=_lib.ZWG_TYPE_F16, table=P, table_stride=4, n_batch=2, n_head_kv=2, d=64, page=16, n_pages=9,
             max_pages=4, page_stride=2 * 16 * 64)
    d.update(kw)
    return _lib.PagedC(*[d[n] for n, _ in _lib.PagedC._fields_])


def tables(**kw):
    d = dict(cos=P, sin=P, n_ctx=64, rot=64, interleaved=0)
    d.update(kw)
    return _lib.RopeTablesC(*[d[n] for n, _ in _lib.RopeTablesC._fields_])


def refused(rc, *words):
    assert rc == _lib.ZWG_ERROR
    for w in words:
        assert w in _lib.last_error(), _lib.last_error()


def ref(x):
    return None if x is None else ctypes.byref(x)


def append(c=None, s=None, tree=None, kind=0, k=None, v=None, t=None, heads=4, q=None, q_out=None):
    return _lib.load().zwg_paged_append(ref(c or cache()), ref(s or seqs()), ref(tree), kind, ref(k or rows()), ref(v or rows()),
                                        ref(t), heads, ref(q), ref(q_out), None)


def attn(c=None, s=None, tree=None, kind=0, heads=4, q=None, out=None, ws=None, size=0):
    return _lib.load().zwg_paged_attn(ref(c or cache()), ref(s or seqs()), ref(tree), kind, heads, ref(q or rows()),
                                      ref(out or rows()), ws, size, None)


def accept(s=None, tree=None, bufs=(P, P, P, P, P)):
    return _lib.load().zwg_tree_accept(ref(s or seqs()), ref(tree or _lib.TreeC(P, 0)), *bufs, None)


def keep(caches=None, s=None, path=P, n_path=P):
    caches = [cache()] if caches is None else caches
    return _lib.load().zwg_paged_keep(b"".join(bytes(c) for c in caches), len(caches), ref(s or seqs()), path, n_path, None)


BAD_CACHE = [
    (dict(k=None), "null cache"), (dict(table=None), "null cache"), (dict(type=0), "F16"), (dict(type=7), "F16"),
    (dict(k=P + 8), "16-byte"), (dict(v=P + 2), "16-byte"), (dict(table=P + 2), "4-byte"), (dict(d=96), "d = 96"),
    (dict(page=8), "page = 8"), (dict(page=24), "page = 24"), (dict(page=512), "page = 512"), (dict(page=0), "page = 0"),
    (dict(n_pages=0), "n_pages"), (dict(n_pages=BIG), "n_pages"), (dict(max_pages=0), "max_pages"), (dict(max_pages=1 << 26), "max_pages"),
    (dict(max_pages=BIG), "max_pages"), (dict(n_head_kv=0), "n_head_kv"), (dict(n_head_kv=40000), "65535"),
    (dict(n_batch=BIG), "65535"), (dict(page_stride=2047), "page_stride"), (dict(page_stride=2056 - 16), "page_stride"),
    (dict(page_stride=2052), "page_stride"), (dict(page_stride=1 << 61), "page_stride"), (dict(table_stride=3), "table_stride"),
    (dict(table_stride=BIG), "table_stride"),
]


@pytest.mark.parametrize("bad,word", BAD_CACHE)
def test_caches_that_every_call_refuses(bad, word):
    for call in (append, attn):
        refused(call(c=cache(**bad)), word)
    refused(keep([cache(**bad)]), word)
    assert _lib.load().zwg_paged_attn_workspace(ref(cache(**bad)), ref(seqs()), 4) == 0


def test_refusals():
    for call in (append, attn):
        refused(call(kind=1), "type")
        refused(call(kind=_lib.ZWG_TYPE_BF16), "f32 rows go with an f16 cache")
        refused(call(c=cache(type=_lib.ZWG_TYPE_BF16)), "f32 rows go with an f16 cache")
        refused(call(s=seqs(n_past=62)), "context full")
        refused(call(s=seqs(n_past=BIG)), "context full")
        refused(call(s=seqs(past=P + 1)), "aligned")
        refused(call(s=seqs(n_batch=3)), "3 sequences")
        refused(call(s=seqs(n=1 << 31)), "too many")
        refused(call(tree=_lib.TreeC(None, 0)), "null parents")
        refused(call(tree=_lib.TreeC(P + 2, 0)), "aligned")
        refused(call(tree=_lib.TreeC(P, BIG)), "stride")
        refused(call(c=cache(max_pages=64, table_stride=64), s=seqs(n=257), tree=_lib.TreeC(P, 0)), "a tree of 257")
        assert call(s=seqs(n=0)) == 0
    refused(append(k=rows(data=None)), "null k")
    refused(append(v=rows(data=P + 1)), "aligned")
    refused(append(k=rows(batch=BIG)), "strides")
    refused(append(t=tables(rot=66)), "rot")
    refused(append(t=tables(n_ctx=7)), "rotary tables")
    refused(append(q=rows()), "without rotary")
    refused(append(q_out=rows()), "q_out without q")
    refused(append(t=tables(), q=rows(data=None)), "null q")
    refused(append(t=tables(), q=rows(), heads=0), "head")
    refused(append(t=tables(), q=rows(), heads=BIG), "head")
    refused(append(t=tables(), q=rows(), q_out=rows(token=255)), "overlap")
    refused(append(t=tables(), q=rows(token=0)), "overlap")
    refused(attn(heads=3), "n_head 3")
    refused(attn(heads=0), "n_head 0")
    refused(attn(heads=1 << 29), "query rows")
    refused(attn(q=rows(data=None)), "null q")
    refused(attn(out=rows(token=128)), "overlap")
    refused(accept(s=seqs(n=300)), "a tree of 300")
    refused(accept(tree=_lib.TreeC(None, 0)), "null parents")
    refused(accept(bufs=(P, P, None, P, P)), "null buffer")
    refused(accept(bufs=(P, P, P, P + 2, P)), "alignment")
    refused(keep(s=seqs(n_batch=3)), "3 sequences")
    refused(keep(s=seqs(n_past=65)), "context full")
    refused(keep(path=None), "null path")
    refused(keep(n_path=None), "null path")
    refused(keep(path=P + 2), "aligned")
    refused(keep([cache(max_pages=64, table_stride=64)], s=seqs(n=257)), "257 tokens")
    refused(keep([cache(), cache(page=32, page_stride=4096)]), "cache 1 differs")
    refused(keep([cache(), cache(), cache(table=P + 16)]), "cache 2 differs")
    assert keep([]) == 0 and keep(s=seqs(n=0)) == 0
    assert _lib.load().zwg_paged_attn(None, ref(seqs()), None, 0, 4, ref(rows()), ref(rows()), None, 0, None) == _lib.ZWG_ERROR
    assert _lib.load().zwg_tree_accept(None, None, P, P, P, P, P, None) == _lib.ZWG_ERROR


def test_one_buffer_twice():
    """Rows that are moved or written twice in one call would race: refused, wherever the buffer comes again."""
    one, two, three = cache(k=P, v=P + 16), cache(k=P + 32, v=P + 48), cache(k=P + 64, v=P)
    refused(keep([one, two, one]), "buffer of cache 2 is given twice")
    refused(keep([one, two, three]), "buffer of cache 2 is given twice")
    refused(keep([two, cache(k=P, v=P)]), "buffer of cache 1 is given twice")
    refused(append(c=cache(k=P, v=P)), "one buffer")


def test_a_tree_of_one_line_is_a_chunk():
    for past, n, first in ((0, 1, 0), (5, 7, 2), (3, 4, 9)):
        line = list(range(-1, n - 1))
        np.testing.assert_array_equal(O.seen_slots(past, n, first, past + n + 2), O.seen_slots(past, n, first, past + n + 2, line))
        np.testing.assert_array_equal(O.positions(past, n), O.positions(past, n, line))


def test_acceptance_by_hand():
    #        0
    #      1   2      tokens below each
    #     3 4   5
    parent = [-1, 0, 0, 1, 1, 2]
    tokens = [9, 4, 7, 1, 2, 2]
    assert O.accept(tokens, [7, 0, 2, 0, 0, 6], parent) == ([0, 2, 5], 6)
    assert O.accept(tokens, [4, 2, 2, 0, 8, 6], parent) == ([0, 1, 4], 8)
    assert O.accept(tokens, [5, 2, 2, 0, 8, 6], parent) == ([0], 5)
    assert O.accept([9, 4, 4], [4, 0, 1], [-1, 0, 0]) == ([0, 1], 0)   # the lower of two equal ones
    assert O.accept([9, 9], [9, 1], [-1, -1]) == ([0], 9)              # another root is never below


def test_the_oracles_attention_is_the_softmax_of_seen_keys():
    rng = np.random.default_rng(0)
    q, k, v = rng.standard_normal((2, 4, 8)), rng.standard_normal((2, 5, 8)), rng.standard_normal((2, 5, 8))
    seen = np.array([[1, 0, 1, 0, 0], [0, 0, 0, 0, 0]], bool)
    out, tol = O.attention(q, k, v, seen, 0, 0.0, False)
    for h in range(4):
        s = np.exp(k[h // 2, [0, 2]] @ q[0, h] / np.sqrt(8))
        np.testing.assert_allclose(out[0, h], s @ v[h // 2, [0, 2]] / s.sum(), rtol=1e-12)
    assert not out[1].any() and (tol > 0).all()


# ---- the integration notes' examples, as tests/test_integration_examples.py takes the others ----

EXAMPLES = [  # the text it starts with, what is there
    ("zwg_paged c = {", "size_t n_seq, size_t n_pages, void* k_pool, void* v_pool, const int32_t* table, zwg_seqs s, zwg_rows q, "
     "zwg_rows k, zwg_rows v, zwg_rows out, zwg_rope_tables tables, void* ws, size_t ws_bytes, void* stream"),
    ("zwg_tree tree = {", "size_t n, size_t n_seq, size_t n_layer, size_t n_vocab, size_t l, const int32_t* parent, zwg_paged* cache, zwg_seqs s, "
     "zwg_rows q, zwg_rows k, zwg_rows v, zwg_rows out, zwg_rope_tables tables, zwg_logit_rules rules, float* logits, int32_t* ids, "
     "const int32_t* tokens, int32_t* path, int32_t* n_path, int32_t* next, void* ws, size_t ws_bytes, void* stream"),
]


@pytest.mark.parametrize("starts,there", EXAMPLES)
def test_c_example(tmp_path, starts, there):
    code, = [b for b in blocks("C") if b.startswith(starts)]
    src = tmp_path / "example.c"
    src.write_text(f"{THERE}\nvoid example({there});\nvoid example({there})\n{{\n{code}\n}}\n")
    out = subprocess.run(["gcc", "-std=c11", "-Wall", "-Wextra", "-Werror", "-Wno-missing-field-initializers", "-Wno-unused-function",
                          "-Wno-unused-parameter", "-fsyntax-only", "-I", os.path.join(ROOT, "include"), str(src)], capture_output=True,
                         text=True)
    assert out.returncode == 0, out.stderr


def test_every_example_is_here():
    assert len(blocks("C")) == len(EXAMPLES)


@pytest.mark.parametrize("zig,c", [("Paged", "zwg_paged"), ("Tree", "zwg_tree")])
def test_zig_structs(zig, c):
    body, = re.findall(r"const " + zig + r" = extern struct \{(.*?)\}", NOTES, flags=re.S)
    got = [tuple(x.strip() for x in m.split(":", 1)) for m in body.split(",") if m.strip()]
    want = header_members(c)
    assert [n for n, _ in got] == [n for n, _ in want]
    for (n, z), (_, k) in zip(got, want):
        assert same_kind(z, k), (n, z, k)


def test_every_call_is_declared_for_zig():
    declared = set(re.findall(r'extern "c" fn (zwg_\w+)\(', NOTES))
    assert {n for n in _lib.SIGNATURES if n.startswith(("zwg_paged", "zwg_tree"))} <= declared

"""The decode step over a cache in 8 bits where no GPU is needed: every refusal of its C entry
points (they check their arguments before they ask for a context, so these calls launch
nothing), the oracle's own properties, and the scaled rotary tables against the formulas."""
import ctypes

import numpy as np
import pytest

from oracle import kv8 as O
from zwhisper_b200 import _lib, ops

P = 1 << 20  # an aligned address that is never read: each call is refused before a launch


def seqs(n_batch=2, n=3, n_past=5, past=None, count=None, first=None):
    return _lib.SeqsC(n_batch, n, n_past, past, count, first)


def rows(data=P, batch=3 * 4 * 64, token=4 * 64):
    return _lib.RowsC(data, batch, token)


def cache(**kw):
    d = dict(k=P, k_scale=P, v=P, v_scale=P, k_open=P, v_open=P, open_block=P, n_batch=2, n_head_kv=2, d=64, n_ctx=64)
    d.update(kw)
    return _lib.Kv8C(*[d[n] for n, _ in _lib.Kv8C._fields_])


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


def call_rope(s=None, t=None, kind=0, d=64, heads=4, q=None, q_out=None, heads_kv=0, k=None, k_out=None):
    return _lib.load().zwg_rope(ref(s or seqs()), ref(t or tables()), kind, d, heads, ref(q or rows()), ref(q_out), heads_kv,
                                ref(k), ref(k_out), None)


def test_rope_refusals():
    refused(call_rope(kind=1), "type")
    refused(call_rope(t=tables(rot=63)), "rot")
    refused(call_rope(t=tables(rot=0)), "rot")
    refused(call_rope(t=tables(rot=66)), "rot")
    refused(call_rope(t=tables(cos=None)), "null rotary")
    refused(call_rope(t=tables(sin=P + 2)), "aligned")
    refused(call_rope(s=seqs(n_past=62)), "context full")
    refused(call_rope(s=seqs(past=P, n_past=65)), "context full")
    refused(call_rope(s=seqs(count=P + 1)), "aligned")
    refused(call_rope(heads=0), "head")
    refused(call_rope(q=rows(data=None)), "null q")
    refused(call_rope(q=rows(data=P + 2)), "aligned")
    refused(call_rope(q=rows(token=255)), "overlap")
    refused(call_rope(q_out=rows(batch=2 * 4 * 64)), "overlap")
    refused(call_rope(q=rows(token=0), q_out=rows(token=0)), "overlap")
    refused(call_rope(k_out=rows()), "k_out without k")
    refused(call_rope(s=seqs(n_batch=1 << 16, n=1 << 16)), "too many")
    # nothing to do is fine without a context; a whole call asks for one
    assert call_rope(s=seqs(n=0)) == 0 and call_rope(s=seqs(n_batch=0)) == 0


def call_append(c=None, s=None, kind=0, k=None, v=None, t=None):
    return _lib.load().zwg_kv8_append(ref(c or cache()), ref(s or seqs()), kind, ref(k or rows()), ref(v or rows()), ref(t), None)


def call_attn(c=None, s=None, kind=0, heads=4, q=None, out=None, ws=None, size=0):
    return _lib.load().zwg_kv8_attn(ref(c or cache()), ref(s or seqs()), kind, heads, ref(q or rows()), ref(out or rows()), ws,
                                    size, None)


def test_kv8_refusals():
    for bad, word in ((dict(k=None), "null cache"), (dict(open_block=None), "null cache"), (dict(v=P + 8), "16-byte"),
                      (dict(k_open=P + 4), "16-byte"), (dict(k_scale=P + 2), "4-byte"), (dict(d=96), "d = 96"),
                      (dict(n_ctx=48), "n_ctx"), (dict(n_ctx=0), "n_ctx"), (dict(n_head_kv=0), "n_head_kv"),
                      (dict(n_head_kv=40000), "65535")):
        refused(call_append(c=cache(**bad)), word)
        refused(call_attn(c=cache(**bad)), word)
        refused(_lib.load().zwg_kv8_read(ref(cache(**bad)), ref(seqs()), P, P, None), word)
        assert _lib.load().zwg_kv8_attn_workspace(ref(cache(**bad)), ref(seqs()), 4) == 0
    for call in (call_append, call_attn):
        refused(call(kind=3), "type")
        refused(call(s=seqs(n_past=62)), "context full")
        refused(call(s=seqs(n_past=1 << 40)), "context full")
        refused(call(s=seqs(n_batch=3)), "3 sequences")
    refused(call_append(k=rows(data=None)), "null k")
    refused(call_append(v=rows(data=P + 1)), "aligned")
    refused(call_append(t=tables(rot=66)), "rot")
    refused(call_append(t=tables(n_ctx=7)), "rotary tables")
    refused(call_attn(heads=3), "n_head 3")
    refused(call_attn(heads=0), "n_head 0")
    refused(call_attn(q=rows(data=None)), "null q")
    refused(call_attn(out=rows(token=128)), "overlap")
    refused(_lib.load().zwg_kv8_read(ref(cache()), ref(seqs()), P + 4, P, None), "16-byte")
    assert call_append(s=seqs(n=0)) == 0 and call_attn(s=seqs(n=0)) == 0


def call_logits(m=2, V=100, stride=100, out=P, out_stride=1, logits=P, **kw):
    r = _lib.LogitRulesC()
    r.repeat = 1.0
    for k, v in kw.items():
        setattr(r, k, v)
    return _lib.load().zwg_llm_logits(logits, m, V, stride, ctypes.byref(r), out, out_stride, None)


def test_logits_refusals():
    refused(call_logits(V=0), "sizes")
    refused(call_logits(logits=None), "null logits")
    refused(call_logits(stride=99), "stride")
    refused(call_logits(n_recent=3, window=3), "recent")
    refused(call_logits(n_bias=2, bias_ids=P), "null biases")
    refused(call_logits(n_bias=4097, bias_ids=P, bias=P), "4096")
    for name in ("repeat", "presence", "frequency"):
        refused(call_logits(**{name: float("nan")}), "finite")
    refused(call_logits(repeat=0.0), "positive")
    refused(call_logits(out_stride=0), "stride")
    refused(call_logits(logits=P + 2), "alignment")
    assert call_logits(m=0) == 0


def test_states_refuse_sizes():
    lib, h = _lib.load(), ctypes.c_void_p()
    assert lib.zwg_llm_state_create_kv8(1, 1, 2, 1, 64, 64, 16, 1e6, None) == _lib.ZWG_ERROR
    assert lib.zwg_llm_state_set_rope(None, P, P, None) == _lib.ZWG_ERROR
    assert lib.zwg_llm_state_kv8(None, 0, ctypes.byref(cache())) == _lib.ZWG_ERROR
    assert not h.value


@pytest.mark.parametrize("split", [[70], [1] * 70, [31, 1, 1, 37], [32, 32, 6], [5, 64, 1]])
def test_oracle_cache_does_not_depend_on_the_split(split):
    rng = np.random.default_rng(0)
    k, v = (rng.standard_normal((2, 70, 2, 64)).astype(np.float32) for _ in range(2))
    whole, parts = O.Cache(2, 2, 64, 96), O.Cache(2, 2, 64, 96)
    whole.append(k, v, [0, 0])
    at = 0
    for n in split:
        parts.append(k[:, at:at + n], v[:, at:at + n], [at, at])
        at += n
    for a, b in ((whole.ints, parts.ints), (whole.scale, parts.scale), (whole.tag, parts.tag)):
        np.testing.assert_array_equal(a, b)
    # a rounding is off by at most half a step of its block
    x = np.stack([k, v]).transpose(0, 1, 3, 2, 4)
    step = np.repeat(whole.scale, 32, -1)[..., :70, None]
    assert (np.abs(whole.values(np.float64)[..., :70, :] - x) <= 0.5001 * step).all()


def test_scaled_rope_tables():
    n, rot, base = 50, 64, 1e4
    plain = ops.rope_tables(n, rot, base)
    for a, b in zip(ops.scaled_rope_tables(n, rot, base), plain):
        np.testing.assert_allclose(a, b, atol=1e-6)  # both are roundings of f64 angles up to 50
    # linear: position 4 p turns as position p
    for a, b in zip(ops.scaled_rope_tables(4 * n, rot, base, "linear", 4.0), plain):
        np.testing.assert_allclose(a[::4], b, atol=1e-6)
    # ntk: the fastest pair stays, the slowest slows by the factor
    i = np.arange(rot // 2)
    inv = base ** (-2.0 * i / rot)

    def speed(*a, **kw):
        cos, sin = ops.scaled_rope_tables(2, rot, base, *a, **kw)
        return np.arctan2(sin[1], cos[1])

    got = speed("ntk", 8.0)
    np.testing.assert_allclose(got[0], 1.0, rtol=1e-6)
    np.testing.assert_allclose(got[-1], inv[-1] / 8, rtol=1e-5)
    got = speed("bands", 8.0, n_train=2048)
    turns = 2048 * inv / (2 * np.pi)
    np.testing.assert_allclose(got[turns > 4], inv[turns > 4], rtol=1e-6)
    np.testing.assert_allclose(got[turns < 1], inv[turns < 1] / 8, rtol=1e-5)
    mid = (turns > 1) & (turns < 4)
    assert mid.any() and (got[mid] < inv[mid]).all() and (got[mid] > inv[mid] / 8).all()
    cos, sin = ops.scaled_rope_tables(3, rot, base, "yarn", 4.0, n_train=2048, low=1.0, high=32.0)
    np.testing.assert_allclose(np.hypot(cos, sin), 0.1 * np.log(4.0) + 1, rtol=1e-6)
    got = speed("yarn", 4.0, n_train=2048, low=1.0, high=32.0, attn_factor=1.0)
    np.testing.assert_allclose(got[turns > 64], inv[turns > 64], rtol=1e-6)
    np.testing.assert_allclose(got[turns < 0.5], inv[turns < 0.5] / 4, rtol=1e-5)
    for bad in (dict(scaling="cubic"), dict(scaling="bands"), dict(factor=0.0)):
        with pytest.raises(ValueError):
            ops.scaled_rope_tables(n, rot, base, **bad)
    with pytest.raises(ValueError):
        ops.scaled_rope_tables(n, 63, base)


def test_oracle_logits():
    x = np.array([1.0, -1.0, 0.0, 2.0], np.float32)
    y, i = O.logits(x, [0, 0, 1], 3, 2.0, 0.5, 0.25, [2, 2], [1.0, 2.0], np.array([0b0111], np.uint32))
    np.testing.assert_allclose(y, [0.5 - 1.0, -2.0 - 0.75, 3.0, -np.inf])
    assert i == 2
    assert O.logits(x, [], 0, 1, 0, 0, [], [], np.zeros(1, np.uint32))[1] == -1

"""The key/value cache in pages on the device (zwg_paged_append, _attn, _keep, zwg_tree_accept) against
oracle/paged.py. Rotated rows and the cache's contents are compared bit for bit: they are the same f32
operations and one rounding. The attention is held to the bound that oracle/paged.py derives for each output."""
import numpy as np
import pytest

from oracle import paged as O
from tests.conftest import has_gpu

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def env():
    if not has_gpu():
        pytest.fail("needs a CUDA device")
    import torch

    from zwhisper_b200 import ops
    ops.set_math("f32")
    return torch, ops


def up(torch, a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a)).to("cuda:0")
    return t if dtype is None else t.to(dtype)


def normal(rng, *shape):
    return rng.standard_normal(shape, dtype=np.float32)


def i32(torch, a):
    return torch.tensor(np.asarray(a).tolist(), dtype=torch.int32, device="cuda:0")


def tree_of(rng, n):
    """Parents: a root, later tokens below earlier ones, a second root now and then."""
    return [-1] + [int(rng.integers(max(0, i - 6), i)) if rng.random() > 0.05 else -1 for i in range(1, n)]


class World:
    """A cache whose pages are handed out in no order, and its contents in the order of slots."""

    def __init__(self, torch, ops, rng, B, Hkv, d, page, slots, bf16, spare=3, joint=False):
        self.torch, self.rng, self.B, self.Hkv, self.d, self.page = torch, rng, B, Hkv, d, page
        per = -(-slots // page)
        self.slots, pool = per * page, B * per + spare
        self.held = torch.bfloat16 if bf16 else torch.float16
        self.row = torch.bfloat16 if bf16 else torch.float32
        table = np.full((B, per + 2), -1, np.int64)
        table[:, :per] = rng.permutation(pool)[: B * per].reshape(B, per)
        self.np_table = table
        pools = up(torch, normal(rng, pool, 2, Hkv, page, d) * np.exp(0.4 * normal(rng, 1, 2, Hkv, 1, d)), self.held)
        k, v = pools[:, 0], pools[:, 1]
        if not joint:
            k, v = k.contiguous(), v.contiguous()
        self.cache = ops.PagedCache(k, v, i32(torch, table))

    def contents(self, dtype=np.float32):
        """k, v [n_batch][n_head_kv][slots][d], the last two pages of a table left out."""
        out = []
        for t in (self.cache.k, self.cache.v):
            x = t.float().cpu().numpy()[np.maximum(self.np_table[:, : self.slots // self.page], 0)]
            out.append(np.moveaxis(x, 2, 1).reshape(self.B, self.Hkv, self.slots, self.d).astype(dtype))
        return out


def check_attn(torch, out, before, world, q, past, count, first, parents, pieces, big=None):
    k, v = world.contents(np.float64)
    qn, got, old = q.float().cpu().numpy(), out.float().cpu().numpy(), before.float().cpu().numpy()
    n, H = q.shape[1], q.shape[2]
    half = 2.0 ** -8 if q.dtype is torch.bfloat16 else 2.0 ** -24
    for b in range(world.B):
        m = int(count[b])
        np.testing.assert_array_equal(got[b, m:], old[b, m:])
        seen = O.seen_slots(int(past[b]), m, int(first[b]), world.slots, None if parents is None else parents[b])
        want, tol = O.attention(qn[b, :m], k[b], v[b], seen, pieces, half, n * H // world.Hkv > 16)
        bad = ~(np.abs(got[b, :m] - want) <= tol)
        assert not bad.any(), (b, np.argwhere(bad)[:3], np.abs(got[b, :m] - want)[bad][:3], tol[bad][:3])


ATTN = [  # batch, n, heads, heads_kv, d, page, past (most), tree
    (1, 1, 1, 1, 64, 16, 0, False), (2, 1, 6, 1, 128, 16, 1, False), (3, 1, 14, 2, 64, 32, 15, False),
    (2, 1, 12, 2, 128, 64, 16, False), (2, 1, 8, 8, 64, 16, 17, False), (1, 1, 16, 1, 128, 256, 300, False),
    (2, 1, 12, 2, 128, 16, 1500, False), (1, 1, 12, 2, 128, 128, 9000, False), (3, 1, 24, 1, 64, 16, 700, False),
    (2, 3, 14, 2, 64, 32, 33, False), (3, 2, 4, 4, 128, 16, 127, False), (2, 5, 12, 2, 128, 64, 259, False),
    (2, 17, 14, 2, 64, 16, 0, False), (2, 40, 4, 2, 128, 32, 100, False), (2, 130, 6, 1, 64, 16, 3, False),
    (1, 97, 12, 2, 128, 256, 1000, False), (2, 256, 2, 1, 64, 64, 130, False), (1, 300, 2, 2, 128, 16, 17, False),
    (1, 1, 6, 1, 64, 16, 0, True), (2, 2, 12, 2, 128, 16, 15, True), (2, 25, 12, 2, 128, 16, 400, True),
    (3, 24, 14, 2, 64, 32, 31, True), (2, 61, 14, 2, 64, 16, 129, True), (1, 64, 4, 4, 128, 128, 1500, True),
    (1, 256, 2, 1, 64, 32, 65, True), (2, 140, 6, 2, 128, 64, 0, True),
]


@pytest.mark.parametrize("B,n,H,Hkv,d,page,most,tree", ATTN)
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("ragged", [False, True])
def test_attn(env, B, n, H, Hkv, d, page, most, tree, bf16, ragged):
    torch, ops = env
    rng = np.random.default_rng(B * n + H + most)
    w = World(torch, ops, rng, B, Hkv, d, page, most + n, bf16, joint=ragged)
    past = rng.integers(0, most + 1, B) if ragged else np.full(B, most)
    count = rng.integers(0, n + 1, B) if ragged else np.full(B, n)
    first = np.minimum(rng.integers(0, most + 3, B), past + n + 2) if ragged else np.zeros(B, int)
    if ragged:
        past[-1], count[0] = most, n
    parents = [tree_of(rng, n) for _ in range(B)] if tree else None
    q = up(torch, 1.5 * normal(rng, B, n, H, d), w.row)
    before = up(torch, normal(rng, B, n, H, d), w.row)
    args = dict(count=i32(torch, count), first=i32(torch, first), max_past=most) if ragged else {}
    if tree:
        args["tree"] = i32(torch, parents)
    out = w.cache.attn(q, i32(torch, past) if ragged else most, out=before.clone(), **args)
    ops.sync()
    check_attn(torch, out, before, w, q, past, count, first, parents, 0 if bf16 else 2)


@pytest.mark.parametrize("B,n,H,Hkv,d,page,most,tree", [a for a in ATTN if a[1] in (1, 25, 40, 97)])
def test_attn_one_piece(env, B, n, H, Hkv, d, page, most, tree):
    torch, ops = env
    rng = np.random.default_rng(7)
    w = World(torch, ops, rng, B, Hkv, d, page, most + n, False)
    parents = [tree_of(rng, n)] * B if tree else None
    q = up(torch, normal(rng, B, n, H, d))
    before = torch.zeros_like(q)
    ops.set_math("tf32")
    try:
        out = w.cache.attn(q, most, **({"tree": i32(torch, parents[0])} if tree else {}))
    finally:
        ops.set_math("f32")
    check_attn(torch, out, before, w, q, np.full(B, most), np.full(B, n), np.zeros(B, int), parents, 1)


APPEND = [  # batch, n, heads, heads_kv, d, page, rot, interleaved, past, tree
    (1, 1, 0, 1, 64, 16, 0, False, 0, False), (3, 1, 14, 2, 64, 16, 64, False, 15, False),
    (2, 5, 12, 2, 128, 32, 128, False, 30, False), (2, 33, 6, 1, 128, 16, 64, True, 7, False),
    (2, 9, 4, 4, 64, 64, 24, False, 60, False), (2, 9, 4, 4, 64, 64, 24, True, 60, False),
    (1, 3, 40, 40, 128, 16, 2, False, 3, False), (2, 130, 2, 1, 64, 256, 16, True, 200, False),
    (2, 24, 14, 2, 64, 16, 64, False, 40, True), (3, 7, 6, 2, 128, 32, 10, True, 0, True),
    (1, 256, 2, 2, 64, 16, 32, False, 5, True), (2, 64, 0, 2, 128, 16, 128, True, 33, True),
]


@pytest.mark.parametrize("B,n,H,Hkv,d,page,rot,inter,most,tree", APPEND)
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("ragged", [False, True])
def test_append(env, B, n, H, Hkv, d, page, rot, inter, most, tree, bf16, ragged):
    torch, ops = env
    rng = np.random.default_rng(B + n + rot)
    w = World(torch, ops, rng, B, Hkv, d, page, most + n, bf16, joint=ragged)
    past = rng.integers(0, most + 1, B) if ragged else np.full(B, most)
    count = rng.integers(0, n + 1, B) if ragged else np.full(B, n)
    parents = [tree_of(rng, n) for _ in range(B)] if tree else [None] * B
    qkv = up(torch, normal(rng, B, n, H + 2 * Hkv, d), w.row)
    q, k, v = qkv[:, :, :H], qkv[:, :, H:H + Hkv], qkv[:, :, H + Hkv:]
    if not rot:
        q = None
    tabs = ops.scaled_rope_tables(most + n, rot or 2, 1e4)
    args = {"rope": (up(torch, tabs[0]), up(torch, tabs[1]), inter)} if rot else {}
    if ragged:
        args.update(count=i32(torch, count), max_past=most)
    if tree:
        args["tree"] = i32(torch, parents)
    want = [x.copy() for x in w.contents()]
    want_q = qkv[:, :, :H].float().cpu().numpy()
    old_q = want_q.copy()
    for b in range(B):
        p, m = int(past[b]), int(count[b])
        pos = O.positions(p, m, parents[b])
        for x, rows, turn in ((want[0], k, True), (want[1], v, False), (want_q, q, True)):
            if rows is None or m == 0:
                continue
            r = rows[b, :m].float().cpu().numpy()
            r = O.rotated(r, *tabs, pos, inter) if turn and rot else r
            if x is want_q:
                x[b, :m] = torch.from_numpy(r).to(w.row).float().numpy()
            else:
                x[b, :, p:p + m] = np.moveaxis(torch.from_numpy(r).to(w.held).float().numpy(), 0, 1)
    untouched = w.cache.k.clone(), w.cache.v.clone()
    at = i32(torch, past) if ragged else most
    if H and rot:
        q_out = up(torch, old_q, w.row)
        w.cache.append(k, v, at, q=q, q_out=q_out, **args)
        np.testing.assert_array_equal(q_out.float().cpu().numpy(), want_q)
        w.cache.append(k, v, at, q=q, **args)  # in place, the same rows again
        np.testing.assert_array_equal(q.float().cpu().numpy(), want_q)
    else:
        w.cache.append(k, v, at, **args)
    ops.sync()
    got = w.contents()
    np.testing.assert_array_equal(got[0], want[0])
    np.testing.assert_array_equal(got[1], want[1])
    # the pool's pages that no sequence has
    free = sorted(set(range(w.cache.k.shape[0])) - set(w.np_table.ravel().tolist()))
    assert torch.equal(w.cache.k[free], untouched[0][free]) and torch.equal(w.cache.v[free], untouched[1][free])


@pytest.mark.parametrize("B,n,Hkv,d,page,layers,bf16", [(1, 1, 1, 64, 16, 1, False), (3, 24, 2, 128, 16, 3, False),
                                                        (2, 61, 2, 64, 32, 70, True), (2, 256, 3, 128, 256, 2, True)])
def test_accept_and_keep(env, B, n, Hkv, d, page, layers, bf16):
    torch, ops = env
    rng = np.random.default_rng(n)
    most = 37
    w = [World(torch, ops, np.random.default_rng(i), B, Hkv, d, page, most + n, bf16) for i in range(layers)]
    for x in w[1:]:
        x.cache.table, x.np_table = w[0].cache.table, w[0].np_table
        x.cache = ops.PagedCache(x.cache.k, x.cache.v, w[0].cache.table)
    past, count = rng.integers(0, most + 1, B), rng.integers(1, n + 1, B)
    count[0] = n
    parents = [tree_of(rng, n) for _ in range(B)]
    tokens = rng.integers(0, 4, (B, n))
    ids = rng.integers(0, 4, (B, n))
    path, kept, following = ops.tree_accept(i32(torch, tokens), i32(torch, ids), i32(torch, parents), count=i32(torch, count))
    want = [x.contents() for x in w]
    for b in range(B):
        m = int(count[b])
        p, nxt = O.accept(tokens[b, :m].tolist(), ids[b, :m].tolist(), parents[b][:m])
        assert path[b].tolist() == p + [-1] * (n - len(p)) and int(kept[b]) == len(p) and int(following[b]) == nxt
        for k, v in want:
            for x in (k, v):
                x[b, :, past[b]:past[b] + len(p)] = x[b][:, [past[b] + i for i in p]]
    ops.paged_keep([x.cache for x in w], path, kept, i32(torch, past), max_past=most)
    ops.sync()
    for x, (k, v) in zip(w, want):
        got = x.contents()
        np.testing.assert_array_equal(got[0], k)
        np.testing.assert_array_equal(got[1], v)

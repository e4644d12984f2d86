"""Calls on the cache in pages that its documentation allows and that are easily refused or answered wrongly: what lies in
slots that a query does not see, pages that are none, entries out of range, rows and pools of any strides, graphs,
streams, and a whole loop of drafts that ends in the tokens of a plain one."""
import numpy as np
import pytest

from oracle import paged as O
from tests.conftest import has_gpu
from tests.test_gpu_seq_paged import World, check_attn, i32, normal, tree_of, up

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def env():
    if not has_gpu():
        pytest.fail("needs a CUDA device")
    import torch

    from zwhisper_b200 import ops
    ops.set_math("f32")
    return torch, ops


SHAPES = [  # n, heads, heads_kv, d, page, past, tree: both kernels, one slot or two of a CTA's rows, splits
    (1, 6, 1, 128, 16, 333, False), (2, 14, 2, 64, 32, 300, False), (40, 12, 2, 64, 16, 100, False), (70, 6, 1, 128, 64, 130, False),
    (256, 2, 1, 128, 16, 60, False), (5, 12, 2, 128, 16, 250, True), (61, 14, 2, 64, 16, 140, True), (25, 8, 2, 128, 32, 2000, True),
    (200, 4, 2, 128, 16, 37, True), (100, 16, 1, 64, 256, 5, True),
]


def poison_of(torch, kind, held):
    return {"nan": float("nan"), "inf": float("inf"), "huge": torch.finfo(held).max}[kind]


@pytest.mark.parametrize("n,H,Hkv,d,page,past,tree", SHAPES)
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("kind", ["nan", "inf", "huge"])
def test_what_no_query_sees_leaves_the_outputs_alone(env, n, H, Hkv, d, page, past, tree, bf16, kind):
    """Slots before first, behind the last token, of pages between, and the rest of the pool."""
    torch, ops = env
    rng = np.random.default_rng(n + d)
    B = 2
    w = World(torch, ops, rng, B, Hkv, d, page, past + n + 20, bf16)
    first = [min(past, 19), 0]
    count = [n, max(1, n - 3)]
    parents = [tree_of(rng, n) for _ in range(B)] if tree else None
    args = dict(first=i32(torch, first), count=i32(torch, count))
    if tree:
        args["tree"] = i32(torch, parents)
    q = up(torch, normal(rng, B, n, H, d), w.row)
    zero = torch.zeros_like(q)
    want = w.cache.attn(q, past, out=zero.clone(), **args)
    bad = poison_of(torch, kind, w.held)
    keep = torch.zeros(w.cache.k.shape[0], page, dtype=torch.bool, device="cuda:0")
    for b in range(B):
        for t in range(first[b], past + count[b]):
            keep[w.np_table[b, t // page], t % page] = True
    for pool in (w.cache.k, w.cache.v):
        pool.masked_fill_(~keep[:, None, :, None], bad)
    got = w.cache.attn(q, past, out=zero.clone(), **args)
    ops.sync()
    assert torch.equal(got, want)


@pytest.mark.parametrize("n,H,Hkv,d,page,past,tree", [s for s in SHAPES if s[0] > 1])
@pytest.mark.parametrize("bf16", [False, True])
def test_a_token_that_only_some_queries_see(env, n, H, Hkv, d, page, past, tree, bf16):
    """An infinity and a NaN among the values of a late token: in the columns of the queries that see it, and nowhere else."""
    torch, ops = env
    rng = np.random.default_rng(n)
    w = World(torch, ops, rng, 1, Hkv, d, page, past + n, bf16)
    parents = [tree_of(rng, n)] if tree else None
    args = {"tree": i32(torch, parents)} if tree else {}
    q = up(torch, normal(rng, 1, n, H, d), w.row)
    want = w.cache.attn(q, past, **args).clone()
    at = n // 2
    t = past + at
    place = (int(w.np_table[0, t // page]), slice(None), t % page)
    w.cache.v[place][:, 3] = float("inf")
    w.cache.v[place][:, 7] = float("nan")
    w.cache.v[place][:, d - 1] = -float("inf")
    got = w.cache.attn(q, past, **args)
    ops.sync()
    seen = torch.from_numpy(O.seen_slots(past, n, 0, past + n, parents[0] if tree else None)[:, t]).cuda()
    assert torch.equal(got[0, ~seen], want[0, ~seen])
    plain = [c for c in range(d) if c not in (3, 7, d - 1)]
    # the sums of the other columns do not know of it
    assert torch.equal(got[0, seen][..., plain], want[0, seen][..., plain])
    assert torch.isnan(got[0, seen][..., 7]).all()
    if bf16:
        assert (got[0, seen][..., 3] == float("inf")).all() and (got[0, seen][..., d - 1] == -float("inf")).all()
    else:
        # a probability is two pieces h + l, l the nearest f16 of what h leaves, so 0 or below it as often as above: where
        # all of a tile's queries see the token, h inf + l inf is NaN for those
        assert not torch.isfinite(got[0, seen][..., [3, d - 1]]).any()


@pytest.mark.parametrize("n,H,Hkv,d,page,past,tree", SHAPES)
@pytest.mark.parametrize("bf16", [False, True])
def test_keys_that_are_not_numbers(env, n, H, Hkv, d, page, past, tree, bf16):
    """A NaN among a key's elements: every output of the queries that see it, and no other's."""
    torch, ops = env
    rng = np.random.default_rng(n)
    w = World(torch, ops, rng, 1, Hkv, d, page, past + n, bf16)
    parents = [tree_of(rng, n)] if tree else None
    args = {"tree": i32(torch, parents)} if tree else {}
    q = up(torch, normal(rng, 1, n, H, d), w.row)
    want = w.cache.attn(q, past, **args).clone()
    t = past + n // 2
    w.cache.k[int(w.np_table[0, t // page]), :, t % page, 5] = float("nan")
    got = w.cache.attn(q, past, **args)
    seen = torch.from_numpy(O.seen_slots(past, n, 0, past + n, parents[0] if tree else None)[:, t]).cuda()
    assert torch.equal(got[0, ~seen], want[0, ~seen]) and torch.isnan(got[0, seen]).all()


@pytest.mark.parametrize("n,H,Hkv,d,page,past,tree", SHAPES)
@pytest.mark.parametrize("bf16", [False, True])
def test_pages_that_are_none(env, n, H, Hkv, d, page, past, tree, bf16):
    torch, ops = env
    from zwhisper_b200._lib import ZwgError
    rng = np.random.default_rng(n)
    B = 2
    w = World(torch, ops, rng, B, Hkv, d, page, past + n, bf16)
    parents = [tree_of(rng, n) for _ in range(B)] if tree else None
    args = {"tree": i32(torch, parents)} if tree else {}
    last = (past + n - 1) // page
    bad = {(0, 0): -1, (0, last): w.cache.k.shape[0], (1, last // 2): -(1 << 31)}
    for (b, i), x in bad.items():
        w.cache.table[b, i] = x
    q = up(torch, normal(rng, B, n, H, d), w.row)
    out = w.cache.attn(q, past, **args)
    with pytest.raises(ZwgError):
        ops.sync()
    k, v = w.contents(np.float64)
    for b in range(B):
        seen = O.seen_slots(past, n, 0, w.slots, parents[b] if tree else None)
        for (bb, i) in bad:
            if bb == b:
                seen[:, i * page:(i + 1) * page] = False
        want, tol = O.attention(q[b].float().cpu().numpy(), k[b], v[b], seen, 0 if bf16 else 2, 2.0 ** (-8 if bf16 else -24),
                                n * H // Hkv > 16)
        assert (np.abs(out[b].float().cpu().numpy() - want) <= tol).all()
    # the append leaves their rows out, and writes the others
    k_new, v_new = (up(torch, normal(rng, B, n, Hkv, d), w.row) for _ in range(2))
    before = w.cache.k.clone(), w.cache.v.clone()
    w.cache.append(k_new, v_new, past, **args)
    with pytest.raises(ZwgError):
        ops.sync()
    for pool, old, new in ((w.cache.k, before[0], k_new), (w.cache.v, before[1], v_new)):
        want = old.clone()
        for b in range(B):
            for i in range(n):
                t = past + i
                if (b, t // page) not in bad:
                    want[int(w.np_table[b, t // page]), :, t % page] = new[b, i].to(w.held)
        assert torch.equal(pool, want)
    # and so does the move of kept rows
    path = i32(torch, [list(range(n))] * B)
    ops.paged_keep(w.cache, path, i32(torch, [n] * B), past)  # nothing moves: no page is looked up
    ops.sync()
    if n > 1:
        path = i32(torch, [[1] + [-1] * (n - 1)] * B)
        ops.paged_keep(w.cache, path, i32(torch, [1, 0]), past)
        if (0, past // page) in bad or (0, (past + 1) // page) in bad:
            with pytest.raises(ZwgError):
                ops.sync()
    ops.set_math("f32")


def test_sequences_out_of_range_are_skipped(env):
    torch, ops = env
    from zwhisper_b200._lib import ZwgError
    rng = np.random.default_rng(0)
    for n, H in ((2, 2), (40, 8)):
        B = 8
        w = World(torch, ops, rng, B, 1, 64, 16, 64, False)
        room = w.cache.n_ctx
        good = [-1] + list(range(n - 1))
        over, under = list(good), list(good)
        over[1], under[-1] = 1, -2
        parents = [good, good, good, over, under, good, good, good]
        past = [3, -1, room - n + 1, 3, 3, 3, 3, 3]
        count = [n, n, n, n, n, n + 1, -1, n]
        first = [0, 0, 0, 0, 0, 0, 0, -1]
        q = up(torch, normal(rng, B, n, H, 64))
        out = torch.full_like(q, 7.0)
        ops.sync()
        args = dict(count=i32(torch, count), tree=i32(torch, parents), max_past=room)
        w.cache.attn(q, i32(torch, past), first=i32(torch, first), out=out, **args)
        with pytest.raises(ZwgError):
            ops.sync()
        assert (out[1:] == 7).all() and not (out[0] == 7).any()
        cos, sin = (up(torch, a) for a in ops.rope_tables(room, 64, 1e4))
        k, v = (up(torch, normal(rng, B, n, 1, 64)) for _ in range(2))
        before, old_q = w.contents(), q.clone()
        w.cache.append(k, v, i32(torch, past), q=q, rope=(cos, sin), **args)
        with pytest.raises(ZwgError):
            ops.sync()
        got = w.contents()
        for a, b in zip(got, before):
            np.testing.assert_array_equal(a[1:7], b[1:7])
            assert (a[0] != b[0]).any() and (a[7] != b[7]).any()
        assert torch.equal(q[1:7], old_q[1:7])
        # a bad tree or count agrees with nothing
        tokens = torch.zeros(B, n, dtype=torch.int32, device="cuda:0")
        path, kept, following = ops.tree_accept(tokens, tokens, args["tree"], count=args["count"])
        with pytest.raises(ZwgError):
            ops.sync()
        assert kept.tolist()[3:7] == [0, 0, 0, 0] and following.tolist()[3:7] == [-1] * 4 and (path[3:7] == -1).all()
        assert kept.tolist()[:3] == [n] * 3  # every token is what the model says: down the line
        # paths that do not rise, or leave the call's tokens
        bad = torch.full((B, n), -1, dtype=torch.int32, device="cuda:0")
        bad[0, :2] = torch.tensor([1, 1])
        bad[1, 0] = n
        bad[2, 0] = -3
        before = w.contents()
        ops.paged_keep(w.cache, bad, i32(torch, [2, 1, 1, 0, 0, 0, 0, n + 1]), 3)
        with pytest.raises(ZwgError):
            ops.sync()
        for a, b in zip(w.contents(), before):
            np.testing.assert_array_equal(a, b)
    ops.sync()


@pytest.mark.parametrize("n,H,Hkv,d,page,past,tree", SHAPES)
@pytest.mark.parametrize("bf16", [False, True])
def test_rows_of_any_strides_and_places(env, n, H, Hkv, d, page, past, tree, bf16):
    """Queries and outputs an element off the wide alignment, tokens outside of sequences, outputs over queries."""
    torch, ops = env
    rng = np.random.default_rng(n)
    B = 2
    w = World(torch, ops, rng, B, Hkv, d, page, past + n, bf16, joint=True)
    parents = [tree_of(rng, n)] * B if tree else None
    args = {"tree": i32(torch, parents[0])} if tree else {}
    q = up(torch, normal(rng, B, n, H, d), w.row)
    want = w.cache.attn(q, past, **args)
    flat = torch.zeros(n * (B * (H * d + 1) + 3) + 8, dtype=w.row, device="cuda:0")
    odd = flat[1:].as_strided((B, n, H, d), (H * d + 1, B * (H * d + 1) + 3, d, 1))
    odd.copy_(q)
    out = torch.zeros_like(flat)
    o = out[1:].as_strided(odd.shape, odd.stride())
    w.cache.attn(odd, past, out=o, **args)
    assert torch.equal(o, want) and int((out != 0).sum()) == int((want != 0).sum())
    w.cache.attn(odd, past, out=odd, **args)
    assert torch.equal(odd, want)
    cos, sin = (up(torch, a) for a in ops.rope_tables(past + n + 1, d, 1e4))
    k, v = (up(torch, normal(rng, B, n, Hkv, d), w.row) for _ in range(2))
    w.cache.append(k, v, past, q=q, rope=(cos, sin), **args)
    after = w.contents()
    w.cache.k.zero_(), w.cache.v.zero_()
    odd.copy_(up(torch, normal(rng, B, n, H, d), w.row))
    plain = odd.clone()
    kv = torch.zeros(2, n * B * (Hkv * d + 1) + 1, dtype=w.row, device="cuda:0")
    ko, vo = (x[1:].as_strided((B, n, Hkv, d), (n * (Hkv * d + 1), Hkv * d + 1, d, 1)) for x in kv)
    ko.copy_(k), vo.copy_(v)
    w.cache.append(ko, vo, past, q=odd, rope=(cos[1:], sin[1:]) if False else (cos, sin), **args)
    got = w.contents()
    for a, b in zip(got, after):
        np.testing.assert_array_equal(a[:, :, past:past + n], b[:, :, past:past + n])
    w.cache.append(k, v, past, q=plain, rope=(cos, sin), **args)
    assert torch.equal(odd, plain)
    ops.sync()


def test_places_beyond_32_bits(env):
    """A pool whose pages lie 2^28 elements apart: rows behind 2^32 bytes and 2^32 elements."""
    torch, ops = env
    rng = np.random.default_rng(1)
    step, pages, page, d = 1 << 28, 20, 16, 128
    store = torch.empty((pages - 1) * step + 2 * page * d, dtype=torch.float16, device="cuda:0")
    k = store.as_strided((pages, 1, page, d), (step, page * d, d, 1))
    v = store[page * d:].as_strided((pages, 1, page, d), (step, page * d, d, 1))
    k.zero_(), v.zero_()
    table = i32(torch, [[19, 0, 18, 17, 1, 16, 2, 15]])
    cache = ops.PagedCache(k, v, table)
    small = ops.PagedCache(torch.zeros(8, 1, page, d, dtype=torch.float16, device="cuda:0"),
                           torch.zeros(8, 1, page, d, dtype=torch.float16, device="cuda:0"), i32(torch, [list(range(8))]))
    for n, H in ((100, 1), (28, 6), (1, 6)):
        rows = [up(torch, normal(rng, 1, n, 1, d)) for _ in range(2)]
        q = up(torch, normal(rng, 1, n, H, d))
        past = {100: 0, 28: 100, 1: 127}[n]
        outs = []
        for c in (cache, small):
            c.append(*rows, past)
            outs.append(c.attn(q, past))
        assert torch.equal(*outs)
    path, kept = i32(torch, [[3, 9, 20] + [-1] * 25]), i32(torch, [3])
    for c in (cache, small):
        ops.paged_keep(c, path, kept, 90)
    assert torch.equal(k[table[0].long()], small.k) and torch.equal(v[table[0].long()], small.v)
    ops.sync()


def test_a_prefix_that_sequences_share(env):
    torch, ops = env
    rng = np.random.default_rng(2)
    w = World(torch, ops, rng, 3, 2, 64, 16, 100, True)
    w.cache.table[1:, :4] = w.cache.table[0, :4]
    w.np_table[1:, :4] = w.np_table[0, :4]
    for n, H in ((1, 4), (36, 14)):
        q = up(torch, normal(rng, 3, n, H, 64), w.row)
        before = torch.zeros_like(q)
        out = w.cache.attn(q, 64, out=before.clone())
        check_attn(torch, out, before, w, q, [64] * 3, [n] * 3, [0] * 3, None, 0)


def test_empty_calls(env):
    torch, ops = env
    rng = np.random.default_rng(3)
    w = World(torch, ops, rng, 2, 1, 64, 16, 32, False)
    q = torch.full((2, 1, 4, 64), 3.0, device="cuda:0")
    # nothing seen: zeros; no tokens: left as they are
    assert not w.cache.attn(q, 5, first=i32(torch, [6, 100])).any()
    out = q.clone()
    w.cache.attn(q, 5, count=i32(torch, [0, 0]), out=out)
    assert torch.equal(out, q)
    big = torch.ones(2, 20, 20, 64, device="cuda:0")
    assert not w.cache.attn(big, 5, first=i32(torch, [26, 25 + 1])).any()
    none = torch.empty(2, 0, 4, 64, device="cuda:0")
    w.cache.attn(none, 5)
    w.cache.append(torch.empty(2, 0, 1, 64, device="cuda:0"), torch.empty(2, 0, 1, 64, device="cuda:0"), 5)
    path, kept, following = ops.tree_accept(*(torch.zeros(2, 1, dtype=torch.int32, device="cuda:0") for _ in range(2)),
                                            i32(torch, [-1]), count=i32(torch, [1, 0]))
    assert kept.tolist() == [1, 0] and path.tolist() == [[0], [-1]] and following.tolist() == [0, -1]
    ops.sync()


def test_wrong_tensors_are_refused(env):
    torch, ops = env
    rng = np.random.default_rng(4)
    w = World(torch, ops, rng, 2, 2, 64, 16, 64, False)
    c = w.cache
    q, k = up(torch, normal(rng, 2, 3, 4, 64)), up(torch, normal(rng, 2, 3, 2, 64))
    tab = tuple(up(torch, a) for a in ops.rope_tables(64, 64, 1e4))
    bad = [
        lambda: c.attn(q.bfloat16(), 1), lambda: c.attn(q[0], 1), lambda: c.attn(q.cpu(), 1), lambda: c.attn(q[:1], 1),
        lambda: c.attn(q, -1), lambda: c.attn(q, 1, out=q.bfloat16()), lambda: c.attn(q, 1, tree=i32(torch, [-1, 0])),
        lambda: c.attn(q, 1, tree=i32(torch, [[-1, 0, 1]] * 3)), lambda: c.attn(q, 1, tree=torch.tensor([-1, 0, 1]).cuda()),
        lambda: c.attn(q, 1, tree=torch.tensor([-1, 0, 1], dtype=torch.int32)), lambda: c.attn(q.transpose(2, 3), 1),
        lambda: c.attn(q, 1, count=i32(torch, [1])), lambda: c.append(k.bfloat16(), k.bfloat16(), 1),
        lambda: c.append(k, k[:, :2], 1), lambda: c.append(k, k, 1, q=q[:, :2], rope=tab), lambda: c.append(k, k, 1, q_out=q),
        lambda: ops.PagedCache(c.k.float(), c.v.float(), c.table), lambda: ops.PagedCache(c.k, c.v[:, :1], c.table),
        lambda: ops.PagedCache(c.k, c.v, c.table.long()), lambda: ops.PagedCache(c.k.transpose(2, 3), c.v.transpose(2, 3), c.table),
        lambda: ops.PagedCache(c.k.cpu(), c.v.cpu(), c.table.cpu()), lambda: ops.PagedCache(c.k[::2], c.v[:c.k[::2].shape[0]], c.table),
        lambda: ops.tree_accept(q, q, None), lambda: ops.tree_accept(i32(torch, [[1]]), i32(torch, [[1]]), None),
        lambda: ops.paged_keep(c, i32(torch, [1, 2]), i32(torch, [1, 1]), 0),
        lambda: ops.paged_keep(c, i32(torch, [[0, 1]] * 2), i32(torch, [1]), 0),
    ]
    for i, call in enumerate(bad):
        with pytest.raises((ValueError, RuntimeError)):
            call()
            pytest.fail(f"call {i} was taken")
    from zwhisper_b200._lib import ZwgError
    with pytest.raises(ZwgError):
        c.attn(q, c.n_ctx - 2)
    with pytest.raises(ZwgError):
        c.append(k, k, 1, q=q)
    with pytest.raises(ZwgError):
        c.attn(q[:, :, :3], 1)
    long = up(torch, normal(rng, 1, 40, 4, 64))
    one = World(torch, ops, rng, 1, 1, 64, 16, 4000, False)
    size = one.cache.attn_workspace_bytes(40, 4, 3000)
    if size:
        with pytest.raises(ZwgError):
            one.cache.attn(long, 3000, workspace=torch.empty(size - 16, dtype=torch.uint8, device="cuda:0"))
    ops.sync()


def greedy(torch, ops, model, w, tables, start, steps, past):
    """Plain decoding: a token at a time."""
    tokens, at = [start], past
    for _ in range(steps):
        x = model["embed"][torch.tensor(tokens[-1], device="cuda:0")].view(1, 1, -1)
        q, k, v = (y.contiguous() for y in model["qkv"](x))
        q = w.cache.append(k, v, at, q=q, rope=tables)
        out = w.cache.attn(q, at)
        tokens.append(int((out.reshape(1, -1) @ model["head"]).argmax()))
        at += 1
    return tokens


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("captured", [False, True])
def test_drafts_end_in_the_tokens_of_plain_decoding(env, bf16, captured):
    """Append, attention over the tree, acceptance and the kept rows, again and again (eagerly, or one captured round that is
    replayed with other drafts): the same tokens as a token at a time, and the same cache. Drafts are right and wrong by
    turns, so that paths of every length come up."""
    torch, ops = env
    rng = np.random.default_rng(5)
    H, Hkv, d, page, steps, past, n, vocab = 6, 2, 64, 16, 60, 21, 12, 50
    width = H * d
    row = torch.bfloat16 if bf16 else torch.float32
    wq, wk, wv = (up(torch, normal(rng, 96, h * d) * 0.2) for h in (H, Hkv, Hkv))
    model = {"embed": up(torch, normal(rng, vocab, 96)), "head": up(torch, normal(rng, width, vocab)).to(row),
             "qkv": lambda x: ((x @ m).view(*x.shape[:2], h, d).to(row) for m, h in ((wq, H), (wk, Hkv), (wv, Hkv)))}
    tables = tuple(up(torch, a) for a in ops.rope_tables(256, d, 1e4))
    seed = np.random.default_rng(6)
    plain, tree = (World(torch, ops, np.random.default_rng(7), 1, Hkv, d, page, 128, bf16) for _ in range(2))
    want = greedy(torch, ops, model, plain, tables, 3, steps, past)
    # one round, on buffers that stay in place
    tokens, parents = (torch.zeros(1, n, dtype=torch.int32, device="cuda:0") for _ in range(2))
    at = i32(torch, [past])
    ws = torch.empty(max(16, tree.cache.attn_workspace_bytes(n, H)), dtype=torch.uint8, device="cuda:0")

    def round_():
        q, k, v = (y.contiguous() for y in model["qkv"](model["embed"][tokens.long()]))
        q = tree.cache.append(k, v, at, q=q, rope=tables, tree=parents, max_past=100)
        out = tree.cache.attn(q, at, tree=parents, max_past=100, workspace=ws)
        ids = (out.reshape(n, -1) @ model["head"]).argmax(1).view(1, n).to(torch.int32)
        path, kept, following = ops.tree_accept(tokens, ids, parents)
        ops.paged_keep(tree.cache, path, kept, at, max_past=100)
        at.add_(kept)
        return path, kept, following

    if captured:
        tokens.fill_(0), parents.copy_(i32(torch, [tree_of(seed, n)]))
        saved = tree.cache.k.clone(), tree.cache.v.clone()
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            round_()
            side.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                result = round_()
        tree.cache.k.copy_(saved[0]), tree.cache.v.copy_(saved[1])
        at.fill_(past)
    got, lengths = [3], set()
    while len(got) <= steps:
        parent, ids = tree_of(seed, n), [got[-1]] + seed.integers(0, vocab, n - 1).tolist()
        true = want[len(got) - 1:]  # what the model will say
        depth = [0] * n
        for i in range(1, n):  # some branches follow it for a while
            if parent[i] < 0:
                parent[i] = 0
            depth[i] = depth[parent[i]] + 1
            if seed.random() < 0.7 and depth[i] < len(true):
                ids[i] = true[depth[i]]
        tokens.copy_(i32(torch, [ids])), parents.copy_(i32(torch, [parent]))
        if captured:
            graph.replay()
            path, kept, following = result
        else:
            path, kept, following = round_()
        m = int(kept)
        lengths.add(m)
        got += [ids[i] for i in path[0, 1:m].tolist()] + [int(following)]
    ops.sync()
    assert got[:steps + 1] == want and len(lengths) > 2
    # the rows of tokens that both caches hold
    half = 2.0 ** (-7 if bf16 else -10)  # one step of the cache's type where two kernels' queries differ in a last bit
    for a, b in zip(tree.contents(), plain.contents()):
        np.testing.assert_allclose(a[:, :, past:past + steps], b[:, :, past:past + steps], rtol=half, atol=1e-6)


def test_captured_calls_read_what_lies_there_at_replay(env):
    """Lengths, counts, pages and trees are read on the device: a graph takes new ones."""
    torch, ops = env
    rng = np.random.default_rng(8)
    B, n, H, most = 3, 20, 12, 300
    w = World(torch, ops, rng, B, 2, 128, 16, most + n, True)
    q = up(torch, normal(rng, B, n, H, 128), w.row)
    before = up(torch, normal(rng, B, n, H, 128), w.row)
    out = before.clone()
    past, count, first = (i32(torch, [0] * B) for _ in range(3))
    tree = i32(torch, [tree_of(rng, n)] * B)
    ws = torch.empty(max(16, w.cache.attn_workspace_bytes(n, H, most)), dtype=torch.uint8, device="cuda:0")
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        w.cache.attn(q, past, count=count, first=first, tree=tree, max_past=most, out=out, workspace=ws)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            w.cache.attn(q, past, count=count, first=first, tree=tree, max_past=most, out=out, workspace=ws)
    for _ in range(4):
        p, c = rng.integers(0, most + 1, B), rng.integers(0, n + 1, B)
        f = np.minimum(rng.integers(0, most, B), p + 3)
        parents = [tree_of(rng, n) for _ in range(B)]
        past.copy_(i32(torch, p)), count.copy_(i32(torch, c)), first.copy_(i32(torch, f)), tree.copy_(i32(torch, parents))
        w.np_table[:] = w.np_table[rng.permutation(B)]
        w.cache.table.copy_(i32(torch, w.np_table))
        out.copy_(before)
        graph.replay()
        check_attn(torch, out, before, w, q, p, c, f, parents, 0)
    ops.sync()


def test_calls_side_by_side_on_streams(env):
    torch, ops = env
    rng = np.random.default_rng(9)
    w = World(torch, ops, rng, 2, 2, 128, 16, 3000, True)
    calls = [(1, 12, 2900), (30, 12, 2000), (200, 4, 700), (2, 12, 2500)]
    qs = [up(torch, normal(rng, 2, n, H, 128), w.row) for n, H, _ in calls]
    want = [w.cache.attn(q, p) for q, (_, _, p) in zip(qs, calls)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    outs = [torch.zeros_like(q) for q in qs]
    for _ in range(10):
        for s, q, o, (_, _, p) in zip(streams, qs, outs, calls):
            with torch.cuda.stream(s):
                w.cache.attn(q, p, out=o)
    torch.cuda.synchronize()
    for o, x in zip(outs, want):
        assert torch.equal(o, x)
    ops.sync()


def test_a_workspace_serves_shorter_calls(env):
    torch, ops = env
    rng = np.random.default_rng(10)
    for B, n, H, Hkv, d, bf16 in ((1, 1, 12, 2, 128, True), (1, 25, 12, 2, 128, False), (2, 61, 14, 2, 64, True), (1, 2, 8, 8, 64, False)):
        w = World(torch, ops, rng, B, Hkv, d, 64, 20000, bf16)
        size = w.cache.attn_workspace_bytes(n, H, 19000)
        ws = torch.empty(max(16, size), dtype=torch.uint8, device="cuda:0")
        q = up(torch, normal(rng, B, n, H, d), w.row)
        for past in (19000, 9001, 3000, 700, 130, 15, 0):
            assert w.cache.attn_workspace_bytes(n, H, past) <= size
            w.cache.attn(q, past, workspace=ws)
    ops.sync()


def test_a_workspace_serves_lengths_of_their_own(env):
    """What attn_workspace_bytes gives for a number of past tokens is enough for lengths on the device, up to it."""
    torch, ops = env
    rng = np.random.default_rng(11)
    for B, n, H, d, bf16, most in ((64, 16, 12, 128, True, 8001), (40, 20, 12, 128, False, 4000), (3, 100, 8, 64, True, 9000)):
        w = World(torch, ops, rng, B, 2, d, 64, most + n, bf16)
        size = w.cache.attn_workspace_bytes(n, H, most)
        ws = torch.empty(max(16, size), dtype=torch.uint8, device="cuda:0")
        q = up(torch, normal(rng, B, n, H, d), w.row)
        for top in (most, most // 2, most // 5, 100):
            past = rng.integers(0, top + 1, B)
            past[0] = top
            out = w.cache.attn(q, i32(torch, past), max_past=top, workspace=ws)
            alone = w.cache.attn(q, top, workspace=ws)
            # a sequence's output does not depend on the others' lengths but for where its keys are cut
            half = 2.0 ** (-7 if bf16 else -18)
            torch.testing.assert_close(out[0].float(), alone[0].float(), rtol=half, atol=half)
    ops.sync()

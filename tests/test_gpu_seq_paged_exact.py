"""Attention over pages to the key (tests/paged_codes.py), over turns, warps, cuts and pages of every length; its accuracy in
norm, by which two f16 pieces of a query are told from one; workspaces with a guard behind them, used again by shorter calls;
and rotary tables that start off the wide alignment."""
import numpy as np
import pytest

from tests.conftest import has_gpu
from tests.paged_codes import bound
from tests.test_gpu_seq_paged import World, i32, normal, tree_of, up

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def env():
    if not has_gpu():
        pytest.fail("needs a CUDA device")
    import torch

    from zwhisper_b200 import ops
    ops.set_math("f32")
    return torch, ops


def launches(torch, call):
    """(threads, CTAs to a row of the grid) of each kernel that the call launches, from a graph it is captured into."""
    from cuda.bindings import driver
    call()
    graph, side = torch.cuda.CUDAGraph(keep_graph=True), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        call()
    raw = driver.CUgraph(graph.raw_cuda_graph())
    err, _, n = driver.cuGraphGetNodes(raw)
    err, nodes, n = driver.cuGraphGetNodes(raw, n)
    assert err == driver.CUresult.CUDA_SUCCESS
    found = []
    for node in nodes[:n]:
        err, kind = driver.cuGraphNodeGetType(node)
        if kind == driver.CUgraphNodeType.CU_GRAPH_NODE_TYPE_KERNEL:
            err, params = driver.cuGraphKernelNodeGetParams(node)
            assert err == driver.CUresult.CUDA_SUCCESS
            found.append((params.blockDimX, params.gridDimX))
    return found


def coded(torch, ops, seed, B, Hkv, d, page, slots, bf16):
    """A cache of `slots` slots a sequence and what its values are: signs [B][Hkv][slots][d]."""
    g = torch.Generator(device="cuda:0")
    g.manual_seed(seed)
    per = -(-slots // page)
    held = torch.bfloat16 if bf16 else torch.float16
    pool = B * per + 3
    table = torch.randperm(pool, generator=g, device="cuda:0")[: B * per].view(B, per)
    k = torch.randn(pool, Hkv, page, d, generator=g, device="cuda:0").to(held)
    v = (torch.randint(0, 2, (pool, Hkv, page, d), generator=g, device="cuda:0", dtype=torch.int8) * 2 - 1).to(held)
    code = v[table].transpose(1, 2).reshape(B, Hkv, per * page, d)
    return ops.PagedCache(k, v, table.to(torch.int32)), code


CODES = [  # batch, n, heads, heads_kv, d, page, past (most), tree, what runs
    (1, 1, 12, 2, 128, 16, 2255, False, "cluster"), (3, 1, 14, 2, 64, 16, 2300, False, "cluster"),
    (2, 1, 6, 1, 64, 32, 777, False, "cluster"), (4, 3, 4, 2, 128, 64, 1501, False, "cluster"), (2, 7, 12, 2, 128, 16, 1999, True, "cluster"),
    (64, 1, 12, 2, 128, 16, 500, False, "any"), (70, 2, 14, 2, 64, 128, 333, False, "any"),
    (1, 1, 12, 2, 128, 128, 9000, False, "cuts"), (2, 1, 12, 2, 128, 128, 131000, False, "cuts"),
    (2, 1, 14, 2, 64, 16, 131000, False, "cuts"), (1, 1, 2, 1, 64, 256, 40003, False, "cuts"), (1, 4, 4, 2, 128, 16, 30011, True, "cuts"),
    (40, 24, 12, 2, 128, 16, 200, False, "chunk"), (40, 21, 12, 2, 128, 32, 1301, False, "chunk"), (64, 16, 14, 2, 64, 16, 150, True, "chunk"),
    (32, 256, 2, 2, 64, 64, 1744, False, "chunk cuts"), (60, 30, 6, 1, 64, 32, 3000, True, "chunk cuts"),
    (80, 256, 2, 2, 64, 64, 1744, False, "chunk"), (80, 61, 12, 2, 128, 16, 777, True, "chunk"),
    (1, 2100, 12, 2, 128, 16, 1, False, "any"), (2, 3001, 2, 1, 64, 32, 200, False, "any"), (1, 700, 8, 8, 64, 64, 77, False, "any"),
    (3, 20, 12, 2, 128, 16, 6000, True, "chunk cuts"), (2, 130, 4, 1, 64, 64, 5000, False, "chunk cuts"),
    (4, 256, 4, 2, 64, 128, 2000, True, "chunk cuts"), (2, 100, 12, 2, 128, 256, 30001, False, "chunk cuts"),
]


@pytest.mark.parametrize("B,n,H,Hkv,d,page,most,tree,kernel", CODES)
@pytest.mark.parametrize("kind", ["f32", "tf32", "bf16"])
@pytest.mark.parametrize("ragged", [False, True])
def test_every_key_counts_once(env, B, n, H, Hkv, d, page, most, tree, kernel, kind, ragged):
    torch, ops = env
    rng = np.random.default_rng(B + n + most)
    cache, code = coded(torch, ops, most + n, B, Hkv, d, page, most + n, kind == "bf16")
    past = (most - rng.integers(0, min(most, 700), B)) if ragged else np.full(B, most)
    past[0] = most
    first = rng.integers(0, np.minimum(past, 400)) if ragged else np.zeros(B, int)
    parents = [tree_of(rng, n) for _ in range(B)] if tree else None
    args = {"tree": i32(torch, parents)} if tree else {}
    if ragged:
        args.update(first=i32(torch, first), max_past=most)
    q = torch.zeros(B, n, H, d, device="cuda:0", dtype=torch.bfloat16 if kind == "bf16" else torch.float32)
    at = i32(torch, past) if ragged else most
    ops.set_math("tf32" if kind == "tf32" else "f32")
    try:
        ran = launches(torch, lambda: cache.attn(q, at, **args))
        out = cache.attn(q, at, **args)
    finally:
        ops.set_math("f32")
    ops.sync()
    rows = n * H // Hkv
    tiles = -(-rows // (256 if ran[0][0] == 640 else 8 if rows <= 8 else 16))
    cuts = ran[0][1] // tiles
    want = {"cluster": ran[0][0] != 640 and 1 < cuts <= 16 and len(ran) == 1, "cuts": ran[0][0] != 640 and cuts > 16 and len(ran) == 2,
            "chunk": ran[0][0] == 640 and (cuts == 1 or ragged), "chunk cuts": ran[0][0] == 640 and cuts > 1 and len(ran) == 2, "any": True}
    assert want[kernel], ran
    half = 2.0 ** -8 if kind == "bf16" else 2.0 ** -24
    for b in range(B):
        p, f = int(past[b]), int(first[b])
        new = code[b, :, p:p + n].double()
        sums = code[b, :, f:p].double().sum(1, keepdim=True)  # [Hkv][1][d]
        if tree:
            above = np.zeros((n, n))
            for i, a in enumerate(parents[b]):
                above[i] = above[a] if a >= 0 else 0
                above[i, i] = 1
            above = up(torch, above).double()
            sums, number = sums + above @ new, p - f + above.sum(1)
        else:
            sums, number = sums + new.cumsum(1), p - f + torch.arange(1, n + 1, device="cuda:0").double()
        sums, number = sums.transpose(0, 1), number[:, None, None]  # [n][Hkv][d]
        tol = bound(sums, number, half).repeat_interleave(H // Hkv, 1)
        off = (out[b].double() - (sums / number).repeat_interleave(H // Hkv, 1)).abs()
        assert (off <= tol).all(), (b, (off > tol).nonzero()[:3], float((off * number).max()))


NORMS = [  # batch, n, heads, heads_kv, d, page, past: cluster, cuts, a few rows, tiles of rows, the chunk kernel, its cuts
    (4, 1, 12, 2, 128, 16, 1500), (1, 1, 12, 2, 128, 128, 9000), (1, 1, 14, 2, 64, 16, 60000), (1, 20, 12, 2, 64, 16, 6000),
    (1, 40, 12, 2, 128, 16, 1000), (16, 60, 12, 2, 128, 64, 2000), (16, 60, 14, 2, 64, 64, 2000), (2, 100, 12, 2, 128, 64, 12000),
]


@pytest.mark.parametrize("B,n,H,Hkv,d,page,past", NORMS)
def test_two_pieces_of_a_query_are_told_from_one(env, B, n, H, Hkv, d, page, past):
    """The error's norm over the output's. A score is off by its products' truncated sums: d / 16 steps in each of two pieces of
    at most 2^-23 of a partial sum, whose size is about 1.5 and which counts half: 16 * 2^-24 * 1.5 = 2^-19.4 at the most, and
    weights are off by that, their values' sum by their mean in squares: below 2^-18. One f16 piece of a probability alone is off by
    2^-12 / sqrt(3) * 0.7 = 2^-13.3 of it (mean in squares): above 2^-15."""
    torch, ops = env
    rng = np.random.default_rng(past)
    w = World(torch, ops, rng, B, Hkv, d, page, past + n, False)
    q = up(torch, 1.5 * normal(rng, B, n, H, d))
    table = w.cache.table[:, : w.slots // page].long()
    k, v = (t[table].transpose(1, 2).reshape(B, Hkv, w.slots, d)[:, :, : past + n].double() for t in (w.cache.k, w.cache.v))
    mask = torch.arange(past + n, device="cuda:0") > past + torch.arange(n, device="cuda:0")[:, None]
    want = torch.empty(B, n, H, d, dtype=torch.float64, device="cuda:0")
    for h in range(H):
        s = (q[:, :, h].double() @ k[:, h // (H // Hkv)].transpose(1, 2) / d ** 0.5).masked_fill(mask, -float("inf"))
        want[:, :, h] = torch.softmax(s, -1) @ v[:, h // (H // Hkv)]
    off = {}
    try:
        for kind in ("f32", "tf32"):
            ops.set_math(kind)
            off[kind] = float((w.cache.attn(q, past).double() - want).norm() / want.norm())
    finally:
        ops.set_math("f32")
    ops.sync()
    assert off["f32"] < 2.0 ** -18 and off["tf32"] > 2.0 ** -15, off


@pytest.mark.parametrize("B,n,H,Hkv,d,bf16,tree", [(1, 1, 12, 2, 128, True, False), (1, 25, 12, 2, 128, False, True), (2, 61, 14, 2, 64, True, True),
                                                   (1, 2, 8, 8, 64, False, False), (2, 1, 2, 1, 128, False, False), (3, 200, 4, 2, 128, False, False)])
@pytest.mark.parametrize("own", [False, True])
def test_a_workspace_used_again_by_shorter_calls(env, B, n, H, Hkv, d, bf16, tree, own):
    """Each call's outputs are those of a workspace of its own, whatever lay in this one, and nothing is written behind it."""
    torch, ops = env
    rng = np.random.default_rng(n)
    w = World(torch, ops, rng, B, Hkv, d, 64, 40000 + n, bf16)
    size = w.cache.attn_workspace_bytes(n, H, 40000)
    store = torch.empty(size + 4096, dtype=torch.uint8, device="cuda:0")
    q = up(torch, normal(rng, B, n, H, d), w.row)
    args = {"tree": i32(torch, tree_of(rng, n))} if tree else {}
    for most in (40000, 19000, 9001, 3000, 700, 130, 15, 0):
        past = most
        if own:  # lengths of their own, on the device
            past, args["max_past"] = i32(torch, [most] + rng.integers(0, most + 1, B - 1).tolist()), most
        want = w.cache.attn(q, past, **args)
        store.fill_(255)  # NaN in every float
        assert torch.equal(w.cache.attn(q, past, workspace=store[:size], **args), want)
        assert torch.equal(w.cache.attn(q, past, workspace=store[:size], **args), want)
        assert (store[size:] == 255).all()
    ops.sync()


@pytest.mark.parametrize("d,rot", [(64, 64), (64, 32), (128, 128), (128, 64)])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("bf16", [False, True])
def test_rotary_tables_that_start_anywhere(env, d, rot, inter, bf16):
    """Tables one, two and three floats off a 16-byte boundary: the same bits."""
    torch, ops = env
    rng = np.random.default_rng(d + rot)
    B, n, H, Hkv, past = 2, 9, 6, 2, 21
    row = torch.bfloat16 if bf16 else torch.float32
    tables = [up(torch, a) for a in ops.scaled_rope_tables(past + n, rot, 1e4)]
    q, k, v = (up(torch, normal(rng, B, n, h, d), row) for h in (H, Hkv, Hkv))

    def off_by(t, floats):
        return torch.zeros(t.numel() + 4, device="cuda:0")[floats:floats + t.numel()].view(t.shape).copy_(t)

    results = []
    for floats in ((0, 0), (1, 1), (2, 2), (3, 3), (0, 1), (2, 0)):
        w = World(torch, ops, np.random.default_rng(1), B, Hkv, d, 16, past + n, bf16)
        out = torch.empty_like(q)
        w.cache.append(k, v, past, q=q, q_out=out, rope=(*(off_by(t, f) for t, f in zip(tables, floats)), inter))
        results.append((out, w.cache.k, w.cache.v))
    ops.sync()
    for other in results[1:]:
        assert all(torch.equal(a, b) for a, b in zip(results[0], other))


@pytest.mark.parametrize("B,n,H,d,slots", [(1, 1, 12, 64, 40000), (1, 100, 12, 128, 4000), (3, 300, 4, 64, 256), (1, 140, 12, 128, 96),
                                           (1, 600, 4, 128, 512)])
@pytest.mark.parametrize("kv8", [False, True])
def test_a_workspace_for_lengths_up_to_the_caches_end(env, B, n, H, d, slots, kv8):
    """Lengths and counts on the device: past tokens up to the cache's end, or more tokens in the call than it holds."""
    torch, ops = env
    rng = np.random.default_rng(slots)
    slots = -(-slots // 32) * 32
    cache = ops.Kv8Cache.empty(B, 2, d, slots) if kv8 else World(torch, ops, rng, B, 2, d, 16, slots - 32, False).cache
    n_ctx, count = cache.n_ctx, rng.integers(1, min(n, 9) + 1, B)
    past = i32(torch, n_ctx - 40 - count if n_ctx > 100 else [0] * B)
    q = up(torch, normal(rng, B, n, H, d))
    want = cache.attn(q, past, count=i32(torch, count), max_past=n_ctx)
    for size in (cache.attn_workspace_bytes(n, H, n_ctx), cache.attn_workspace_bytes(n, H)):
        ws = torch.empty(max(16, size), dtype=torch.uint8, device="cuda:0")
        assert torch.equal(cache.attn(q, past, count=i32(torch, count), max_past=n_ctx, workspace=ws, out=torch.zeros_like(q)), want)
    ops.sync()


SOME = [(2, 1, 12, 2, 128, 16, 700), (1, 1, 14, 2, 64, 16, 30000), (2, 6, 12, 2, 64, 32, 300), (40, 24, 12, 2, 128, 16, 200), (2, 100, 12, 2, 128, 64, 5000)]


@pytest.mark.parametrize("B,n,H,Hkv,d,page,past", SOME)
@pytest.mark.parametrize("bf16", [False, True])
def test_a_query_that_is_no_number_spoils_its_own_row(env, B, n, H, Hkv, d, page, past, bf16):
    torch, ops = env
    rng = np.random.default_rng(n)
    w = World(torch, ops, rng, B, Hkv, d, page, past + n, bf16)
    q = up(torch, normal(rng, B, n, H, d), w.row)
    want = w.cache.attn(q, past)
    bad = torch.zeros(B, n, H, dtype=torch.bool, device="cuda:0")
    for i, x in enumerate((float("nan"), float("inf"), -float("inf"))):
        b, t, h = B - 1, (i * n) // 3, (5 * i + 1) % H
        q[b, t, h, (7 * i) % d] = x
        bad[b, t, h] = True
    got = w.cache.attn(q, past)
    ops.sync()
    assert torch.equal(got[~bad], want[~bad]) and not torch.isfinite(got[bad]).any()


@pytest.mark.parametrize("B,n,H,Hkv,d,page,past", SOME)
@pytest.mark.parametrize("bf16", [False, True])
def test_a_table_that_is_part_of_a_wider_one(env, B, n, H, Hkv, d, page, past, bf16):
    """Rows of the table further apart than they are long, and not from a 16-byte boundary on."""
    torch, ops = env
    rng = np.random.default_rng(n)
    w = World(torch, ops, rng, B, Hkv, d, page, past + n, bf16)
    wide = torch.full((B + 2, w.cache.table.shape[1] + 5), 1 << 30, dtype=torch.int32, device="cuda:0")
    part = wide[1:B + 1, 3:3 + w.cache.table.shape[1]]
    part.copy_(w.cache.table)
    pools = [x.clone() for x in (w.cache.k, w.cache.v)]
    other = ops.PagedCache(*pools, part)
    q, k, v = (up(torch, normal(rng, B, n, h, d), w.row) for h in (H, Hkv, Hkv))
    path, kept = i32(torch, [[n - 1] + [-1] * (n - 1)] * B), i32(torch, [1] * B)
    out = []
    for c in (w.cache, other):
        c.append(k, v, past)
        out.append(c.attn(q, past))
        ops.paged_keep(c, path, kept, past)
    ops.sync()
    assert torch.equal(*out) and torch.equal(other.k, w.cache.k) and torch.equal(other.v, w.cache.v)

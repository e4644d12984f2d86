"""Attention over pages where the tcgen05 kernel is the one that runs (many rows of many sequences, or a long cache), which
each test sees to by the kernel's size: against the oracle, in every form it has: both d, f32 in two pieces and one, bf16,
128 rows and more, cut keys, trees, ragged batches; and what lies where a query does not look."""
import numpy as np
import pytest

from oracle import paged as O
from tests.conftest import has_gpu
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


def attend(torch, cache, q, *args, **kw):
    """cache.attn, which must have launched the kernel of 640 threads: the call is captured as well, into a graph whose
    nodes tell (a profiler's trace would, too, but one that was first opened a minute ago loses records)."""
    from cuda.bindings import driver
    out = cache.attn(q, *args, **kw)
    graph, side = torch.cuda.CUDAGraph(keep_graph=True), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        cache.attn(q, *args, **{**kw, "out": torch.empty_like(out)})
    raw = driver.CUgraph(graph.raw_cuda_graph())
    err, _, n = driver.cuGraphGetNodes(raw)
    err, nodes, n = driver.cuGraphGetNodes(raw, n)
    assert err == driver.CUresult.CUDA_SUCCESS
    threads = []
    for node in nodes[:n]:
        err, kind = driver.cuGraphNodeGetType(node)
        if kind == driver.CUgraphNodeType.CU_GRAPH_NODE_TYPE_KERNEL:
            err, params = driver.cuGraphKernelNodeGetParams(node)
            assert err == driver.CUresult.CUDA_SUCCESS
            threads.append(params.blockDimX)
    assert 640 in threads, threads
    return out


def contents(w, b):
    """k and v [n_head_kv][slots][d] of sequence b, in 64 bits."""
    pages = np.maximum(w.np_table[b, : w.slots // w.page], 0).tolist()
    return [np.moveaxis(t[pages].double().cpu().numpy(), 1, 0).reshape(w.Hkv, w.slots, w.d) for t in (w.cache.k, w.cache.v)]


def check_attn(torch, out, before, w, q, past, count, first, parents, pieces):
    """Some of the sequences against the oracle; rows behind every sequence's last one as they were."""
    half = 2.0 ** -8 if q.dtype is torch.bfloat16 else 2.0 ** -24
    for b in sorted({0, 1, w.B // 3, w.B // 2, w.B - 1}):
        m = int(count[b])
        seen = O.seen_slots(past[b], m, int(first[b]), w.slots, None if parents is None else parents[b])
        want, tol = O.attention(q[b, :m].float().cpu().numpy(), *contents(w, b), seen, pieces, half, True)
        got = out[b, :m].float().cpu().numpy()
        bad = ~(np.abs(got - want) <= tol)
        assert not bad.any(), (b, np.argwhere(bad)[:3], np.abs(got - want)[bad][:3], tol[bad][:3])
    behind = torch.arange(q.shape[1], device=q.device) >= torch.tensor([int(c) for c in count], device=q.device)[:, None]
    assert torch.equal(out[behind], before[behind])


SHAPES = [  # batch, n, heads, heads_kv, d, page, past, tree
    (40, 24, 12, 2, 128, 16, 200, False),    # a slot of 128 rows and one of 16
    (40, 21, 12, 2, 128, 32, 301, False),    # 126 rows: both slots take them
    (64, 16, 14, 2, 64, 16, 150, True),      # 112
    (40, 61, 14, 2, 64, 16, 140, True),      # two CTAs of rows
    (3, 20, 12, 2, 128, 16, 6000, True),     # cut keys, both slots
    (2, 130, 4, 1, 64, 64, 5000, False),     # cut keys, three CTAs of rows
    (5, 40, 16, 2, 128, 256, 3000, False), (4, 256, 4, 2, 64, 128, 2000, True), (70, 128, 2, 1, 128, 64, 77, False),
    (60, 30, 6, 1, 64, 32, 3000, True),      # more cuts than fit at once where lengths differ
    (100, 40, 8, 2, 64, 256, 0, False), (90, 100, 8, 2, 128, 16, 0, True),
]


@pytest.mark.parametrize("B,n,H,Hkv,d,page,most,tree", SHAPES)
@pytest.mark.parametrize("kind", ["f32", "tf32", "bf16"])
@pytest.mark.parametrize("ragged", [False, True])
def test_chunks(env, B, n, H, Hkv, d, page, most, tree, kind, ragged):
    torch, ops = env
    rng = np.random.default_rng(B * n + H + most)
    w = World(torch, ops, rng, B, Hkv, d, page, most + n, kind == "bf16", joint=ragged)
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
    ops.set_math("tf32" if kind == "tf32" else "f32")
    try:
        out = attend(torch, w.cache, q, i32(torch, past) if ragged else most, out=before.clone(), **args)
    finally:
        ops.set_math("f32")
    ops.sync()
    check_attn(torch, out, before, w, q, past, count, first, parents, {"f32": 2, "tf32": 1, "bf16": 0}[kind])


@pytest.mark.parametrize("B,n,H,Hkv,d,page,past,tree", [s for s in SHAPES if s[6]])
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("kind", ["nan", "inf", "huge"])
def test_what_no_query_sees(env, B, n, H, Hkv, d, page, past, tree, bf16, kind):
    torch, ops = env
    rng = np.random.default_rng(n + d)
    w = World(torch, ops, rng, B, Hkv, d, page, past + n + 20, bf16)
    first = rng.integers(0, min(past, 150) + 1, B)
    count = rng.integers(max(1, n - 4), n + 1, B)
    parents = [tree_of(rng, n) for _ in range(B)] if tree else None
    args = dict(first=i32(torch, first), count=i32(torch, count))
    if tree:
        args["tree"] = i32(torch, parents)
    q = up(torch, normal(rng, B, n, H, d), w.row)
    zero = torch.zeros_like(q)
    want = attend(torch, w.cache, q, past, out=zero.clone(), **args)
    bad = {"nan": float("nan"), "inf": float("inf"), "huge": torch.finfo(w.held).max}[kind]
    keep = np.zeros((w.cache.k.shape[0], page), bool)
    for b in range(B):
        t = np.arange(first[b], past + count[b])
        keep[w.np_table[b, t // page], t % page] = True
    keep = torch.from_numpy(keep).cuda()
    for pool in (w.cache.k, w.cache.v):
        pool.masked_fill_(~keep[:, None, :, None], bad)
    got = attend(torch, w.cache, q, past, out=zero.clone(), **args)
    ops.sync()
    assert torch.equal(got, want)


@pytest.mark.parametrize("B,n,H,Hkv,d,page,past,tree", SHAPES)
@pytest.mark.parametrize("bf16", [False, True])
def test_a_token_that_only_some_queries_see(env, B, n, H, Hkv, d, page, past, tree, bf16):
    torch, ops = env
    rng = np.random.default_rng(n)
    w = World(torch, ops, rng, B, Hkv, d, page, past + n, bf16)
    parents = [tree_of(rng, n) for _ in range(B)] if tree else None
    args = {"tree": i32(torch, parents)} if tree else {}
    q = up(torch, normal(rng, B, n, H, d), w.row)
    want = attend(torch, w.cache, q, past, **args).clone()
    seen = np.zeros((B, n), bool)
    for b in range(B):
        t = past + (b * 7) % n
        place = (int(w.np_table[b, t // page]), slice(None), t % page)
        w.cache.v[place][:, 3] = float("inf")
        w.cache.v[place][:, d - 7] = float("nan")
        w.cache.v[place][:, d - 1] = -float("inf")
        seen[b] = O.seen_slots(past, n, 0, past + n, parents[b] if tree else None)[:, t]
    got = attend(torch, w.cache, q, past, **args)
    ops.sync()
    seen = torch.from_numpy(seen).cuda()
    assert torch.equal(got[~seen], want[~seen])
    plain = [c for c in range(d) if c not in (3, d - 7, d - 1)]
    assert torch.equal(got[seen][..., plain], want[seen][..., plain])
    assert torch.isnan(got[seen][..., d - 7]).all()
    if bf16:
        assert (got[seen][..., 3] == float("inf")).all() and (got[seen][..., d - 1] == -float("inf")).all()
    else:
        # a probability is two pieces h + l, l the nearest f16 of what h leaves, so 0 or below it as often as above: where
        # all of a tile's queries see the token, h inf + l inf is NaN for those
        assert not torch.isfinite(got[seen][..., [3, d - 1]]).any()


@pytest.mark.parametrize("B,n,H,Hkv,d,page,past,tree", [s for s in SHAPES if s[6] > s[5]])
@pytest.mark.parametrize("bf16", [False, True])
def test_pages_that_are_none(env, B, n, H, Hkv, d, page, past, tree, bf16):
    torch, ops = env
    from zwhisper_b200._lib import ZwgError
    rng = np.random.default_rng(n)
    w = World(torch, ops, rng, B, Hkv, d, page, past + n, bf16)
    parents = [tree_of(rng, n) for _ in range(B)] if tree else None
    args = {"tree": i32(torch, parents)} if tree else {}
    last = (past + n - 1) // page
    bad = {(0, 0): -1, (0, last): w.cache.k.shape[0], (1, last // 2): -(1 << 31), (B - 1, max(0, last - 1)): 1 << 30}
    for (b, i), x in bad.items():
        w.cache.table[b, i] = x
    q = up(torch, normal(rng, B, n, H, d), w.row)
    ops.sync()
    out = attend(torch, w.cache, q, past, **args)
    with pytest.raises(ZwgError):
        ops.sync()
    for b in {0, 1, B - 1, B // 2}:
        k, v = contents(w, b)
        seen = O.seen_slots(past, n, 0, w.slots, parents[b] if tree else None)
        for (bb, i) in bad:
            if bb == b:
                seen[:, i * page:(i + 1) * page] = False
        want, tol = O.attention(q[b].float().cpu().numpy(), k, v, seen, 0 if bf16 else 2, 2.0 ** (-8 if bf16 else -24), True)
        assert (np.abs(out[b].float().cpu().numpy() - want) <= tol).all()


@pytest.mark.parametrize("bf16", [False, True])
def test_scores_of_any_size(env, bf16):
    """Maxima that grow along the keys (sums are taken over again), and scores so far apart that one key is all there is."""
    torch, ops = env
    rng = np.random.default_rng(3)
    for size in (0.01, 8.0, 60.0):
        w = World(torch, ops, rng, 40, 2, 128, 16, 700, bf16)
        for b in range(40):
            for i in range(44):
                w.cache.k[int(w.np_table[b, i])] *= size * (0.2 + i / 44)
        q = up(torch, normal(rng, 40, 20, 12, 128), w.row)
        before = torch.zeros_like(q)
        out = attend(torch, w.cache, q, 680, out=before.clone())
        check_attn(torch, out, before, w, q, [680] * 40, [20] * 40, [0] * 40, None, 0 if bf16 else 2)


@pytest.mark.parametrize("B", [2, 3, 255, 256, 257, 300])
@pytest.mark.parametrize("bad", [False, True])
def test_every_sequence_of_many_lengths_is_taken_once(env, B, bad):
    """CTAs take up to 256 sequences in the order of their lengths, many of them alike here; an entry out of range is left
    out, and the others stand."""
    torch, ops = env
    rng = np.random.default_rng(B)
    n, most = (130 if B > 3 else 250), (90 if B > 3 else 3000)
    w = World(torch, ops, rng, B, 1, 64, 16, most + n, True)
    past = rng.choice([0, 1, 40, most - 1, most], B)
    q = up(torch, 1.5 * normal(rng, B, n, 2, 64), w.row)
    before = up(torch, normal(rng, B, n, 2, 64), w.row)
    given, count = past.copy(), np.full(B, n)
    if bad:
        given[B // 2], count[B // 2] = most + 7, 0  # (count: of what check_attn expects)
        if B > 3:
            given[1], count[1] = -(2 ** 31), 0
    out = attend(torch, w.cache, q, i32(torch, given), max_past=most, out=before.clone())
    if bad:
        with pytest.raises(RuntimeError):
            ops.sync()
    else:
        ops.sync()
    for b in range(B):  # rows that are written differ from those that were there
        same = (out[b] == before[b]).all(-1).all(-1).sum().item()
        assert same == n - count[b], (b, same)
    check_attn(torch, out, before, w, q, past, count, np.zeros(B, int), None, 0)

"""Attention over pages of which those before a sequence's `first` have been given back (their entries are -1): no query
needs them, so the outputs stay and the device error word stays clear."""
import numpy as np
import pytest

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


SHAPES = [  # batch, n, heads, heads_kv, d, page, past, tree: steps, few rows and chunks, alone and in cuts
    (2, 1, 14, 2, 64, 16, 333, False), (1, 1, 6, 1, 64, 16, 9000, False), (2, 1, 12, 2, 128, 16, 333, False),
    (2, 5, 14, 2, 64, 16, 300, True), (2, 1, 2, 1, 64, 32, 333, False), (40, 40, 12, 2, 64, 16, 330, False),
    (3, 20, 12, 2, 128, 32, 3000, True), (40, 24, 12, 2, 128, 128, 500, False),
]


@pytest.mark.parametrize("B,n,H,Hkv,d,page,past,tree", SHAPES)
@pytest.mark.parametrize("bf16", [False, True])
def test_pages_before_the_first_key_are_not_needed(env, B, n, H, Hkv, d, page, past, tree, bf16):
    torch, ops = env
    rng = np.random.default_rng(n + d)
    w = World(torch, ops, rng, B, Hkv, d, page, past + n, bf16)
    args = {"tree": i32(torch, [tree_of(rng, n) for _ in range(B)])} if tree else {}
    q = up(torch, normal(rng, B, n, H, d), w.row)
    at = past // page
    for first in (page, page + 1, 2 * page - 1, at * page, at * page - 1, past):
        w.cache.table.copy_(i32(torch, w.np_table))
        mine = i32(torch, [max(0, first - 16 * b) for b in range(B)])
        want = w.cache.attn(q, past, first=mine, **args)
        ops.sync()
        for b in range(B):
            w.cache.table[b, : max(0, first - 16 * b) // page] = -1
        got = w.cache.attn(q, past, first=mine, **args)
        ops.sync()  # raises where a page was missed
        assert torch.equal(got, want)


@pytest.mark.parametrize("n,H,d", [(1, 6, 64), (1, 6, 128), (3, 40, 64), (40, 12, 64), (40, 12, 128)])
def test_a_sequence_that_sees_no_key_needs_no_page(env, n, H, d):
    torch, ops = env
    rng = np.random.default_rng(n)
    B, past = 40, 37
    w = World(torch, ops, rng, B, 1, d, 16, past + n, True)
    w.cache.table[1] = -1
    first = [0] * B
    first[1] = past + n
    out = w.cache.attn(up(torch, normal(rng, B, n, H, d), w.row), past, first=i32(torch, first))
    ops.sync()
    assert not out[1].any() and out[0].any() and out[2].any()

"""Calls on the 8-bit cache that its documentation allows and that are easily refused or answered wrongly."""
import numpy as np
import pytest

from oracle import kv8 as O
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


def i32(torch, a):
    return torch.tensor(list(a), dtype=torch.int32, device="cuda:0")


def test_ragged_append_with_tables_shorter_than_the_cache(env):
    """Sequences within the tables are appended; those that end or start behind them are left out and reported."""
    torch, ops = env
    from zwhisper_b200._lib import ZwgError
    rng = np.random.default_rng(0)
    B, n, past = 5, 3, [0, 29, 30, 33, 7]  # of 32 positions
    cos, sin = (torch.from_numpy(a).cuda() for a in ops.rope_tables(32, 64, 1e4))
    k, v = (rng.standard_normal((B, n, 1, 64), dtype=np.float32) for _ in range(2))
    cache, want = ops.Kv8Cache.empty(B, 1, 64, 64), O.Cache(B, 1, 64, 64)
    ops.sync()
    # within the tables: no error
    cache.append(torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda(), i32(torch, [0, 29, 0, 0, 7]), count=i32(torch, [3, 3, 0, 0, 3]),
                 rope=(cos, sin))
    ops.sync()
    cache = ops.Kv8Cache.empty(B, 1, 64, 64)
    cache.append(torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda(), i32(torch, past), rope=(cos, sin))
    with pytest.raises(ZwgError):
        ops.sync()
    turned = k.copy()
    for b in (0, 1, 4):
        turned[b] = O.rope(k[b], cos.cpu().numpy(), sin.cpu().numpy(), past[b] + np.arange(n), False)
    want.append(turned, v, past, [3, 3, 0, 0, 3])
    np.testing.assert_array_equal(cache.k.cpu().numpy().reshape(B, 1, 64, 64), want.ints[0])
    np.testing.assert_array_equal(cache.v_scale.cpu().numpy(), want.scale[1])
    np.testing.assert_array_equal(cache.open_block.cpu().numpy(), want.tag)
    # a bound of the caller's own, as attn has
    cache = ops.Kv8Cache.empty(B, 1, 64, 64)
    cache.append(torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda(), i32(torch, past), rope=(cos, sin), max_past=7)
    with pytest.raises(ZwgError):
        ops.sync()
    assert cache.open_block.flatten().tolist() == [0, -1, -1, -1, 0]
    with pytest.raises(ZwgError):
        cache.append(torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda(), i32(torch, past), rope=(cos, sin), max_past=33)
    ops.sync()


@pytest.mark.parametrize("B,n_ctx", [(1, 2048), (1, 4096), (2, 1024), (3, 1056), (8, 4096), (12, 2048), (64, 2048)])
@pytest.mark.parametrize("n", [1, 2, 40, 200])
def test_workspace_for_any_length_serves_positions_on_the_device(env, B, n_ctx, n):
    """attn_workspace_bytes without a length is enough for a call whose positions only the device knows."""
    torch, ops = env
    g = torch.Generator(device="cuda:0").manual_seed(n)
    cache = ops.Kv8Cache.empty(B, 2, 64, n_ctx)
    k, v = (torch.randn(B, n_ctx, 2, 64, device="cuda:0", generator=g) for _ in range(2))
    cache.append(k, v, 0)
    q = torch.randn(B, n, 12, 64, device="cuda:0", generator=g)
    size = cache.attn_workspace_bytes(n, 12)
    ws = torch.full((size + 256,), 77, dtype=torch.uint8, device="cuda:0")
    at = i32(torch, [n_ctx - n] * B)
    out = cache.attn(q, at, workspace=ws[:size])
    assert torch.equal(out, cache.attn(q, at))
    assert (ws[size:] == 77).all()
    ops.sync()


def test_rotary_tables_on_another_device_are_refused(env):
    torch, ops = env
    st = ops.LlmState(1, 1, 2, 1, 64, 64, kv8=True)
    t = torch.ones(64, 32, device="cuda:0")
    st.set_rope(t, t)
    st.device = 1  # as if the state were there
    with pytest.raises(ValueError, match="cuda:1"):
        st.set_rope(t, t)
    st.device = 0
    st.close()


@pytest.mark.parametrize("B,n,past,d", [(1, 1, 4000, 64), (2, 1, 20000, 128), (3, 5, 300, 64), (1, 64, 4000, 64), (40, 150, 2000, 64),
                                        (12, 256, 1700, 128)])
@pytest.mark.parametrize("bf16", [False, True])
def test_output_in_the_place_of_the_queries(env, B, n, past, d, bf16):
    """Whole, cut and joined keys, and sums that wait in the output's place."""
    torch, ops = env
    g = torch.Generator(device="cuda:0").manual_seed(n)
    cache = ops.Kv8Cache.empty(B, 1, d, (past + n + 31) // 32 * 32)
    cache.append(*(torch.randn(B, past + n, 1, d, device="cuda:0", generator=g) for _ in range(2)), 0)
    q = torch.randn(B, n, 6, d, device="cuda:0", generator=g).to(torch.bfloat16 if bf16 else torch.float32)
    want = cache.attn(q, past)
    assert cache.attn(q, past, out=q) is q and torch.equal(q, want)
    ops.sync()


def test_a_cache_whose_offsets_pass_32_bits(env):
    """A sequence of more than 2^28 tokens of d 128 (34 GB of keys, as many of values): append, read, a step and a chunk."""
    torch, ops = env
    rng = np.random.default_rng(1)
    d, n_ctx, past = 128, 2 ** 28 + 4096, 2 ** 28 + 1003
    cache = ops.Kv8Cache.empty(1, 1, d, n_ctx)
    cache.k_scale.fill_(1.0)
    cache.v.fill_(64)
    cache.v_scale.fill_(1.0 / 64)
    k, v = (rng.standard_normal((1, 5, 1, d), dtype=np.float32) for _ in range(2))
    cache.append(torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda(), past)
    assert int(cache.open_block[0, 0]) == past // 32 and past // 32 == (past + 4) // 32
    # the open block goes on from the cache's own values in front of the new tokens: zeros and ones
    want = O.Cache(1, 1, d, 32)
    want.append(np.zeros((1, past % 32, 1, d), np.float32), np.ones((1, past % 32, 1, d), np.float32), [0])
    want.append(k, v, [past % 32])
    gk, gv = cache.read(5, past)
    for got, side in ((gk, 0), (gv, 1)):
        np.testing.assert_array_equal(got[0, :, 0].cpu().numpy(), want.values()[side][0, 0, past % 32:past % 32 + 5])
    # a step that sees the last 200 tokens alone
    q = rng.standard_normal((1, 1, 6, d), dtype=np.float32)
    out = cache.attn(torch.from_numpy(q).cuda(), past + 4, first=i32(torch, [past - 195])).cpu().numpy()
    kk, vv = (x[0, :, 0].cpu().numpy()[None, None].astype(np.float64) for x in cache.read(200, past - 195))
    exact, tol = O.attention(q, kk, vv, [199], None, None, 2, 2.0 ** -24)
    assert (np.abs(out - exact) <= tol).all()
    # block 5 alone has keys that count: every query of a step and of a chunk gives its values
    cache.k[0, 0, 5] = 100
    cache.v[0, 0, 5] = 32
    for n in (1, 16):
        out = cache.attn(torch.ones(1, n, 6, d, device="cuda:0"), past)
        assert (out - 0.5).abs().max() < 1e-6
    ops.sync()
    del cache
    torch.cuda.empty_cache()

"""The key/value cache in 8 bits on the device (zwg_kv8_append, _read, _attn, zwg_rope and the
states that keep such caches) against oracle/kv8.py. Rotated rows, int8 values, scales and read-back
values are compared bit for bit: they are the same f32 (or exactly rounded) operations. The
attention is held to the bound that oracle/kv8.py derives for each output from the arithmetic."""
import numpy as np
import pytest

from oracle import kv8 as O
from oracle import qwen
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
    return torch.tensor(list(a), dtype=torch.int32, device="cuda:0")


# ---- rotary positions -------------------------------------------------------------------

ROPE = [  # batch, n, heads, heads_kv, d, rot, interleaved, bf16
    (1, 1, 1, 1, 64, 64, False, False), (3, 5, 14, 2, 64, 64, False, True), (2, 33, 12, 2, 128, 64, True, False),
    (4, 2, 6, 1, 128, 128, True, True), (2, 3, 4, 4, 80, 20, False, False), (2, 3, 4, 4, 80, 20, True, True),
    (2, 4, 3, 1, 10, 6, True, False), (2, 4, 3, 1, 10, 2, False, True), (1, 300, 2, 2, 64, 24, False, True),
]


@pytest.mark.parametrize("B,n,H,Hkv,d,rot,inter,bf16", ROPE)
@pytest.mark.parametrize("ragged", [False, True])
def test_rope(env, B, n, H, Hkv, d, rot, inter, bf16, ragged):
    torch, ops = env
    rng = np.random.default_rng(B * n + rot)
    n_ctx = n + 40
    cos, sin = (up(torch, a) for a in ops.scaled_rope_tables(n_ctx, rot, 1e4, "linear", 2.5))
    kind = torch.bfloat16 if bf16 else torch.float32
    past = rng.integers(0, 41, B)
    count = rng.integers(0, n + 1, B)
    # the three parts of a packed row, read and written in place
    qkv = up(torch, normal(rng, B, n, H + 2 * Hkv, d), kind)
    want = qkv.float().cpu().numpy()
    for b in range(B):
        m = int(count[b]) if ragged else n
        pos = (int(past[b]) if ragged else 17) + np.arange(m)
        want[b, :m, :H + Hkv] = O.rope(want[b, :m, :H + Hkv], cos.cpu().numpy(), sin.cpu().numpy(), pos, inter)
    want = torch.from_numpy(want).to(kind)
    before = qkv.clone()
    args = dict(count=i32(torch, count)) if ragged else {}
    at = i32(torch, past) if ragged else 17
    q, k = qkv[:, :, :H], qkv[:, :, H:H + Hkv]
    qo, ko = ops.rope(q, cos, sin, at, k=k, interleaved=inter, inplace=False, q_out=q.clone().contiguous(),
                      k_out=k.clone().contiguous(), **args)
    assert torch.equal(qkv, before)
    ops.rope(q, cos, sin, at, k=k, interleaved=inter, **args)
    assert torch.equal(qkv.cpu(), want)
    assert torch.equal(qo, qkv[:, :, :H]) and torch.equal(ko, qkv[:, :, H:H + Hkv])
    ops.sync()


def test_rope_unaligned_rows_and_turn_back(env):
    torch, ops = env
    rng = np.random.default_rng(1)
    cos, sin = (up(torch, a) for a in ops.rope_tables(64, 64, 1e4))
    flat = up(torch, normal(rng, 2 * 5 * (3 * 64 + 1) + 1))
    x = flat[1:].view(2, 5, 3 * 64 + 1)[..., :192].view(2, 5, 3, 64)
    want = np.stack([O.rope(a, cos.cpu().numpy(), sin.cpu().numpy(), 3 + np.arange(5), False) for a in x.cpu().numpy()])
    ops.rope(x, cos, sin, 3)
    np.testing.assert_array_equal(x.cpu().numpy(), want)
    # the rotation by the other angle, its transpose, takes it back: the rows' own gradient
    back = ops.rope(x.contiguous(), cos, -sin, 3)
    orig = np.stack([O.rope(a, cos.cpu().numpy(), -sin.cpu().numpy(), 3 + np.arange(5), False) for a in want])
    np.testing.assert_array_equal(back.cpu().numpy(), orig)


def test_rope_out_of_range_sequence_is_skipped(env):
    torch, ops = env
    from zwhisper_b200._lib import ZwgError
    cos, sin = (up(torch, a) for a in ops.rope_tables(32, 64, 1e4))
    x = torch.randn(4, 3, 2, 64, device="cuda:0")
    before = x.clone()
    ops.sync()
    ops.rope(x, cos, sin, i32(torch, [0, 30, -1, 33]))
    with pytest.raises(ZwgError):
        ops.sync()
    assert torch.equal(x[1:], before[1:]) and not torch.equal(x[0], before[0])
    ops.sync()


# ---- append and read --------------------------------------------------------------------

def same(torch, cache, want):
    """The device cache holds the oracle's (the int8 values, scales, open rows and tags)."""
    B, H, n_ctx, d = want.ints[0].shape
    k = cache.k.cpu().numpy().reshape(B, H, n_ctx, d)
    v = cache.v.cpu().numpy().transpose(0, 1, 2, 4, 3).reshape(B, H, n_ctx, d)
    np.testing.assert_array_equal(k, want.ints[0])
    np.testing.assert_array_equal(v, want.ints[1])
    np.testing.assert_array_equal(cache.k_scale.cpu().numpy(), want.scale[0])
    np.testing.assert_array_equal(cache.v_scale.cpu().numpy(), want.scale[1])
    np.testing.assert_array_equal(cache.k_open.cpu().numpy(), want.open[0])
    np.testing.assert_array_equal(cache.v_open.cpu().numpy(), want.open[1])
    np.testing.assert_array_equal(cache.open_block.cpu().numpy(), want.tag)


APPENDS = [  # batch, heads_kv, d, n_ctx, positions and lengths of the calls (going back included)
    (1, 1, 64, 32, [(0, 1)]),
    (2, 2, 64, 128, [(0, 32), (32, 1), (33, 30), (63, 1), (64, 64)]),
    (2, 1, 128, 160, [(0, 5), (5, 1), (6, 100), (106, 54)]),
    (1, 3, 128, 96, [(0, 96)]),
    # back into a full block, into the open one, and to the start
    (2, 2, 128, 128, [(0, 70), (40, 3), (43, 2), (42, 1), (64, 40), (0, 2), (2, 40)]),
    (1, 1, 64, 128, [(0, 64), (63, 2), (31, 1)]),
]


@pytest.mark.parametrize("B,H,d,n_ctx,calls", APPENDS)
@pytest.mark.parametrize("bf16", [False, True])
def test_append_and_read(env, B, H, d, n_ctx, calls, bf16):
    torch, ops = env
    rng = np.random.default_rng(n_ctx + d)
    cache, want = ops.Kv8Cache.empty(B, H, d, n_ctx), O.Cache(B, H, d, n_ctx)
    for past, n in calls:
        kind = torch.bfloat16 if bf16 else torch.float32
        k, v = (up(torch, normal(rng, B, n, H, d) * np.exp(normal(rng, B, n, H, 1)), kind) for _ in range(2))
        cache.append(k, v, past)
        want.append(k.float().cpu().numpy(), v.float().cpu().numpy(), [past] * B)
        same(torch, cache, want)
        gk, gv = cache.read(past + n, 0)
        for got, side in ((gk, 0), (gv, 1)):
            np.testing.assert_array_equal(got.cpu().numpy(), want.values()[side][:, :, :past + n].transpose(0, 2, 1, 3))
    past, n = calls[-1]
    gk, _ = cache.read(n, past)
    np.testing.assert_array_equal(gk.cpu().numpy(), want.values()[0][:, :, past:past + n].transpose(0, 2, 1, 3))
    ops.sync()


def test_append_ragged_and_strided(env):
    torch, ops = env
    rng = np.random.default_rng(5)
    B, H, d, n_ctx, n = 5, 2, 64, 160, 37
    cache, want = ops.Kv8Cache.empty(B, H, d, n_ctx), O.Cache(B, H, d, n_ctx)
    past = np.zeros(B, np.int64)
    for count in ([37, 0, 1, 32, 36], [1, 1, 1, 1, 1], [0, 37, 31, 30, 37]):
        packed = up(torch, normal(rng, n, B, 3 * H, d))  # token-major: the batch is the inner stride
        k, v = packed[:, :, :H].transpose(0, 1), packed[:, :, 2 * H:].transpose(0, 1)
        cache.append(k, v, i32(torch, past), count=i32(torch, count))
        want.append(k.cpu().numpy(), v.cpu().numpy(), past, count)
        past = past + np.array(count)
        same(torch, cache, want)
    gk, gv = cache.read(20, i32(torch, past - 20 * (past >= 20)), count=i32(torch, [20 * (p >= 20) for p in past]))
    for b in range(B):
        if past[b] >= 20:
            np.testing.assert_array_equal(gv[b].cpu().numpy(), want.values()[1][b, :, past[b] - 20:past[b]].transpose(1, 0, 2))
    ops.sync()


def test_append_values_at_borders_and_odd_blocks(env):
    """Ties between two integers, blocks of zeros, tiny, huge, infinite and NaN values."""
    torch, ops = env
    rng = np.random.default_rng(6)
    B, H, d, n_ctx = 1, 8, 64, 32
    k = normal(rng, B, 32, H, d)
    k[:, :, 0] = rng.integers(-254, 255, (B, 32, d)) / np.float32(2)  # 127 / max = 1: halves are ties
    k[0, 3, 0, 5] = 127
    k[:, :, 0] = np.clip(k[:, :, 0], -127, 127)
    k[:, :, 1] = 0
    k[:, :, 2] *= np.float32(1e-42)
    k[:, :, 3] *= np.float32(1e37)
    k[0, 7, 4, 9] = np.inf
    k[0, 8, 5, 9] = np.nan
    k[0, 1, 6] = -np.float32(3.0)
    k[:, :, 7] = np.where(rng.random((B, 32, d)) < 0.5, 0.5, -1.0)  # half of the largest: 63.5 exactly
    cache, want = ops.Kv8Cache.empty(B, H, d, n_ctx), O.Cache(B, H, d, n_ctx)
    cache.append(up(torch, k), up(torch, -k), 0)
    want.append(k, -k, [0])
    same(torch, cache, want)
    got, _ = cache.read(32, 0)
    assert torch.isnan(got[0, :, 4:6]).all() and torch.isfinite(got[0, :, :4]).all()
    # filled anew from its start, a block reads as finite again
    cache.append(up(torch, k[:, :1]), up(torch, k[:, :1]), 0)
    got, _ = cache.read(1, 0)
    assert torch.isfinite(got).all()
    ops.sync()


@pytest.mark.parametrize("inter,rot", [(False, 64), (True, 64), (False, 32), (True, 6)])
def test_append_rotates(env, inter, rot):
    torch, ops = env
    rng = np.random.default_rng(7)
    B, H, d, n_ctx = 2, 2, 64, 128
    cos, sin = (up(torch, a) for a in ops.rope_tables(n_ctx, rot, 1e4))
    a, b = ops.Kv8Cache.empty(B, H, d, n_ctx), ops.Kv8Cache.empty(B, H, d, n_ctx)
    for past, n in ((0, 40), (40, 1), (41, 70)):
        k, v = (up(torch, normal(rng, B, n, H, d)) for _ in range(2))
        a.append(k, v, past, rope=(cos, sin, inter))
        b.append(ops.rope(k.clone(), cos, sin, past, interleaved=inter), v, past)
    for x, y in zip(a._keep, b._keep):
        assert torch.equal(x, y)
    ops.sync()


def test_append_out_of_range_is_skipped(env):
    torch, ops = env
    from zwhisper_b200._lib import ZwgError
    cache = ops.Kv8Cache.empty(4, 1, 64, 64)
    x = torch.randn(4, 3, 1, 64, device="cuda:0")
    ops.sync()
    cache.append(x, x, i32(torch, [0, 62, -5, 3]), count=i32(torch, [3, 3, 3, 4]))
    with pytest.raises(ZwgError):
        ops.sync()
    assert cache.open_block.flatten().tolist() == [0, -1, -1, -1]
    assert (cache.k[1:] == 0).all() and (cache.k_open[1:] == 0).all()
    # tables that are too short for the positions refuse a uniform call, and skip a ragged one
    cos, sin = (up(torch, a) for a in ops.rope_tables(8, 64, 1e4))
    with pytest.raises(ZwgError):
        cache.append(x, x, 6, rope=(cos, sin))
    ops.sync()


# ---- attention --------------------------------------------------------------------------

def fill(torch, ops, rng, B, H, d, n_ctx, length, spread=0.4):
    """A cache of random values, `length` tokens a sequence; what lies behind them is garbage."""
    k, v = (normal(rng, B, n_ctx, H, d) * np.exp(spread * normal(rng, B, n_ctx // 32, H, 1).repeat(32, 1)) for _ in range(2))
    cache, want = ops.Kv8Cache.empty(B, H, d, n_ctx), O.Cache(B, H, d, n_ctx)
    cache.append(up(torch, k), up(torch, v), 0, count=i32(torch, length))
    want.append(k, v, [0] * B, length)
    for b in range(B):
        blk = (int(length[b]) + 31) // 32
        cache.k[b, :, blk:] = 113
        cache.v[b, :, blk:] = -77
        cache.k_scale[b, :, blk:] = float("nan")
        cache.v_scale[b, :, blk:] = float("inf")
    return cache, want


def check_attn(torch, ops, rng, cache, want, H, past, n, bf16=False, math="f32", count=None, first=None, size=1.5, tensor=True,
               max_past=None):
    B, Hkv, _, d = want.ints[0].shape
    kind = torch.bfloat16 if bf16 else torch.float32
    q = up(torch, normal(rng, B, n, H, d) * np.float32(size), kind)
    out = torch.full((B, n, H, d), 7.0, dtype=kind, device="cuda:0")
    ops.set_math(math)
    try:
        got = cache.attn(q, i32(torch, past) if tensor else int(past[0]), count=None if count is None else i32(torch, count),
                         first=None if first is None else i32(torch, first), max_past=max_past, out=out)
    finally:
        ops.set_math("f32")
    assert got is out
    vals = want.values(np.float64)
    exact, tol = O.attention(q.float().cpu().numpy(), vals[0], vals[1], past, count, first,
                             0 if bf16 else {"f32": 2, "tf32": 1}[math], 2.0 ** -8 if bf16 else 2.0 ** -24)
    got = out.float().cpu().numpy().astype(np.float64)
    left = np.isnan(exact)
    assert (got[left] == 7.0).all()
    over = (np.abs(got - exact) - tol)[~left].max(initial=-1.0)
    assert over <= 0, f"off by {np.abs(got - exact)[~left].max()}, {over} more than the bound"
    ops.sync()
    return q, out


ATTN = [  # batch, heads, heads_kv, d, n, past
    (1, 1, 1, 64, 1, [0]),
    (1, 12, 2, 128, 1, [700]),
    (3, 14, 2, 64, 1, [31, 32, 33]),
    (2, 8, 8, 128, 1, [95, 1]),
    (2, 16, 1, 64, 1, [200, 3]),
    (2, 9, 1, 128, 1, [64, 127]),
    (2, 14, 2, 64, 3, [61, 0]),
    (1, 12, 2, 128, 5, [250]),
    (2, 4, 2, 64, 40, [0, 30]),
    (1, 14, 2, 64, 130, [77]),
    (1, 6, 1, 128, 67, [90]),
    (1, 3, 3, 128, 256, [0]),
    (1, 40, 1, 64, 2, [31]),
    (2, 16, 2, 128, 5, [300, 2]),
    (1, 16, 2, 64, 6, [1500]),
    (1, 13, 1, 128, 20, [40]),
]


@pytest.mark.parametrize("B,H,Hkv,d,n,past", ATTN)
@pytest.mark.parametrize("mode", ["f32", "tf32", "bf16"])
def test_attention(env, B, H, Hkv, d, n, past, mode):
    torch, ops = env
    rng = np.random.default_rng(B * H + n)
    length = [p + n for p in past]
    cache, want = fill(torch, ops, rng, B, Hkv, d, (max(length) + 63) // 32 * 32, length)
    check_attn(torch, ops, rng, cache, want, H, past, n, bf16=mode == "bf16", math="tf32" if mode == "tf32" else "f32",
               tensor=len(set(past)) > 1)


@pytest.mark.parametrize("d,n", [(64, 1), (128, 4), (64, 50), (128, 140)])
def test_attention_padded_rows_and_empty_masks(env, d, n):
    """count leaves rows as they are, first hides keys; where it hides all of them a row is zero."""
    torch, ops = env
    rng = np.random.default_rng(d + n)
    B, H, Hkv = 6, 4, 2
    past = np.array([40, 0, 100, 64, 5, 33])
    count = np.array([n, max(1, n - 1), 0, n, max(1, n // 2), n])
    first = np.array([0, 0, 50, 64 + n // 2, 5 + n, 1000])
    cache, want = fill(torch, ops, rng, B, Hkv, d, 288, past + count)
    check_attn(torch, ops, rng, cache, want, H, past, n, count=count, first=first)
    check_attn(torch, ops, rng, cache, want, H, past, n, bf16=True, count=count, first=first, max_past=100)


@pytest.mark.parametrize("d", [64, 128])
def test_attention_long_context_splits(env, d):
    torch, ops = env
    rng = np.random.default_rng(d)
    cache, want = fill(torch, ops, rng, 2, 1, d, 9024, [9001, 4321])
    check_attn(torch, ops, rng, cache, want, 6, [9000, 4320], 1)
    check_attn(torch, ops, rng, cache, want, 6, [8995, 4315], 6, first=[17, 4000])
    check_attn(torch, ops, rng, cache, want, 6, [8937, 4257], 64)


@pytest.mark.parametrize("B,n,lengths", [(1, 1, (500, 770, 1000, 1600, 2050)), (6, 1, (900, 1500, 3000)), (8, 1, (1600, 3100)),
                                         (12, 1, (1100, 1700)), (24, 1, (770, 1300)), (8, 2, (1000, 2200))])
def test_attention_however_the_keys_are_cut(env, B, n, lengths):
    """Batches and lengths on both sides of where the number and the size of the cuts change."""
    torch, ops = env
    rng = np.random.default_rng(B + n)
    n_ctx = (max(lengths) + 31) // 32 * 32
    cache, want = fill(torch, ops, rng, B, 2, 64, n_ctx, [max(lengths)] * B)
    for past in lengths:
        ends = [max(past - n - 37 * b, 0) for b in range(B)]
        check_attn(torch, ops, rng, cache, want, 12, ends, n, max_past=past - n)
    check_attn(torch, ops, rng, cache, want, 12, ends, n, bf16=True, max_past=past - n)


def test_attention_workspace_serves_shorter_caches(env):
    torch, ops = env
    for B in (1, 2, 3, 5, 7, 8, 9, 12, 16, 24, 64):
        cache = ops.Kv8Cache.empty(B, 2, 64, 32768 if B < 9 else 4096)
        for n in (1, 2, 7, 200):
            sizes = [cache.attn_workspace_bytes(n, 12, n_past=p) for p in range(0, cache.n_ctx - n, 151)]
            assert sizes == sorted(sizes)
            assert sizes[-1] <= cache.attn_workspace_bytes(n, 12)


@pytest.mark.parametrize("B,H,d,n,past,pad", [(40, 2, 64, 150, 2000, 0), (40, 2, 128, 131, 1700, 4), (1, 2, 128, 130, 4000, 0)])
def test_attention_sums_do_not_drift_with_the_keys(env, B, H, d, n, past, pad):
    """Two pieces keep the accuracy of f32 sums over thousands of keys: within 2.5e-6 of the exact output in
    norm. Rows behind the 128th of a tile, unaligned rows (pad), whole and partial tiles."""
    torch, ops = env
    rng = np.random.default_rng(d)
    n_ctx = (past + n + 31) // 32 * 32
    k, v = (up(torch, normal(rng, B, past + n, 1, d)) for _ in range(2))
    cache = ops.Kv8Cache.empty(B, 1, d, n_ctx)
    cache.append(k, v, 0)
    q = up(torch, normal(rng, B, n, H, d))
    rows = torch.full((B, n, H * d + pad // 2), 7.0, device="cuda:0")
    out = rows[..., :H * d].unflatten(-1, (H, d))
    cache.attn(q, past, out=out)
    kk, vv = (x[:, :, 0].double() for x in cache.read(past + n, 0))
    s = torch.einsum("bnhd,bkd->bnhk", q.double(), kk) / d ** 0.5
    hidden = torch.arange(past + n, device="cuda:0")[None] > past + torch.arange(n, device="cuda:0")[:, None]
    exact = torch.einsum("bnhk,bkd->bnhd", s.masked_fill(hidden[:, None], float("-inf")).softmax(-1), vv)
    # runs of 768 keys: 96 truncated sums (half a step of 2^-23 each, 48 of them behind an average key) and
    # as many in the scores' and the last roundings' share: 48 * 0.36 * 2^-23 = 2.1e-6 at the most
    assert (out.double() - exact).norm() < 2.5e-6 * exact.norm()
    assert (rows[..., H * d:] == 7.0).all()
    ops.sync()


@pytest.mark.parametrize("d,n", [(64, 17), (128, 17), (64, 43), (128, 43)])
@pytest.mark.parametrize("mode", ["f32", "tf32", "bf16"])
def test_attention_chunks_of_large_batches(env, d, n, mode):
    """Batches large enough that 256 rows and 128 keys at a time are the faster way: ragged, padded, empty rows."""
    torch, ops = env
    rng = np.random.default_rng(d + n)
    B, H = 96 if n < 40 else 48, 12
    past = rng.integers(0, 300, B)
    past[:3] = [0, 299, 128]
    count = rng.integers(1, n + 1, B)
    count[:4] = [n, n, 0, 1]
    first = rng.integers(0, 40, B)
    first[:5] = [0, 290, 0, 500, past[4] + n // 2]
    cache, want = fill(torch, ops, rng, B, 2, d, 384, past + count)
    check_attn(torch, ops, rng, cache, want, H, past, n, bf16=mode == "bf16", math="tf32" if mode == "tf32" else "f32",
               count=count, first=first, max_past=299)


@pytest.mark.parametrize("d", [64, 128])
def test_attention_nan_blocks_in_large_batches(env, d):
    torch, ops = env
    rng = np.random.default_rng(d)
    B, n, H = 96, 17, 6
    k, v = (normal(rng, B, 160, 1, d) for _ in range(2))
    k[5, 40, 0, 3] = np.inf
    v[7, 100, 0, 1] = np.nan
    cache, want = ops.Kv8Cache.empty(B, 1, d, 192), O.Cache(B, 1, d, 192)
    cache.append(up(torch, k), up(torch, v), 0)
    q = normal(rng, B, n, H, d)
    first = np.zeros(B, np.int64)
    first[7] = 128  # behind the block of NaN
    out = cache.attn(up(torch, q), 160 - n, first=i32(torch, first)).cpu().numpy()
    assert np.isnan(out[5]).all()
    others = np.arange(B) != 5
    assert np.isfinite(out[others]).all()
    k[5, 40, 0, 3] = 0
    v[7, 100, 0, 1] = 0
    want.append(k, v, [0] * B)
    vals = want.values(np.float64)
    exact, tol = O.attention(q, vals[0], vals[1], [160 - n] * B, None, first, 2, 2.0 ** -24)
    assert (np.abs(out - exact) <= tol)[others].all()
    ops.sync()


def test_attention_sharp_and_flat_scores(env):
    """One key that takes all the weight, equal keys, zero queries, queries of very different sizes."""
    torch, ops = env
    rng = np.random.default_rng(3)
    cache, want = fill(torch, ops, rng, 2, 2, 64, 512, [500, 500], spread=1.5)
    for size in (0.0, 1e-30, 1e-4, 30.0, 200.0):
        check_attn(torch, ops, rng, cache, want, 4, [499, 499], 1, size=size, tensor=False)
        check_attn(torch, ops, rng, cache, want, 4, [460, 460], 40, size=size, tensor=False)


@pytest.mark.parametrize("n", [1, 3, 70])
def test_attention_scores_of_any_size_stay_finite(env, n):
    """Scores up to the largest that f32 holds: the key they belong to takes all the weight, nothing overflows."""
    torch, ops = env
    rng = np.random.default_rng(n)
    k, v = normal(rng, 1, 160, 1, 64), normal(rng, 1, 160, 1, 64)
    k[0, 37] = 9 * np.sign(k[0, 37])
    cache = ops.Kv8Cache.empty(1, 1, 64, 160)
    cache.append(up(torch, k), up(torch, v), 0)
    ck, cv = cache.read(160, 0)
    for size in (1e3, 1e8, 1e20, 1e33):
        q = up(torch, np.broadcast_to(np.sign(k[0, 37]), (1, n, 2, 64)) * np.float32(size))
        out = cache.attn(q, 160 - n)
        assert torch.equal(out, cv[0, 37].expand_as(out)) or torch.allclose(out, cv[0, 37].expand_as(out), rtol=1e-5, atol=0)
    # values of very different sizes in the blocks that a query weighs alike
    for scale in (1e-30, 1e30):
        v2 = v.copy()
        v2[0, 64:] *= np.float32(scale)
        cache = ops.Kv8Cache.empty(1, 1, 64, 160)
        cache.append(up(torch, k), up(torch, v2), 0)
        _, cv = cache.read(160, 0)
        q = torch.zeros(1, n, 2, 64, device="cuda:0")
        out = cache.attn(q, 160 - n)
        for i in range(n):
            want = cv[0, :160 - n + i + 1].double().mean(0).float()
            top = cv[0, :160 - n + i + 1].abs().max()
            assert ((out[0, i] - want).abs() <= 1e-6 * top).all()
    ops.sync()


def test_attention_out_of_range_sequence_is_skipped(env):
    torch, ops = env
    from zwhisper_b200._lib import ZwgError
    rng = np.random.default_rng(11)
    cache, want = fill(torch, ops, rng, 4, 1, 64, 320, [300] * 4)
    for n in (1, 70):
        q = up(torch, normal(rng, 4, n, 2, 64))
        good = cache.attn(q, i32(torch, [200] * 4), max_past=200)
        out = torch.full_like(q, 5.0)
        ops.sync()
        cache.attn(q, i32(torch, [200, 201, -1, 200]), first=i32(torch, [0, 0, 0, -1]), max_past=200, out=out)
        with pytest.raises(ZwgError):
            ops.sync()
        assert torch.equal(out[0], good[0]) and (out[1:] == 5).all()
    ops.sync()


def test_attention_on_two_streams_at_once(env):
    torch, ops = env
    rng = np.random.default_rng(12)
    cache, _ = fill(torch, ops, rng, 2, 2, 64, 4096, [4000, 4000])
    qs = [up(torch, normal(rng, 2, n, 8, 64)) for n in (1, 1, 40, 40)]
    want = [cache.attn(q, 4000 - q.shape[1]) for q in qs]
    streams = [torch.cuda.Stream() for _ in qs]
    torch.cuda.synchronize()
    got = [[] for _ in qs]
    for _ in range(10):
        for i, (q, s) in enumerate(zip(qs, streams)):
            with torch.cuda.stream(s):
                got[i].append(cache.attn(q, 4000 - q.shape[1]))
    torch.cuda.synchronize()
    for i, w in enumerate(want):
        assert all(torch.equal(w, g) for g in got[i])


def test_attention_nan_blocks_reach_only_the_queries_that_see_them(env):
    torch, ops = env
    rng = np.random.default_rng(4)
    for side in (0, 1):
        k, v = (normal(rng, 1, 128, 1, 64) for _ in range(2))
        (k, v)[side][0, 100] = np.nan  # block 3: tokens 96 .. 127
        cache = ops.Kv8Cache.empty(1, 1, 64, 128)
        cache.append(up(torch, k), up(torch, v), 0)
        q = up(torch, normal(rng, 1, 60, 2, 64))
        out = cache.attn(q, 60)  # positions 60 .. 119
        assert torch.isfinite(out[0, :36]).all() and torch.isnan(out[0, 36:]).all()
        out = cache.attn(q, 60, first=i32(torch, [96]))
        assert (out[0, :36] == 0).all() and torch.isnan(out[0, 36:]).all()
    # a query that is not finite spoils its own row alone
    cache, want = fill(torch, ops, rng, 1, 1, 64, 64, [50])
    for bad in (float("nan"), float("inf")):
        q = up(torch, normal(rng, 1, 4, 2, 64))
        good = cache.attn(q, 46)
        q[0, 1, 1, 3] = bad
        out = cache.attn(q, 46)
        out[0, 1, 1], good[0, 1, 1] = 0, 0
        assert torch.equal(out, good)
    ops.sync()


def test_attention_strides_streams_and_graphs(env):
    torch, ops = env
    rng = np.random.default_rng(8)
    B, H, Hkv, d, n = 3, 6, 2, 64, 2
    cache, want = fill(torch, ops, rng, B, Hkv, d, 1056, [1002] * B)
    packed = up(torch, normal(rng, n, B, H + 5, d))
    q = packed[:, :, :H].transpose(0, 1)
    dense = cache.attn(q.contiguous(), 1000)
    wide = torch.full((B, n, H + 1, d), 3.0, device="cuda:0")
    cache.attn(q, 1000, out=wide[:, :, :H])
    assert torch.equal(wide[:, :, :H], dense) and (wide[:, :, H] == 3).all()
    odd = torch.zeros(q.numel() + 1, device="cuda:0")[1:].view(B, n, H, d)
    odd.copy_(q)
    assert torch.equal(cache.attn(odd, 1000), dense)
    # another stream, and a graph whose positions live on the device
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = cache.attn(q, 1000)
    s.synchronize()
    assert torch.equal(other, dense)
    past, ws = i32(torch, [1000] * B), torch.empty(cache.attn_workspace_bytes(n, H), dtype=torch.uint8, device="cuda:0")
    k, v = (up(torch, normal(rng, B, n, Hkv, d)) for _ in range(2))
    out, q0 = torch.zeros(B, n, H, d, device="cuda:0"), q.contiguous()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.append(k, v, past)
        cache.attn(q0, past, out=out, workspace=ws)
        past += n
    graph.replay()
    graph.replay()
    torch.cuda.synchronize()
    assert past.tolist() == [1004] * B
    cache.append(k, v, 1000)
    cache.append(k, v, 1002)
    # the same call outside the graph (with n_past a number the keys may be cut at other places)
    assert torch.equal(cache.attn(q0, i32(torch, [1002] * B)), out)
    ops.sync()


@pytest.mark.parametrize("B,n,past,kv", [(40, 150, 2000, 1), (8, 96, 2000, 2), (1, 64, 4000, 1), (2, 1, 9000, 1)])
def test_attention_chunks_captured_and_on_another_stream(env, B, n, past, kv):
    """Calls that drain sums, cut keys into a workspace or join many partials: a replayed graph, another stream and
    a second replay give what the plain call gave, bit for bit; the graph follows positions on the device."""
    torch, ops = env
    d, H = 64, 6 * kv
    n_ctx = (past + n + 63) // 32 * 32
    g = torch.Generator(device="cuda:0").manual_seed(B)
    rows = lambda heads, tokens: torch.randn(B, tokens, heads, d, device="cuda:0", generator=g)
    cache = ops.Kv8Cache.empty(B, kv, d, n_ctx)
    cache.append(rows(kv, past + n), rows(kv, past + n), 0)
    q = rows(H, n)
    at = torch.full((B,), past, dtype=torch.int32, device="cuda:0")
    want = cache.attn(q, at, max_past=past)
    short = cache.attn(q, at - 77, max_past=past)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = cache.attn(q, at, max_past=past)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, want)
    out = torch.zeros_like(q)
    ws = torch.empty(max(1, cache.attn_workspace_bytes(n, H, n_past=past)), dtype=torch.uint8, device="cuda:0")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.attn(q, at, max_past=past, out=out, workspace=ws)
    for shift, expect in ((0, want), (77, short), (0, want)):
        at.fill_(past - shift)
        out.fill_(5.0)
        graph.replay()
        assert torch.equal(out, expect)
    ops.sync()


def test_attention_is_the_same_every_time(env):
    torch, ops = env
    rng = np.random.default_rng(9)
    cache, _ = fill(torch, ops, rng, 2, 2, 128, 4096, [4000, 3000])
    q = up(torch, normal(rng, 2, 1, 12, 128))
    past = i32(torch, [3999, 2999])
    outs = [cache.attn(q, past) for _ in range(5)]
    assert all(torch.equal(outs[0], o) for o in outs[1:])


def test_python_refusals(env):
    torch, ops = env
    from zwhisper_b200._lib import ZwgError
    cache = ops.Kv8Cache.empty(2, 2, 64, 64)
    q = torch.zeros(2, 1, 4, 64, device="cuda:0")
    x = torch.zeros(2, 1, 2, 64, device="cuda:0")
    for call in (lambda: cache.attn(q.double(), 0), lambda: cache.attn(q.cpu(), 0), lambda: cache.attn(q[:1], 0),
                 lambda: cache.attn(q[..., :32], 0), lambda: cache.attn(q, -1), lambda: cache.attn(q, 0, out=q.bfloat16()),
                 lambda: cache.attn(q, i32(torch, [0])), lambda: cache.attn(q, 0, count=i32(torch, [1])),
                 lambda: cache.attn(q, 0, first=torch.zeros(2, device="cuda:0")), lambda: cache.append(x, x.bfloat16(), 0),
                 lambda: cache.append(x[:, :, :1], x, 0), lambda: cache.append(x.transpose(2, 3), x, 0),
                 lambda: cache.read(1, 0, k=x[:1]), lambda: ops.Kv8Cache.empty(1, 1, 96, 64),
                 lambda: ops.Kv8Cache.empty(1, 1, 64, 40), lambda: ops.rope(q, x[0, 0], x[0, 0].half()),
                 lambda: ops.Kv8Cache(cache.k, cache.v_scale, cache.v, cache.v_scale, cache.k_open, cache.v_open[:1],
                                      cache.open_block)):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: cache.attn(q, 64), lambda: cache.attn(torch.zeros(2, 1, 3, 64, device="cuda:0"), 0),
                 lambda: cache.append(x, x, 64), lambda: cache.read(65, 0)):
        with pytest.raises(ZwgError):
            call()
    big = ops.Kv8Cache.empty(1, 1, 64, 32768)
    q1 = torch.zeros(1, 1, 4, 64, device="cuda:0")
    with pytest.raises(ZwgError):
        big.attn(q1, 32000, workspace=torch.empty(16, dtype=torch.uint8, device="cuda:0"))
    ops.sync()


def test_workspace_elsewhere_is_refused(env):
    torch, ops = env
    cache = ops.Kv8Cache.empty(1, 1, 64, 32768)
    q = torch.zeros(1, 1, 4, 64, device="cuda:0")
    size = cache.attn_workspace_bytes(1, 4, n_past=32000)
    assert size > 0
    for ws in (torch.empty(size, dtype=torch.uint8), torch.empty(2 * size, dtype=torch.uint8, device="cuda:0")[::2]):
        with pytest.raises(ValueError):
            cache.attn(q, 32000, workspace=ws)
    ops.sync()


# ---- the states that keep such caches ----------------------------------------------------

@pytest.mark.parametrize("d,B,math", [(64, 2, "f32"), (128, 1, "f32"), (64, 2, "tf32")])
def test_llm_state_in_8_bits(env, d, B, math):
    """append_rope + attn of a state: the prompt in chunks, then steps, against the oracle's cache."""
    torch, ops = env
    rng = np.random.default_rng(d + B)
    H, Hkv, n_ctx = 14, 2, 256
    st = ops.LlmState(2, B, H, Hkv, d, n_ctx, rope_base=1e6, kv8=True, n_chunk=64)
    cos, sin = (up(torch, a) for a in ops.scaled_rope_tables(n_ctx, d, 1e6, "ntk", 4.0))
    st.set_rope(cos, sin)
    want = O.Cache(B, Hkv, d, n_ctx)
    past = 0
    for n in (64, 64, 13, 1, 1):
        q, k, v = (normal(rng, B, n, h, d) for h in (H, Hkv, Hkv))
        tq = up(torch, q)
        st.append_rope(1, tq, up(torch, k), up(torch, v), past)
        ops.set_math(math)
        try:
            out = st.attn(1, tq, past)
        finally:
            ops.set_math("f32")
        pos = past + np.arange(n)
        tables = cos.cpu().numpy(), sin.cpu().numpy()
        qr, kr = (np.stack([O.rope(x, *tables, pos, False) for x in y]) for y in (q, k))
        np.testing.assert_array_equal(tq.cpu().numpy().reshape(qr.shape), qr)
        want.append(kr, v, [past] * B)
        same(torch, st.kv8_cache(1), want)
        vals = want.values(np.float64)
        exact, tol = O.attention(qr, vals[0], vals[1], [past] * B, None, None, 2 if math == "f32" else 1, 2.0 ** -24)
        assert (np.abs(out.cpu().numpy().reshape(exact.shape) - exact) <= tol).all()
        past += n
    assert (st.kv8_cache(0).open_block == -1).all()
    st.close()


@pytest.mark.parametrize("B", [1, 3])
def test_llm_forward_in_8_bits(env, B):
    """A whole model over 8-bit caches, prompt and greedy steps with the logit rules: the q/k/v product's
    staging gives the cache that append gives, logits are near those over f32 caches, and the
    tokens follow the rules applied to the logits."""
    torch, ops = env
    m = qwen.make_model(5, n_layer=2, n_vocab=96, n_head=4, n_head_kv=2, d=64, n_ff=128, n_ctx=96)
    W = ops.LlmWeightsQ8(m["layers"], m["embd"], None, m["output_norm"], m["cfg"]["eps"])
    st8 = ops.LlmState(2, B, 4, 2, 64, 96, rope_base=m["cfg"]["rope_base"], kv8=True, n_chunk=20)
    st32 = ops.LlmState(2, B, 4, 2, 64, 96, rope_base=m["cfg"]["rope_base"])
    rng = np.random.default_rng(B)
    toks = rng.integers(0, 96, (B, 45)).astype(np.int32)
    allow = i32(torch, [-1, -1, 0x7FFFFFFF])
    history, past = toks.copy(), 0
    for n in (20, 17, 1, 3, 1, 1, 1, 1):
        t = up(torch, history[:, past:past + n])
        _, a = st8.forward_q8(W, t, past)
        _, b = st32.forward_q8(W, t, past)
        past += n
        kt, v32 = st32.cache_views(0)
        # layer 0's keys and values do not go through a cache: the 8-bit ones are their quantised rows
        want = O.Cache(B, 2, 64, 96)
        want.append(kt[..., :past].permute(0, 3, 1, 2).cpu().numpy(), v32.view(B, 96, 2, 64)[:, :past].cpu().numpy(), [0] * B)
        got, cached = st8.kv8_cache(0).read(past, 0), want.values()
        for x, side in zip(got, cached):
            np.testing.assert_array_equal(x.cpu().numpy(), side[:, :, :past].transpose(0, 2, 1, 3))
        # scores and values move by half a step of 127: a few parts in a hundred of the hidden state
        scale = b.abs().max()
        assert (a - b).abs().max() < 0.1 * scale
        raw = a.clone()
        ids = ops.llm_logits(a, recent=up(torch, history[:, :past]), window=16, repeat=1.1, presence=0.01, allow=allow)
        for r in range(B):
            y, i = O.logits(raw[r].cpu().numpy(), history[r, :past], 16, 1.1, 0.01, 0.0, [], [], allow.cpu().numpy())
            np.testing.assert_array_equal(a[r].cpu().numpy(), y)
            assert int(ids[r]) == i
        if past >= 41 and past < 45:
            history[:, past] = ids.cpu().numpy()
    st8.close()
    st32.close()
    ops.sync()


def test_llm_state_in_8_bits_refusals(env):
    torch, ops = env
    from zwhisper_b200._lib import ZwgError
    for bad in (dict(d=96), dict(n_ctx=100), dict(n_head_kv=3)):
        with pytest.raises(ZwgError):
            ops.LlmState(**{**dict(n_layer=1, n_batch=1, n_head=4, n_head_kv=2, d=64, n_ctx=64, kv8=True), **bad})
    st = ops.LlmState(1, 1, 4, 2, 64, 64, kv8=True, n_chunk=8)
    q = torch.zeros(1, 9, 256, device="cuda:0")
    k = torch.zeros(1, 9, 128, device="cuda:0")
    for call in (lambda: st.append_rope(0, q, k, k, 0), lambda: st.attn(0, q, 0), lambda: st.cache_ptrs(0),
                 lambda: st.kv8_cache(1), lambda: st.append_rope(0, q[:, :8], k[:, :8], k[:, :8], 60)):
        with pytest.raises(ZwgError):
            call()
    with pytest.raises(ValueError):
        st.set_rope(q, q)
    st.close()
    plain = ops.LlmState(1, 1, 4, 2, 64, 64)
    with pytest.raises(ZwgError):
        plain.kv8_cache(0)
    plain.close()

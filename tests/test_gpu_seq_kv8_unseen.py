"""Attention over the 8-bit cache where the tokens behind a query, which it does not see, have values
far larger than those it sees: they change nothing of its output. Against oracle/kv8.py with the
unseen values taken out, so that its bound goes by the values a query sees."""
import numpy as np
import pytest

from oracle import kv8 as O
from tests.conftest import has_gpu

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("B,H,n", [(1, 1, 40), (1, 6, 8), (96, 6, 40)])  # both kernels, shared tiles of rows
@pytest.mark.parametrize("mode", ["f32", "tf32", "bf16"])
def test_values_that_a_query_does_not_see(d, B, H, n, mode):
    if not has_gpu():
        pytest.fail("needs a CUDA device")
    import torch

    from zwhisper_b200 import ops
    rng = np.random.default_rng(d + n)
    past, step = 96 - 4 * n // 5, 96  # a query at position p < step sees no large value
    k, v = (rng.standard_normal((B, 192, 1, d), dtype=np.float32) for _ in range(2))
    v[:, step:] *= np.float32(2.0 ** 40)
    cache, held = ops.Kv8Cache.empty(B, 1, d, 192), O.Cache(1, 1, d, 192)
    cache.append(torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda(), 0)
    held.append(k[:1], v[:1], [0])
    kk, vv = held.values(np.float64)
    q = torch.from_numpy(rng.standard_normal((B, n, H, d), dtype=np.float32)).cuda()
    if mode == "bf16":
        q = q.bfloat16()
    ops.set_math("tf32" if mode == "tf32" else "f32")
    try:
        out = cache.attn(q, past).float().cpu().numpy()
    finally:
        ops.set_math("f32")
    pieces, half = {"f32": (2, 2.0 ** -24), "tf32": (1, 2.0 ** -24), "bf16": (0, 2.0 ** -8)}[mode]
    small = np.where(np.arange(192)[:, None] < step, vv, 0)
    checked = 0
    for i in range(n):
        large = past + i >= step
        exact, tol = O.attention(q[:1, i:i + 1].float().cpu().numpy(), kk, vv if large else small, [past + i], None, None, pieces, half)
        # more than 48 rows to a kv head: the smallest step of a probability's last piece is 2^-36 of the largest value
        tol = tol + (past + i + 1) * 2.0 ** -36 * np.abs(vv if large else small)[0, 0, :past + i + 1].max()
        assert (np.abs(out[0, i] - exact[0, 0]) <= tol[0, 0]).all(), (i, np.abs(out[0, i] - exact[0, 0]).max())
        checked += not large
    assert 0 < checked < n
    ops.sync()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("B,n", [(1, 3), (96, 40)])  # both kernels
@pytest.mark.parametrize("size_q,size_k", [(2e38, 3e-39), (4e37, 1e-38), (2e-38, 2e37), (1e-39, 3e38)])
def test_queries_at_the_ends_of_f32(d, B, n, size_q, size_k):
    """Queries whose largest element is near f32's largest or smallest numbers, and keys that make ordinary scores of them."""
    if not has_gpu():
        pytest.fail("needs a CUDA device")
    import torch

    from zwhisper_b200 import ops
    rng = np.random.default_rng(d + n)
    H, past = 6, 60
    clipped = lambda *s: np.clip(rng.standard_normal(s), -1.1, 1.1)  # noqa: E731
    k, v = (clipped(B, past + n, 1, d) * size_k).astype(np.float32), clipped(B, past + n, 1, d).astype(np.float32)
    q = (clipped(B, n, H, d) * size_q).astype(np.float32)
    cache, held = ops.Kv8Cache.empty(B, 1, d, 128), O.Cache(1, 1, d, 128)
    cache.append(torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda(), 0)
    held.append(k[:1], v[:1], [0])
    ops.set_math("f32")
    out = cache.attn(torch.from_numpy(q).cuda(), past).cpu().numpy()
    kk, vv = held.values(np.float64)
    exact, tol = O.attention(q[:1], kk, vv, [past], None, None, 2, 2.0 ** -24)
    # the factor of a row's scores, down to 2^-129, is rounded to a multiple of 2^-149: 2^-21 of a score of at most 8
    tol = tol + 2 * 2.0 ** -21 * 8 * np.abs(v).max()
    assert (np.abs(out[:1] - exact) <= tol).all(), np.abs(out[:1] - exact).max()
    ops.sync()

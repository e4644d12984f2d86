"""The rules on a step's logits (zwg_llm_logits) against oracle/kv8.py, bit for bit: the kernel
makes the same f32 operations."""
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


def words(rng, rows, V, share):
    bits = (rng.random((rows, (V + 31) // 32, 32)) < share).astype(np.uint64)
    return (bits << np.arange(32, dtype=np.uint64)).sum(-1).astype(np.uint32).view(np.int32)


CASES = [  # m, vocab, recent, window, biases, share of tokens allowed (None: no mask)
    (1, 1, 1, 1, 0, None), (1, 31, 5, 3, 2, 0.5), (3, 33, 40, 40, 7, 0.3), (2, 1000, 0, 0, 0, 0.01),
    (5, 8193, 200, 64, 300, None), (2, 65538, 3000, 2500, 1000, 0.7), (1, 151936, 300, 256, 32, 0.5),
    (64, 4099, 17, 100, 1, 0.999), (2, 262147, 10, 10, 4096, 0.2), (3, 500, 0, 0, 5, None), (2, 777, 9, 0, 0, None),
]


@pytest.mark.parametrize("m,V,n_recent,window,n_bias,share", CASES)
def test_rules(env, m, V, n_recent, window, n_bias, share):
    torch, ops = env
    rng = np.random.default_rng(V + m)
    x = (3 * rng.standard_normal((m, V))).astype(np.float32)
    recent = (rng.random((m, n_recent)) ** 4 * V).astype(np.int32)
    ids = (rng.random((m, n_bias)) ** 2 * V).astype(np.int32)
    bias = rng.standard_normal((m, n_bias)).astype(np.float32)
    allow = None if share is None else words(rng, m, V, share)
    t = lambda a: torch.from_numpy(a.copy()).to("cuda:0")  # noqa: E731
    y = t(x)
    kw = dict(bias_ids=t(ids), bias=t(bias)) if n_bias else {}
    out = ops.llm_logits(y, recent=t(recent) if n_recent else None, window=window, repeat=1.3, presence=0.4, frequency=0.15,
                         allow=None if allow is None else t(allow), **kw)
    for r in range(m):
        want, best = O.logits(x[r], recent[r], window, 1.3, 0.4, 0.15, ids[r], bias[r], None if allow is None else allow[r])
        np.testing.assert_array_equal(y[r].cpu().numpy(), want)
        assert int(out[r]) == best
    ops.sync()


def test_lists_of_rows_that_differ(env):
    """Lengths of the rows' histories on the device, padding, one bias list and mask for all rows,
    rows of a wider buffer, the choice written into a column."""
    torch, ops = env
    rng = np.random.default_rng(0)
    m, V = 4, 501
    wide = torch.from_numpy(rng.standard_normal((m, 512)).astype(np.float32)).to("cuda:0")
    x, before = wide[:, :V], wide.clone()
    recent = rng.integers(0, V, (m, 20)).astype(np.int32)
    recent[1, 3:9] = -1
    n = np.array([20, 15, 0, 1], np.int32)
    ids, bias = np.array([7, 7, 7, 500, 7], np.int32), np.array([1e8, 1.0, -1e8, 2.0, 0.5], np.float32)
    allow = words(rng, 1, V, 0.8)[0]
    t = lambda a: torch.from_numpy(a).to("cuda:0")  # noqa: E731
    tokens = torch.full((m, 3), -7, dtype=torch.int32, device="cuda:0")
    ops.llm_logits(x, recent=t(recent), n_recent=t(n), window=10, repeat=0.8, presence=-0.1, frequency=0.2, bias_ids=t(ids),
                   bias=t(bias), allow=t(allow), out=tokens[:, 1])
    for r in range(m):
        want, best = O.logits(before[r, :V].cpu().numpy(), recent[r, :n[r]], 10, 0.8, -0.1, 0.2, ids, bias, allow)
        np.testing.assert_array_equal(x[r].cpu().numpy(), want)
        assert tokens[r].tolist() == [-7, best, -7]
    assert torch.equal(wide[:, V:], before[:, V:])
    ops.sync()


def test_extreme_logits(env):
    torch, ops = env
    inf, nan = float("inf"), float("nan")
    rows = torch.tensor([[nan, 1.0, nan, 1.0], [-inf, -inf, nan, -inf], [inf, 2.0, inf, nan], [-inf, -3e38, -inf, -inf]],
                        device="cuda:0")
    assert ops.llm_logits(rows.clone()).tolist() == [1, -1, 0, 1]
    # a mask that leaves nothing, and one that leaves the last token
    x = torch.randn(2, 70, device="cuda:0")
    allow = torch.tensor([[0, 0, 0], [0, 0, 1 << 5]], dtype=torch.int32, device="cuda:0")
    assert ops.llm_logits(x, allow=allow).tolist() == [-1, 69]
    assert torch.isinf(x[0]).all()
    # ties: the first index, wherever the row is cut
    x = torch.zeros(3, 20000, device="cuda:0")
    x[1, 19999] = x[1, 2500] = x[1, 2499] = 1
    x[2] = -inf
    x[2, 12345:] = -5
    assert ops.llm_logits(x).tolist() == [0, 2499, 12345]
    ops.sync()


def test_ids_out_of_range_are_left_out(env):
    torch, ops = env
    from zwhisper_b200._lib import ZwgError
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda:0")  # noqa: E731
    x = torch.randn(1, 50, device="cuda:0")
    ops.sync()
    for kw in (dict(recent=i32([[50, 1]])), dict(bias_ids=i32([60, 1]), bias=torch.ones(2, device="cuda:0")),
               dict(bias_ids=i32([-1, 1]), bias=torch.ones(2, device="cuda:0")),
               dict(recent=i32([[1, 1]]), n_recent=i32([3])), dict(recent=i32([[2, 2]]), n_recent=i32([-1]))):
        y = x.clone()
        ops.llm_logits(y, repeat=2.0, **kw)
        with pytest.raises(ZwgError):
            ops.sync()
        differ = (y != x)[0].nonzero().flatten().tolist()
        assert differ == ([] if kw.get("n_recent") is not None and int(kw["n_recent"]) < 0 else [1])
    ops.sync()


def test_refusals(env):
    torch, ops = env
    from zwhisper_b200._lib import ZwgError
    x = torch.zeros(2, 50, device="cuda:0")
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda:0")  # noqa: E731
    for kw in (dict(recent=i32(3, 4)), dict(recent=i32(2, 4).long()), dict(recent=i32(2, 4), n_recent=5),
               dict(recent=i32(2, 4), n_recent=i32(3)), dict(bias_ids=i32(3)), dict(bias_ids=i32(3), bias=torch.zeros(2, device="cuda:0")),
               dict(allow=i32(1)), dict(allow=i32(2, 1)), dict(out=i32(3)), dict(recent=i32(2, 4).cpu())):
        with pytest.raises(ValueError):
            ops.llm_logits(x, **kw)
    with pytest.raises(ValueError):
        ops.llm_logits(x.t())
    for kw in (dict(repeat=0.0), dict(presence=float("inf")), dict(bias_ids=i32(5000), bias=torch.zeros(5000, device="cuda:0"))):
        with pytest.raises(ZwgError):
            ops.llm_logits(x, **kw)


def test_graph(env):
    torch, ops = env
    x0 = torch.randn(3, 5000, device="cuda:0")
    recent = torch.randint(0, 5000, (3, 30), dtype=torch.int32, device="cuda:0")
    x, out = x0.clone(), torch.zeros(3, dtype=torch.int32, device="cuda:0")
    want = ops.llm_logits(x0.clone(), recent=recent, repeat=1.2)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        x.copy_(x0)
        ops.llm_logits(x, recent=recent, repeat=1.2, out=out)
    graph.replay()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)

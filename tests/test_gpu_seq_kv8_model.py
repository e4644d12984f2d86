"""The model's own path over 8-bit caches, piece by piece: what the q/k/v product leaves in the caches by
way of its staging is, bit for bit, the quantised rows that it writes into f32 caches, and a whole
forward pass is the pass put together from the public calls (whose attention over such a cache is held
to the oracle elsewhere)."""
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


def model(ops, d):
    m = qwen.make_model(d, n_layer=2, n_vocab=96, n_head=4, n_head_kv=2, d=d, n_ff=128, n_ctx=128)
    return m, ops.LlmWeightsQ8(m["layers"], m["embd"], None, m["output_norm"], m["cfg"]["eps"])


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("B", [1, 3])
def test_staged_rows_become_the_cache(env, d, B):
    """Chunks that start and end inside a block, of lengths that are no multiple of four, one token, a cut back."""
    torch, ops = env
    m, W = model(ops, d)
    rng = np.random.default_rng(d + B)
    st8 = ops.LlmState(2, B, 4, 2, d, 128, rope_base=m["cfg"]["rope_base"], kv8=True, n_chunk=50)
    st32 = ops.LlmState(2, B, 4, 2, d, 128, rope_base=m["cfg"]["rope_base"])
    want = [O.Cache(B, 2, d, 128) for _ in range(2)]
    for past, n in ((0, 33), (33, 1), (34, 50), (84, 3), (87, 1), (40, 9), (49, 2)):
        x = torch.from_numpy(rng.standard_normal((B, n, 4 * d), dtype=np.float32)).cuda()
        for layer in range(2):
            q8, q32 = (st.qkv_q8(layer, x, W, past) for st in (st8, st32))
            assert torch.equal(q8, q32)
            kt, v = st32.cache_views(layer)
            k = kt[..., past:past + n].permute(0, 3, 1, 2).cpu().numpy()
            want[layer].append(k, v.view(B, 128, 2, d)[:, past:past + n].cpu().numpy(), [past] * B)
            got, c = st8.kv8_cache(layer), want[layer]
            np.testing.assert_array_equal(got.k.cpu().numpy().reshape(c.ints[0].shape), c.ints[0])
            np.testing.assert_array_equal(got.v.cpu().numpy().transpose(0, 1, 2, 4, 3).reshape(c.ints[1].shape), c.ints[1])
            np.testing.assert_array_equal(got.k_scale.cpu().numpy(), c.scale[0])
            np.testing.assert_array_equal(got.v_scale.cpu().numpy(), c.scale[1])
            np.testing.assert_array_equal(got.k_open.cpu().numpy(), c.open[0])
            np.testing.assert_array_equal(got.v_open.cpu().numpy(), c.open[1])
            np.testing.assert_array_equal(got.open_block.cpu().numpy(), c.tag)
    st8.close()
    st32.close()
    ops.sync()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("B", [1, 3])
def test_forward_is_its_pieces(env, d, B):
    torch, ops = env
    m, W = model(ops, d)
    rng = np.random.default_rng(d + B)
    make = lambda: ops.LlmState(2, B, 4, 2, d, 128, rope_base=m["cfg"]["rope_base"], kv8=True, n_chunk=50)  # noqa: E731
    whole, parts = make(), make()
    past = 0
    for n in (50, 1, 17, 1, 1):
        t = torch.from_numpy(rng.integers(0, 96, (B, n)).astype(np.int32)).cuda()
        hidden, logits = whole.forward_q8(W, t, past)
        x = ops.embed_q8(t, *W.embd).view(B * n, 4 * d)
        for i, L in enumerate(W.layers):
            q = parts.qkv_q8(i, ops.rms_norm(x, L["attn_norm"], W.eps), W, past)
            ops.linear_q8_add(parts.attn(i, q.view(B, n, 4 * d), past).view(B * n, 4 * d), *L["wo"], x)
            g = ops.linear_q8_silu_mul(ops.rms_norm(x, L["ffn_norm"], W.eps), L["w_gate"], L["w_up"])
            ops.linear_q8_add(g, *L["w_down"], x)
        assert torch.equal(hidden.view(B * n, 4 * d), x)
        last = x.view(B, n, 4 * d)[:, -1].contiguous()
        assert torch.equal(logits, ops.linear_q8(ops.rms_norm(last, W.output_norm, W.eps), *W.output))
        past += n
    whole.close()
    parts.close()
    ops.sync()


@pytest.mark.parametrize("d,B,n", [(64, 16, 1), (128, 16, 1), (64, 3, 50), (128, 8, 33)])
def test_forward_replayed(env, d, B, n):
    """A captured pass, whose kernels start before their predecessors end and share the state's staging and
    workspace, gives the eager pass's bits at every replay."""
    torch, ops = env
    m = qwen.make_model(d, n_layer=4, n_vocab=96, n_head=4, n_head_kv=2, d=d, n_ff=128, n_ctx=640)
    W = ops.LlmWeightsQ8(m["layers"], m["embd"], None, m["output_norm"], m["cfg"]["eps"])
    rng = np.random.default_rng(d)
    st = ops.LlmState(4, B, 4, 2, d, 640, rope_base=m["cfg"]["rope_base"], kv8=True, n_chunk=64)
    for past in range(0, 512, 64):
        st.forward_q8(W, torch.from_numpy(rng.integers(0, 96, (B, 64)).astype(np.int32)).cuda(), past)
    t = torch.from_numpy(rng.integers(0, 96, (B, n)).astype(np.int32)).cuda()
    x, logits = (a.clone() for a in st.forward_q8(W, t, 512))
    xo, lo, scratch = torch.empty_like(x), torch.empty_like(logits), st.scratch(n, W.n_ff)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        st.forward_q8(W, t, 512, x=xo, logits=lo, scratch=scratch)
    for _ in range(20):
        lo.fill_(float("nan"))
        graph.replay()
        assert torch.equal(xo, x) and torch.equal(lo, logits)
    del graph
    st.close()
    ops.sync()

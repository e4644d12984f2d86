"""Positions of a state's calls: a negative one, which reaches the C entry points as a huge one, is refused
like any other that has no room, also where position and length together wrap to a small number."""
import pytest

from oracle import qwen
from tests.conftest import has_gpu

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def env():
    if not has_gpu():
        pytest.fail("needs a CUDA device")
    import torch

    from zwhisper_b200 import ops
    return torch, ops


@pytest.mark.parametrize("kv8", [False, True])
def test_llm_state(env, kv8):
    torch, ops = env
    from zwhisper_b200._lib import ZwgError
    m = qwen.make_model(5, n_layer=2, n_vocab=96, n_head=4, n_head_kv=2, d=64, n_ff=128, n_ctx=96)
    W = ops.LlmWeightsQ8(m["layers"], m["embd"], None, m["output_norm"], m["cfg"]["eps"])
    st = ops.LlmState(2, 1, 4, 2, 64, 96, kv8=kv8)
    for n, past in ((1, -1), (2, -1), (2, -2), (3, -2), (1, 96), (97, 0), (2, 95)):
        x, k = torch.zeros(1, n, 256, device="cuda:0"), torch.zeros(1, n, 128, device="cuda:0")
        tokens = torch.zeros(1, n, dtype=torch.int32, device="cuda:0")
        for call in (lambda: st.append_rope(0, x, k, k, past), lambda: st.attn(0, x, past), lambda: st.qkv_q8(0, x, W, past),
                     lambda: st.layer_q8(0, W, x, past), lambda: st.forward_q8(W, tokens, past)):
            with pytest.raises(ZwgError, match="context full"):
                call()
    ops.sync()
    st.close()


def test_decoder_state(env):
    torch, ops = env
    from zwhisper_b200._lib import ZwgError
    st = ops.DecoderState(1, 1, 128, 2, 64, 100)
    for n, past in ((1, -1), (2, -1), (3, -2), (1, 64), (65, 0)):
        x = torch.zeros(1, n, 128, device="cuda:0")
        with pytest.raises(ZwgError, match="context full"):
            st.self_attn(0, x, x, x, past)
    ops.sync()
    st.close()


def test_rope_append(env):
    torch, ops = env
    from zwhisper_b200 import _lib
    ops.sync()
    x = torch.zeros(64 * 64, device="cuda:0").data_ptr()
    for n, past in ((1, -1), (2, -1), (2, -2), (33, 0), (1, 32)):
        rc = _lib.load().zwg_rope_kt_append(1, n, past, 1, 1, 64, 32, x, x, x, x, x, x, x, 64 * n, 64 * n, 64 * 32, None)
        assert rc == _lib.ZWG_ERROR and "context full" in _lib.last_error()
    ops.sync()


def test_sizes_whose_products_wrap_are_refused(env):
    torch, ops = env
    from zwhisper_b200._lib import ZwgError
    fine = dict(n_layer=1, n_batch=1, n_head=2, n_head_kv=1, d=64, n_ctx=64, kv8=True, n_chunk=8)
    ops.LlmState(**fine).close()
    for bad in (dict(n_batch=1 << 33, n_head=1 << 33, n_head_kv=1 << 33), dict(n_batch=1 << 63, n_head_kv=2), dict(n_layer=1 << 62),
                dict(n_layer=65535, n_batch=60000, n_ctx=1 << 25), dict(n_chunk=-1), dict(n_chunk=0)):
        with pytest.raises(ZwgError, match="bad sizes|too large"):
            ops.LlmState(**{**fine, **bad})
    ops.sync()

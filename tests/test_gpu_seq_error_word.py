"""The device error word: an entry out of range (which only leaves its sequence or token out) neither
hides a later timeout nor cuts the waits of later kernels short. The timeout is the library's own
bounded wait on a barrier that nothing completes (zwg_selftest_timeout); nothing faults."""
import pytest

from tests.conftest import has_gpu

pytestmark = pytest.mark.gpu


def test_a_timeout_behind_an_entry_out_of_range_is_reported():
    if not has_gpu():
        pytest.fail("needs a CUDA device")
    import torch

    from zwhisper_b200 import _lib, ops
    _lib.ensure_init(0)
    lib = _lib.load()
    ops.sync()
    x = torch.zeros(1, 40, device="cuda:0")
    ops.llm_logits(x, recent=torch.tensor([[40]], dtype=torch.int32, device="cuda:0"))  # no such token
    torch.cuda.synchronize()
    # the wait's early end, as for any error, would leave the word as it was: an error, not a timeout
    assert lib.zwg_selftest_timeout() == _lib.ZWG_TIMEOUT, _lib.last_error()
    assert lib.zwg_sync() == _lib.ZWG_OK
    # alone, the entry is reported as what it is
    ops.llm_logits(x, recent=torch.tensor([[40]], dtype=torch.int32, device="cuda:0"))
    torch.cuda.synchronize()
    assert lib.zwg_sync() == _lib.ZWG_ERROR
    assert lib.zwg_sync() == _lib.ZWG_OK

"""The bound of tests/paged_codes.py tells a key that is lost, doubled or taken for another, at every length that
tests/test_gpu_seq_paged_exact.py uses."""
import numpy as np
import pytest

from tests.paged_codes import bound


@pytest.mark.parametrize("number", [3, 40, 700, 2256, 9001, 131001])
@pytest.mark.parametrize("half_step", [2.0 ** -24, 2.0 ** -8])
@pytest.mark.parametrize("d", [64, 128])
def test_one_key_is_told(number, half_step, d):
    rng = np.random.default_rng(number + d)
    code = (rng.integers(0, 2, (number, d), dtype=np.int8) * 2 - 1).astype(np.int8)
    sums = code.sum(0, dtype=np.int64)
    tol = bound(sums.astype(float), number, half_step)
    right = sums / number
    rounded = right * (1 + rng.uniform(-1, 1, d) * half_step)
    assert (np.abs(rounded - right) <= tol).all()
    for key in rng.integers(0, number, 20):
        other = int(rng.integers(0, number))
        lost, twice = (sums - code[key]) / (number - 1), (sums + code[key]) / (number + 1)
        for wrong in (lost, twice) + (((sums - code[key] + code[other]) / number,) if (code[key] != code[other]).any() else ()):
            assert (np.abs(wrong * (1 + rng.uniform(-1, 1, d) * half_step) - right) > tol).any()

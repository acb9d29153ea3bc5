"""Temperatures so small that the factor of the scores, log2(e) / T, is no number are refused before anything is launched."""
import numpy as np
import pytest

from paligemma_multimodal_system_b200 import _lib, build

P = 0x1000  # an address that nothing reads: every call below is refused


@pytest.fixture(scope="module")
def library():
    build.build()
    return _lib.lib()


def _refused(library, temperature):
    return library.pg_token_logprobs(P, 10, P, P, P, P, P, P, 2, 10, 3, temperature, 0) == -1  # PG_ERR_ARG


def test_the_factor_that_is_used_has_to_be_finite(library):
    with np.errstate(over="ignore"):
        for t in (1e-45, 2.9e-39, 2.95e-39, 3.5e-39, 4.2e-39, 4.23e-39):
            assert not np.isfinite(np.float32(1.0) / np.float32(t) * np.float32(1.4426950408889634)) and _refused(library, t), t

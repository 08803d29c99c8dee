"""Sizes, addresses and arguments at which the embedding, list and AdamW operators stop, before anything reaches a
device."""
import numpy as np
import pytest

from recommend_amd import _ffi


def refused(name, *args, error=""):
    assert getattr(_ffi.load(), name)(*args) == _ffi.RK_ERR_ARG
    assert error in _ffi.last_error(), _ffi.last_error()


@pytest.mark.parametrize("D", [(1 << 31) - (1 << 24), (1 << 31) - 1])
def test_columns_that_pass_32_bits_are_refused(D):
    b = _ffi.ptr(np.zeros(64, np.float64))
    refused("rk_embedding_fwd", b, D, 4, D, 0, b, 8, 1, 1.0, b, None, error="2^31 columns")
    refused("rk_embedding_bwd", b, 0, b, 8, 1, 4, D, 1.0, -1, b, b, 1 << 40, None, error="2^31 columns")

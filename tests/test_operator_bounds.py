"""Sizes, addresses and arguments at which the embedding, list and AdamW operators stop, before anything reaches a
device."""
import numpy as np
import pytest
import torch

from recommend_amd import _ffi
from recommend_amd.loss import preference_loss


def refused(name, *args, error=""):
    assert getattr(_ffi.load(), name)(*args) == _ffi.RK_ERR_ARG
    assert error in _ffi.last_error(), _ffi.last_error()


@pytest.mark.parametrize("D", [(1 << 31) - (1 << 24), (1 << 31) - 1])
def test_columns_that_pass_32_bits_are_refused(D):
    b = _ffi.ptr(np.zeros(64, np.float64))
    refused("rk_embedding_fwd", b, D, 4, D, 0, b, 8, 1, 1.0, b, None, error="2^31 columns")
    refused("rk_embedding_bwd", b, 0, b, 8, 1, 4, D, 1.0, -1, b, b, 1 << 40, None, error="2^31 columns")


def test_reference_values_that_require_a_gradient_are_refused():
    """They would get none.  Detached, or where nothing is recorded, the call goes on to the next check."""
    scores, items, ref = torch.zeros(2, 3, 5), torch.zeros(2, 3, dtype=torch.int64), torch.zeros(2, requires_grad=True)
    with pytest.raises(ValueError, match="detach"):
        preference_loss(scores, items, ref)
    with pytest.raises(_ffi.RkError, match="HIP device"):
        preference_loss(scores, items, ref.detach())
    with torch.no_grad(), pytest.raises(_ffi.RkError, match="HIP device"):
        preference_loss(scores, items, ref)
    with torch.autograd.forward_ad.dual_level(), pytest.raises(NotImplementedError, match="ref_logps"):
        preference_loss(scores, items, torch.autograd.forward_ad.make_dual(torch.zeros(2), torch.ones(2)))


def test_list_calls_refuse_addresses_that_are_not_8_byte_aligned():
    buf, lib = np.zeros(4096, np.float64), _ffi.load()
    b, odd = _ffi.ptr(buf), buf.ctypes.data + 4
    need = lib.rk_list_logps_ws_bytes(4, 3, 5)
    geo = (b, 0, 4, 3, 5, 15, 5, b, 3, -100, 0)
    for stat, ws in ((odd, b), (b, odd)):
        refused("rk_list_logps_fwd", *geo, stat, b, b, ws, need, None, error="8-byte aligned")
        refused("rk_preference_fwd", *geo, b, 0.1, 0.0, 0, stat, b, b, b, b, ws, need, None, error="8-byte aligned")
    refused("rk_list_logps_bwd", *geo, odd, b, b, b, b, b, None, error="8-byte aligned")

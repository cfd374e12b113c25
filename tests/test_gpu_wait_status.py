"""What the status words say of a wait that gave up: its kind, and its thread block's number in a grid of two dimensions."""
import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_the_thread_block_of_a_grid_of_two_dimensions():
    import dsv3_b200
    from dsv3_b200 import _lib
    stream = torch.cuda.current_stream().cuda_stream
    _lib.check(_lib.lib.dsv3_selftest_bounded_wait(2_000_000, stream))
    detail = (ctypes.c_uint32 * 4)()
    assert _lib.lib.dsv3_check_device_status(stream, detail) == _lib.ERR_DEVICE_TIMEOUT
    assert list(detail) == [1, 9, 0, 5]                                     # block (1, 2) of 2 x 3
    message = _lib.lib.dsv3_last_error().decode()
    assert "cta=5" in message and "11-15 latent attention" in message
    dsv3_b200.check_device_status()

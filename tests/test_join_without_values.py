"""Joins of rows that have no values: nothing to do, and logarithms of them are refused rather than left unwritten."""
import pytest
import torch

from test_expanded_refusals import _lib, vp


def test_rows_without_values():
    lib, names = _lib()
    outs, lses = (vp * 2)(1024, 1024), (vp * 2)(512, 512)
    join = lambda rows, lse: lib.dsv3_attention_join(outs, lses, 2, rows, 0, 2048, lse, None)  # noqa: E731
    assert join(4, None) == join(0, None) == join(0, 4096) == names.OK
    assert join(4, 4096) == names.ERR_UNSUPPORTED


@pytest.mark.gpu
def test_rows_without_values_in_python():
    from dsv3_b200 import attention_join
    out, lse = torch.zeros(3, 0, dtype=torch.bfloat16, device="cuda"), torch.zeros(3, device="cuda")
    assert attention_join([out, out], [lse, lse]).shape == (3, 0)
    with pytest.raises(NotImplementedError):
        attention_join([out, out], [lse, lse], return_lse=True)
    joined, joined_lse = attention_join([out[:0]], [lse[:0]], return_lse=True)
    assert joined.shape == (0, 0) and joined_lse.shape == (0,)

"""What the 8-bit attention operators hand to the library, without a GPU: the
entry points are recorded instead of called, the tensors are the host's."""
import ctypes

import pytest
import torch

from qmoe_b200 import attention, capi, quantize_int8


class Ctx:
    device, handle = 0, None


@pytest.fixture
def calls(monkeypatch):
    got = []
    monkeypatch.setattr(attention, "_on", lambda ctx, name, t: None)
    monkeypatch.setattr(attention, "_use_stream", lambda ctx: None)
    monkeypatch.setattr(capi, "call", lambda name, *a: got.append((name, a)))
    return got


VIEWS = {
    "packed": lambda x: x[:64].reshape(2, 32),
    "apart": lambda x: x[:96].reshape(2, 48)[:, 5:37],
    "one row repeated": lambda x: x[:32].expand(4, 32),
    "overlapping rows": lambda x: x[:80].unfold(0, 32, 8),
    "rows one apart": lambda x: x[:35].unfold(0, 32, 1),
    "columns apart": lambda x: x[:128].reshape(2, 64)[:, ::2],
    "one column": lambda x: x[:20].reshape(10, 2)[:, 1:],
    "one column repeated": lambda x: x[:1].expand(7, 1),
    "one row": lambda x: x[3:35][None],
}


@pytest.mark.parametrize("view", list(VIEWS))
def test_quantize_hands_over_the_rows_of_a_view(monkeypatch, calls, view):
    """Row r of the call, at r * row_stride from its pointer, is row r of x."""
    whole = torch.arange(128, dtype=torch.float32)
    x = VIEWS[view](whole)
    rows, cols = x.shape

    def call(name, ctx, ptr, dtype, n, width, stride, codes, scales):
        assert (name, dtype, n, width) == ("qmoe_quantize_int8", capi.QMOE_DTYPE_F32, rows, cols)
        # where x is handed over itself, before any of it is read
        if whole.data_ptr() <= ptr < whole.data_ptr() + 4 * whole.numel():
            assert ptr == x.data_ptr() and (rows == 1 or stride == x.stride(0)) and (cols == 1 or x.stride(1) == 1)
        else:
            assert stride == cols
        assert rows == 1 or stride >= cols
        for r in range(rows):
            assert list((ctypes.c_float * cols).from_address(ptr + 4 * r * stride)) == x[r].tolist()
        calls.append(name)

    monkeypatch.setattr(capi, "call", call)
    codes, scales = quantize_int8(x, Ctx())
    assert len(calls) == 1 and codes.shape == x.shape and scales.shape == x.shape[:1]

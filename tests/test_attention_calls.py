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


def scratch_bytes(dtype, T, R, heads, kv_heads, dims, block, max_blocks, max_kv=0):
    cache = capi.KvCacheC(4096, 4096, 4096, 4096, max_blocks, block, kv_heads, *dims)
    n = ctypes.c_int64()
    assert capi.lib().qmoe_kv_attend_workspace(ctypes.byref(cache), dtype, T, R, heads, max_blocks, max_kv,
                                               ctypes.byref(n)) == capi.QMOE_OK
    return n.value


F32, BF16 = capi.QMOE_DTYPE_F32, capi.QMOE_DTYPE_BF16


@pytest.mark.parametrize("heads,kv_heads,dims", [(32, 8, (128, 128)), (64, 8, (128, 128)), (128, 1, (64, 64)), (16, 16, (192, 128)),
                                                 (8, 8, (64, 64)), (112, 16, (128, 128))])
@pytest.mark.parametrize("R", [1, 2, 7, 64, 300, 4096])
def test_attention_scratch_stays_small(heads, kv_heads, dims, R):
    """Long prompts over a wide table: what is cut into pieces has scratch, not every
    token of the batch.  Pieces are cut for at most 16 CTAs on each of 148 SMs, of up
    to 32 columns (heads by tokens) with 130 floats each: 39.4 MB; in f32 128 MiB for
    the requests of several tokens come on top."""
    few, many = 16 * 148 * 32 * 130 * 4, 128 << 20
    for T in (1, 2, R, R + 1, 3 * R, 700, 8192, 65536):
        for tokens in (64, 4096, 131072, 1 << 20):
            args = (T, R, heads, kv_heads, dims, 64, tokens // 64)
            assert scratch_bytes(BF16, *args) <= few, args
            assert scratch_bytes(F32, *args) <= few + many, args


def test_attention_scratch_of_few_rows():
    # nothing is cut: no scratch; two rows after 131072 tokens: pieces of both
    assert scratch_bytes(BF16, 5, 1, 32, 8, (128, 128), 64, 1) == 0
    n = scratch_bytes(BF16, 2, 2, 32, 8, (128, 128), 64, 2048)
    assert n > 0 and n % (2 * 32 * 130 * 4) == 0


class Library:
    """The one entry point of a library whose stream others may set as well."""

    def __init__(self):
        self.stream = None

    def qmoe_ctx_set_stream(self, handle, stream):
        self.stream = getattr(stream, "value", stream) or 0
        return capi.QMOE_OK


def context(monkeypatch):
    from qmoe_b200 import Context, layer
    lib = Library()
    monkeypatch.setattr(capi, "lib", lambda: lib)
    monkeypatch.setattr(attention, "_fns", {})
    ctx = Context.__new__(Context)
    ctx.handle, ctx.device = None, 0
    return lib, ctx, layer


def test_every_call_sets_its_own_stream(monkeypatch):
    """Whatever another thread or a C call left there, a call runs on the current stream."""
    lib, ctx, layer = context(monkeypatch)

    class Current:
        cuda_stream = 70

    monkeypatch.setattr(attention, "_raw_stream", lambda device: 70)
    monkeypatch.setattr(layer.torch.cuda, "is_available", lambda: True)
    monkeypatch.setattr(layer.torch.cuda, "current_stream", lambda device: Current)
    for use in (lambda: attention._use_stream(ctx), ctx.use_current_torch_stream, lambda: ctx.use_stream(70)):
        for other in (0, 90):
            use()
            assert lib.stream == 70
            capi.lib().qmoe_ctx_set_stream(None, other)
        use()
        assert lib.stream == 70


def test_two_threads_whose_sets_cross(monkeypatch):
    """One thread sets, another sets before the first is done: from the next call on
    each is on its own stream again."""
    import threading
    lib, ctx, _ = context(monkeypatch)
    crossed = []

    class Crossing(Library):
        def qmoe_ctx_set_stream(self, handle, stream):
            Library.qmoe_ctx_set_stream(self, handle, stream)
            if not crossed:
                crossed.append(True)
                t = threading.Thread(target=lambda: ctx.use_stream(2))
                t.start()
                t.join()
            return capi.QMOE_OK

    lib = Crossing()
    monkeypatch.setattr(capi, "lib", lambda: lib)
    monkeypatch.setattr(attention, "_fns", {})
    current = [1]
    monkeypatch.setattr(attention, "_raw_stream", lambda device: current[0])
    attention._use_stream(ctx)
    for s in (1, 2, 1, 1, 2, 2):
        current[0] = s
        attention._use_stream(ctx)
        assert lib.stream == s


def test_rows_too_long_for_the_quantiser_are_refused():
    """Columns are counted in 32 bits, in steps of a thread block."""
    ctx = ctypes.cast(ctypes.create_string_buffer(256), ctypes.c_void_p)
    for cols in ((1 << 30) + 1, (1 << 31) - 256, (1 << 31) - 1, 1 << 31):
        assert capi.lib().qmoe_quantize_int8(ctx, 64, F32, 1, cols, cols, 64, 64) == capi.QMOE_ERR_INVALID, cols

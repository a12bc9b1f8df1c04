"""What the 8-bit attention operators refuse, without a GPU: the C entry
points' checks come before any launch, and the Python ones before the C call."""
import ctypes

import pytest
import torch

from qmoe_b200 import capi, Int8Tensor, KVCache, quantize_int8, plan_pages
from qmoe_b200.attention import layer_norm


def rc(name, *args):
    return getattr(capi.lib(), name)(*args), capi.lib().qmoe_last_error().decode()


@pytest.fixture
def ctx():
    # the layout of a context is the library's own; any non-NULL pointer reaches the
    # checks, which read nothing of it before they refuse
    return ctypes.cast(ctypes.create_string_buffer(256), ctypes.c_void_p)


def cache(**kw):
    c = dict(k=4096, v=4096, k_range=4096, v_range=4096, num_blocks=4, block_size=16, kv_heads=2, k_dim=64, v_dim=64)
    c.update(kw)
    return ctypes.pointer(capi.KvCacheC(*c.values()))


BAD_CACHES = [(dict(block_size=8), capi.QMOE_ERR_INVALID), (dict(block_size=24), capi.QMOE_ERR_INVALID),
              (dict(block_size=272), capi.QMOE_ERR_INVALID), (dict(block_size=0), capi.QMOE_ERR_INVALID),
              (dict(num_blocks=-1), capi.QMOE_ERR_INVALID), (dict(num_blocks=1 << 27), capi.QMOE_ERR_INVALID),
              (dict(kv_heads=0), capi.QMOE_ERR_INVALID), (dict(k_dim=96), capi.QMOE_ERR_UNSUPPORTED),
              (dict(k_dim=128), capi.QMOE_ERR_UNSUPPORTED), (dict(v_dim=128), capi.QMOE_ERR_UNSUPPORTED),
              (dict(k=None), capi.QMOE_ERR_INVALID), (dict(v_range=None), capi.QMOE_ERR_INVALID),
              (dict(k=4104), capi.QMOE_ERR_INVALID)]


@pytest.mark.parametrize("change,code", BAD_CACHES, ids=lambda v: str(v))
def test_caches(ctx, change, code):
    n = ctypes.c_int64()
    got, msg = rc("qmoe_kv_attend_workspace", cache(**change), 0, 1, 1, 2, 4, 0, ctypes.byref(n))
    assert got == code and msg
    got, _ = rc("qmoe_kv_append", ctx, cache(**change), 4096, 4096, 0, 1, 128, 128, 4096)
    assert got == code
    got, _ = rc("qmoe_kv_attend", ctx, cache(**change), 4096, 0, 1, 128, 2, 4096, 4096, 1, 4096, 4, 0, 1.0, 4096, 128,
                None, 0)
    assert got == code


def test_append_arguments(ctx):
    ok = [ctx, cache(), 4096, 4096, 0, 2, 128, 128, 4096]
    for i, v in ((0, None), (1, None), (2, None), (3, None), (4, 2), (5, -1), (5, 1 << 31), (6, 127), (7, 64), (8, None)):
        a = list(ok)
        a[i] = v
        assert rc("qmoe_kv_append", *a)[0] == capi.QMOE_ERR_INVALID, (i, v)
    assert rc("qmoe_kv_append", *ok[:2], None, None, 0, 0, 0, 0, None)[0] == capi.QMOE_OK


def test_attend_arguments(ctx):
    ok = [ctx, cache(), 4096, 0, 3, 256, 4, 4096, 4096, 2, 4096, 4, 0, 1.0, 4096, 256, None, 0]
    for i, v in ((0, None), (1, None), (2, None), (3, 7), (4, -1), (4, 1 << 25), (5, 255), (6, 3), (6, 0), (7, None),
                 (8, None), (9, -1), (10, None), (11, -1), (11, 1 << 27), (13, float("nan")), (13, float("inf")),
                 (14, None), (15, 255)):
        a = list(ok)
        a[i] = v
        assert rc("qmoe_kv_attend", *a)[0] == capi.QMOE_ERR_INVALID, (i, v)


def test_plan_arguments(ctx):
    ok = [ctx, 64, 64, 2, 16, 64, 4, 8, 64, 4, 3, 64, 64, 64, 64, 64]
    for i, v in ((0, None), (1, None), (2, None), (3, -1), (4, 15), (4, 0), (5, None), (6, -1), (7, -1), (7, 1 << 27), (8, None),
                 (9, -1), (9, 1 << 27), (10, -1), (10, 1 << 31), (11, None), (12, None), (13, None), (14, None), (15, None)):
        a = list(ok)
        a[i] = v
        assert rc("qmoe_kv_plan", *a)[0] == capi.QMOE_ERR_INVALID, (i, v)


def test_int8_arguments(ctx):
    h = ctypes.c_void_p()
    ok = [ctx, 64, 64, 4, 4, 0, ctypes.byref(h)]
    for i, v, code in ((0, None, 1), (1, None, 1), (2, None, 1), (3, 0, 1), (4, -1, 1), (5, 9, 1),
                       (4, capi.QMOE_INT8_MAX_IN_FEATURES + 1, 3), (3, 1 << 31, 3)):
        a = list(ok)
        a[i] = v
        assert rc("qmoe_int8_create", *a)[0] == code, (i, v)
    assert rc("qmoe_int8_forward", None, 64, 0, 1, 4, None, 64, 128, 1 << 20)[0] == capi.QMOE_ERR_INVALID
    assert rc("qmoe_int8_workspace", None, 1, None)[0] == capi.QMOE_ERR_INVALID
    assert rc("qmoe_int8_destroy", None)[0] == capi.QMOE_OK
    for bad in ((None, 64, 0, 2, 4, 4, 64, 64), (ctx, 64, 5, 2, 4, 4, 64, 64), (ctx, 64, 0, -2, 4, 4, 64, 64),
                (ctx, 64, 0, 2, 0, 4, 64, 64), (ctx, 64, 0, 2, 4, 3, 64, 64), (ctx, None, 0, 2, 4, 4, 64, 64)):
        assert rc("qmoe_quantize_int8", *bad)[0] == capi.QMOE_ERR_INVALID, bad
    for bad in ((None, 64, 0, 2, 64, 64, 64, 1e-6, 64), (ctx, 64, 3, 2, 64, 64, 64, 1e-6, 64),
                (ctx, 64, 0, 2, 65, 64, 64, 1e-6, 64), (ctx, None, 0, 2, 64, 64, 64, 1e-6, 64),
                (ctx, 68, 0, 2, 64, 64, 64, 1e-6, 64)):
        assert rc("qmoe_layer_norm", *bad)[0] == capi.QMOE_ERR_INVALID, bad


def test_python_refuses_host_tensors():
    x = torch.zeros(2, 64)
    i = torch.zeros(2, dtype=torch.int32)

    class Ctx:                                    # a context that must not be reached
        device, handle = 0, None

    with pytest.raises(TypeError):
        quantize_int8(x, Ctx())
    with pytest.raises(TypeError):
        layer_norm(x, x[0], x[0], ctx=Ctx())
    with pytest.raises(TypeError):
        plan_pages(i, i, i.reshape(2, 1), i, 16, 2, 2, ctx=Ctx())
    with pytest.raises(TypeError):
        KVCache.from_tensors(x, x, x, x, Ctx())
    with pytest.raises(ValueError):
        KVCache(4, 20, 2, 64, ctx=Ctx())
    with pytest.raises(ValueError):
        Int8Tensor.from_bytes(torch.zeros(4, 4), (4, 4), torch.zeros(4), Ctx())
    with pytest.raises(ValueError):
        Int8Tensor.from_bytes(torch.zeros(4, 4, dtype=torch.int8), (4, 5), torch.zeros(4), Ctx())

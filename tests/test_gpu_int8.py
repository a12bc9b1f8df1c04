"""The 8-bit integer product and the row quantiser against 64-bit arithmetic."""
import numpy as np
import pytest
import torch

import attn_ref as ref

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def weights(n, k, seed):
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(-127, 128, (n, k), generator=g, dtype=torch.int8)
    scales = torch.rand(n, generator=g) * 0.01 + 1e-4
    return codes, scales


def rows(t, k, dt, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(t, k, generator=g) * torch.exp(torch.randn(t, 1, generator=g))
    return x.to(dt)


def check_product(y, want, dt, k):
    # the sum is exact; its conversion, two products, the scale's division and the
    # residual add round in f32 (5 half steps of 2^-24), the result to dt
    half = torch.finfo(dt).eps / 2
    tol = (5 * 2.0 ** -24 + half) * want.abs() + 2.0 ** -24 * want.abs().max()
    assert (y.cpu().double() - want).abs().le(tol * 1.01).all(), (y.cpu().double() - want).abs().max()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("t,k,n", [(1, 2048, 2048), (1, 1, 1), (3, 17, 5), (16, 128, 128), (17, 129, 127), (33, 1411, 1001),
                                   (64, 256, 640), (129, 1000, 300), (257, 384, 129), (520, 7168, 256), (5, 16384, 512)])
def test_product(dtype, t, k, n):
    from qmoe_b200 import Int8Tensor
    dt = DT[dtype]
    codes, scales = weights(n, k, 7 * t + k)
    x = rows(t, k, dt, t + n)
    w = Int8Tensor.from_bytes(codes.cuda(), (n, k), scales.cuda())
    y = w.forward(x.cuda())
    assert y.shape == (t, n) and y.dtype == dt
    check_product(y, ref.product(x, codes, scales), dt, k)
    res = rows(t, n, dt, 5)
    y = w.forward(x.cuda(), residual=res.cuda())
    want = ref.product(x, codes, scales, res)
    half = torch.finfo(dt).eps / 2
    big = ref.product(x, codes, scales).abs() + res.double().abs()
    assert (y.cpu().double() - want).abs().le(big * 6 * 2.0 ** -24 + want.abs() * half * 1.01).all()


def test_product_in_place_views_and_host_weights():
    from qmoe_b200 import Int8Tensor
    codes, scales = weights(256, 192, 1)
    w = Int8Tensor.from_bytes(codes.numpy(), (256, 192), scales.numpy())
    big = rows(40, 512, torch.bfloat16, 2).cuda()
    view = big[:, 100:292]                       # rows 512 apart, start not 16-byte aligned
    want = ref.product(view.cpu(), codes, scales)
    check_product(w.forward(view), want, torch.bfloat16, 192)
    y3 = w.forward(view.unflatten(0, (4, 10)))
    assert y3.shape == (4, 10, 256)
    check_product(y3.flatten(0, 1), want, torch.bfloat16, 192)
    res = rows(40, 256, torch.bfloat16, 3).cuda()
    fresh = w.forward(view, residual=res)
    same = w.forward(view, residual=res, out=res)
    assert same.data_ptr() == res.data_ptr() and torch.equal(same, fresh)
    assert w.forward(big[:0, :192]).shape == (0, 256)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_rows_that_are_not_finite_or_nothing(dtype):
    from qmoe_b200 import Int8Tensor
    codes, scales = weights(130, 200, 4)
    x = rows(6, 200, DT[dtype], 5)
    x[1] = 0
    x[2, 199] = float("nan")
    x[3, 0] = float("-inf")
    x[4] *= 1e30
    x[5] *= 1e-30
    y = Int8Tensor.from_bytes(codes.cuda(), (130, 200), scales.cuda()).forward(x.cuda()).cpu()
    assert y[2].isnan().all() and y[3].isnan().all()
    assert (y[1] == 0).all()
    keep = [0, 1, 4, 5]
    check_product(y[keep], ref.product(x[keep], codes, scales), DT[dtype], 200)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("t,k", [(1, 1), (5, 1000), (7, 4097), (300, 64), (2, 131072)])
def test_quantize_rows_exactly(dtype, t, k):
    from qmoe_b200 import quantize_int8
    x = rows(t, k, DT[dtype], k)
    if k > 1000:                                  # values on and next to borders between two codes
        m = x[0].abs().max().item()
        edges = (torch.arange(-126, 126) + 0.5) / 127 * m
        x[0, 1:253] = edges.to(x.dtype)
        x[0, 253:505] = torch.nextafter(edges.float(), torch.zeros(()) + 1e9).to(x.dtype)
        x[0, 505] = m / 2
    codes, scales = quantize_int8(x.cuda())
    c, r = ref.quantize(x)
    assert torch.equal(codes.cpu().double(), c)
    assert torch.equal(scales.cpu(), (r.float() / torch.tensor(127.0)))


def test_from_float_is_rows_of_the_weight():
    from qmoe_b200 import Int8Tensor
    w = rows(300, 500, torch.float32, 9)
    c, r = ref.quantize(w)
    x = rows(9, 500, torch.float32, 10)
    y = Int8Tensor.from_float(w.cuda()).forward(x.cuda())
    check_product(y, ref.product(x, c, (r / 127).float()), torch.float32, 500)


def test_repeats_streams_and_graph():
    from qmoe_b200 import Int8Tensor
    codes, scales = weights(2048, 1024, 11)
    w = Int8Tensor.from_bytes(codes.cuda(), (2048, 1024), scales.cuda())
    xs = [rows(t, 1024, torch.bfloat16, t).cuda() for t in (3, 100)]
    want = [w.forward(x) for x in xs]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = [w.forward(x) for x in xs]
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graphs, outs = [], []
    for x in xs:                                  # two graphs, replayed in turn
        out = torch.empty(x.shape[0], 2048, dtype=torch.bfloat16, device="cuda")
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            w.forward(x, out=out)
        graphs.append(graph)
        outs.append(out)
    for _ in range(3):
        for o in outs:
            o.zero_()
        for gr in graphs:
            gr.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, outs))


def test_large_matches_exact_integers():
    """A product of many tiles: whole numbers that f32 holds come out exactly."""
    from qmoe_b200 import Int8Tensor
    g = torch.Generator().manual_seed(3)
    codes = torch.randint(-3, 4, (1200, 2000), generator=g, dtype=torch.int8)
    w = Int8Tensor.from_bytes(codes.cuda(), (1200, 2000), torch.ones(1200).cuda())
    x = torch.randint(-126, 127, (1500, 2000), generator=g).float()
    x[:, 0] = 127
    y = w.forward(x.cuda()).cpu()
    assert np.array_equal(y.numpy(), (x.double() @ codes.double().T).numpy())


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("t,k,n", [(2000, 96, 5000), (700, 130, 4200), (301, 2624, 64), (190, 5000, 4097)])
def test_wide_products_add_in_place(dtype, t, k, n):
    """Tiles of 256 and 128 tokens, several a CTA, with ragged ends both ways and a
    residual that is the output itself."""
    from qmoe_b200 import Int8Tensor
    dt = DT[dtype]
    codes, scales = weights(n, k, t)
    x, res = rows(t, k, dt, n), rows(t, n, dt, 9)
    w = Int8Tensor.from_bytes(codes.cuda(), (n, k), scales.cuda())
    y = res.cuda()
    fresh = w.forward(x.cuda(), residual=y)
    w.forward(x.cuda(), residual=y, out=y)
    assert torch.equal(y, fresh)
    plain, want = ref.product(x, codes, scales), ref.product(x, codes, scales, res)
    # five f32 roundings of the parts, one of the result
    tol = (plain.abs() + res.double().abs()) * 6 * 2.0 ** -24 + want.abs() * torch.finfo(dt).eps / 2 * 1.01
    assert (y.cpu().double() - want).abs().le(tol).all()
    check_product(w.forward(x.cuda()), plain, dt, k)

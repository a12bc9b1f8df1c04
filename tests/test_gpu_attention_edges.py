"""Edges of the 8-bit attention operators: views, poison, rows of nobody, long
and padded batches, values far from one.  Plain forms in 64 bits (attn_ref)."""
import pytest
import torch

import attn_ref as ref

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def i32(v, *shape):
    return torch.tensor(v, dtype=torch.int32).reshape(shape or (len(v),)).cuda()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_quantize_views_whose_rows_repeat_or_overlap(dtype):
    from qmoe_b200 import Int8Tensor, quantize_int8
    x = torch.randn(4096, generator=torch.Generator().manual_seed(1)).to(DT[dtype]).cuda()
    views = [x[:200].expand(64, 200), x[:640].unfold(0, 128, 8), x[:71].unfold(0, 64, 1), x[:1].expand(9, 1),
             x[:2048].reshape(8, 256)[:, 3:131], x[:512].reshape(4, 128)[:, ::2]]
    for v in views:
        codes, scales = quantize_int8(v)
        c, r = ref.quantize(v.cpu())
        assert torch.equal(codes.cpu().double(), c) and torch.equal(scales.cpu(), r.float() / torch.tensor(127.0))
    w = Int8Tensor.from_float(views[1])
    assert w.shape == tuple(views[1].shape)
    assert torch.equal(w.forward(x[:128][None]), Int8Tensor.from_float(views[1].contiguous()).forward(x[:128][None]))

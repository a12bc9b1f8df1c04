"""The operators together: a decoder layer's attention half, whole layers in a
chain, prompts and single tokens over one cache, planned on the GPU."""
import pytest
import torch

import attn_ref as ref

pytestmark = pytest.mark.gpu
HID, HEADS, KVH, DK, DV, BS = 128, 4, 2, 64, 64, 16


def int8_weight(out_f, in_f, g):
    w = torch.randn(out_f, in_f, generator=g) / in_f ** 0.5
    c, r = ref.quantize(w)
    return c.to(torch.int8), (r / 127).float()


def make_half(seed, rotate=None):
    from qmoe_b200 import AttentionBlock, Int8Tensor, KVCache
    g = torch.Generator().manual_seed(seed)
    rows = HEADS * DK + KVH * (DK + DV)
    qkv, out = int8_weight(rows, HID, g), int8_weight(HID, HEADS * DV, g)
    norm = (1 + 0.1 * torch.randn(HID, generator=g), 0.1 * torch.randn(HID, generator=g), 1e-6)
    cache = KVCache(40, BS, KVH, DK, DV)
    block = AttentionBlock(cache, Int8Tensor.from_bytes(qkv[0], (rows, HID), qkv[1]),
                           Int8Tensor.from_bytes(out[0], (HID, HEADS * DV), out[1]), HEADS,
                           (norm[0].cuda(), norm[1].cuda(), norm[2]), rotate=rotate)
    return block, dict(qkv=qkv, out=out, norm=norm)


class Plain:
    """The half in 64 bits, with a cache of its own."""

    def __init__(self, w):
        self.w = w
        self.k, self.v = (torch.zeros(40, KVH, BS, d, dtype=torch.float64) for d in (DK, DV))
        self.kr, self.vr = (torch.zeros(40, KVH, dtype=torch.float64) for _ in range(2))

    def forward(self, x, plan):
        w, b, eps = self.w["norm"]
        y = torch.nn.functional.layer_norm(x.double(), (HID,), w.double(), b.double(), eps)
        qkv = ref.product(y, *self.w["qkv"])
        q, k, v = qkv.split([HEADS * DK, KVH * DK, KVH * DV], 1)
        ref.append(self.k, self.kr, k.reshape(-1, KVH, DK), plan["slots"], BS)
        ref.append(self.v, self.vr, v.reshape(-1, KVH, DV), plan["slots"], BS)
        o = torch.zeros(x.shape[0], HEADS, DV, dtype=torch.float64)
        ref.attend(q.reshape(-1, HEADS, DK), self.k, self.kr, self.v, self.vr, plan["q_start"], plan["kv_lens"],
                   plan["table"], BS, DK ** -0.5, o)
        return ref.product(o.reshape(-1, HEADS * DV), *self.w["out"], residual=x)


STEPS = [  # (new tokens of the requests, rows of the buffer): prompts, a chunk, single tokens, a padded batch
    ([20, 7, 33], 60), ([1, 25, 1], 27), ([1, 1, 1], 3), ([1, 1, 1], 8), ([0, 1, 15], 16)]


def run_steps(forward, plain, dtype, tol):
    from qmoe_b200 import plan_pages
    g = torch.Generator().manual_seed(4)
    cached, free = [0, 0, 0], list(range(39, -1, -1))
    table = torch.full((3, 8), -1, dtype=torch.int32, device="cuda")
    ptable = [[-1] * 8 for _ in range(3)]
    dev = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    for new, rows in STEPS:
        x = torch.randn(rows, HID, generator=g).to(dtype)
        p = plan_pages(dev(cached), dev(new), table, dev(free), BS, rows, 40)
        want_p = ref.plan(cached, new, ptable, free, BS, rows, 40)
        assert p.slots.tolist() == want_p["slots"] and p.block_table.tolist() == ptable
        got = forward(x.cuda(), p)
        want = plain(x, want_p)
        live = sum(new)
        err = (got.cpu().double() - want)[:live].abs().max().item()
        assert err <= tol * want[:live].abs().max().item(), err
        free = free[p.taken.item():]
        cached = [c + n for c, n in zip(cached, new)]


# Both sides quantise their own y, k, v and o: an error e in front of a quantiser
# may move a value across a border, one step of 2/127 of the row's range for an
# element. In f32 (e about 2^-20) that is rare and one of K = 128 or more elements:
# below 2/127 * 3 sigma / sqrt(128) of a row's size. In bf16 (qkv and o rounded,
# 2^-9 of their value and less than half a step on average) every element may be
# off by that half step: the four quantised quantities add at most 4 / 127 of the
# attention half's size, which the residual and its rounding (2^-8) dominate.
TOL = {torch.float32: 2.0 / 127, torch.bfloat16: 4.0 / 127 + 2.0 ** -8}


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_attention_half(dtype):
    block, w = make_half(1)
    plain = Plain(w)
    run_steps(block.forward, plain.forward, dtype, TOL[dtype])


def test_rotate_sees_positions():
    seen = []

    def rotate(q, k, positions):
        seen.append(positions.clone())
        return q * 1.0, k * 1.0                  # packed copies in place of the views

    block, w = make_half(1, rotate)
    run_steps(block.forward, Plain(w).forward, torch.float32, TOL[torch.float32])
    assert seen[1].tolist() == [20] + list(range(7, 32)) + [33]
    assert seen[3].tolist()[3:] == [-1] * 5


def moe_layer(seed):
    from qmoe_b200 import MoEConfig, PackedExpert, QMoELayer
    g = torch.Generator().manual_seed(seed)
    E, inter = 4, 64
    pk = lambda o, i: (torch.randint(0, 256, (o, i // 4), generator=g, dtype=torch.uint8).numpy(),  # noqa: E731
                       (torch.rand(o, generator=g) * 0.05).numpy())
    experts = [PackedExpert(pk(inter, HID), pk(inter, HID), pk(HID, inter)) for _ in range(E)]
    layer = QMoELayer(MoEConfig(E, 2, HID, inter), torch.randn(E, HID, generator=g).numpy(), experts)
    layer.set_norm(torch.ones(HID).numpy(), torch.zeros(HID).numpy())
    return layer


def test_chain_runs_whole_layers():
    from qmoe_b200 import BlockChain, plan_pages
    dev = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    halves = [make_half(s)[0] for s in (1, 2)]
    others = [make_half(s)[0] for s in (1, 2)]
    layers = [moe_layer(s) for s in (3, 4)]
    chain = BlockChain(layers, attention=halves)
    table = torch.full((2, 4), -1, dtype=torch.int32, device="cuda")
    g = torch.Generator().manual_seed(4)
    cached = [0, 0]
    free = list(range(40))
    for new in ([9, 20], [1, 1]):
        x = torch.randn(sum(new), HID, generator=g).cuda()
        p = plan_pages(dev(cached), dev(new), table, dev(free), BS, sum(new), 40)
        out = torch.empty_like(x)
        got = chain.forward(x, plan=p, out=out)
        assert got.data_ptr() == out.data_ptr()
        y = x
        for a, L in zip(others, layers):
            y = L.forward_block(a.forward(y, p))
        assert torch.equal(got, y)
        free, cached = free[p.taken.item():], [c + n for c, n in zip(cached, new)]
    with pytest.raises(ValueError):
        chain.forward(x)
    with pytest.raises(ValueError):
        BlockChain(layers).forward(x, plan=p)
    with pytest.raises(ValueError):
        BlockChain(layers, attention=halves[:1])


def test_decode_step_in_a_graph():
    """plan, projections, append and attention captured once; lengths, tables and inputs change in place."""
    from qmoe_b200 import plan_pages
    dev = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    block, _ = make_half(5)
    eager, _ = make_half(5)
    state = {}
    for b in (block, eager):                     # a prompt of each request first
        table = torch.full((3, 6), -1, dtype=torch.int32, device="cuda")
        x = torch.randn(40, HID, generator=torch.Generator().manual_seed(1)).cuda()
        p = plan_pages(dev([0, 0, 0]), dev([10, 14, 16]), table, dev(list(range(40))), BS, 40, 40)
        b.forward(x, p)
        state[b] = table
    cached, new, free = dev([10, 14, 16]), dev([1, 1, 1]), dev(list(range(39, 2, -1)))
    x = torch.zeros(3, HID, device="cuda")
    block.forward(x, plan_pages(cached, dev([0, 0, 0]), state[block].clone(), free, BS, 3, 40))   # loads every kernel
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        p = plan_pages(cached, new, state[block], free, BS, 3, 40)
        y = block.forward(x, p)
    at = 0
    for step in range(20):
        x.copy_(torch.randn(3, HID, generator=torch.Generator().manual_seed(step)))
        graph.replay()
        q = plan_pages(cached, new, state[eager], free, BS, 3, 40)
        want = eager.forward(x, q)
        assert torch.equal(y, want) and torch.equal(p.slots, q.slots)
        cached += 1
        at += p.taken.item()
        free.copy_(torch.cat([dev(list(range(39, 2, -1)))[at:], dev([0] * at)]))
    assert at == 3 + 2                            # 10, 14, 16 -> 30, 34, 36 tokens in blocks of 16

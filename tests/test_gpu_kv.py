"""Plan, append and attention of the 8-bit paged cache against plain 64-bit forms."""
import random

import pytest
import torch

import attn_ref as ref

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def i32(v, *shape):
    return torch.tensor(v, dtype=torch.int32).reshape(shape or (len(v),)).cuda()


# ---- plan ---------------------------------------------------------------------

def run_plan(cached, new, table, free, bs, cap, nb):
    from qmoe_b200 import plan_pages
    width = len(table[0]) if table else 0
    t = i32([x for row in table for x in row], len(table), width)
    p = plan_pages(i32(cached), i32(new), t, i32(free), bs, cap, nb)
    got = {k: getattr(p, k).tolist() for k in ("q_start", "kv_lens", "slots", "positions", "taken")}
    got["table"] = p.block_table.tolist()
    return got


def make_plan(R, bs, seed, new_max, cached_max, spare=3):
    g = random.Random(seed)
    cached = [g.choice([0, 1, bs - 1, bs, bs + 1, g.randint(0, cached_max)]) for _ in range(R)]
    new = [g.choice([0, 1, 1, g.randint(0, new_max)]) for _ in range(R)]
    width = -(-(cached_max + bs + 1 + new_max) // bs) + 1
    ids = list(range(sum(-(-c // bs) for c in cached) + sum(-(-n // bs) + 1 for n in new) + spare))
    g.shuffle(ids)
    table = []
    for c in cached:
        have = -(-c // bs)
        table.append([ids.pop() for _ in range(have)] + [-1] * (width - have))
    return cached, new, table, ids


@pytest.mark.parametrize("R,bs,new_max,cached_max", [(1, 16, 1, 0), (1, 16, 40, 100), (7, 16, 40, 100), (32, 64, 1, 300),
                                                     (300, 32, 9, 200), (1500, 48, 5, 120), (2100, 128, 3, 300), (5000, 16, 2, 40)])
@pytest.mark.parametrize("room", ["all", "short", "none"])
def test_plan(R, bs, new_max, cached_max, room):
    cached, new, table, free = make_plan(R, bs, R + bs, new_max, cached_max)
    need = sum(-(-(c + n) // bs) - -(-c // bs) for c, n in zip(cached, new))
    free = free if room == "all" else free[:need // 2] if room == "short" else []
    nb = 10 ** 6
    cap = sum(new) + (5 if room == "all" else 0)
    want = ref.plan(cached, new, [list(r) for r in table], free, bs, cap, nb)
    got = run_plan(cached, new, table, free, bs, cap, nb)
    assert got == want
    if room == "all":
        assert got["taken"] == [need] and all(v == c + n for v, c, n in zip(got["kv_lens"], cached, new))


def test_plan_denials_and_bad_entries():
    bs = 16
    # too long for its row; negative; fits; rows behind the capacity; entry -1 and one past the cache
    cached = [40, -1, 5, 10, 20, 3]
    new = [60, 2, 2, -3, 1, 1]
    table = [[0, 1, 2, -1], [-1] * 4, [-1, -1, -1, -1], [3, -1, -1, -1], [4, 99, -1, -1], [5, -1, -1, -1]]
    for cap in (64, 65, 66, 3, 0):
        want = ref.plan(cached, new, [list(r) for r in table], [6, 7], bs, cap, 10)
        assert run_plan(cached, new, table, [6, 7], bs, cap, 10) == want, cap


def test_plan_of_nothing():
    from qmoe_b200 import plan_pages
    e = torch.empty(0, dtype=torch.int32, device="cuda")
    p = plan_pages(e, e, torch.empty(0, 4, dtype=torch.int32, device="cuda"), e, 16, 3, 8)
    assert p.q_start.tolist() == [0] and p.slots.tolist() == [-1] * 3 and p.taken.tolist() == [0]


# ---- append ---------------------------------------------------------------------

def make_cache(nb, bs, H, dk, dv, seed):
    from qmoe_b200 import KVCache
    g = torch.Generator().manual_seed(seed)
    k = torch.randint(-127, 128, (nb, H, dk // 64, bs, 64), generator=g, dtype=torch.int8)
    v = torch.randint(-127, 128, (nb, H, bs // 16, dv, 16), generator=g, dtype=torch.int8)
    kr, vr = torch.rand(nb, H, generator=g) * 3 + 0.5, torch.rand(nb, H, generator=g) * 3 + 0.5
    return KVCache.from_tensors(k.cuda(), v.cuda(), kr.cuda(), vr.cuda()), k, v, kr, vr


def check_append(cache, k0, v0, kr0, vr0, k, v, slots):
    bs = cache.block_size
    for flat, got, gr, codes, ranges, x in ((ref.k_flat, cache.k, cache.k_range, k0, kr0, k),
                                            (ref.v_flat, cache.v, cache.v_range, v0, vr0, v)):
        want, r = flat(codes).double(), ranges.double()
        ref.append(want, r, x, slots, bs)
        assert torch.equal(gr.cpu().double(), r)
        assert torch.equal(flat(got.cpu()).double(), want)


def runs_to_slots(runs, bs, order):
    slots = []
    for off, n in runs:                          # each run in blocks of its own
        while n > 0:
            b, m = order.pop(), min(n, bs - off)
            slots += [b * bs + off + i for i in range(m)]
            off, n = 0, n - m
    return slots


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("bs,H,dk,dv", [(16, 1, 64, 64), (16, 3, 192, 128), (48, 2, 128, 128), (64, 8, 128, 128),
                                        (256, 2, 192, 128)])
def test_append(dtype, bs, H, dk, dv):
    runs = [(0, 1), (bs - 1, 1), (5, 3), (3, bs), (0, 2 * bs + 7), (bs // 2, 1), (1, 1)]
    nb = sum(-(-(o + n) // bs) for o, n in runs) + 2
    order = list(range(nb))
    random.Random(bs).shuffle(order)
    slots = runs_to_slots(runs, bs, order)
    slots[5:5] = [-1]                             # a row of nobody between two runs
    slots += [-1, nb * bs, -7]
    T = len(slots)
    cache, *start = make_cache(nb, bs, H, dk, dv, bs + dk)
    g = torch.Generator().manual_seed(1)
    x = torch.randn(T, H * (dk + dv) + 11, generator=g) * torch.exp(torch.randn(T, 1, generator=g))
    x[[t for t, s in enumerate(slots) if not 0 <= s < nb * bs]] = float("nan")
    x = x.to(DT[dtype])
    for shift in (0, 3):                          # packed, and a view that starts at an odd place
        k = x[:, shift:shift + H * dk].unflatten(1, (H, dk))
        v = x[:, shift + H * dk:shift + H * (dk + dv)].unflatten(1, (H, dv))
        cache, *start = make_cache(nb, bs, H, dk, dv, bs + dk)
        xd = x.cuda()
        cache.append(xd[:, shift:shift + H * dk].unflatten(1, (H, dk)),
                     xd[:, shift + H * dk:shift + H * (dk + dv)].unflatten(1, (H, dv)), i32(slots))
        check_append(cache, *start, k, v, slots)


def test_append_token_by_token_and_again():
    """A block filled one token a call: the range grows, earlier codes follow; repeating a call changes nothing."""
    bs, H = 32, 2
    cache, k0, v0, kr0, vr0 = make_cache(3, bs, H, 128, 128, 5)
    g = torch.Generator().manual_seed(2)
    flat = [ref.k_flat(k0).double(), kr0.double(), ref.v_flat(v0).double(), vr0.double()]
    for i in range(bs):
        k = (torch.randn(1, H, 128, generator=g) * 1.1 ** i).bfloat16()
        v = (torch.randn(1, H, 128, generator=g) * (0 if i < 3 else 1)).bfloat16()
        for _ in range(2):
            cache.append(k.cuda(), v.cuda(), i32([bs + i]))
        ref.append(flat[0], flat[1], k, [bs + i], bs)
        ref.append(flat[2], flat[3], v, [bs + i], bs)
    assert torch.equal(ref.k_flat(cache.k.cpu()).double(), flat[0])
    assert torch.equal(ref.v_flat(cache.v.cpu()).double(), flat[2])
    assert torch.equal(cache.k_range.cpu().double(), flat[1]) and torch.equal(cache.v_range.cpu().double(), flat[3])


def test_append_values_that_are_not_finite():
    """They poison their block and head alone, until the block starts anew."""
    cache, k0, v0, kr0, vr0 = make_cache(2, 16, 2, 64, 64, 6)
    k, v = torch.randn(2, 2, 64), torch.randn(2, 2, 64)
    k[1, 0, 5] = float("inf")
    v[0, 1, 63] = float("nan")
    cache.append(k.cuda(), v.cuda(), i32([3, 4]))
    assert cache.k_range.isnan().tolist() == [[True, False], [False, False]]
    assert cache.v_range.isnan().tolist() == [[False, True], [False, False]]
    assert (cache.k[0, 0, :, :5] == 0).all() and (cache.k[0, 0, :, 5:] == k0[0, 0, :, 5:].cuda()).all()
    k[1, 0, 5] = v[0, 1, 63] = 1.0
    cache.append(k.cuda(), v.cuda(), i32([0, 1]))
    assert not cache.k_range.isnan().any() and not cache.v_range.isnan().any()


# ---- attention --------------------------------------------------------------------

def attend_case(dtype, bs, H, G, dk, dv, lens, seed, pad=0, spread=0.5, holes=False):
    """lens: (kv tokens, new tokens) of each request."""
    g = random.Random(seed)
    width = max([-(-kv // bs) for kv, _ in lens] + [0]) + 1
    nb = sum(-(-kv // bs) for kv, _ in lens) + 2
    cache, k, v, kr, vr = make_cache(nb, bs, H, dk, dv, seed)
    ids = list(range(nb))
    g.shuffle(ids)
    table = []
    for kv, _ in lens:
        have = -(-kv // bs)
        table.append([ids.pop() for _ in range(have)] + [-1] * (width - have))
    if holes:
        for row in table:
            for j in range(len(row)):
                if row[j] >= 0 and g.random() < 0.4:
                    row[j] = g.choice([-1, nb, 2 ** 30])
    starts = [0]
    for _, n in lens:
        starts.append(starts[-1] + n)
    gen = torch.Generator().manual_seed(seed)
    q = (torch.randn(starts[-1] + pad, H * G, dk, generator=gen) * spread).to(DT[dtype])
    return cache, (ref.k_flat(k), kr, ref.v_flat(v), vr), q, starts, [kv for kv, _ in lens], table


def check_attend(got, want, vr, dtype):
    bound = ref.attend_bound(DT[dtype]) * vr.max().item()
    err = (got.cpu().double() - want).abs().max().item()
    assert err <= bound, (err, bound)


SHAPES = [(16, 1, 1, 64, 64), (16, 2, 1, 192, 128), (32, 2, 4, 128, 128), (64, 1, 7, 128, 128), (128, 2, 16, 128, 128),
          (48, 1, 20, 64, 64), (16, 1, 40, 192, 128)]
LENS = {
    "one token": [(1, 1)],
    "decode": [(1, 1), (15, 1), (16, 1), (17, 1), (0, 1), (63, 1), (64, 1), (65, 1), (200, 1), (333, 1)],
    "long": [(2000, 1), (700, 1)],
    "prompts": [(37, 37), (90, 20), (0, 3), (129, 64), (5, 0), (300, 17)],
}


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("lens", list(LENS))
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_attend(dtype, lens, shape):
    bs, H, G, dk, dv = shape
    cache, flat, q, starts, kv, table = attend_case(dtype, bs, H, G, dk, dv, LENS[lens], 3, pad=4)
    q[starts[-1]:] = float("nan")
    scale = ref.new_scale(dk)
    width = len(table[0])
    want = ref.attend(q, *flat, starts, kv, table, bs, scale, torch.full((q.shape[0], H * G, dv), 0.25, dtype=torch.float64))
    for max_kv in (0, max(kv)):                   # cut into pieces by the table's width, by the longest request
        out = torch.full((q.shape[0], H * G, dv), 0.25, dtype=q.dtype, device="cuda")
        got = cache.attend(q.cuda(), i32(starts), i32(kv), i32([x for r in table for x in r], len(table), width),
                           max_kv=max_kv, out=out)
        assert got.data_ptr() == out.data_ptr()
        check_attend(got, want, flat[3], dtype)
        assert (got[starts[-1]:] == 0.25).all()   # rows of nobody stay
        for r, (k, n) in enumerate(LENS[lens]):
            if k == 0:
                assert (got[starts[r]:starts[r + 1]] == 0).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape", [(16, 1, 1, 64, 64), (48, 1, 2, 192, 128), (32, 1, 7, 128, 128), (128, 2, 2, 128, 128)],
                         ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("lens", [[(257, 257), (1, 1), (130, 129)], [(900, 300), (0, 40), (64, 64), (333, 33)],
                                  [(1, 1)] * 40 + [(600, 70)] + [(20, 20)] * 9])
def test_attend_prompts(dtype, shape, lens):
    """Prompts and chunks over several tiles of keys and rows, single tokens between them."""
    bs, H, G, dk, dv = shape
    cache, flat, q, starts, kv, table = attend_case(dtype, bs, H, G, dk, dv, lens, 5, pad=3, spread=1.5)
    q[starts[-1]:] = float("nan")
    scale = ref.new_scale(dk)
    out = torch.full((q.shape[0], H * G, dv), 0.25, dtype=q.dtype, device="cuda")
    got = cache.attend(q.cuda(), i32(starts), i32(kv), i32([x for r in table for x in r], len(table), len(table[0])), out=out)
    want = ref.attend_dense(q, *flat, starts, kv, table, bs, scale, torch.full(out.shape, 0.25, dtype=torch.float64))
    check_attend(got, want, flat[3], dtype)
    assert (got[starts[-1]:] == 0.25).all()
    for _ in range(2):
        assert torch.equal(cache.attend(q.cuda(), i32(starts), i32(kv), i32([x for r in table for x in r], len(table),
                                                                           len(table[0])), out=out.clone()), got)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attend_bad_pages_views_and_empty_blocks(dtype):
    bs, H, G, dk, dv = 16, 2, 4, 128, 128
    cache, flat, q, starts, kv, table = attend_case(dtype, bs, H, G, dk, dv, [(100, 1), (40, 9), (7, 1)], 8, holes=True)
    table[2][0] = -5                              # a request without any page left
    # ranges far apart, and a block of zeros that another writer gave the range 0
    cache.v_range[0] = 1e-12
    cache.v_range[1] = 0.0
    cache.v[1] = 0
    vr = cache.v_range.cpu()
    flat = (flat[0], flat[1], ref.v_flat(cache.v.cpu()), vr)
    wide = torch.zeros(q.shape[0], 3 * H * G * dk, dtype=q.dtype, device="cuda")
    view = wide[:, H * G * dk:2 * H * G * dk].unflatten(1, (H * G, dk))
    view.copy_(q)
    out = torch.zeros(q.shape[0], 2 * H * G * dv, dtype=q.dtype, device="cuda")
    got = cache.attend(view, i32(starts), i32(kv), i32([x for r in table for x in r], len(table), len(table[0])),
                       scale=0.07, out=out[:, :H * G * dv].unflatten(1, (H * G, dv)))
    want = ref.attend(q, *flat, starts, kv, table, bs, 0.07, torch.zeros(q.shape[0], H * G, dv, dtype=torch.float64))
    check_attend(got, want, vr, dtype)
    assert (out[:, H * G * dv:] == 0).all()
    assert (got[starts[2]:] == 0).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attend_extreme_scores(dtype):
    """One key far above the rest: the softmax is its value; and q of zero: the mean."""
    bs, H, dk = 32, 1, 128
    cache, flat, q, starts, kv, table = attend_case(dtype, bs, H, 1, dk, 128, [(500, 1), (500, 1), (500, 1)], 9)
    kval = flat[0].double() * (flat[1].double() / 127)[:, :, None, None]
    j = 321
    q[0, 0] = (kval[table[0][j // bs], 0, j % bs] * 30).to(q.dtype)
    q[1] = 0
    q[2] = q[2] * 1e-30
    args = (i32(starts), i32(kv), i32([x for r in table for x in r], len(table), len(table[0])))
    got = cache.attend(q.cuda(), *args, scale=1.0).cpu().double()
    vval = flat[2].double() * (flat[3].double() / 127)[:, :, None, None]
    half = torch.finfo(DT[dtype]).eps / 2
    one = vval[table[0][j // bs], 0, j % bs]
    assert (got[0, 0] - one).abs().le(one.abs() * half * 1.01 + 1e-5).all()
    mean = ref.attend(q, *flat, starts, kv, table, bs, 1.0, torch.zeros(3, 1, 128, dtype=torch.float64))
    assert (got[1:] - mean[1:]).abs().max() <= ref.attend_bound(DT[dtype]) * flat[3].max()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("scale", [-0.11, 0.0, None])
def test_attend_views_scales_and_wrong_hints(dtype, scale):
    """q and out that start at odd places, negative and zero scales, and a max_kv below the truth."""
    bs, H, G, dk, dv = 32, 2, 3, 128, 128
    cache, flat, q, starts, kv, table = attend_case(dtype, bs, H, G, dk, dv, [(700, 1), (90, 70), (400, 5), (2, 2)], 12)
    width = H * G * dk
    wide = torch.zeros(q.shape[0], width + 9, dtype=q.dtype, device="cuda")
    view = wide[:, 3:3 + width].unflatten(1, (H * G, dk))
    view.copy_(q)
    out = torch.zeros(q.shape[0], H * G * dv + 7, dtype=q.dtype, device="cuda")
    args = (i32(starts), i32(kv), i32([x for r in table for x in r], len(table), len(table[0])))
    got = cache.attend(view, *args, scale=scale, max_kv=16, out=out[:, 1:1 + H * G * dv].unflatten(1, (H * G, dv)))
    s = ref.new_scale(dk) if scale is None else scale
    want = ref.attend_dense(q, *flat, starts, kv, table, bs, s, torch.zeros(q.shape[0], H * G, dv, dtype=torch.float64))
    check_attend(got, want, flat[3], dtype)
    assert (out[:, 0] == 0).all() and (out[:, 1 + H * G * dv:] == 0).all()


@pytest.mark.parametrize("G", [33, 100, 160])
def test_attend_many_heads_to_one(G):
    cache, flat, q, starts, kv, table = attend_case("bf16", 16, 1, G, 64, 64, [(50, 1), (70, 9), (33, 2)], 13)
    got = cache.attend(q.cuda(), i32(starts), i32(kv), i32([x for r in table for x in r], 3, len(table[0])))
    want = ref.attend_dense(q, *flat, starts, kv, table, 16, ref.new_scale(64), torch.zeros(q.shape[0], G, 64, dtype=torch.float64))
    check_attend(got, want, flat[3], "bf16")


def test_attend_poisoned_rows_stay_apart():
    """A NaN query row and a poisoned block reach their own outputs alone."""
    bs = 16
    cache, flat, q, starts, kv, table = attend_case("bf16", bs, 2, 2, 64, 64, [(40, 3), (20, 1)], 10)
    args = (i32(starts), i32(kv), i32([x for r in table for x in r], 2, len(table[0])))
    clean = cache.attend(q.cuda(), *args)
    q[1, 0, 3] = float("nan")
    cache.k_range[table[1][0], 1] = float("nan")
    got = cache.attend(q.cuda(), *args)
    bad = torch.zeros_like(got, dtype=torch.bool)
    bad[1, 0] = True
    bad[3, 2:] = True
    assert got[bad].isnan().all() and torch.equal(got[~bad], clean[~bad])


def test_attend_repeats_streams_and_graphs():
    bs, H, G, dk, dv = 64, 4, 4, 128, 128
    cache, flat, q, starts, kv, table = attend_case("bf16", bs, H, G, dk, dv, [(900, 1)] * 3 + [(300, 40)], 11)
    args = (i32(starts), i32(kv), i32([x for r in table for x in r], len(table), len(table[0])))
    q = q.cuda()
    want = cache.attend(q, *args)
    for _ in range(3):
        assert torch.equal(cache.attend(q, *args), want)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = cache.attend(q, *args)
    side.synchronize()
    assert torch.equal(got, want)
    graphs = []
    for rows in (q, q * 2):
        out = torch.zeros_like(want)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            cache.attend(rows, *args, out=out)
        graphs.append((g, out, cache.attend(rows, *args)))
    for _ in range(2):
        for g, out, _ in graphs:
            out.zero_()
            g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for _, o, w in graphs)


def test_attend_of_nothing():
    cache, *_ = make_cache(2, 16, 2, 64, 64, 1)
    e = torch.empty(0, dtype=torch.int32, device="cuda")
    q = torch.empty(0, 4, 64, device="cuda")
    assert cache.attend(q, i32([0]), e, torch.empty(0, 1, dtype=torch.int32, device="cuda")).shape == (0, 4, 64)
    q = torch.ones(3, 4, 64, device="cuda")
    assert (cache.attend(q, i32([0]), e, torch.empty(0, 1, dtype=torch.int32, device="cuda")) == 0).all()
    none = cache.attend(q, i32([0, 3]), i32([0]), torch.empty(1, 0, dtype=torch.int32, device="cuda"))
    assert (none == 0).all()
    cache.append(q[:0, :2], q[:0, :2], e)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape", [(16, 16, 8, 64, 64), (64, 8, 4, 128, 128)], ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("lens", [[(310, 300), (1, 1), (3, 2), (60, 7), (260, 259)], [(700, 650), (90, 1), (40, 40)]])
def test_attend_prompts_that_fill_the_device(dtype, shape, lens):
    """Query tiles by the hundred, with every other kind of request beside them,
    written by a launch right in front and read by one right behind."""
    bs, H, G, dk, dv = shape
    cache, flat, q, starts, kv, table = attend_case(dtype, bs, H, G, dk, dv, lens, 8, pad=2, spread=1.0)
    q[starts[-1]:] = 0.0
    args = i32(starts), i32(kv), i32([x for r in table for x in r], len(table), len(table[0]))
    want = ref.attend_dense(q, *flat, starts, kv, table, bs, ref.new_scale(dk), torch.zeros(q.shape[0], H * G, dv, dtype=torch.float64))
    src, out = q.cuda(), torch.zeros(q.shape[0], H * G, dv, dtype=q.dtype, device="cuda")
    graph, side, buf = torch.cuda.CUDAGraph(), torch.cuda.Stream(), torch.empty_like(src)
    copies = [torch.empty_like(out) for _ in range(3)]
    with torch.cuda.graph(graph, stream=side):
        for c in copies:
            buf.copy_(src)
            cache.attend(buf, *args, out=out)
            c.copy_(out)
            buf.fill_(float("nan"))
            out.zero_()
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    check_attend(copies[0], want, flat[3], dtype)
    assert torch.equal(copies[0], copies[1]) and torch.equal(copies[0], copies[2])

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


# ---- attention: poisoned blocks and rows of nobody --------------------------------

def attend_case(dtype, bs, H, G, dk, dv, lens, seed, pad=0, spread=1.0, ranges=(0.5, 3.5)):
    """A cache, its 64-bit parts, q and the lists of a batch; lens: (kv tokens, new tokens)."""
    from qmoe_b200 import KVCache
    g = torch.Generator().manual_seed(seed)
    blocks = [-(-kv // bs) for kv, _ in lens]
    nb, width = sum(blocks) + 2, max(blocks + [0]) + 1
    k = torch.randint(-127, 128, (nb, H, dk // 64, bs, 64), generator=g, dtype=torch.int8)
    v = torch.randint(-127, 128, (nb, H, bs // 16, dv, 16), generator=g, dtype=torch.int8)
    kr, vr = (torch.rand(nb, H, generator=g) * (ranges[1] - ranges[0]) + ranges[0] for _ in range(2))
    ids = torch.randperm(nb, generator=g).tolist()
    table = [[ids.pop() for _ in range(b)] + [-1] * (width - b) for b in blocks]
    starts = [0]
    for _, n in lens:
        starts.append(starts[-1] + n)
    q = (torch.randn(starts[-1] + pad, H * G, dk, generator=g) * spread).to(DT[dtype])
    cache = KVCache.from_tensors(k.cuda(), v.cuda(), kr.cuda(), vr.cuda())
    return cache, (ref.k_flat(k), kr, ref.v_flat(v), vr), q, starts, [kv for kv, _ in lens], table


def device_args(starts, kv, table):
    return i32(starts), i32(kv), i32([x for r in table for x in r], len(table), len(table[0]))


def check_rows(got, want, vr, dtype, slack=0.0):
    """Element by element: half a step of the result, and of the largest value what
    the weights may be off by, once each in numerator and denominator.  P in fp16:
    2^-12 (two terms 2^-22).  Exponents: at most 16 additions in f32, each off by a
    step, 2^-23 of a partial sum below 8: 2^-16.  `slack`: what a case adds to that."""
    half = torch.finfo(DT[dtype]).eps / 2
    w = (2.0 ** -11 if dtype == "bf16" else 2.0 ** -22) + 2.0 ** -16
    err = (got.cpu().double() - want).abs()
    bound = half * 1.01 * want.abs() + 2 * (w + slack) * vr.max().item()
    assert (err <= bound).all(), ((err - bound).max().item(), err.max().item())


# requests of one kind each beside a single token: tiles of the matrix kernel and
# few tokens' rows (bf16), the streaming kernel's tiles (f32)
POISONED = [[(300, 300), (5, 1)], [(700, 100), (5, 1)], [(90, 9), (5, 1)], [(40, 7), (5, 1)], [(86, 9), (5, 1)], [(35, 7), (5, 1)]]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("lens", POISONED, ids=str)
@pytest.mark.parametrize("shape", [(16, 2, 1, 64, 64), (16, 1, 4, 128, 128), (32, 2, 2, 192, 128)], ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("which", ["k", "v"])
def test_poison_reaches_only_rows_that_see_it(dtype, shape, lens, which):
    """A block whose range is NaN, in the middle of a request's new tokens and at
    their end: the tokens before it keep their bits."""
    bs, H, G, dk, dv = shape
    cache, flat, q, starts, kv, table = attend_case(dtype, bs, H, G, dk, dv, lens, 21)
    args = device_args(starts, kv, table)
    clean = cache.attend(q.cuda(), *args)
    assert not clean.isnan().any()
    total, new = lens[0]
    for token in (total - 1, total - 1 - new // 2):
        block = token // bs
        ranges = getattr(cache, which + "_range")
        old = ranges[table[0][block], H - 1].item()
        ranges[table[0][block], H - 1] = float("nan")
        got = cache.attend(q.cuda(), *args)
        ranges[table[0][block], H - 1] = old
        bad = torch.zeros_like(got, dtype=torch.bool)
        first = max(0, block * bs - (total - new))   # the first new token that sees the block
        bad[first:new, (H - 1) * G:] = True
        assert got[bad].isnan().all()
        assert torch.equal(got[~bad], clean[~bad])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("lens", [[(3000, 1), (1500, 1)], [(3000, 3), (1500, 1), (60, 40)], [(2000, 0), (1500, 1), (900, 2), (5, 0)]], ids=str)
@pytest.mark.parametrize("first", [1, 6])
def test_rows_in_front_of_the_first_request_stay(dtype, lens, first):
    """A later part of a batch: q_start does not begin at 0, the rows before and behind it are others'."""
    bs, H, G, dk, dv = 16, 2, 2, 128, 128
    cache, flat, q, starts, kv, table = attend_case(dtype, bs, H, G, dk, dv, lens, 31, pad=first + 3)
    starts = [s + first for s in starts]
    live = slice(first, starts[-1])
    q[:first] = q[starts[-1]:] = float("nan")
    want = ref.attend_dense(q, *flat, starts, kv, table, bs, ref.new_scale(dk), torch.zeros(q.shape[0], H * G, dv, dtype=torch.float64))
    out = torch.full((q.shape[0], H * G, dv), 0.25, dtype=q.dtype, device="cuda")
    cache.attend(q.cuda(), *device_args(starts, kv, table), out=out)
    assert (out[:first] == 0.25).all() and (out[starts[-1]:] == 0.25).all()
    check_rows(out[live], want[live], flat[3], dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("G,lens", [
    (4, [(9000, 1), (4000, 70), (3000, 5), (2500, 1), (700, 33)]),          # every kind, all of them in pieces
    (1, [(20000, 2), (30, 30)]), (16, [(16500, 1)]), (2, [(5000, 12)] * 5 + [(40, 0)] * 90 + [(6000, 1)]),
], ids=str)
def test_many_pieces_of_every_kind(dtype, G, lens):
    """Requests of one, few and many tokens of one batch, each with many pieces of scratch to itself."""
    bs, H, dk, dv = 64, 1, 128, 128
    cache, flat, q, starts, kv, table = attend_case(dtype, bs, H, G, dk, dv, lens, 41, pad=2)
    q[starts[-1]:] = float("nan")
    args = device_args(starts, kv, table)
    want = ref.attend_dense(q, *flat, starts, kv, table, bs, ref.new_scale(dk), torch.full((q.shape[0], H * G, dv), 0.25, dtype=torch.float64))
    for max_kv in (0, 200):                       # by the table's width; told far too little
        out = torch.full((q.shape[0], H * G, dv), 0.25, dtype=q.dtype, device="cuda")
        cache.attend(q.cuda(), *args, max_kv=max_kv, out=out)
        assert (out[starts[-1]:] == 0.25).all()
        check_rows(out[:starts[-1]], want[:starts[-1]], flat[3], dtype)


def test_scratch_is_all_that_is_written():
    """A workspace of just the bytes asked for, with a guard behind it."""
    import ctypes
    from qmoe_b200 import capi
    for dtype in ("bf16", "f32"):
        cache, flat, q, starts, kv, table = attend_case(dtype, 64, 2, 4, 128, 128, [(9000, 1), (4000, 70), (3000, 5), (10, 0), (2500, 1)], 42)
        args = device_args(starts, kv, table)
        want = cache.attend(q.cuda(), *args)
        T, R, width, code = q.shape[0], len(kv), len(table[0]), capi.QMOE_DTYPE_BF16 if dtype == "bf16" else capi.QMOE_DTYPE_F32
        n = ctypes.c_int64()
        capi.call("qmoe_kv_attend_workspace", cache._p, code, T, R, 8, width, 0, ctypes.byref(n))
        assert n.value > 0
        ws = torch.full((n.value + 4096,), 171, dtype=torch.uint8, device="cuda")
        qd, out = q.cuda(), torch.zeros_like(want)
        cache.ctx.use_current_torch_stream()
        a = [cache.ctx.handle, cache._p, qd.data_ptr(), code, T, 8 * 128, 8, *(x.data_ptr() for x in args[:2]), R,
             args[2].data_ptr(), width, 0, 128 ** -0.5, out.data_ptr(), 8 * 128, ws.data_ptr()]
        capi.call("qmoe_kv_attend", *a, n.value)
        assert torch.equal(out, want) and (ws[n.value:] == 171).all()
        assert capi.lib().qmoe_kv_attend(*a, n.value - 1) == capi.QMOE_ERR_INVALID


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("G,lens", [(4, [(300, 150)]), (1, [(700, 133), (90, 32), (80, 1), (140, 140)]), (16, [(1, 1)] * 30 + [(2100, 170)])], ids=str)
def test_prompts_among_more_places_than_tokens(dtype, G, lens):
    """A captured step's batch: more requests than rows, nearly all of them empty.
    Prompts of more than 128 tokens among them go by tiles like any other: the same
    bits as without the empty places (bf16; in f32 the places change how the keys
    are cut)."""
    bs, H, dk, dv = 16, 2, 128, 128
    tokens = sum(n for _, n in lens)
    places = [lens[0]] + [(50, 0)] * (tokens + 3 - len(lens)) + lens[1:]
    cache, flat, q, starts, kv, table = attend_case(dtype, bs, H, G, dk, dv, places, 51, pad=2)
    q[tokens:] = float("nan")
    assert q.shape[0] <= len(kv)
    out = torch.full((q.shape[0], H * G, dv), 0.25, dtype=q.dtype, device="cuda")
    cache.attend(q.cuda(), *device_args(starts, kv, table), out=out)
    want = ref.attend_dense(q, *flat, starts, kv, table, bs, ref.new_scale(dk), torch.zeros(q.shape[0], H * G, dv, dtype=torch.float64))
    check_rows(out[:tokens], want[:tokens], flat[3], dtype)
    assert (out[tokens:] == 0.25).all()
    if dtype == "bf16":
        full = [i for i, (_, n) in enumerate(places) if n]
        few = cache.attend(q.cuda(), *device_args([starts[i] for i in full] + [tokens], [kv[i] for i in full], [table[i] for i in full]))
        for i, (_, n) in enumerate(places):
            if n > 128:
                assert torch.equal(out[starts[i]:starts[i + 1]], few[starts[i]:starts[i + 1]])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_a_request_longer_than_the_buffer(dtype):
    """Rows that the buffer does not hold are left out, however few it holds."""
    for T, n in ((20, 40), (50, 90), (20, 20), (150, 190)):
        cache, flat, q, starts, kv, table = attend_case(dtype, 16, 2, 2, 64, 64, [(200, n)] + [(0, 0)] * 159, 52)
        want = ref.attend_dense(q, *flat, starts, kv, table, 16, ref.new_scale(64), torch.zeros(q.shape[0], 4, 64, dtype=torch.float64))
        for places in (160, 1):
            got = cache.attend(q[:T].cuda(), *device_args(starts[:places + 1], kv[:places], table[:places]))
            check_rows(got, want[:T], flat[3], dtype)


@pytest.mark.parametrize("mean", [0.0, 8.0, 32.0])
@pytest.mark.parametrize("G,new", [(1, 1), (4, 1), (12, 1), (20, 1), (4, 5), (4, 200)])
@pytest.mark.parametrize("dk", [64, 128, 192])
def test_scores_of_rows_with_a_mean(mean, G, new, dk):
    """q with a common offset and one outlying key in each block, whose range the small
    codes of the others share: bf16 scores are as exact as f32 sums of q . k."""
    from qmoe_b200 import KVCache
    g = torch.Generator().manual_seed(61)
    bs, kv, dv = 16, 640, 128 if dk > 64 else 64
    nb = kv // bs
    k = torch.randint(-1, 2, (nb, 1, dk // 64, bs, 64), generator=g, dtype=torch.int8)
    k[:, :, :, 7] = -127
    v = torch.randint(-127, 128, (nb, 1, 1, dv, 16), generator=g, dtype=torch.int8)
    kr, vr = torch.full((nb, 1), 20.0), torch.full((nb, 1), 2.0)
    q = (torch.randn(new, G, dk, generator=g) + mean).bfloat16()
    others = (ref.k_flat(k).double() * (20 / 127))[:, 0, [i for i in range(bs) if i != 7]].reshape(-1, dk)
    scale = 8.0 / 1.4427 / (q.double().reshape(-1, dk) @ others.T).std().item()   # exponents of 8 or so
    cache = KVCache.from_tensors(k.cuda(), v.cuda(), kr.cuda(), vr.cuda())
    table = list(range(nb))
    got = cache.attend(q.cuda(), i32([0, new]), i32([kv]), i32(table, 1, nb), scale=scale)
    want = ref.attend_dense(q, ref.k_flat(k), kr, ref.v_flat(v), vr, [0, new], [kv], [table], bs, scale,
                            torch.zeros(new, G, dv, dtype=torch.float64))
    # at most 16 additions, each off by a step of a partial sum, which no sum of
    # magnitudes over the dims passes; nor the base of the exponential, the largest score
    largest = (q.double().abs().reshape(-1, dk) @ others.abs().T).max().item() * scale * 1.4427
    check_rows(got, want, vr, "bf16", slack=16 * 2.0 ** -23 * largest)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("G,lens", [(2, [(300, 1)]), (2, [(3000, 1), (90, 7)]), (4, [(400, 150), (70, 1)])], ids=str)
def test_rows_of_q_far_from_one(dtype, G, lens):
    """2^n q with the scale 2^-n scale: the same bits, up to the type's largest values."""
    cache, flat, q, starts, kv, table = attend_case(dtype, 16, 2, G, 128, 128, lens, 71)
    args = device_args(starts, kv, table)
    scale = ref.new_scale(128)
    clean = cache.attend(q.cuda(), *args, scale=scale)
    assert q.abs().max() < 8
    for n in (-90, 60, 100, 110, 122):
        got = cache.attend(q.cuda() * 2.0 ** n, *args, scale=scale * 2.0 ** -n)
        assert torch.equal(got, clean), n


# ---- product ------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("t,k,n", [(3, 200, 130), (40, 2048, 640), (700, 130, 4200), (1, 4096, 256), (300, 5000, 300)])
def test_product_of_rows_far_from_one(dtype, t, k, n):
    """2^a x with weights of 2^b: 2^(a + b) times the result, bit for bit, wherever that
    is in range, some rows and not others; codes times a row's scale alone are not."""
    from qmoe_b200 import Int8Tensor
    g = torch.Generator().manual_seed(t + k)
    dt = DT[dtype]
    codes = torch.randint(-127, 128, (n, k), generator=g, dtype=torch.int8).cuda()
    scales = (torch.rand(n, generator=g) * 0.01 + 1e-4).cuda()
    x = torch.randn(t, k, generator=g).to(dt).cuda()
    res = torch.randn(t, n, generator=g).to(dt).cuda()
    w = Int8Tensor.from_bytes(codes, (n, k), scales)
    clean, added = w.forward(x), w.forward(x, residual=res)
    assert x.abs().max() < 32
    for a, b in ((122, -100), (122, -60), (-50, 100), (60, 40)):
        far = Int8Tensor.from_bytes(codes, (n, k), scales * 2.0 ** b)
        y = far.forward(x * 2.0 ** a).double() * 2.0 ** -(a + b)
        assert torch.equal(y, clean.double()), (a, b)
        y = far.forward(x * 2.0 ** a, residual=(res.double() * 2.0 ** (a + b)).to(dt)).double() * 2.0 ** -(a + b)
        assert torch.equal(y, added.double()), (a, b)
        mixed = x.clone()
        mixed[::2] *= 2.0 ** a
        y = far.forward(mixed).double() * 2.0 ** -b
        y[::2] *= 2.0 ** -a
        keep = torch.isfinite(clean.double() * 2.0 ** b)
        assert torch.equal(y[::2], clean[::2].double())
        assert torch.equal(y[1::2], clean[1::2].double()) and keep.all()


def test_shape_comes_from_the_handle():
    from qmoe_b200 import Int8Tensor
    w = Int8Tensor.from_bytes(torch.zeros(5 * 17, dtype=torch.int8).cuda(), (5, 17), torch.ones(5).cuda())
    assert w.shape == (5, 17) and w.forward(torch.ones(2, 17).cuda()).shape == (2, 5)


def test_plan_keeps_the_position_where_a_table_entry_is_no_block():
    from qmoe_b200 import plan_pages
    p = plan_pages(i32([20, 16]), i32([2, 1]), i32([3, -1, 9, 4, 99, 7], 2, 3), i32([5]), 16, 4, 8)
    assert p.slots.tolist() == [-1, -1, 5 * 16, -1]           # rows of entry -1; of a new block; of nobody
    assert p.positions.tolist() == [20, 21, 16, -1] and p.kv_lens.tolist() == [22, 17] and p.taken.tolist() == [1]


# ---- attention: nothing left out, nothing rounded twice ---------------------------------

@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape", [(16, 1, 1, 64, 64), (48, 1, 2, 192, 128), (64, 2, 4, 128, 128), (128, 1, 8, 128, 128)],
                         ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("lens", [[(900, 300), (700, 33), (333, 1)], [(2000, 500), (1500, 9), (40, 40)], [(3000, 129)]], ids=str)
def test_every_group_of_keys_counts_once(dtype, shape, lens):
    """V one value over each 16 tokens and another in each group: a group left out or
    taken twice moves a row far beyond what roundings do."""
    bs, H, G, dk, dv = shape
    cache, flat, q, starts, kv, table = attend_case(dtype, bs, H, G, dk, dv, lens, 81, spread=0.5)
    g = torch.Generator().manual_seed(82)
    nb = cache.num_blocks
    groups = (torch.randint(0, 2, (nb, H, bs // 16, 1, 1), generator=g) * 254 - 127).to(torch.int8)
    cache.v.copy_(groups.expand(nb, H, bs // 16, dv, 16))
    flat = (*flat[:2], ref.v_flat(cache.v.cpu()), flat[3])
    want = ref.attend_dense(q, *flat, starts, kv, table, bs, ref.new_scale(dk), torch.zeros(q.shape[0], H * G, dv, dtype=torch.float64))
    check_rows(cache.attend(q.cuda(), *device_args(starts, kv, table)), want, flat[3], dtype)


@pytest.mark.parametrize("lens", [[(900, 1), (700, 1), (600, 1)], [(800, 60), (700, 3)]], ids=str)
@pytest.mark.parametrize("G,dk,dv", [(1, 128, 128), (4, 192, 128), (2, 64, 64)])
def test_f32_keeps_its_second_terms(lens, G, dk, dv):
    """Root mean square of the error over many keys.  Weights are off by 2^-22 (P) and
    their exponents by four (root of 16 additions) times 2^-24 of sums below 8, 2^-19;
    both average over some 80 keys or more of like weight, to 2^-22 of the largest |v|.
    P in one fp16 term: 2^-11 at most, 2^-12.3 in the mean, 2^-17 averaged."""
    cache, flat, q, starts, kv, table = attend_case("f32", 64, 2, G, dk, dv, lens, 91)
    got = cache.attend(q.cuda(), *device_args(starts, kv, table)).cpu().double()
    want = ref.attend_dense(q, *flat, starts, kv, table, 64, ref.new_scale(dk), torch.zeros(q.shape[0], 2 * G, dv, dtype=torch.float64))
    rms = (got - want).pow(2).mean().sqrt().item()
    assert rms <= 2.0 ** -20 * flat[3].max().item(), rms


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("G,lens", [(1, [(134500, 1)]), (2, [(134500, 3)]), (5, [(65600, 1), (131072, 1)])], ids=str)
def test_the_most_pieces(dtype, G, lens):
    """Long caches of one kv head: as many pieces as the join takes, and more keys than those would hold."""
    cache, flat, q, starts, kv, table = attend_case(dtype, 128, 1, G, 64, 64, lens, 95)
    want = ref.attend_dense(q, *flat, starts, kv, table, 128, ref.new_scale(64), torch.zeros(q.shape[0], G, 64, dtype=torch.float64))
    for max_kv in (0, max(kv), 3000):
        check_rows(cache.attend(q.cuda(), *device_args(starts, kv, table), max_kv=max_kv), want, flat[3], dtype)

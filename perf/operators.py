"""The 8-bit attention half of a decoder layer, operator by operator, as measured work.

Four operators: the matrix product in 8-bit integers with a scale for each
token and output channel; the block table and slot map of a paged cache, built
from request lengths; the append of new keys and values to that cache, held in
8 bits with a range for each block of tokens and head; and attention over it.

`run(state)` with `own` false computes them in elementary torch operations,
with `own` true through the package.  `exact(case, seed)` gives the same
results from the definitions in 64 bits.

Layouts (shared with the package):
  k codes  int8 [blocks, kv_heads, k_dim / 64, block, 64]
  v codes  int8 [blocks, kv_heads, block / 16, v_dim, 16]
  ranges   f32  [blocks, kv_heads]; a code c stands for c * range / 127
"""
import math
import os
import random
import sys

import torch

own = False

FLOOR = 127.0 * 2.0 ** -64  # the smallest range: a scale of 2^-64
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


# --------------------------------------------------------------------------
# cases
# --------------------------------------------------------------------------

def listed():
    return [
        # the output projection of one decoded token at hidden size 2048: latency alone
        dict(name="product, one token", op="product", tokens=1, k=2048, n=2048, dtype="bf16", add=True),
        # a decode batch through a 16384 -> 7168 output projection: 117 MB of weights stream once
        dict(name="product, 32 tokens", op="product", tokens=32, k=16384, n=7168, dtype="bf16", add=True),
        # ragged everything, f32 activations: a small odd projection over part of a prompt
        dict(name="product, odd sizes", op="product", tokens=777, k=1411, n=1001, dtype="f32", add=False),
        # a prompt chunk through a 7168 -> 16384 query projection: the tensor cores' rate
        dict(name="product, prompt", op="product", tokens=4096, k=7168, n=16384, dtype="bf16", add=False),
        # the decode step of 32 requests
        dict(name="plan, 32 single tokens", op="plan", requests=32, new=1, cached=4000, block=64, tokens=32, short=False, mix=1),
        # thousands of requests of a mixed batch, prompts among them, and a pool that runs dry
        dict(name="plan, 4096 mixed", op="plan", requests=4096, new=120, cached=6000, block=16, tokens=262144, short=True, mix=2),
        # the decode step of 64 requests with 8 heads of 128
        dict(name="append, 64 single tokens", op="append", requests=64, new=1, cached=5000, block=64, kv_heads=8, k_dim=128,
             v_dim=128, dtype="bf16", fused=8, pad=0, mix=3),
        # two prompts of about 4000 tokens, keys of 192 and values of 128 in 16 heads, f32
        dict(name="append, prompts", op="append", requests=2, new=4099, cached=37, block=16, kv_heads=16, k_dim=192, v_dim=128,
             dtype="f32", fused=0, pad=5, mix=4),
        # one token of one request, keys of 192 and values of 128, f32: latency
        dict(name="attend, one token", op="attend", requests=1, new=1, cached=999, block=16, heads=16, kv_heads=16, k_dim=192,
             v_dim=128, dtype="f32", fused=False, pad=0, even=True, mix=5),
        # the decode step of 64 requests of ragged lengths, four query heads to each kv head
        dict(name="attend, 64 requests", op="attend", requests=64, new=1, cached=8192, block=64, heads=32, kv_heads=8, k_dim=128,
             v_dim=128, dtype="bf16", fused=True, pad=3, even=False, mix=6),
        # two requests far into a long context, eight query heads to each kv head
        dict(name="attend, two long", op="attend", requests=2, new=1, cached=131071, block=128, heads=64, kv_heads=8, k_dim=128,
             v_dim=128, dtype="bf16", fused=False, pad=0, even=True, mix=7),
        # chunks of three prompts behind what they have cached already
        dict(name="attend, prompts", op="attend", requests=3, new=2048, cached=6000, block=64, heads=32, kv_heads=8, k_dim=128,
             v_dim=128, dtype="bf16", fused=True, pad=0, even=False, mix=8),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["product", "product", "plan", "append", "attend", "attend"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    mix = rng.randrange(1 << 20)
    if op == "product":
        t, k, n = _log(rng, 1, 4096), _log(rng, 17, 16384), _log(rng, 5, 16384)
        if rng.random() < 0.5:
            k, n = -(-k // 64) * 64, -(-n // 64) * 64
        while t * k * n > 4096 * 7168 * 16384:
            t = (t + 1) // 2
        return dict(op=op, tokens=t, k=k, n=n, dtype=dtype, add=rng.random() < 0.5)
    block = rng.choice([16, 32, 48, 64, 128])
    if op == "plan":
        r = _log(rng, 1, 6000)
        new = rng.choice([1, 1, _log(rng, 2, 100)])
        return dict(op=op, requests=r, new=new, cached=_log(rng, 1, 6000), block=block, tokens=r * new + rng.choice([0, 3, 64]),
                    short=rng.random() < 0.4, mix=mix)
    kv = rng.choice([1, 2, 4, 8, 16])
    kd, vd = rng.choice([(64, 64), (128, 128), (128, 128), (192, 128)])
    if op == "append":
        r = _log(rng, 1, 256)
        new = rng.choice([1, _log(rng, 2, 8192)])
        while r * new > 8192:
            r = (r + 1) // 2
            new = max(1, new // 2)
        return dict(op=op, requests=r, new=new, cached=_log(rng, 1, 4000), block=block, kv_heads=kv, k_dim=kd, v_dim=vd,
                    dtype=dtype, fused=rng.choice([0, kv]), pad=rng.choice([0, 0, 7]), mix=mix)
    heads = kv * rng.choice([1, 2, 4, 7, 8, 16])
    r, cached = _log(rng, 1, 64), _log(rng, 1, 65536)
    new = rng.choice([1, 1, _log(rng, 2, 16), _log(rng, 17, 2048)])
    while r * heads * new * (cached + new) > 2 ** 30 or r * kv * (cached + new) * 256 > 2 ** 31:
        if r > 1:
            r = (r + 1) // 2
        elif cached > 64:
            cached //= 2
        else:
            new = (new + 1) // 2
    return dict(op=op, requests=r, new=new, cached=cached, block=block, heads=heads, kv_heads=kv, k_dim=kd, v_dim=vd, dtype=dtype,
                fused=rng.random() < 0.5, pad=rng.choice([0, 0, 5]), even=rng.random() < 0.3, mix=mix)


def _lens(c):
    """(tokens cached, new tokens) of each request, from the case alone."""
    g = random.Random(c["mix"])
    r, new, cached = c["requests"], c["new"], c["cached"]
    if c.get("even"):
        return [cached] * r, [new] * r
    a = [int(cached * g.random() ** 1.5) for _ in range(r)]
    b = [new if new == 1 else 1 + int(new * g.random() ** (4.0 if c["op"] == "plan" else 0.5)) for _ in range(r)]
    b = [min(x, new) for x in b]
    a[0], b[0] = cached, new
    return a, b


# --------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed & 0x7FFFFFFF)


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)


def _rows(g, t, width):
    """Activations: a spread of row sizes and a few outlying channels, as a decoder's residual stream has."""
    x = _normal(g, t, width) * torch.exp(0.5 * _normal(g, t, 1))
    return x * torch.exp((_normal(g, 1, width) - 2.0).clamp_min(0.0))


def _codes(g, *shape):
    return (_normal(g, *shape) * 42.0).round().clamp_(-127, 127).to(torch.int8)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _package():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "qmoe-rs_b200", "python")
    if at not in sys.path:
        sys.path.insert(0, at)
    import qmoe_b200
    return qmoe_b200


def prepare(case, seed):
    g = _gen(seed)
    s = dict(case)
    if case["op"] == "product":
        dt = DTYPES[case["dtype"]]
        s["x"] = _rows(g, case["tokens"], case["k"]).to(dt)
        s["w"] = _codes(g, case["n"], case["k"])
        s["ws"] = torch.exp(0.3 * _normal(g, case["n"])) * (0.02 / 42.0)
        s["res"] = _normal(g, case["tokens"], case["n"]).to(dt) if case["add"] else None
        if own:  # the weights as the package keeps them, laid out once
            s["tensor"] = _package().Int8Tensor.from_bytes(s["w"], (case["n"], case["k"]), s["ws"])
        return s
    cached, new = _lens(case)
    bs = case["block"]
    if case["op"] == "plan":
        have = [-(-c // bs) for c in cached]
        need = [-(-(c + n) // bs) - h for c, n, h in zip(cached, new, have)]
        width = -(-(case["cached"] + case["new"]) // bs) + 1
        pool = sum(have) + sum(need) + 8
        order = torch.randperm(pool, generator=g, device="cuda").to(torch.int32)
        table = torch.full((case["requests"], width), -1, dtype=torch.int32, device="cuda")
        col = torch.arange(width, device="cuda")[None]
        h = _ints(have).long()
        at = (h.cumsum(0) - h)[:, None] + col
        table = torch.where(col < h[:, None], order[at.clamp(max=pool - 1)], table)
        free = order[sum(have):]
        s["free"] = free[: len(free) // 2].clone() if case["short"] else free.clone()
        s.update(cached_lens=_ints(cached), new_lens=_ints(new), table=table.contiguous(), pool=pool)
        return s
    H, kd, vd, dt = case["kv_heads"], case["k_dim"], case["v_dim"], DTYPES[case["dtype"]]
    kv = [c + n for c, n in zip(cached, new)]
    if case["op"] == "attend" and case["requests"] > 2 and not case["even"]:
        kv[1] = 0  # a request that the pool had no room for: its rows see nothing
    blocks = [-(-x // bs) for x in kv]
    if case["op"] == "append":  # only the blocks that the new tokens touch
        first = [c // bs for c in cached]
        blocks = [b - f for b, f in zip(blocks, first)]
    pool = sum(blocks) + 3
    order = torch.randperm(pool, generator=g, device="cuda").to(torch.int32)
    s["kc"] = _codes(g, pool, H, kd // 64, bs, 64)
    s["vc"] = _codes(g, pool, H, bs // 16, vd, 16)
    s["kr"] = 3.0 * torch.exp(0.25 * _normal(g, pool, H))
    s["vr"] = 3.0 * torch.exp(0.5 * _normal(g, pool, H))
    tokens = sum(new)
    rows = tokens + case["pad"]
    if case["op"] == "append":
        per_request = torch.repeat_interleave(torch.arange(case["requests"], device="cuda"), _ints(new).long())
        start = _ints(new).long().cumsum(0) - _ints(new).long()
        base = _ints(blocks).long().cumsum(0) - _ints(blocks).long()
        off = _ints([c % bs for c in cached]).long()
        p = torch.arange(tokens, device="cuda") - start[per_request] + off[per_request]
        slot = order.long()[base[per_request] + p // bs] * bs + p % bs
        s["slots"] = torch.cat([slot.to(torch.int32), torch.full((case["pad"],), -1, dtype=torch.int32, device="cuda")])
        q = case["fused"] * kd
        x = _normal(g, rows, q + H * (kd + vd)) * torch.exp(0.3 * _normal(g, rows, 1))
        x[tokens:] = float("nan")  # rows that no request has hold anything
        x = x.to(dt)
        k, v = x[:, q:q + H * kd], x[:, q + H * kd:]
        if not case["fused"]:
            k, v = k.contiguous(), v.contiguous()
        s["k"], s["v"] = k.unflatten(1, (H, kd)), v.unflatten(1, (H, vd))
    else:
        width = max(blocks) + 1
        base = [0]
        for b in blocks:
            base.append(base[-1] + b)
        col = torch.arange(width, device="cuda")[None]
        at = (_ints(base[:-1]).long()[:, None] + col).clamp(max=pool - 1)
        s["table"] = torch.where(col < _ints(blocks)[:, None], order[at], torch.full_like(at, -1, dtype=torch.int32)).contiguous()
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        s["q_start"], s["kv_lens"] = _ints(starts), _ints(kv)
        s["max_new"], s["max_kv"], s["scale"] = max(new), max(kv), kd ** -0.5
        hq = case["heads"]
        extra = H * (kd + vd) if case["fused"] else 0
        x = _normal(g, rows, hq * kd + extra) * torch.exp(0.5 * _normal(g, 1, 1))
        x[tokens:] = float("nan")
        s["q"] = x.to(dt)[:, :hq * kd].unflatten(1, (hq, kd))
        s["out"] = torch.full((rows, hq, vd), 0.5, dtype=dt, device="cuda")
    if own:  # a view of the same memory
        s["cache"] = _package().KVCache.from_tensors(s["kc"], s["vc"], s["kr"], s["vr"])
    return s


# --------------------------------------------------------------------------
# one pass
# --------------------------------------------------------------------------

def run(s):
    if s["op"] == "product":
        return s["tensor"].forward(s["x"], residual=s["res"]) if own else _product(s)
    if s["op"] == "plan":
        if own:
            p = _package().plan_pages(s["cached_lens"], s["new_lens"], s["table"], s["free"], s["block"], s["tokens"], s["pool"])
            return dict(table=p.block_table, q_start=p.q_start, kv_lens=p.kv_lens, slots=p.slots, positions=p.positions,
                        taken=p.taken)
        return _plan(s)
    if s["op"] == "append":
        if own:
            s["cache"].append(s["k"], s["v"], s["slots"])
        else:
            _append(s)
        # what the codes stand for
        return dict(k=torch.mul(s["kc"], (s["kr"] / 127.0)[:, :, None, None, None]),
                    v=torch.mul(s["vc"], (s["vr"] / 127.0)[:, :, None, None, None]), k_range=s["kr"], v_range=s["vr"])
    if own:
        return s["cache"].attend(s["q"], s["q_start"], s["kv_lens"], s["table"], scale=s["scale"], max_kv=s["max_kv"], out=s["out"])
    return _attend(s)


def _product(s):
    x = s["x"].float()
    r = x.abs().amax(1, keepdim=True).clamp_min(FLOOR)
    codes = torch.round(x.double() * 127.0 / r.double()).float()  # in 64 bits: values next to a border between two codes
    y = (codes @ s["w"].float().T) * (r / torch.full_like(r, 127.0)) * s["ws"][None]
    if s["res"] is not None:
        y = y + s["res"].float()
    return y.to(s["x"].dtype)


def _plan(s):
    cached, new, table, free, bs = s["cached_lens"].long(), s["new_lens"].long(), s["table"], s["free"], s["block"]
    width, cap, pool = table.shape[1], s["tokens"], s["pool"]
    end = new.clamp_min(0).cumsum(0)
    q_start = torch.cat([torch.zeros_like(end[:1]), end])
    ok = (cached >= 0) & (new >= 0) & (cached + new <= width * bs) & (end <= cap)
    have = (cached + bs - 1) // bs
    need = torch.where(ok, (cached + new + bs - 1) // bs - have, 0)
    upto = need.cumsum(0)
    ok = ok & ((need == 0) | (upto <= free.numel()))
    need_ok = torch.where(ok, need, 0)
    taken = torch.where(ok & (need > 0), upto, 0).amax().reshape(1)
    col = torch.arange(width, device=table.device)[None]
    at = (upto - need)[:, None] + col - have[:, None]
    fresh = (col >= have[:, None]) & (col < (have + need_ok)[:, None])
    table.copy_(torch.where(fresh, free[at.clamp(0, free.numel() - 1)], table))
    kv = torch.where(ok, cached + new, 0)
    t = torch.arange(cap, device=table.device)
    r = torch.searchsorted(end, t, right=True).clamp(max=len(end) - 1)
    pos = cached[r] + t - q_start[r]
    live = (t < end[-1]) & ok[r]
    block = table[r, (pos // bs).clamp(0, width - 1)].long()
    good = live & (block >= 0) & (block < pool)
    i32 = torch.int32
    return dict(table=table, q_start=q_start.to(i32), kv_lens=kv.to(i32), slots=torch.where(good, block * bs + pos % bs, -1).to(i32),
                positions=torch.where(live, pos, -1).to(i32), taken=taken.to(i32))


def _append_one(x, codes, ranges, slots, bs, at):
    """x [tokens, heads, dim] into `codes`, through `at`: codes as [blocks, heads, block, dim]."""
    x = x.float()
    nb, H = ranges.shape
    live = slots >= 0
    blk, off = torch.where(live, slots // bs, nb).long(), torch.where(live, slots % bs, bs).long()
    first = torch.full((nb + 1,), bs, dtype=torch.long, device=x.device).scatter_reduce(0, blk, off, "amin")[:nb]
    amax = torch.where(live[:, None], x.abs().amax(2), 0.0)
    seen = torch.zeros(nb + 1, H, device=x.device).scatter_reduce(0, blk[:, None].expand(-1, H), amax, "amax")[:nb]
    touched = (first < bs)[:, None]
    old = torch.where((first > 0)[:, None], ranges, 0.0)
    new = torch.where(touched, torch.maximum(old, seen).clamp_min(FLOOR), ranges)
    before = touched[:, :, None, None] & (torch.arange(bs, device=x.device)[None, :] < first[:, None])[:, None, :, None]
    grid = at(codes)
    # codes in 64 bits: values next to a border between two codes
    moved = torch.round(grid.double() * ranges.double()[:, :, None, None] / new.double()[:, :, None, None])
    moved = torch.where(before, moved, grid.double())
    moved = torch.cat([moved, torch.zeros_like(moved[:1])])  # the tokens without a slot go to a block that is dropped
    mine = torch.cat([new, torch.ones_like(new[:1])])[blk].double()
    moved[blk, :, off.clamp(max=bs - 1)] = torch.round(x.double() * 127.0 / mine[:, :, None])
    ranges.copy_(new)
    return moved[:nb].to(torch.int8)


def _append(s):
    kc, vc, bs = s["kc"], s["vc"], s["block"]
    nb, H, kd, vd = kc.shape[0], kc.shape[1], s["k_dim"], s["v_dim"]
    k = _append_one(s["k"], kc, s["kr"], s["slots"], bs, lambda c: c.permute(0, 1, 3, 2, 4).reshape(nb, H, bs, kd))
    kc.copy_(k.reshape(nb, H, bs, kd // 64, 64).permute(0, 1, 3, 2, 4))
    v = _append_one(s["v"], vc, s["vr"], s["slots"], bs, lambda c: c.permute(0, 1, 2, 4, 3).reshape(nb, H, bs, vd))
    vc.copy_(v.reshape(nb, H, bs // 16, 16, vd).permute(0, 1, 2, 4, 3))


def _attend(s):
    q, bs, out = s["q"], s["block"], s["out"]
    rows, hq, kd = q.shape
    H, vd, n, n_max = s["kv_heads"], s["v_dim"], s["requests"], s["max_new"]
    nb = -(-s["max_kv"] // bs)
    idx = s["table"][:, :nb].clamp(0, s["kc"].shape[0] - 1).long()
    ks = (s["kr"][idx] / 127.0).permute(0, 2, 1).repeat_interleave(bs, 2)[..., None]
    vs = (s["vr"][idx] / 127.0).permute(0, 2, 1).repeat_interleave(bs, 2)[..., None]
    k = s["kc"][idx].permute(0, 2, 1, 4, 3, 5).reshape(n, H, nb * bs, kd).float() * ks
    v = s["vc"][idx].permute(0, 2, 1, 3, 5, 4).reshape(n, H, nb * bs, vd).float() * vs
    start, kv = s["q_start"].long(), s["kv_lens"].long()
    i = torch.arange(n_max, device=q.device)
    t = (start[:-1, None] + i).clamp(max=rows - 1)
    qs = q[t].float().reshape(n, n_max, H, hq // H, kd).permute(0, 2, 3, 1, 4).reshape(n, H, -1, kd)
    sc = (qs @ k.transpose(2, 3)).mul_(s["scale"]).reshape(n, H, hq // H, n_max, nb * bs)
    pos = (kv - (start[1:] - start[:-1]))[:, None] + i
    hidden = torch.arange(nb * bs, device=q.device) > pos[:, :, None]
    sc.masked_fill_(hidden[:, None, None], float("-inf"))
    top = sc.amax(4, keepdim=True)
    p = sc.sub_(torch.where(top == float("-inf"), 0.0, top)).exp_()
    total = p.sum(4, keepdim=True)
    o = (p.reshape(n, H, -1, nb * bs) @ v).reshape(n, H, hq // H, n_max, vd) / torch.where(total == 0, 1.0, total)
    o = o.permute(0, 3, 1, 2, 4).reshape(n, n_max, hq, vd).to(q.dtype)
    row = torch.arange(rows, device=q.device)
    r = torch.searchsorted(start[1:], row, right=True).clamp(max=n - 1)
    out.copy_(torch.where((row < start[-1])[:, None, None], o[r, (row - start[r]).clamp(max=n_max - 1)], out))
    return out


# --------------------------------------------------------------------------
# the least that a pass reads, writes and computes
# --------------------------------------------------------------------------

def work(case):
    if case["op"] == "product":
        t, k, n = case["tokens"], case["k"], case["n"]
        e = 2 if case["dtype"] == "bf16" else 4
        return dict(bytes=t * k * e + n * k + 4 * n + t * n * e * (2 if case["add"] else 1), flops=2 * t * k * n)
    cached, new = _lens(case)
    bs = case["block"]
    if case["op"] == "plan":
        r, t = case["requests"], case["tokens"]
        need = sum(-(-(c + n) // bs) - -(-c // bs) for c, n in zip(cached, new))
        return dict(bytes=4 * (4 * r + 1 + 2 * t + 2 * need), flops=0)
    H, kd, vd = case["kv_heads"], case["k_dim"], case["v_dim"]
    e = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "append":
        t = sum(new)
        # x in, codes and what they stand for out, for the tokens and the pool's values
        pool = sum(-(-(c + n) // bs) - c // bs for c, n in zip(cached, new)) + 3
        return dict(bytes=t * H * (kd + vd) * (e + 1) + 4 * t + pool * H * (bs * (kd + vd) * 5 + 16), flops=0)
    kv = [c + n for c, n in zip(cached, new)]
    if case["requests"] > 2 and not case["even"]:
        kv[1] = 0
    pairs = sum(sum(x - n + i + 1 for i in range(n)) for x, n in zip(kv, new) if x)
    t = sum(new)
    return dict(bytes=sum(kv) * H * (kd + vd) + sum(-(-x // bs) for x in kv) * (8 * H + 4) + t * case["heads"] * (kd + vd) * e,
                flops=2 * pairs * case["heads"] * (kd + vd))


# --------------------------------------------------------------------------
# the definitions in 64 bits
# --------------------------------------------------------------------------

def exact(case, seed):
    global own
    if case["op"] == "plan":
        return None  # whole numbers only
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    if case["op"] == "product":
        x = s["x"].double()
        r = torch.maximum(x.abs().max(dim=1).values, torch.tensor(FLOOR, dtype=torch.float64, device="cuda"))
        c = (127.0 * x / r.unsqueeze(1)).round()
        parts = []
        for a in range(0, case["n"], 4096):
            w = s["w"][a:a + 4096].double() * s["ws"][a:a + 4096].double().unsqueeze(1)
            parts.append(torch.einsum("tk,nk->tn", c, w))
        y = torch.cat(parts, dim=1) * (r / 127.0).unsqueeze(1)
        return y + s["res"].double() if s["res"] is not None else y
    bs, H, kd, vd = case["block"], case["kv_heads"], case["k_dim"], case["v_dim"]
    if case["op"] == "append":
        slots, runs = s["slots"].tolist(), {}
        for t, slot in enumerate(slots):
            if slot >= 0:
                runs.setdefault(slot // bs, []).append((slot % bs, t))
        out = {}
        for name, x, codes, ranges, dim in (("k", s["k"], s["kc"], s["kr"], kd), ("v", s["v"], s["vc"], s["vr"], vd)):
            c, r, x = codes.double(), ranges.double(), x.double()
            for b, members in runs.items():
                lo, ts = members[0][0], [t for _, t in members]
                y = x[ts[0]:ts[-1] + 1].transpose(0, 1)  # heads, tokens, dim
                top = y.abs().flatten(1).max(dim=1).values
                if lo > 0:
                    top = torch.maximum(top, r[b])
                top = top.clamp(min=FLOOR)
                new = (127.0 * y / top[:, None, None]).round()
                if name == "k":
                    flat = c[b].transpose(1, 2).reshape(H, bs, dim)
                else:
                    flat = c[b].transpose(2, 3).reshape(H, bs, dim)
                flat = flat.clone()
                if lo > 0:
                    flat[:, :lo] = (flat[:, :lo] * r[b][:, None, None] / top[:, None, None]).round()
                flat[:, lo:lo + len(ts)] = new
                c[b] = flat.reshape(H, bs, dim // 64, 64).transpose(1, 2) if name == "k" else flat.reshape(H, bs // 16, 16, dim).transpose(2, 3)
                r[b] = top
            out[name] = c * (r / 127.0)[:, :, None, None, None]
            out[name + "_range"] = r
        return out
    out = s["out"].double()
    heads = case["heads"]
    table, kv, start = s["table"].tolist(), s["kv_lens"].tolist(), s["q_start"].tolist()
    for b in range(case["requests"]):
        n, length = start[b + 1] - start[b], kv[b]
        if n == 0:
            continue
        if length == 0:
            out[start[b]:start[b + 1]] = 0.0
            continue
        pages = torch.tensor(table[b][:-(-length // bs)], device="cuda")
        live = torch.arange(length, device="cuda").unsqueeze(0) <= torch.arange(length - n, length, device="cuda").unsqueeze(1)
        for h in range(H):
            k = s["kc"][pages, h].double() * (s["kr"][pages, h].double() / 127.0)[:, None, None, None]
            v = s["vc"][pages, h].double() * (s["vr"][pages, h].double() / 127.0)[:, None, None, None]
            k = k.transpose(1, 2).reshape(-1, kd)[:length]
            v = v.transpose(2, 3).reshape(-1, vd)[:length]
            for j in range(h * (heads // H), (h + 1) * (heads // H)):
                a = torch.einsum("nd,ld->nl", s["q"][start[b]:start[b + 1], j].double(), k) * s["scale"]
                a = torch.where(live, a, torch.full_like(a, -math.inf))
                a = torch.exp(a - torch.logsumexp(a, dim=1, keepdim=True))
                out[start[b]:start[b + 1], j] = torch.einsum("nl,ld->nd", a, v)
    return out

"""Plain 64-bit restatements of the 8-bit attention operators (CPU tensors)."""
import math

import torch

FLOOR = 127.0 * 2.0 ** -64
D = torch.float64


def quantize(x, floor=None):
    """(codes, range) of the last dimension's rows in f64; `floor`: ranges at least that."""
    x = x.to(D)
    r = x.abs().amax(-1).clamp_min(FLOOR)
    if floor is not None:
        r = torch.maximum(r, floor)
    return torch.round(127.0 * x / r[..., None]), r


def product(x, codes, scales, residual=None):
    c, r = quantize(x)
    y = (c @ codes.to(D).T) * (r / 127.0)[:, None] * scales.to(D)[None]
    return y + residual.to(D) if residual is not None else y


def plan(cached, new, table, free, bs, capacity, num_blocks):
    """Lists in, dict of lists out; `table` (list of lists) is updated."""
    width = len(table[0]) if table else 0
    q_start, kv_lens, slots, positions = [0], [], [], []
    lacking = taken = 0
    for r, (c, n) in enumerate(zip(cached, new)):
        rows = max(n, 0)
        end = q_start[-1] + rows
        ok = c >= 0 and n >= 0 and c + n <= width * bs and end <= capacity
        need = -(-(c + n) // bs) - -(-c // bs) if ok else 0
        first, lacking = lacking, lacking + need
        ok = ok and (need == 0 or lacking <= len(free))
        if ok:
            have = -(-c // bs)
            for j in range(need):
                table[r][have + j] = free[first + j]
            taken = max(taken, lacking if need else 0)
        kv_lens.append(c + n if ok else 0)
        for i in range(rows):
            if q_start[-1] + i >= capacity:
                break
            pos = c + i if ok else -1
            b = table[r][pos // bs] if ok else -1
            slots.append(b * bs + pos % bs if 0 <= b < num_blocks else -1)
            positions.append(pos)
        q_start.append(end)
    slots += [-1] * (capacity - len(slots))
    positions += [-1] * (capacity - len(positions))
    return dict(q_start=q_start, kv_lens=kv_lens, slots=slots, positions=positions, taken=[taken], table=table)


# codes as [blocks, heads, tokens, dim]
def k_flat(k):
    nb, H, ch, bs, w = k.shape
    return k.permute(0, 1, 3, 2, 4).reshape(nb, H, bs, ch * w)


def v_flat(v):
    nb, H, g, dim, w = v.shape
    return v.permute(0, 1, 2, 4, 3).reshape(nb, H, g * w, dim)


def append(flat, ranges, x, slots, bs):
    """One of K, V: flat codes (f64, updated), ranges [blocks, heads] (f64, updated), x [T, heads, dim]."""
    runs = {}
    for t, s in enumerate(slots):
        if 0 <= s < flat.shape[0] * bs:
            runs.setdefault(s // bs, []).append((s % bs, t))
    for b, ts in runs.items():
        off = ts[0][0]
        y = x[[t for _, t in ts]].to(D).transpose(0, 1)            # heads, n, dim
        r = y.abs().flatten(1).amax(1).clamp_min(FLOOR)
        if off:
            r = torch.maximum(r, ranges[b])
            flat[b, :, :off] = torch.round(flat[b, :, :off] * ranges[b][:, None, None] / r[:, None, None])
        flat[b, :, off:off + len(ts)] = torch.round(127.0 * y / r[:, None, None])
        ranges[b] = r


def attend(q, kf, kr, vf, vr, q_start, kv_lens, table, bs, scale, out):
    """q [T, heads, dk]; flat codes and ranges; lists; `out` (f64) updated."""
    T, heads, _ = q.shape
    H = kf.shape[1]
    kval = kf.to(D) * (kr.to(D) / 127.0)[:, :, None, None]
    vval = vf.to(D) * (vr.to(D) / 127.0)[:, :, None, None]
    nb = kf.shape[0]
    for r in range(len(kv_lens)):
        n = q_start[r + 1] - q_start[r]
        for i in range(n):
            t = q_start[r] + i
            if t >= T:
                continue
            L = kv_lens[r] - n + i + 1
            toks = [j for j in range(max(L, 0)) if 0 <= table[r][j // bs] < nb]
            if not toks:
                out[t] = 0.0
                continue
            b = torch.tensor([table[r][j // bs] for j in toks])
            o = torch.tensor([j % bs for j in toks])
            for h in range(heads):
                kh = h // (heads // H)
                s = (kval[b, kh, o] @ q[t, h].to(D)) * scale
                p = torch.softmax(s, 0)
                out[t, h] = p @ vval[b, kh, o]
    return out


def attend_dense(q, kf, kr, vf, vr, q_start, kv_lens, table, bs, scale, out):
    """attend() for tables without holes, a request and head at a time."""
    heads, H = q.shape[1], kf.shape[1]
    for r, kv in enumerate(kv_lens):
        a, b = q_start[r], q_start[r + 1]
        if a == b:
            continue
        if kv == 0:
            out[a:b] = 0.0
            continue
        pages = torch.tensor(table[r][:-(-kv // bs)])
        hidden = torch.arange(kv)[None] > torch.arange(kv - (b - a), kv)[:, None]
        for h in range(heads):
            kh = h // (heads // H)
            k = (kf[pages, kh].to(D) * (kr[pages, kh].to(D) / 127.0)[:, None, None]).flatten(0, 1)[:kv]
            v = (vf[pages, kh].to(D) * (vr[pages, kh].to(D) / 127.0)[:, None, None]).flatten(0, 1)[:kv]
            s = (q[a:b, h].to(D) @ k.T * scale).masked_fill(hidden, -math.inf)
            out[a:b, h] = torch.softmax(s, 1) @ v
    return out


def attend_bound(dtype):
    """Largest |error| of an attention output relative to the largest |v| of its head.

    Scores: q in fp16 by a power of two a row, exact for bf16 (2^-28 of the row's
    largest), 2^-23 with two terms; the f32 sums of at most 24 products-of-16 steps
    and the softmax's own roundings stay below 2^-18 of |score| <= 2^4 here: 2^-14
    in p's exponent at worst, relative 2^-14.  P in fp16: 2^-12 relative a term
    (2^-22 with two).  The sums are convex, so the output is off by at most twice
    (numerator and denominator) that of the largest |v|, and half a step of the
    output type: bf16 2^-8.
    """
    p = 2.0 ** -12 if dtype == torch.bfloat16 else 2.0 ** -22
    s = 2.0 ** -14
    return 2 * (p + s) + (2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -23)


def new_scale(dim):
    return 1.0 / math.sqrt(dim)

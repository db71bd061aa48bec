"""The cache operators from their definitions, in 64 bits and one sequence at a time (torch on the
CPU, or on the device of the tensors): step, release, append and attention."""
import math

import torch

F64 = torch.float64


def step(ctx, new, tables, free, count, page, num_tokens):
    """(tables, seq_lens, cu, granted, slots, positions, count) of one step; lists and CPU tensors."""
    tables, count0 = tables.clone(), count
    batch, blocks = len(ctx), tables.shape[1]
    seq_lens, cu, granted, slots, positions = [], [0], [], [-1] * num_tokens, [-1] * num_tokens
    needed = taken = 0
    for b in range(batch):
        c, n = ctx[b], new[b]
        ok = c >= 0 and n >= 0
        n = n if ok else 0
        end = cu[-1] + n
        want, have = -(-(c + n) // page), -(-c // page)
        ok = ok and want <= blocks and end <= num_tokens
        need = want - have if ok else 0
        needed += need
        ok = ok and (need == 0 or needed <= count0)
        if ok:
            for j in range(need):
                tables[b, have + j] = free[count0 - 1 - (needed - need + j)]
            taken += need
            for i in range(n):
                pos = c + i
                slots[cu[-1] + i] = int(tables[b, pos // page]) * page + pos % page
                positions[cu[-1] + i] = pos
        seq_lens.append(c + n if ok else 0)
        granted.append(int(ok))
        cu.append(end)
    cu = [min(x, num_tokens) for x in cu]
    return tables, seq_lens, cu, granted, slots, positions, count0 - taken


def rotate(x, positions, cos, sin, interleaved):
    """x [tokens, heads, dim] in 64 bits, rounded to f32."""
    y = x.to(F64).clone()
    half = cos.shape[1]
    c, s = cos.to(F64)[positions][:, None], sin.to(F64)[positions][:, None]
    lo = torch.arange(half, device=x.device)
    a, b = (2 * lo, 2 * lo + 1) if interleaved else (lo, lo + half)
    u, w = y[..., a].clone(), y[..., b].clone()
    y[..., a], y[..., b] = u * c - w * s, u * s + w * c
    return y.float()


def block_scale(x, kind):
    """The scale of one (page, head)'s new values x (f32)."""
    amax = x.abs().max().item() if x.numel() else 0.0
    if not torch.isfinite(x).all():
        return math.nan
    if amax == 0:
        return 0.0
    if kind == "int8":
        return max(torch.tensor(amax / 127, dtype=F64).float().item(), 2.0 ** -126)
    m, e = math.frexp(amax)
    return 2.0 ** max(e - 8 if m > 0.875 else e - 9, -126)


def codes(x, scale, kind):
    """x (64 bits) as codes under scale, as their values in 64 bits."""
    if not scale > 0:
        return torch.zeros_like(x)
    q = x / scale
    if kind == "int8":
        return q.round().clamp(-127, 127)
    return q.float().to(torch.float8_e4m3fn).to(F64)


def append(k_codes, v_codes, k_scales, v_scales, kind, k, v, slots, page):
    """Codes (as 64-bit values, k [pages, heads, page, dim], v [pages, heads, dim, page]) and scales
    after appending k and v (f32 [tokens, heads, dim], k rotated already) to slots."""
    k_codes, v_codes, k_scales, v_scales = (t.clone() for t in (k_codes, v_codes, k_scales, v_scales))
    t = 0
    while t < len(slots):
        if slots[t] < 0:
            t += 1
            continue
        pg, o, m = slots[t] // page, slots[t] % page, 1
        while t + m < len(slots) and slots[t + m] == slots[t] + m and slots[t + m] // page == pg:
            m += 1
        for store, scales, x, is_v in ((k_codes, k_scales, k, False), (v_codes, v_scales, v, True)):
            for h in range(x.shape[1]):
                rows = x[t: t + m, h]
                was = scales[pg, h].item() if o else 0.0
                fresh = block_scale(rows, kind)
                now = math.nan if math.isnan(was) or math.isnan(fresh) else max(was, fresh)
                block = store[pg, h].t() if is_v else store[pg, h]  # [page, dim]
                if now > was > 0:
                    block[:o] = codes(block[:o] * was, now, kind)
                block[o: o + m] = codes(rows.to(F64), now, kind)
                scales[pg, h] = now
        t += m
    return k_codes, v_codes, k_scales, v_scales


def attention(q, k_codes, v_codes, k_scales, v_scales, tables, seq_lens, cu, scale, causal=True, window=0):
    """(out, sum_j p_j |v_j|, largest |v|, largest sum_d |q_d k_d| scale) in 64 bits, over codes given as
    values; the largest |v| is over the keys that a row's sequence shows to any of its rows.  Rows no
    sequence owns are zero."""
    page, dev = k_codes.shape[2], q.device
    heads, kv = q.shape[1], k_codes.shape[1]
    out = torch.zeros(q.shape, dtype=F64, device=dev)
    mag, most = torch.zeros_like(out), torch.zeros_like(out)
    reach = 0.0
    for b in range(len(seq_lens)):
        t0, t1, n = cu[b], cu[b + 1], seq_lens[b]
        if t1 <= t0 or n <= 0:
            continue
        blocks = tables[b, : -(-n // page)].long()
        there = ((blocks >= 0) & (blocks < k_codes.shape[0])).repeat_interleave(page)[:n]
        at = blocks.clamp(0, k_codes.shape[0] - 1)
        for h in range(kv):
            g = heads // kv
            ks = (k_codes[at, h].to(F64) * k_scales[at, h].to(F64)[:, None, None]).reshape(-1, q.shape[2])[:n]
            vs = (v_codes[at, h].to(F64) * v_scales[at, h].to(F64)[:, None, None]).transpose(1, 2).reshape(-1, q.shape[2])[:n]
            rows = q[t0:t1, h * g:(h + 1) * g].to(F64)
            s = rows @ ks.t() * scale
            seen = there[None].expand(t1 - t0, n)
            if causal:
                pos = n - (t1 - t0) + torch.arange(t1 - t0, device=dev)[:, None]
                j = torch.arange(n, device=dev)
                seen = seen & (j <= pos)
                if window:
                    seen = seen & (j > pos - window)
            s = s.masked_fill(~seen[:, None], -math.inf)
            top = s.amax(-1, keepdim=True)
            w = (s - torch.where(top == -math.inf, 0.0, top)).exp()
            w = torch.where(seen[:, None], w, 0.0)
            total = w.sum(-1, keepdim=True)
            w = w / torch.where(total == 0, 1.0, total)
            vz = torch.where(seen.any(0)[:, None], vs, 0.0)
            out[t0:t1, h * g:(h + 1) * g] = w @ vz
            mag[t0:t1, h * g:(h + 1) * g] = w @ vz.abs()
            most[t0:t1, h * g:(h + 1) * g] = torch.nan_to_num(vz).abs().max()
            big = (rows.abs() @ torch.where(seen.any(0)[:, None], ks, 0.0).abs().t()) * abs(scale)
            reach = max(reach, torch.nan_to_num(big).max().item())
    return out, mag, most, reach


def attention_bound(dtype, mag, most, out, reach, keys):
    """How far an output may be from the 64-bit one, element by element.

    f32: a logit is a sum of dim products whose operands are held to 2^-22 of the row's largest and
    whose running sum is rounded at most 20 times, so it is off by (2^-22 + 20 * 2^-24) sum |q k| scale;
    a weight by twice that (its own logit and the sum's) and the exponential's few last bits (16 * 2^-24);
    the weighted sum over the keys is rounded once per 16 keys and per join, 2^-24 each.  16-bit types:
    the weights are rounded to f16 (half a step: 2^-11) and the result to its type.

    All types: a weight goes into the product as f16 parts of 2^9 w s / r, where w is relative to a base
    that the row's largest logit is at or up to 6 above (so the weights' sum is at least 1 and w at most
    2^6), s its page's scale and r the power of two next above the largest scale so far.  The parts are
    off by half the smallest f16 step, 2^-25, whatever the weight's size: 2^-34 r |code| of the result for
    each key, and r |code| < 2 s_max |code|_max.  s_max |code|_max is at most 127 (448 for e4m3) s_max, which
    the tests' blocks of random codes reach to within a factor of 2: 2^-34 * 4 * the largest |v|, for each key."""
    rel = 2 * (2.0 ** -22 + 20 * 2.0 ** -24) * reach + (16 + keys / 16 + 64) * 2.0 ** -24
    step_half = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}[dtype]
    if dtype != torch.float32:
        rel += 2.0 ** -11
    tiny = {torch.float32: 0.0, torch.float16: 2.0 ** -25, torch.bfloat16: 0.0}[dtype]
    return rel * mag + keys * 2.0 ** -32 * most + step_half * out.abs() + tiny + 1e-37

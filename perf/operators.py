"""The cache operators' work: block tables, appends to an 8-bit key/value cache, attention over it.

Each case is one pass through one operator:

* ``step``    block tables, slot maps and positions of a serving step, from the requests' lengths
* ``append``  the step's keys and values, rotated, quantised and written into the cache's pages,
              and the queries rotated
* ``attend``  causal attention of the step's queries over the cache: prompts and single tokens
* ``cross``   attention of a decoder's queries over an encoder's cached states

Head layouts are the benchmark's (32 query heads, 8 key/value heads of 128) and generic ones; 16 sequences
are the reference server's slots and 512 tokens its prefill chunk.  Keys and values are normal with a few
channels several times as large, as a transformer's are; a sequence's lengths go by the case alone.
"""
from __future__ import annotations

import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
KINDS = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
THETA = 500000.0


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed() -> list[dict]:
    llama = {"heads": 32, "kv_heads": 8, "dim": 128}
    return [
        # a token step of the server's 16 slots: latency counts
        {"name": "step_decode16", "op": "step", "batch": 16, "active": 16, "new": 1, "ctx": 4096, "page": 64},
        # four prefill chunks among the slots, in small pages
        {"name": "step_chunks", "op": "step", "batch": 16, "active": 4, "new": 512, "ctx": 1500, "page": 16},
        # a large batch with prompts of several thousand tokens in it
        {"name": "step_batch600", "op": "step", "batch": 600, "active": 600, "new": 50, "ctx": 2000, "page": 32},
        # one token of one sequence: the smallest append
        {"name": "append_decode1", "op": "append", "kind": "int8", "dtype": "f32", "batch": 1, "active": 1, "new": 1,
         "ctx": 1000, "page": 64, "rot": 128, "pairs": "halves", **llama},
        # a batch of tokens; half the channels rotated, in neighbouring pairs
        {"name": "append_decode64_e4m3", "op": "append", "kind": "e4m3", "dtype": "bf16", "batch": 64, "active": 64, "new": 1,
         "ctx": 900, "page": 32, "rot": 64, "pairs": "neighbours", **llama},
        # four prefill chunks that continue partly filled pages
        {"name": "append_chunks", "op": "append", "kind": "int8", "dtype": "f32", "batch": 4, "active": 4, "new": 512,
         "ctx": 777, "page": 64, "rot": 128, "pairs": "halves", **llama},
        # one token of one sequence with a short context
        {"name": "attend_decode1", "op": "attend", "kind": "int8", "dtype": "f32", "batch": 1, "active": 1, "new": 1,
         "ctx": 1000, "page": 64, "window": 0, **llama},
        # a batch of tokens, ragged contexts
        {"name": "attend_decode32", "op": "attend", "kind": "int8", "dtype": "f32", "batch": 32, "active": 32, "new": 1,
         "ctx": 4096, "page": 64, "window": 0, **llama},
        # one token of one sequence with a very long context
        {"name": "attend_long", "op": "attend", "kind": "e4m3", "dtype": "f32", "batch": 1, "active": 1, "new": 1,
         "ctx": 131071, "page": 128, "window": 0, **llama},
        # four prefill chunks with their contexts
        {"name": "attend_chunks", "op": "attend", "kind": "int8", "dtype": "f32", "batch": 4, "active": 4, "new": 512,
         "ctx": 1500, "page": 64, "window": 0, **llama},
        # a long prompt in 16 bits with a sliding window of no round length
        {"name": "attend_prompt_bf16", "op": "attend", "kind": "e4m3", "dtype": "bf16", "batch": 1, "active": 1, "new": 8000,
         "ctx": 0, "page": 64, "window": 5000, **llama},
        # a decoder's prompts over an encoder's 1500 states
        {"name": "cross_encoder", "op": "cross", "kind": "int8", "dtype": "f16", "batch": 8, "active": 8, "new": 220,
         "ctx": 1500, "page": 16, "heads": 20, "kv_heads": 20, "dim": 64},
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    """A whole number in [lo, hi], spread over the logarithm."""
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng) -> dict:
    op = rng.choice(("step", "append", "append", "attend", "attend", "attend", "cross"))
    page = rng.choice((16, 32, 64, 128))
    if op == "step":
        batch = _log_int(rng, 1, 600)
        return {"op": op, "batch": batch, "active": rng.randint(1, batch), "new": _log_int(rng, 1, max(1, 16000 // batch)),
                "ctx": _log_int(rng, 1, 8192) - 1, "page": page}
    kv_heads = rng.choice((1, 2, 4, 5, 8))
    case = {"op": op, "kind": rng.choice(("int8", "e4m3")), "dtype": rng.choice(("f32", "f32", "f16", "bf16")), "page": page,
            "heads": kv_heads * rng.choice((1, 2, 3, 4, 7, 8)), "kv_heads": kv_heads, "dim": rng.choice((64, 96, 128, 128, 192, 256))}
    if op == "append":
        batch = _log_int(rng, 1, 64)
        rot = rng.choice((case["dim"], case["dim"], case["dim"] // 2))
        return {**case, "batch": batch, "active": rng.randint(1, batch), "new": _log_int(rng, 1, max(1, 2048 // batch)),
                "ctx": _log_int(rng, 1, 2048) - 1, "rot": rot, "pairs": rng.choice(("halves", "neighbours"))}
    if op == "cross":
        batch = _log_int(rng, 1, 8)
        return {**case, "batch": batch, "active": batch, "new": _log_int(rng, 1, 256), "ctx": _log_int(rng, 1, 1500)}
    window = rng.choice((0, 0, 0, _log_int(rng, 16, 2048)))
    if rng.random() < 0.6:  # single tokens, or a few at once
        batch = _log_int(rng, 1, 32)
        return {**case, "batch": batch, "active": rng.randint(1, batch), "new": rng.choice((1, 1, 1, 2, 5)),
                "ctx": _log_int(rng, 1, 32768 // batch) - 1, "window": window}
    batch = _log_int(rng, 1, 4)
    return {**case, "batch": batch, "active": batch, "new": _log_int(rng, 16, 1024), "ctx": _log_int(rng, 1, 1024) - 1, "window": window}


def _lengths(case) -> tuple[list[int], list[int]]:
    """(tokens in the cache before, new tokens) of each sequence; a row that is not active has no new ones."""
    ctx, new = [], []
    for i in range(case["batch"]):
        on = i * case["active"] // case["batch"] != (i - 1) * case["active"] // case["batch"] or case["active"] == case["batch"]
        c, n = case["ctx"], case["new"]
        ctx.append(c - (i * 7919) % (c // 2 + 1))
        new.append(n - (i * 4793) % (n // 2 + 1) if on else 0)
    return ctx, new


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _gen(seed: int) -> torch.Generator:
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _states(g, tokens: int, heads: int, dim: int, dtype) -> torch.Tensor:
    """Queries, keys or values [tokens, heads, dim]: normal, a few channels several times as large."""
    x = torch.randn(tokens, heads, dim, generator=g, device="cuda")
    loud = torch.rand(heads, dim, generator=g, device="cuda") < 0.03
    return (x * torch.where(loud, 6.0, 1.0)).to(dtype)


def _cache(g, case, pages: int) -> dict:
    """Codes and scales of a cache whose pages are all in use."""
    h, p, d = case["kv_heads"], case["page"], case["dim"]
    k = torch.randn(pages, h, p, d, generator=g, device="cuda")
    v = torch.randn(pages, h, d, p, generator=g, device="cuda")
    far = 0.03 if case["kind"] == "int8" else 2.0 ** -6
    vary = torch.rand(2, pages, h, generator=g, device="cuda")
    if case["kind"] == "int8":
        k, v = (k * 32).round().clamp_(-127, 127).to(torch.int8), (v * 32).round().clamp_(-127, 127).to(torch.int8)
        scales = far * (0.6 + 0.8 * vary)
    else:
        k, v = (k * 64).clamp_(-448, 448).to(torch.float8_e4m3fn), (v * 64).clamp_(-448, 448).to(torch.float8_e4m3fn)
        scales = torch.where(vary < 0.5, far, far / 2)
    return {"k": k, "v": v, "k_scales": scales[0].contiguous(), "v_scales": scales[1].contiguous()}


def _layout(case, g) -> dict:
    """A step's block tables and maps over randomly placed pages, and how many pages there are."""
    ctx, new = _lengths(case)
    b, p = case["batch"], case["page"]
    lens = list(ctx) if case["op"] == "cross" else [c + n for c, n in zip(ctx, new)]
    blocks = max(1, max(-(-n // p) for n in lens))
    used = sum(-(-n // p) for n in lens)
    order = torch.randperm(used, generator=g, device="cuda").to(torch.int32)
    starts = [sum(-(-n // p) for n in lens[:i]) for i in range(b)]
    i = torch.arange(blocks, device="cuda")
    at = torch.tensor(starts, device="cuda")[:, None] + i
    live = i < torch.tensor([-(-n // p) for n in lens], device="cuda")[:, None]
    tables = torch.where(live, order[at.clamp(max=used - 1)], -1).to(torch.int32) if used else torch.full((b, blocks), -1, dtype=torch.int32, device="cuda")
    rows = [(s, j) for s in range(b) for j in range(new[s])]
    seq = torch.tensor([r[0] for r in rows], device="cuda")
    at = torch.tensor([r[1] for r in rows], device="cuda")
    pos = at + torch.tensor(ctx, device="cuda")[seq]
    lay = {"tables": tables, "pages": used + 1, "seq": seq, "at": at, "positions": pos.to(torch.int32), "tokens": len(rows),
           "cu": torch.tensor([sum(new[:s]) for s in range(b + 1)], dtype=torch.int32, device="cuda"),
           "lens": torch.tensor(lens, dtype=torch.int32, device="cuda"), "longest": max(lens), "most": max(new)}
    if case["op"] != "cross":
        lay["slots"] = tables[seq, pos // p].to(torch.int64) * p + pos % p
    return lay


def prepare(case, seed) -> dict:
    g, op, p = _gen(seed), case["op"], case["page"]
    ctx, new = _lengths(case)
    s = {"case": case}
    if op == "step":
        blocks = max(1, max(-(-(c + n) // p) for c, n in zip(ctx, new)))
        held = sum(-(-c // p) for c in ctx)
        more = sum(-(-(c + n) // p) for c, n in zip(ctx, new)) - held
        order = torch.randperm(held + more + 7, generator=g, device="cuda").to(torch.int32)
        tables = torch.full((case["batch"], blocks), -1, dtype=torch.int32, device="cuda")
        have = torch.arange(blocks, device="cuda") < torch.tensor([-(-c // p) for c in ctx], device="cuda")[:, None]
        tables[have] = order[:held]
        s |= {"tables": tables, "free": order.roll(-held).contiguous(), "free_count": torch.tensor([more + 7], dtype=torch.int32, device="cuda"),
              "ctx": torch.tensor(ctx, dtype=torch.int32, device="cuda"), "new": torch.tensor(new, dtype=torch.int32, device="cuda"),
              "tokens": sum(new)}
        if own:  # the framework's handle on these tables: nothing is computed
            from lightbulb_amd import attention as at
            s["pages"] = at.PageTable.wrap(s["tables"], s["free"], s["free_count"], p)
        return s
    s |= _layout(case, g)
    t, dtype = s["tokens"], TYPES[case["dtype"]]
    cache = _cache(g, case, s["pages"])
    s |= {"q": _states(g, t, case["heads"], case["dim"], dtype), "cache": cache}
    if op == "append":
        s["k_new"] = _states(g, t, case["kv_heads"], case["dim"], dtype)
        s["v_new"] = _states(g, t, case["kv_heads"], case["dim"], dtype)
        half = case["rot"] // 2
        angle = torch.arange(s["longest"], dtype=torch.float64, device="cuda")[:, None] * THETA ** (
            -torch.arange(half, dtype=torch.float64, device="cuda") / half)
        s |= {"cos": angle.cos().float(), "sin": angle.sin().float()}
    else:
        s["scale"] = case["dim"] ** -0.5
    if own:  # the framework's handles on these tensors: nothing is computed
        from lightbulb_amd import attention as at
        s["kv"] = at.KvCache.wrap(cache["k"], cache["v"], cache["k_scales"], cache["v_scales"])
        s["step"] = at.Step(s["tables"], s["lens"], s["cu"], s.get("slots"), s["positions"] if op == "append" else None, page_size=p,
                            num_tokens=t, max_len=s["longest"], max_new=s["most"])
        if op == "append":
            s["rotary"] = at.Rotary(s["cos"], s["sin"], interleaved=case["pairs"] == "neighbours")
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(s):
    op = s["case"]["op"]
    if own:
        from lightbulb_amd import attention as at
        if op == "step":
            # a scheduler that asks whether a step fits takes no pages yet
            t = s["pages"].step(s["ctx"], s["new"], s["tokens"], commit=False)
            return [s["tables"], t.seq_lens, t.cu_new, t.granted, t.slots, t.positions, t.free_count]
        if op == "append":
            c = s["cache"]
            q = s["kv"].append(s["k_new"], s["v_new"], s["step"], rotary=s["rotary"], q=s["q"])
            return [q, c["k"], c["v"], c["k_scales"], c["v_scales"]]
        if op == "cross":
            return at.paged_attention(s["q"], s["kv"], s["step"], scale=s["scale"], causal=False)
        return at.paged_attention(s["q"], s["kv"], s["step"], scale=s["scale"], window=s["case"]["window"])
    return {"step": _plain_step, "append": _plain_append, "attend": _plain_attend, "cross": _plain_attend}[op](s)


def _plain_step(s):
    p, t, tables, free = s["case"]["page"], s["tokens"], s["tables"], s["free"]
    b, blocks = tables.shape
    ctx, new, count = s["ctx"].long(), s["new"].long(), s["free_count"].long()
    have, want = (ctx + p - 1) // p, (ctx + new + p - 1) // p
    ends = new.cumsum(0)
    fits = (want <= blocks) & (ends <= t)
    need = torch.where(fits, want - have, 0)
    cum = need.cumsum(0)
    granted = fits & ((need == 0) | (cum <= count))
    # the pages' places in the tables
    j = torch.arange(blocks, device=tables.device)
    fresh = granted[:, None] & (j >= have[:, None]) & (j < want[:, None])
    nth = (cum - need)[:, None] + j - have[:, None]
    tables.copy_(torch.where(fresh, free[(count - 1 - nth).clamp(0, free.numel() - 1)], tables))
    # the tokens' slots and positions
    cu = torch.cat([ends.new_zeros(1), ends])
    tok = torch.arange(t, device=tables.device)
    seq = torch.searchsorted(cu, tok, right=True) - 1
    pos = ctx[seq] + tok - cu[seq]
    slots = tables[seq, pos // p].long() * p + pos % p
    ok = granted[seq]
    return [tables, torch.where(granted, ctx + new, 0).int(), cu.int(), granted.int(), torch.where(ok, slots, -1),
            torch.where(ok, pos, -1).int(), (count - torch.where(granted, need, 0).sum()).int()]


def _plain_rotate(x, positions, cos, sin, rot: int, pairs: str):
    """Rotated in 64 bits, rounded to 32."""
    c, n = cos[positions.long()].double()[:, None], sin[positions.long()].double()[:, None]
    y = x.double()
    r = y[..., :rot]
    a, b = (r[..., : rot // 2], r[..., rot // 2:]) if pairs == "halves" else (r[..., 0::2], r[..., 1::2])
    u, w = a * c - b * n, b * c + a * n
    r = torch.cat([u, w], -1) if pairs == "halves" else torch.stack([u, w], -1).flatten(-2)
    return torch.cat([r, y[..., rot:]], -1).float()


def _plain_scale(amax, kind: str):
    """The scale of a block whose largest magnitude is amax."""
    if kind == "int8":
        s = (amax.double() / 127).float().clamp(min=2.0 ** -126)
    else:
        m, e = torch.frexp(amax)
        n = torch.where(m > 0.875, e - 8, e - 9).clamp(min=-126)
        s = torch.ldexp(torch.ones_like(amax), n)
    return torch.where(amax > 0, s, 0.0)


def _plain_codes(x, s, kind: str):
    """x / s as codes; zero where the scale is."""
    r = torch.where(s > 0, x.double() / torch.where(s > 0, s, 1.0).double(), 0.0)
    return r.round().clamp(-127, 127).to(torch.int8) if kind == "int8" else r.float().to(torch.float8_e4m3fn)


def _plain_append(s):
    case, c = s["case"], s["cache"]
    p, kind, t = case["page"], case["kind"], s["tokens"]
    q = _plain_rotate(s["q"], s["positions"], s["cos"], s["sin"], case["rot"], case["pairs"]).to(s["q"].dtype)
    k = _plain_rotate(s["k_new"], s["positions"], s["cos"], s["sin"], case["rot"], case["pairs"])
    # the runs of new tokens that share a page: at most cu[i+1] // p - cu[i] // p + 2 of them in sequence i
    b = case["batch"]
    cu, lens = s["cu"].long(), s["lens"].long()
    start = cu // p + 2 * torch.arange(b + 1, device=cu.device)
    x = torch.arange(t // p + 2 * b, device=cu.device)
    seq = (torch.searchsorted(start, x, right=True) - 1).clamp(max=b - 1)
    before = lens - (cu[1:] - cu[:-1])
    first = (before[seq] // p + x - start[seq]) * p  # the position at which the run's page begins
    live = (first < lens[seq]) & (cu[seq + 1] > cu[seq])
    page = torch.where(live, s["tables"][seq, (first // p).clamp(0, s["tables"].shape[1] - 1)].long(), s["pages"] - 1)
    place = first[:, None] + torch.arange(p, device=cu.device)  # the positions of the page's places
    fresh = live[:, None] & (place >= before[seq][:, None]) & (place < lens[seq][:, None])
    kept = live[:, None] & (place < before[seq][:, None])
    tok = (cu[seq][:, None] + place - before[seq][:, None]).clamp(0, t - 1)
    for name, new in (("k", k), ("v", s["v_new"].float())):
        codes, scales = c[name], c[name + "_scales"]
        block = new[tok].transpose(1, 2)  # [runs, heads, places, dim]
        is_new, is_old = fresh[:, None, :, None], kept[:, None, :, None]
        amax = torch.where(is_new, block.abs(), 0.0).amax((2, 3))
        old = codes.view(torch.int8)[page]
        old = (old if name == "k" else old.transpose(2, 3)).contiguous().view(codes.dtype)
        was = torch.where(is_old.any(2)[..., 0], scales[page], 0.0)
        now = torch.where(live[:, None], torch.maximum(was, _plain_scale(amax, kind)), scales[page])
        put = torch.where(is_new, _plain_codes(block, now[..., None, None], kind).view(torch.int8),
                          torch.where(is_old, _plain_codes(old.double() * was.double()[..., None, None], now[..., None, None], kind).view(torch.int8),
                                      old.view(torch.int8)))
        codes.view(torch.int8)[page] = put if name == "k" else put.transpose(2, 3)
        scales[page] = now
    return [q, c["k"], c["v"], c["k_scales"], c["v_scales"]]


def _plain_attend(s):
    case, c = s["case"], s["cache"]
    b, p, h, d = case["batch"], case["page"], case["kv_heads"], case["dim"]
    g, most = case["heads"] // h, s["most"]
    at = s["tables"].clamp(min=0).long()
    length = at.shape[1] * p
    k = c["k"].view(torch.int8)[at].view(c["k"].dtype).float() * c["k_scales"][at][..., None, None]  # [batch, blocks, heads, page, dim]
    v = c["v"].view(torch.int8)[at].view(c["v"].dtype).float() * c["v_scales"][at][..., None, None]
    k = k.transpose(1, 2).reshape(b, h, length, d)
    v = v.permute(0, 2, 1, 4, 3).reshape(b, h, length, d)
    q = torch.zeros(b, most, h * g, d, device=k.device)
    q[s["seq"], s["at"]] = s["q"].float()
    q = q.view(b, most, h, g, d).permute(0, 2, 3, 1, 4).reshape(b, h, g * most, d)
    scores = (q @ k.transpose(2, 3)).view(b, h, g, most, length) * s["scale"]
    j = torch.arange(length, device=k.device)
    lens = s["lens"].long()
    seen = (j < lens[:, None])[:, None].expand(b, most, length)
    if case["op"] == "attend":
        pos = (lens - (s["cu"][1:] - s["cu"][:-1]))[:, None] + torch.arange(most, device=k.device)
        seen = seen & (j <= pos[..., None])
        if case["window"]:
            seen = seen & (j > pos[..., None] - case["window"])
    scores = torch.where(seen[:, None, None], scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    w = (scores - torch.where(top > -math.inf, top, 0.0)).exp()
    total = w.sum(-1, keepdim=True)
    o = (w.view(b, h, g * most, length) @ v).view(b, h, g, most, d) / torch.where(total > 0, total, 1.0)
    return o.permute(0, 3, 1, 2, 4).reshape(b, most, h * g, d)[s["seq"], s["at"]].to(s["q"].dtype)


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    if case["op"] == "step":
        return None  # whole numbers
    s = prepare(case, seed)
    return _exact_append(case, s) if case["op"] == "append" else _exact_attention(case, s)


def _exact_turn(x, s, case):
    y = x.double().clone()
    half = case["rot"] // 2
    c, n = s["cos"].double()[s["positions"].long()], s["sin"].double()[s["positions"].long()]
    for i in range(half):
        a, b = (i, i + half) if case["pairs"] == "halves" else (2 * i, 2 * i + 1)
        u, w = x[..., a].double(), x[..., b].double()
        y[..., a] = u * c[:, i, None] - w * n[:, i, None]
        y[..., b] = u * n[:, i, None] + w * c[:, i, None]
    return y


def _exact_append(case, s):
    ctx, new = _lengths(case)
    p, kind = case["page"], case["kind"]
    q = _exact_turn(s["q"], s, case)
    turned = _exact_turn(s["k_new"], s, case).float()
    out = []
    for name, x in (("k", turned), ("v", s["v_new"].float())):
        codes = s["cache"][name].double()
        codes = codes if name == "k" else codes.transpose(2, 3).contiguous()
        scales = s["cache"][name + "_scales"].double()
        t = 0
        for b, (c, n) in enumerate(zip(ctx, new)):
            pos = c
            while pos < c + n:
                page, o = int(s["tables"][b, pos // p]), pos % p
                m = min(p - o, c + n - pos)
                rows = x[t: t + m].double().transpose(0, 1)  # [heads, tokens, dim]
                amax = rows.abs().amax((1, 2))
                if kind == "int8":
                    scale = (amax / 127).float().double()
                else:
                    scale = torch.exp2(torch.ceil(torch.log2(amax / 448)))
                was = scales[page] if o else torch.zeros_like(scale)
                scale = torch.maximum(scale, was)
                both = torch.cat([codes[page][:, :o] * was[:, None, None], rows], 1) / scale[:, None, None]
                codes[page][:, : o + m] = both.round() if kind == "int8" else both.to(torch.float8_e4m3fn).double()
                scales[page] = scale
                pos, t = pos + m, t + m
        out.append((codes if name == "k" else codes.transpose(2, 3).contiguous(), scales))
    (k, ks), (v, vs) = out
    return [q, None if kind == "int8" else k, None if kind == "int8" else v, ks, vs]


def _exact_attention(case, s):
    ctx, new = _lengths(case)
    p, h, g = case["page"], case["kv_heads"], case["heads"] // case["kv_heads"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    codes = {name: s["cache"][name].double() for name in ("k", "v")}
    t = 0
    for b, (c, n) in enumerate(zip(ctx, new)):
        length = c if case["op"] == "cross" else c + n
        if n and length:
            pages = s["tables"][b, : -(-length // p)].long()
            for i in range(h):
                k = (codes["k"][pages, i] * s["cache"]["k_scales"][pages, i].double()[:, None, None]).reshape(-1, case["dim"])[:length]
                v = (codes["v"][pages, i] * s["cache"]["v_scales"][pages, i].double()[:, None, None]).transpose(1, 2).reshape(-1, case["dim"])[:length]
                rows = s["q"][t: t + n, i * g: (i + 1) * g].double()
                e = torch.einsum("tgd,ld->tgl", rows, k) * s["scale"]
                if case["op"] == "attend":
                    at = c + torch.arange(n, device="cuda")[:, None, None]
                    j = torch.arange(length, device="cuda")
                    e = e.masked_fill(j > at, -math.inf)
                    if case["window"]:
                        e = e.masked_fill(j <= at - case["window"], -math.inf)
                out[t: t + n, i * g: (i + 1) * g] = torch.softmax(e, -1) @ v
        t += n
    return out


# ---------------------------------------------------------------------------
# the work that a pass cannot do without
# ---------------------------------------------------------------------------
def work(case) -> dict:
    ctx, new = _lengths(case)
    t, p = sum(new), case["page"]
    if case["op"] == "step":
        more = sum(-(-(c + n) // p) - -(-c // p) for c, n in zip(ctx, new))
        held = sum(len({j // p for j in (c, c + n - 1)} if n else ()) for c, n in zip(ctx, new))
        # lengths, free pages and table entries read; table entries, slots, positions and lengths written
        return {"bytes": 8 * len(ctx) + 4 * held + 8 * more + 12 * t + 12 * len(ctx), "flops": 0}
    size = TYPES[case["dtype"]].itemsize
    h, kv, d = case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "append":
        # q, k, v read, q and the codes written, the angles' rows, slots and positions read
        return {"bytes": t * (2 * h * d * size + 2 * kv * d * size + 2 * kv * d + 4 * case["rot"] + 12), "flops": t * (3 * case["rot"] * (h + kv) + 4 * kv * d)}
    pairs = held = 0
    for c, n in zip(ctx, new):
        if case["op"] == "cross":
            pairs, held = pairs + n * c, held + (c if n else 0)
        else:
            w = case["window"] or c + n
            pairs += sum(min(w, c + i + 1) for i in range(n))
            held += min(c + n, w + n - 1) if n else 0
    return {"bytes": held * kv * 2 * (d + 4 / p) + 2 * t * h * d * size, "flops": 4 * pairs * h * d}

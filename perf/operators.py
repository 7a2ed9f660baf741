"""Cases of the paged key-value cache: the plan of a step (block tables and slot maps), the append of
new rows, the read-back of stored rows, and the attention of one new token over the pages.

A cache holds, for every layer, ``n_pages`` pages of ``page_size`` positions, laid out
``[layer][page][kv_head][slot][head_dim]``: fp16, or Q4_0 blocks of 32 along head_dim as a nibble
plane (byte j of a block: element j low, element j + 16 high) and an fp16 scale plane.  A request's
position p lives in page ``table[request][p // page_size]`` at slot ``p % page_size``.

``own = False`` computes the operators from elementary torch operations in 32 bits, ``own = True``
through bmo_jetson_b200.paged.
"""
import math
import random

import numpy as np
import torch

own = False

ACT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
THETA = 10000.0
# drawn cases stay below the largest listed one's traffic (attn_64_sessions_f16)
MAX_BYTES = 1.4e9


# --------------------------------------------------------------------------- cases

def listed():
    return [
        # one frame of 64 sessions: one position each, one in sixteen starts a page
        {"name": "plan_64_sessions", "op": "plan", "requests": 64, "page_size": 16, "min_len": 0, "max_len": 2999,
         "min_new": 1, "max_new": 1, "end_every": 0, "window": 0, "shape": 1},
        # sessions joining with a history of odd length while others end, sliding window of 500 positions
        {"name": "plan_histories", "op": "plan", "requests": 61, "page_size": 24, "min_len": 0, "max_len": 1500,
         "min_new": 0, "max_new": 2999, "end_every": 7, "window": 500, "shape": 2},
        # one session's frame: the smallest call, all latency
        {"name": "append_1_session_f16", "op": "append", "tokens": 1, "heads": 32, "kv_heads": 32, "head_dim": 128,
         "page_size": 16, "kv": "f16", "act": "f32", "rope": True, "shape": 3},
        # a batched frame's rows, straight from the QKV projection's output, into a Q4_0 cache
        {"name": "append_64_sessions_q4", "op": "append", "tokens": 64, "heads": 32, "kv_heads": 32, "head_dim": 128,
         "page_size": 16, "kv": "q4_0", "act": "f32", "rope": True, "shape": 4},
        # eight histories imported at once, fewer key heads than query heads, odd count
        {"name": "append_histories_bf16", "op": "append", "tokens": 23993, "heads": 32, "kv_heads": 8,
         "head_dim": 128, "page_size": 64, "kv": "f16", "act": "bf16", "rope": True, "shape": 5},
        # a few rows looked at
        {"name": "read_7_rows_f16", "op": "read", "tokens": 7, "kv_heads": 32, "head_dim": 128, "page_size": 16,
         "kv": "f16", "act": "f32", "shape": 6},
        # a whole session taken out of a Q4_0 cache to move it
        {"name": "read_session_q4", "op": "read", "tokens": 2999, "kv_heads": 32, "head_dim": 128, "page_size": 16,
         "kv": "q4_0", "act": "f32", "shape": 7},
        # batch 1 over the 512 positions of the temporal transformer's window
        {"name": "attn_1_session_512", "op": "attn", "rows": 1, "heads": 32, "kv_heads": 32, "head_dim": 128,
         "page_size": 16, "kv": "f16", "act": "f32", "min_len": 701, "max_len": 701, "window": 512, "shape": 8},
        # short and empty sessions, pages of an odd size, eight query heads to a key head, heads of 64
        {"name": "attn_ragged_short", "op": "attn", "rows": 37, "heads": 16, "kv_heads": 2, "head_dim": 64,
         "page_size": 24, "kv": "f16", "act": "f16", "min_len": 0, "max_len": 300, "window": 0, "shape": 9},
        # 64 sessions at positions uniform in [0, 3000), Q4_0 cache, window of 512
        {"name": "attn_64_sessions_q4", "op": "attn", "rows": 64, "heads": 32, "kv_heads": 32, "head_dim": 128,
         "page_size": 16, "kv": "q4_0", "act": "f32", "min_len": 1, "max_len": 3000, "window": 512, "shape": 10},
        # the same sessions over their whole history in fp16: the largest
        {"name": "attn_64_sessions_f16", "op": "attn", "rows": 64, "heads": 32, "kv_heads": 32, "head_dim": 128,
         "page_size": 16, "kv": "f16", "act": "f32", "min_len": 1, "max_len": 3000, "window": 0, "shape": 11},
        # one long context, four query heads to a key head: the work is split over the length
        {"name": "attn_long_context_gqa", "op": "attn", "rows": 1, "heads": 32, "kv_heads": 8, "head_dim": 128,
         "page_size": 64, "kv": "f16", "act": "bf16", "min_len": 131071, "max_len": 131071, "window": 0, "shape": 12},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["plan", "append", "read", "attn", "attn", "attn"])
    page = rng.choice([8, 16, 16, 24, 32, 64, 128])
    shape = rng.randrange(1 << 30)
    if op == "plan":
        prompt = rng.random() < 0.5
        return {"op": op, "requests": _log_int(rng, 1, 400), "page_size": page, "min_len": 0,
                "max_len": _log_int(rng, 10, 3000), "min_new": 0 if prompt else 1,
                "max_new": _log_int(rng, 2, 3000) if prompt else 1, "end_every": rng.choice([0, 3, 7]),
                "window": rng.choice([0, 0, 500, 512, 1000]), "shape": shape}
    head_dim = rng.choice([64, 128, 128])
    kv = rng.choice(["f16", "q4_0"])
    act = rng.choice(["f32", "f32", "f16", "bf16"])
    kv_heads = rng.choice([1, 2, 4, 8, 16, 32])
    heads = kv_heads * rng.choice([1, 2, 4, 8] if kv_heads <= 4 else [1, 2, 4] if kv_heads <= 8 else [1])
    case = {"op": op, "kv_heads": kv_heads, "head_dim": head_dim, "page_size": page, "kv": kv, "act": act,
            "shape": shape}
    if op != "attn":
        case["tokens"] = _log_int(rng, 1, 24000)
        if op == "append":
            case |= {"heads": heads, "rope": rng.random() < 0.8}
        while work(case)["bytes"] > 3e8:
            case["tokens"] = max(1, case["tokens"] // 2 - 1)
        return case
    longest = _log_int(rng, 1, 131072)
    case |= {"heads": heads, "rows": _log_int(rng, 1, 64), "max_len": longest,
             "min_len": rng.choice([0, 1, longest // 2, longest]),
             "window": rng.choice([0, 0, 500, 512, 1000])}
    # the plain form gathers every row at the longest row's length
    def padded(c):
        return c["rows"] * min(c["max_len"], c["window"] or c["max_len"]) * c["kv_heads"] * c["head_dim"]

    while padded(case) > MAX_BYTES / 4 or not sum(_lens(case)):
        if padded(case) > MAX_BYTES / 4:
            case["max_len"] = max(1, case["max_len"] // 2 + 1)
            case["rows"] = max(1, case["rows"] - case["rows"] // 8)
        else:
            case["max_len"] = case["min_len"] = 1
        case["min_len"] = min(case["min_len"], case["max_len"])
    return case


def _lens(case):
    """The lengths of a case's requests: part of its shape, the same for every seed."""
    r = random.Random(case["shape"])
    return [r.randint(case["min_len"], case["max_len"]) for _ in range(case.get("requests") or case["rows"])]


def _new(case):
    """The new positions of a case's requests (-1: the request ends)."""
    r = random.Random(case["shape"] + 1)
    n = [r.randint(case["min_new"], case["max_new"]) for _ in range(case["requests"])]
    e = case["end_every"]
    return [-1 if e and i % e == e - 1 else x for i, x in enumerate(n)]


def _cdiv(a, b):
    return -(-a // b)


def _row_bytes(case):
    """Bytes of one position's keys of one head in the cache."""
    return case["head_dim"] * (2 if case["kv"] == "f16" else 18 / 32)


def work(case):
    ps = case["page_size"]
    if case["op"] == "plan":
        lens, new, w = _lens(case), _new(case), case["window"]
        first = lambda n: max(0, n - w) // ps if w else 0  # noqa: E731
        moved = sum(_cdiv(a, ps) - first(a) if n < 0 else _cdiv(a + n, ps) - _cdiv(a, ps) + first(a + n) - first(a)
                    for a, n in zip(lens, new))
        # lens and n_new in, lens and offsets out; a page id read and written; slot, position, request of a token
        return {"bytes": 16 * len(lens) + 8 * moved + 12 * sum(max(0, n) for n in new) + 32, "flops": 0}
    size = ACT[case["act"]].itemsize
    if case["op"] == "attn":
        n = sum(min(a, case["window"] or a) for a in _lens(case))
        dim = case["heads"] * case["head_dim"]
        return {"bytes": 2 * n * case["kv_heads"] * _row_bytes(case) + case["rows"] * (2 * dim * size + 4 * case["heads"])
                + 4 * _cdiv(n, ps), "flops": 4 * n * dim}
    t, kv = case["tokens"], case["kv_heads"] * case["head_dim"]
    stored = 2 * case["kv_heads"] * _row_bytes(case)
    back = stored + 2 * kv * (2 if case["kv"] == "f16" else 4)
    if case["op"] == "read":
        return {"bytes": t * (4 + stored + 2 * kv * size), "flops": 0}
    # the pass stores the rows and reads them back as the values they stand for
    q = case["heads"] * case["head_dim"] * size if case["rope"] else 0
    return {"bytes": t * (12 + 2 * kv * size + 2 * q + stored + back), "flops": t * 3 * (kv + q // size)}


# --------------------------------------------------------------------------- inputs

def _pack(x):
    """Q4_0 of the last axis: (nibble bytes, fp16 scales)."""
    b = x.reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    lane = torch.arange(32, device=x.device)
    first = torch.where(b.abs() == b.abs().amax(-1, keepdim=True), lane, 32).amin(-1, keepdim=True)
    d = torch.gather(b, -1, first) / -8.0
    inv = torch.where(d != 0, 1.0 / d, torch.zeros_like(d))
    n = (b * inv + 8.5).trunc().clamp(max=15).to(torch.uint8)
    bytes_ = n[..., :16] | (n[..., 16:] << 4)
    return bytes_.reshape(*x.shape[:-1], x.shape[-1] // 2), d[..., 0].half()


def _pool(case, n_pages, gen):
    """A cache of one layer whose pages hold keys and values of N(0, 1)."""
    shape = (1, n_pages, case["kv_heads"], case["page_size"], case["head_dim"])
    f16 = case["kv"] == "f16"
    s = {}
    for name in ("k", "v"):
        s[name] = torch.empty(shape if f16 else shape[:-1] + (shape[-1] // 2,), dtype=torch.float16 if f16 else torch.uint8,
                              device="cuda")
        s[name + "_scale"] = None if f16 else torch.empty(shape[:-1] + (shape[-1] // 32,), dtype=torch.float16,
                                                          device="cuda")
        per = max(1, (1 << 26) // math.prod(shape[2:]))
        for i in range(0, n_pages, per):
            x = torch.randn((min(per, n_pages - i),) + shape[2:], device="cuda", generator=gen)
            if f16:
                s[name][0, i:i + per] = x.half()
            else:
                s[name][0, i:i + per], s[name + "_scale"][0, i:i + per] = _pack(x)
    return s


def _gen(seed):
    return torch.Generator("cuda").manual_seed(seed)


def _int(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _book(case, lens, n_pages, max_blocks, gen):
    """The block table of requests of these lengths on pages in random order, and the ring of free pages."""
    w, ps = case.get("window", 0), case["page_size"]
    order = torch.randperm(n_pages, generator=gen, device="cuda").int().cpu()
    table = torch.full((len(lens), max_blocks), -1, dtype=torch.int32)
    used = 0
    for r, n in enumerate(lens):
        first, last = (max(0, n - w) // ps if w else 0), _cdiv(n, ps)
        table[r, first:last] = order[used:used + last - first]
        used += last - first
    free = torch.cat([order[used:], order[:used]])  # the entries past the count are stale
    return {"table": table.cuda(), "lens": _int(lens), "free": free.cuda(), "book": _int([0, n_pages - used, 0, 0])}


def prepare(case, seed):
    gen = _gen(seed)
    ps = case["page_size"]
    s = {"case": case, "window": case.get("window", 0), "page_size": ps}
    if case["op"] == "plan":
        lens, new, w = _lens(case), _new(case), case["window"]
        need = sum(_cdiv(n + max(0, m), ps) + 1 for n, m in zip(lens, new))
        blocks = max(_cdiv(n + max(0, m), ps) for n, m in zip(lens, new)) + 1
        s |= _book(case, lens, 2 * need + 5, blocks, gen)
        tokens = sum(max(0, m) for m in new)
        tokens += tokens // 8 + 3  # room for more than this step's
        s["n_new"] = _int(new)
        s |= {n: torch.empty(tokens, dtype=torch.int32, device="cuda") for n in ("slot", "pos", "req")}
        s |= {"offsets": torch.empty(len(lens) + 1, dtype=torch.int32, device="cuda"),
              "lens_out": torch.empty_like(s["lens"]), "book_out": torch.empty_like(s["book"])}
        return s
    act = ACT[case["act"]]
    if case["op"] == "attn":
        lens, w = _lens(case), case["window"]
        held = sum(_cdiv(n, ps) - (max(0, n - w) // ps if w else 0) for n in lens)
        s |= _pool(case, held + 3, gen)
        s |= _book(case, lens, held + 3, _cdiv(max(1, case["max_len"]), ps), gen)
        shape = (case["rows"], case["heads"], case["head_dim"])
        s["q"] = torch.randn(shape, device="cuda", generator=gen).to(act)
        s["out"] = torch.empty_like(s["q"])
        s["lse"] = torch.empty(shape[:2], device="cuda")
        return s
    t = case["tokens"]
    pages = _cdiv(t, ps) + 3
    s |= _pool(case, pages, gen)
    s |= _book(case, [], pages, 1, gen)
    s["table"], s["lens"] = _int([[-1]]), _int([0])
    s["slot"] = torch.randperm(pages * ps, generator=gen, device="cuda")[:t].int()
    # rows stored are read back in the type that holds them: fp16, or Q4_0's values as floats
    back = act if case["op"] == "read" else torch.float16 if case["kv"] == "f16" else torch.float32
    s |= {n: torch.empty((t, case["kv_heads"], case["head_dim"]), dtype=back, device="cuda") for n in ("k_out", "v_out")}
    if case["op"] == "append":
        h, kv, hd = case["heads"], case["kv_heads"], case["head_dim"]
        # q, k and v are slices of the projection's output
        qkv = torch.randn((t, (h + 2 * kv) * hd), device="cuda", generator=gen).to(act)
        s["q"] = qkv[:, :h * hd].unflatten(1, (h, hd))
        s["k_new"] = qkv[:, h * hd:(h + kv) * hd].unflatten(1, (kv, hd))
        s["v_new"] = qkv[:, (h + kv) * hd:].unflatten(1, (kv, hd))
        s["pos"] = torch.randint(0, 3000, (t,), generator=gen, device="cuda").int()
        s["q_out"] = torch.empty((t, h, hd), dtype=act, device="cuda")
    return s


# --------------------------------------------------------------------------- plain forms

def _plain_plan(s):
    lens, new, ps, w = s["lens"].long(), s["n_new"].long(), s["page_size"], s["window"]
    blocks, n_pages, n_req = s["table"].shape[1], s["free"].numel(), lens.numel()
    head, count = s["book"][0].long(), s["book"][1].long()
    first = lambda n: torch.clamp(n - w, min=0) // ps if w else torch.zeros_like(n)  # noqa: E731
    ends, add = new < 0, new.clamp(min=0)
    after = torch.where(ends, 0, lens + add)
    have = (lens + ps - 1) // ps
    take = torch.where(ends, 0, (after + ps - 1) // ps - have)
    give = torch.where(ends, have, first(after)) - first(lens)
    ok = (take.sum() <= count) & ((after + ps - 1) // ps <= blocks).all() & (add.sum() <= s["slot"].numel())
    take, give, add = (torch.where(ok, x, 0) for x in (take, give, add))
    take_end, give_end, add_end = take.cumsum(0), give.cumsum(0), add.cumsum(0)
    cells = torch.cat([s["table"].reshape(-1), s["table"].new_zeros(1)])
    ring = torch.cat([s["free"], s["free"].new_zeros(1)])

    def items(ends_, starts, n):  # (item number, request, number within the request, whether there is such an item)
        i = torch.arange(n, device="cuda")
        r = torch.searchsorted(ends_, i, right=True).clamp(max=n_req - 1)
        return i, r, i - starts[r], i < ends_[-1]

    i, r, j, real = items(take_end, take_end - take, n_pages)
    cells[torch.where(real, r * blocks + have[r] + j, n_req * blocks)] = ring[(head + i) % n_pages]
    i, r, j, real = items(give_end, give_end - give, n_pages)
    page = cells[torch.where(real, r * blocks + first(lens)[r] + j, n_req * blocks)]
    ring[torch.where(real, (head + count + i) % n_pages, n_pages)] = page
    i, r, j, real = items(add_end, add_end - add, s["slot"].numel())
    pos = lens[r] + j
    slot = cells[torch.where(real, r * blocks + pos // ps, n_req * blocks)].long() * ps + pos % ps
    minus = torch.full_like(i, -1)
    book = torch.stack([(head + take.sum()) % n_pages, count - take.sum() + give.sum(), torch.zeros_like(head), add.sum()])
    return {"table": cells[:-1].view_as(s["table"]), "free": ring[:-1], "lens": torch.where(ok, after, lens).int(),
            "book": book.int(), "slot": torch.where(real, slot, minus).int(), "pos": torch.where(real, pos, minus).int(),
            "req": torch.where(real, r, minus).int(),
            "offsets": torch.cat([torch.zeros(1, dtype=torch.int64, device="cuda"), add_end]).int()}


def _plain_rope(x, pos, dim):
    """Pairs (2i, 2i + 1) turned by pos * theta^(-2i / dim); the angle in 32 bits, as the decode step has it."""
    e = torch.arange(0, dim, 2, device="cuda", dtype=torch.float32) / float(dim)
    freq = torch.pow(torch.tensor(THETA, dtype=torch.float64, device="cuda"), -e.double()).float()
    angle = (pos.float()[:, None] * freq).double()
    c, sn = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    re, im = x[..., 0::2], x[..., 1::2]
    return torch.stack([re * c - im * sn, re * sn + im * c], -1).flatten(-2)


def _unpack(nibbles, scale):
    b = nibbles.reshape(*nibbles.shape[:-1], nibbles.shape[-1] // 16, 16)
    n = torch.cat([b & 15, b >> 4], -1).float() - 8.0
    return (n * scale.float()[..., None]).flatten(-2)


def _rows(s, name, page, slot):
    """Rows [..., kv_head, head_dim] of layer 0 in 32 bits, by page and slot."""
    x = s[name][0][page, :, slot]
    return x.float() if s[name + "_scale"] is None else _unpack(x, s[name + "_scale"][0][page, :, slot])


def _plain_read(s):
    page, slot = s["slot"].long() // s["page_size"], s["slot"].long() % s["page_size"]
    return {n: _rows(s, n, page, slot).to(s[n + "_out"].dtype) for n in ("k", "v")}


def _plain_append(s):
    page, slot = s["slot"].long() // s["page_size"], s["slot"].long() % s["page_size"]
    q, k, v = s["q"].float(), s["k_new"].float(), s["v_new"].float()
    if s["case"]["rope"]:
        q, k = _plain_rope(q, s["pos"], q.shape[-1]), _plain_rope(k, s["pos"], k.shape[-1])
    if s["k_scale"] is None:
        s["k"][0][page, :, slot], s["v"][0][page, :, slot] = k.half(), v.half()
    else:
        s["k"][0][page, :, slot], s["k_scale"][0][page, :, slot] = _pack(k)
        s["v"][0][page, :, slot], s["v_scale"][0][page, :, slot] = _pack(v)
    return _plain_read(s) | ({"q": q.to(s["q"].dtype)} if s["case"]["rope"] else {})


def _plain_attn(s):
    lens, ps, w, case = s["lens"].long(), s["page_size"], s["window"], s["case"]
    start = torch.clamp(lens - w, min=0) if w else torch.zeros_like(lens)
    j = start[:, None] + torch.arange(max(1, min(case["max_len"], w or case["max_len"])), device="cuda")
    real = j < lens[:, None]
    page = torch.gather(s["table"].long(), 1, (j // ps).clamp(max=s["table"].shape[1] - 1))
    page = torch.where(real, page, 0)
    rows, kv, hd = case["rows"], case["kv_heads"], case["head_dim"]
    q = s["q"].float().view(rows, kv, -1, hd)
    k = _rows(s, "k", page, j % ps).permute(0, 2, 3, 1)  # [row][kv head][head_dim][position]
    score = torch.matmul(q, k) / math.sqrt(hd)
    del k
    score = torch.where(real[:, None, None], score, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    v = _rows(s, "v", page, j % ps).permute(0, 2, 1, 3)
    out = torch.matmul(p, v) / torch.where(total == 0, 1.0, total)
    return {"out": out.view(rows, -1, hd).to(s["q"].dtype), "lse": (top + torch.log(total)).view(rows, -1)}


# --------------------------------------------------------------------------- one pass

def _cache(s):
    """The handle that a user's program makes once over its buffers: the book alone, or the cache."""
    if "cache" not in s:
        from bmo_jetson_b200.paged import PageBook, PagedKV
        book = PageBook(s["table"], s["lens"], s["free"], s["book"], page_size=s["page_size"], window=s["window"])
        s["cache"] = book if s["case"]["op"] == "plan" else PagedKV(book, s["k"], s["v"], k_scale=s["k_scale"],
                                                                    v_scale=s["v_scale"])
    return s["cache"]


def run(s):
    op = s["case"]["op"]
    if not own:
        return {"plan": _plain_plan, "append": _plain_append, "read": _plain_read, "attn": _plain_attn}[op](s)
    c = _cache(s)
    if op == "plan":
        c.plan(s["n_new"], s["slot"], s["pos"], s["req"], s["offsets"], lens_out=s["lens_out"], state_out=s["book_out"])
        return {"table": s["table"], "free": s["free"], "lens": s["lens_out"], "book": s["book_out"], "slot": s["slot"],
                "pos": s["pos"], "req": s["req"], "offsets": s["offsets"]}
    if op == "attn":
        c.attention(0, s["q"], s["out"], lse=s["lse"])
        return {"out": s["out"], "lse": s["lse"]}
    if op == "append":
        if s["case"]["rope"]:
            c.append(0, s["k_new"], s["v_new"], s["slot"], pos=s["pos"], q=s["q"], q_out=s["q_out"], theta=THETA)
        else:
            c.append(0, s["k_new"], s["v_new"], s["slot"])
    c.read(0, s["slot"], s["k_out"], s["v_out"])
    got = {"k": s["k_out"], "v": s["v_out"]}
    return got | ({"q": s["q_out"]} if op == "append" and s["case"]["rope"] else {})


# --------------------------------------------------------------------------- 64 bits

def _exact_rows(s, name, page, slot):
    x = s[name][0, page, :, slot].cpu().numpy()
    if s[name + "_scale"] is None:
        return x.astype(np.float64)
    d = s[name + "_scale"][0, page, :, slot].cpu().numpy().astype(np.float64)
    y = np.empty(x.shape[:-1] + (2 * x.shape[-1],))
    for b in range(d.shape[-1]):
        part = x[..., 16 * b:16 * b + 16].astype(np.int64)
        y[..., 32 * b:32 * b + 16] = ((part % 16) - 8) * d[..., b:b + 1]
        y[..., 32 * b + 16:32 * b + 32] = ((part // 16) - 8) * d[..., b:b + 1]
    return y


def _exact_turn(x, pos):
    """Complex multiplication by e^(i angle), the angle rounded to 32 bits as the operator defines it."""
    dim = x.shape[-1]
    e = (np.arange(0, dim, 2, dtype=np.float32) / np.float32(dim)).astype(np.float64)
    angle = pos.astype(np.float32)[:, None] * (THETA ** -e).astype(np.float32)
    z = (x[..., 0::2] + 1j * x[..., 1::2]) * np.exp(1j * angle.astype(np.float64))[:, None]
    y = np.empty(x.shape)
    y[..., 0::2], y[..., 1::2] = z.real, z.imag
    return y


def exact(case, seed):
    if case["op"] == "plan":
        return None  # whole numbers
    s = prepare(case, seed)
    ps = case["page_size"]
    if case["op"] == "attn":
        w, lens, table = case["window"], s["lens"].tolist(), s["table"].cpu()
        rows, h, kv, hd = case["rows"], case["heads"], case["kv_heads"], case["head_dim"]
        out, lse = torch.zeros((rows, h, hd), dtype=torch.float64), torch.full((rows, h), -math.inf, dtype=torch.float64)
        for r, n in enumerate(lens):
            at = np.arange(max(0, n - w) if w else 0, n)
            if not at.size:
                continue
            page, slot = table[r].numpy()[at // ps], at % ps
            if s["k_scale"] is None:
                page, slot = torch.from_numpy(page).long().cuda(), torch.from_numpy(slot).cuda()
                k, v = s["k"][0, page, :, slot].double(), s["v"][0, page, :, slot].double()
            else:
                k, v = (torch.from_numpy(_exact_rows(s, n_, page, slot)).cuda() for n_ in ("k", "v"))
            q = s["q"][r].double().view(kv, h // kv, hd)
            x = torch.einsum("kgd,jkd->kgj", q, k) * hd ** -0.5
            lse[r] = torch.logsumexp(x, -1).reshape(h).cpu()
            out[r] = torch.einsum("kgj,jkd->kgd", torch.softmax(x, -1), v).reshape(h, hd).cpu()
        return {"out": out, "lse": lse}
    page, slot = (x.numpy() for x in (s["slot"].cpu().long() // ps, s["slot"].cpu().long() % ps))
    if case["op"] == "read":
        return {n: _exact_rows(s, n, page, slot) for n in ("k", "v")}
    q, k, v = (s[n].double().cpu().numpy() for n in ("q", "k_new", "v_new"))
    if case["rope"]:
        pos = s["pos"].cpu().numpy()
        q, k = _exact_turn(q, pos), _exact_turn(k, pos)
    # a Q4_0 block's codes are defined by 32-bit operations: its rows have no value in 64 bits
    got = {"k": None, "v": None} if case["kv"] == "q4_0" else {"k": k, "v": v}
    return got | ({"q": q} if case["rope"] else {})

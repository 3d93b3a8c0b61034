"""Performance cases of the operators around a KV cache held in 4 bits: page tables, append, read-back and attention.

A cache is a uint8 tensor [pages, kv heads, page size / 16, 18 * head size]: blocks of 16 positions of one head, each the
4-bit codes of K (8 * head size bytes), those of V, then K's and V's fp16 scales and biases (head size bytes each).  A
position's codes are head size / 2 bytes, low nibble first; the 16-byte piece at byte o of a code region stands at
o ^ (16 * (o / 128 mod 8)).  Scales and biases are [64-value group][16 scales, 16 biases].  An element is worth
fp16(code * scale + bias): the affine group-64 scheme of the framework's weights.

The kinds of case:

  plan     page tables, slot map, positions and row offsets of a step, on the GPU, from the requests' lengths
  append   query and key norm, rotation by one or three position axes, K and V into their slots; the rows are read back
  read     K and V of given slots as fp16 (a prefix on its way to a host blob)
  attend   attention of a ragged batch of query rows over the cache, a row for each request or many
"""
import math

import torch

own = False

F16, F32, F64, I32, I64 = torch.float16, torch.float32, torch.float64, torch.int32, torch.int64
GROUP, BLOCK = 64, 16
EPS, THETA = 1e-6, 1e7


# ---------------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # a decode step of a full batch: 64 requests take a position each, some a page with it
        {"name": "plan_64", "op": "plan", "batch": 64, "page": 64, "past": 2000, "new": 1},
        # prompts admitted together with decoding requests, many of them, in small pages, some requests ended
        {"name": "plan_700", "op": "plan", "batch": 700, "page": 16, "past": 4001, "new": 509},
        # the framework's own head geometry, one decode row: launches and latency
        {"name": "append_1", "op": "append", "rows": 1, "heads": 16, "kv_heads": 2, "dim": 256, "rope": 64, "axes": 1, "page": 64, "norm": True},
        # image and text rows of a prompt chunk: three position axes, the whole head rotated
        {"name": "append_4093", "op": "append", "rows": 4093, "heads": 32, "kv_heads": 8, "dim": 128, "rope": 128, "axes": 3, "page": 32, "norm": True},
        # a shared 1024-position prefix of the framework's geometry
        {"name": "read_1024", "op": "read", "rows": 1024, "kv_heads": 2, "dim": 256, "page": 64},
        # a long conversation's state, odd length
        {"name": "read_30001", "op": "read", "rows": 30001, "kv_heads": 8, "dim": 128, "page": 128},
        # single-user decode after the benchmark's 512-position prompt, gated output as in the framework's model
        {"name": "attend_1", "op": "attend", "batch": 1, "heads": 16, "kv_heads": 2, "dim": 256, "page": 64, "new": 1, "past": 512, "ragged": False, "causal": True, "gate": True},
        # a decode step of a full batch, lengths up to 8192
        {"name": "attend_64", "op": "attend", "batch": 64, "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "new": 1, "past": 8191, "ragged": True, "causal": True, "gate": False},
        # verify rows of a speculative step, seven requests, small odd pages
        {"name": "attend_verify", "op": "attend", "batch": 7, "heads": 32, "kv_heads": 8, "dim": 128, "page": 48, "new": 4, "past": 1999, "ragged": False, "causal": True, "gate": False},
        # a prompt call of 1024 rows at the end of a long context, the framework's geometry
        {"name": "attend_chunk", "op": "attend", "batch": 1, "heads": 16, "kv_heads": 2, "dim": 256, "page": 64, "new": 1024, "past": 7168, "ragged": False, "causal": True, "gate": True},
        # ragged prompts without a past
        {"name": "attend_prompts", "op": "attend", "batch": 4, "heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "new": 2900, "past": 0, "ragged": True, "causal": True, "gate": False},
        # a decoder's rows over an encoder's states of another length
        {"name": "attend_cross", "op": "attend", "batch": 16, "heads": 12, "kv_heads": 12, "dim": 64, "page": 32, "new": 77, "past": 1500, "ragged": True, "causal": False, "gate": False},
    ]


def draw(rng):
    def size(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))

    op = rng.choice(["plan", "append", "read", "attend", "attend", "attend"])
    if op == "plan":
        return {"op": op, "batch": size(1, 700), "page": rng.choice([16, 32, 64, 128]), "past": size(1, 4001), "new": size(1, 509)}
    if op == "read":
        return {"op": op, "rows": size(1, 30001), "kv_heads": rng.choice([1, 2, 4, 8]), "dim": rng.choice([64, 128]), "page": rng.choice([16, 48, 64, 256])}
    kv, dim = rng.choice([1, 2, 4, 8]), rng.choice([64, 128, 256])
    heads = min(32, kv * rng.choice([1, 2, 3, 4, 7, 8])) // kv * kv
    if op == "append":
        rope = rng.choice([dim, dim // 2, dim // 4, 0])
        return {"op": op, "rows": size(1, 4093 * 128 // max(dim, 128)), "heads": heads, "kv_heads": kv, "dim": dim, "rope": rope,
                "axes": rng.choice([1, 3]) if rope else 1, "page": rng.choice([16, 32, 64, 112]), "norm": rng.random() < 0.8}
    c = {"op": op, "batch": 1, "heads": heads, "kv_heads": kv, "dim": dim, "page": rng.choice([16, 32, 48, 64, 128]), "new": 1, "past": 0,
         "ragged": rng.random() < 0.6, "causal": rng.random() < 0.85, "gate": rng.random() < 0.4}
    kind = rng.choice(["decode", "decode", "verify", "prompt"])
    if kind == "decode":
        c["batch"], c["past"] = size(1, 64), size(1, 8191)
    elif kind == "verify":
        c["batch"], c["past"], c["new"] = size(1, 16), size(16, 8191), size(2, 17)
    else:
        c["batch"], c["new"], c["past"] = size(1, 4), size(18, 2900), rng.choice([0, 0, size(64, 4096)])
    if not c["causal"]:
        c["past"] = max(c["past"], 1)
    top = {d["name"]: _cost(d) for d in listed()}["attend_chunk"]
    while _cost(c) > top:
        c["new"], c["past"] = max(1, c["new"] * 2 // 3), max(1, c["past"] * 2 // 3)
    return c


def _cost(c):
    w = work(c)
    return w["bytes"] / 6e12 + w["flops"] / 1e15


def _spread(n, most):
    """n lengths up to `most`, the first of them `most`: what requests of different ages have."""
    return [most if i == 0 else max(1, round(most * (0.25 + 0.75 * ((i * 0.6180339887498949) % 1.0)))) for i in range(n)]


def _lengths(c):
    """Rows and keys of each request of an attend case."""
    n, past = c["batch"], c["past"]
    news = _spread(n, c["new"]) if c["ragged"] else [c["new"]] * n
    pasts = ([0] * n if not past else _spread(n, past)[::-1]) if c["ragged"] else [past] * n
    return news, [p + m for p, m in zip(pasts, news)] if c["causal"] else pasts


def _plan_lengths(c):
    """Lengths and rows to come of each request of a plan case: one in 16 has ended, of a large batch nine in ten decode."""
    lens = [v - 1 for v in _spread(c["batch"], c["past"] + 1)]
    news = [-1 if i % 16 == 15 else (m if c["new"] == 1 or i % 10 == 0 else 1) for i, m in enumerate(_spread(c["batch"], c["new"]))]
    return lens, news


def work(case):
    c = case
    if c["op"] == "plan":
        lens, news = _plan_lengths(c)
        rows = sum(max(0, m) for m in news)
        grown = sum(-(-(v + m) // c["page"]) - -(-v // c["page"]) for v, m in zip(lens, news) if m > 0)
        ended = sum(-(-v // c["page"]) for v, m in zip(lens, news) if m < 0)
        return {"bytes": 16 * c["batch"] + 12 * rows + 8 * (grown + ended) + 4 * c["batch"], "flops": 4 * rows}
    cell = c["kv_heads"] * c["dim"] * 9 // 8                               # bytes of K and V of a position
    if c["op"] == "append":
        h, d = c["heads"], c["dim"]
        return {"bytes": c["rows"] * ((2 * h + 2 * c["kv_heads"]) * d * 2 + cell + 8 + 4 * c["axes"]), "flops": c["rows"] * d * (8 * (h + c["kv_heads"]) + 12 * c["kv_heads"])}
    if c["op"] == "read":
        return {"bytes": c["rows"] * (cell + c["kv_heads"] * c["dim"] * 4 + 8), "flops": c["rows"] * c["kv_heads"] * c["dim"] * 4}
    news, keys = _lengths(c)
    pairs = sum(m * (k - m) + m * (m + 1) // 2 if c["causal"] else m * k for m, k in zip(news, keys))
    rows = sum(news) * c["heads"] * c["dim"] * 2
    return {"bytes": rows * (3 if c["gate"] else 2) + sum(keys) * cell, "flops": 4 * c["dim"] * c["heads"] * pairs}


# ---------------------------------------------------------------------------------------------- inputs
def _tables(counts, page, gen, spare=5):
    """Block tables of requests with that many positions over shuffled pages: (table, number of pages, pages not used)."""
    need = [-(-v // page) for v in counts]
    pages = sum(need) + spare
    order = torch.randperm(pages, generator=gen, device="cuda").to(I32)
    table = torch.zeros((len(counts), max(max(need), 1)), dtype=I32, device="cuda")
    n, wide = torch.tensor(need, device="cuda"), torch.arange(table.shape[1], device="cuda")
    table[wide < n[:, None]] = order[: sum(need)]
    return table, pages, order[sum(need):]


def _filled(pages, kv, page, dim, gen):
    """A cache that holds normally distributed K and V: codes of a normal value each, scales a sixth off one another, biases that centre them."""
    blocks, groups = pages * kv * (page // BLOCK), dim // GROUP
    out = torch.empty((blocks, 18 * dim), dtype=torch.uint8, device="cuda")
    step = max(1, (1 << 24) // dim)
    for at in range(0, blocks, step):
        n = min(step, blocks - at)
        s = torch.empty((n, 2, groups, 1, BLOCK), device="cuda").uniform_(0.27, 0.36, generator=gen).to(F16)
        b = (s.float() * -7.5).to(F16)
        x = torch.randn((n, 2, groups, GROUP, BLOCK), generator=gen, device="cuda")
        code = ((x - b.float()) / s.float()).round_().clamp_(0, 15).to(torch.uint8).permute(0, 1, 4, 2, 3).reshape(n, 2, BLOCK * dim)
        code = code[..., 0::2] | code[..., 1::2] << 4
        out[at:at + n, : 16 * dim] = code[:, :, _swizzled(8 * dim)].reshape(n, 16 * dim)
        out[at:at + n, 16 * dim:] = torch.cat([s, b], 3).reshape(n, -1).view(torch.uint8)
    return out.view(pages, kv, page // BLOCK, 18 * dim)


def _swizzled(n):
    """Where byte o of a code region of n bytes stands (its own inverse)."""
    o = torch.arange(n, device="cuda")
    return o ^ ((o >> 7 & 7) << 4)


def prepare(case, seed):
    c = dict(case)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    ints = lambda v, t=I32: torch.tensor(v, dtype=t, device="cuda")  # noqa: E731
    normal = lambda *shape: torch.randn(shape, generator=gen, device="cuda").to(F16)  # noqa: E731
    if c["op"] == "plan":
        lens, news = _plan_lengths(c)
        held, pages, _ = _tables(lens, c["page"], gen, 0)
        most = max(-(-(v + max(0, m)) // c["page"]) for v, m in zip(lens, news))
        table = torch.zeros((c["batch"], most + 3), dtype=I32, device="cuda")
        table[:, : held.shape[1]] = held
        grown = sum(-(-(v + m) // c["page"]) for v, m in zip(lens, news) if m > 0)
        free = torch.zeros(pages + grown, dtype=I32, device="cuda")
        free[:grown] = torch.randperm(grown, generator=gen, device="cuda").to(I32) + pages
        rows = -(-sum(max(0, m) for m in news) // 64) * 64
        return {**c, "lens": ints(lens), "news": ints(news), "table": table, "free": free, "count": ints([grown]), "max_rows": rows}
    if c["op"] == "append":
        h, kv, d, n = c["heads"], c["kv_heads"], c["dim"], c["rows"]
        pages = -(-n // c["page"]) + 2
        cache = _filled(pages, kv, c["page"], d, gen)
        row = normal(n, (h + 2 * kv) * d)                                  # one projection's output: q | k | v
        past = torch.arange(n, device="cuda") + 1000                       # text positions, of an image's rows its grid's
        pos = torch.stack([past, past // 3 * 2 + 7, past * 5 // 4 - 11][: c["axes"]]).to(I32)
        slots = torch.randperm(pages * c["page"], generator=gen, device="cuda")[:n]
        w = lambda: (1 + 0.2 * torch.randn(d, generator=gen, device="cuda")).to(F16)  # noqa: E731
        return {**c, "cache": cache, "slots": slots, "q": row[:, : h * d].view(n, h, d), "k": row[:, h * d: (h + kv) * d].view(n, kv, d), "v": row[:, (h + kv) * d:].view(n, kv, d),
                "q_norm": w() if c["norm"] else None, "k_norm": w() if c["norm"] else None, "pos": pos,
                # the frequencies are dealt out to the axes in turn, as far as two thirds of them go; the rest follow time
                "axis_of": [i % 3 if i < c["rope"] // 3 else 0 for i in range(c["rope"] // 2)] if c["axes"] == 3 else None}
    if c["op"] == "read":
        pages = -(-c["rows"] // c["page"])
        cache = _filled(pages, c["kv_heads"], c["page"], c["dim"], gen)
        order = torch.randperm(pages, generator=gen, device="cuda")        # a request's pages, its positions in order
        at = torch.arange(c["rows"], device="cuda")
        return {**c, "cache": cache, "slots": order[at // c["page"]] * c["page"] + at % c["page"]}
    news, keys = _lengths(c)
    table, pages, _ = _tables(keys, c["page"], gen)
    starts = [0]
    for m in news:
        starts.append(starts[-1] + m)
    return {**c, "cache": _filled(pages, c["kv_heads"], c["page"], c["dim"], gen), "table": table, "kv_len": ints(keys), "q_start": ints(starts),
            "max_q": max(news), "q": normal(starts[-1], c["heads"], c["dim"]) * 1.5, "g": normal(starts[-1], c["heads"], c["dim"]) if c["gate"] else None}


# ---------------------------------------------------------------------------------------------- the operators
def run(state):
    return {"plan": _plan, "append": _append, "read": _read, "attend": _attend}[state["op"]](state)


def _plan(s):
    if own:
        from qwisp_b200 import ops
        p = ops.kv_plan(s["lens"], s["news"], s["table"], s["free"], s["count"], s["page"], s["max_rows"])
        return [p.kv_len, p.q_start, p.slots, p.pos, p.free_count, p.status, s["table"], s["free"]]
    page, table, free, n = s["page"], s["table"], s["free"], s["max_rows"]
    lens, news, count = s["lens"].to(I64), s["news"].to(I64), s["count"].to(I64)
    ended = news < 0
    have, rows = (lens + page - 1) // page, news.clamp(min=0)
    need = torch.where(ended, 0, (lens + rows + page - 1) // page)
    back, grown = torch.where(ended, have, 0), torch.where(ended, 0, need - have)
    back_at, grown_at = count + back.cumsum(0) - back, grown.cumsum(0) - grown
    q_start = torch.nn.functional.pad(rows.cumsum(0), (1, 0))
    # the pages of ended requests go onto the stack, those that others need come off its top, request by request
    wide = torch.arange(table.shape[1], device="cuda")
    freed = ended[:, None] & (wide < have[:, None])
    stack = torch.cat([free, free.new_zeros(1)]).scatter(0, torch.where(freed, back_at[:, None] + wide, free.numel()).flatten(), table.flatten())[:-1]
    top = count + back.sum()
    takes = ~ended[:, None] & (wide >= have[:, None]) & (wide < need[:, None])
    popped = stack[(top - 1 - (grown_at[:, None] + wide - have[:, None])).clamp(0, free.numel() - 1)]
    status = torch.stack([(grown.sum() - top[0]).clamp(min=0), ((lens < 0) | (need > table.shape[1])).sum(), (q_start[-1] - n).clamp(min=0)])
    fine = status.sum() == 0
    tables = torch.where(fine & takes, popped, table)
    at = torch.arange(n, device="cuda")
    b = (torch.searchsorted(q_start, at, right=True) - 1).clamp(max=lens.numel() - 1)
    live = fine & (at < q_start[-1])
    pos = torch.where(live, lens[b] + at - q_start[b], 0)
    slots = torch.where(live, tables[b, (pos // page).clamp(max=table.shape[1] - 1)].to(I64) * page + pos % page, -1)
    return [torch.where(fine & ended, 0, torch.where(fine, lens + rows, lens)).to(I32), torch.where(fine, q_start, 0).to(I32), slots, pos.to(I32),
            torch.where(fine, top - grown.sum(), count).to(I32), status.to(I32), tables, torch.where(fine, stack, free)]


def _away(x):
    """Rounded to the nearest whole number, halves away from zero, in 64 bits: x + 0.5 can round up in 32."""
    x = x.double()
    return (x.abs() + 0.5).floor() * x.sign()


def _quantised(x):
    """(codes, scale, bias) of values [..., 64] that fp16 holds: 32-bit arithmetic, every operation rounded once."""
    x = x.float()
    lo, hi = x.amin(-1, True), x.amax(-1, True)
    scale = ((hi - lo) / torch.full_like(lo, 15.0)).clamp(min=1e-7)
    side = lo.abs() > hi.abs()
    scale, edge = torch.where(side, scale, -scale), torch.where(side, lo, hi)
    q0 = _away(edge / scale).float()
    scale, bias = torch.where(q0 == 0, scale, edge / torch.where(q0 == 0, 1.0, q0)), torch.where(q0 == 0, 0.0, edge)
    return _away((x - bias) / scale).clamp(0, 15).to(torch.uint8), scale.to(F16), bias.to(F16)


def _stored(s, name, at, x):
    """Quantises x [rows, heads, dim] into the cache's region of that name, at (block, position in it) of every row and head."""
    cache, dim = s["cache"], s["dim"]
    block, inside = at
    second = name == "v"
    code, scale, bias = _quantised(x.reshape(*x.shape[:2], dim // GROUP, GROUP))
    code = code.reshape(*x.shape[:2], dim)
    o = inside[..., None] * (dim // 2) + torch.arange(dim // 2, device="cuda")
    cache.view(-1, 18 * dim)[block[..., None], 8 * dim * second + (o ^ ((o >> 7 & 7) << 4))] = code[..., 0::2] | code[..., 1::2] << 4
    o = 8 * dim + dim // 2 * second + torch.arange(dim // GROUP, device="cuda") * 2 * BLOCK + inside[..., None]
    halves = cache.view(-1, 18 * dim).view(F16)
    halves[block[..., None], o] = scale[..., 0]
    halves[block[..., None], o + BLOCK] = bias[..., 0]


def _places(s):
    """(block, position in it) of every row's slot and head."""
    page, kv = s["page"], s["kv_heads"]
    slots, head = s["slots"][:, None], torch.arange(kv, device="cuda")
    inside = slots % page
    return (slots // page * kv + head) * (page // BLOCK) + inside // BLOCK, (inside % BLOCK).expand(-1, kv)


def _append(s):
    if own:
        from qwisp_b200 import ops
        q = ops.kv4_append(s["cache"], s["slots"], s["q"], s["k"], s["v"], q_norm=s["q_norm"], k_norm=s["k_norm"], eps=EPS,
                           pos=s["pos"], rope_dims=s["rope"], rope_theta=THETA, axis_of=s["axis_of"])
        return [q, *ops.kv4_read(s["cache"], s["slots"])]
    rope = s["rope"]
    # angles in 64 bits: a far position's has few digits left in 32.  Keys stay in 64 bits up to their one rounding to fp16, so that
    # a code next to a border does not go by the order of a sum.
    axis = torch.tensor(s["axis_of"] or [0] * (rope // 2), dtype=I64, device="cuda")
    angle = s["pos"].double()[axis].T * THETA ** (torch.arange(rope // 2, dtype=F64, device="cuda") * (-2.0 / max(rope, 1)))

    def turned(x, w):
        if w is not None:
            x = x * torch.rsqrt(x.square().mean(-1, True) + EPS) * w.to(x.dtype)
        if not rope:
            return x
        c, n = angle.cos().to(x.dtype)[:, None], angle.sin().to(x.dtype)[:, None]
        a, b, rest = x[..., : rope // 2], x[..., rope // 2: rope], x[..., rope:]
        return torch.cat([a * c - b * n, a * n + b * c, rest], -1)

    q = turned(s["q"].float(), s["q_norm"]).to(F16)
    k = turned(s["k"].double(), s["k_norm"]).float().to(F16)
    at = _places(s)
    _stored(s, "k", at, k)
    _stored(s, "v", at, s["v"])
    return [q, *_read(s)]


def _read(s):
    if own:
        from qwisp_b200 import ops
        return list(ops.kv4_read(s["cache"], s["slots"]))
    dim = s["dim"]
    block, inside = _places(s)
    rows, halves = s["cache"].view(-1, 18 * dim), s["cache"].view(-1, 18 * dim).view(F16)
    o = inside[..., None] * (dim // 2) + torch.arange(dim // 2, device="cuda")
    o = o ^ ((o >> 7 & 7) << 4)
    sb = 8 * dim + torch.arange(dim // GROUP, device="cuda") * 2 * BLOCK + inside[..., None]

    def values(second):
        code = rows[block[..., None], 8 * dim * second + o]
        code = torch.stack([code & 15, code >> 4], -1).reshape(*block.shape, dim // GROUP, GROUP)
        scale, bias = halves[block[..., None], sb + dim // 2 * second], halves[block[..., None], sb + dim // 2 * second + BLOCK]
        return (code * scale[..., None].float() + bias[..., None].float()).to(F16).reshape(*block.shape, dim)

    return [values(0), values(1)]


def _attend(s):
    if own:
        from qwisp_b200 import ops
        return ops.kv4_attention(s["cache"], s["table"], s["kv_len"], s["q"], s["q_start"], s["max_q"], causal=s["causal"], gate=s["g"])
    dim, kv, n, most = s["dim"], s["kv_heads"], s["batch"], s["max_q"]
    span = s["table"].shape[1] * s["page"]
    blocks = s["cache"][s["table"].to(I64)].transpose(1, 2).reshape(n, kv, -1, 18 * dim)
    where = _swizzled(8 * dim)

    def values(second):
        code = blocks[..., 8 * dim * second: 8 * dim * (second + 1)][..., where]
        code = torch.stack([code & 15, code >> 4], -1).reshape(n, kv, -1, BLOCK, dim // GROUP, GROUP)
        at = 16 * dim + dim * second
        sb = blocks[..., at: at + dim].contiguous().view(F16).view(n, kv, -1, dim // GROUP, 2, BLOCK).transpose(3, 5).float()
        return (code * sb[..., 0, :, None] + sb[..., 1, :, None]).to(F16).float().reshape(n, kv, span, dim)

    # the requests' rows side by side, padded to the longest
    first, rows = s["q_start"][:-1].to(I64), (s["q_start"][1:] - s["q_start"][:-1]).to(I64)
    each = torch.arange(most, device="cuda")
    q = s["q"][(first[:, None] + each).clamp(max=s["q"].shape[0] - 1)].float().view(n, most, kv, -1, dim).permute(0, 2, 3, 1, 4)
    keys = s["kv_len"].to(I64)
    sees = keys[:, None] - rows[:, None] + each + 1 if s["causal"] else keys[:, None].expand(-1, most)
    hidden = torch.arange(span, device="cuda") >= sees[..., None]
    p = (q.reshape(n, kv, -1, dim) @ values(0).transpose(2, 3)).view(n, kv, -1, most, span).mul_(dim ** -0.5).masked_fill_(hidden[:, None, None], -math.inf)
    p = p.sub_(p.amax(-1, True).clamp(min=-1e30)).exp_()
    total = p.sum(-1)
    o = (p.view(n, kv, -1, span) @ values(1)).view(n, kv, -1, most, dim) / torch.where(total == 0, 1.0, total)[..., None]
    at = torch.arange(s["q"].shape[0], device="cuda")
    b = torch.searchsorted(s["q_start"].to(I64), at, right=True) - 1
    o = o.permute(0, 3, 1, 2, 4).reshape(n, most, -1, dim)[b, at - first[b]]
    return (o * torch.sigmoid(s["g"].float()) if s["gate"] else o).to(F16)


# ---------------------------------------------------------------------------------------------- the definitions in 64 bits
def _cell(block, name):
    """Values [16, dim] in 64 bits of K or V of blocks [..., 18 * dim], read word by word."""
    dim = block.shape[-1] // 18
    first = 0 if name == "k" else 8 * dim
    o = torch.arange(8 * dim, device=block.device)
    code = block[..., first + (o ^ ((o >> 7) % 8 * 16))].view(*block.shape[:-1], BLOCK, dim // 2, 1)
    code = torch.cat([code % 16, code // 16], -1).reshape(*block.shape[:-1], BLOCK, dim).double()
    first = 16 * dim if name == "k" else 17 * dim
    sb = block[..., first: first + dim].clone().view(F16).double().view(*block.shape[:-1], dim // GROUP, 2 * BLOCK)
    scale, bias = (t.transpose(-1, -2).repeat_interleave(GROUP, -1) for t in sb.split(BLOCK, -1))
    return (code * scale + bias).half().double()


def _exact_read(s):
    page = s["page"]
    out = []
    for name in "kv":
        parts = []
        for slots in s["slots"].split(2048):
            v = _cell(s["cache"][slots // page, :, slots % page // BLOCK], name)
            parts.append(v[torch.arange(len(slots), device="cuda"), :, slots % page % BLOCK])
        out.append(torch.cat(parts))
    return out


def _affine(x):
    """What values [..., 64] are worth in the cache: the scheme's scale and bias are fp16, its codes the nearest."""
    lo, hi = x.min(-1, True).values, x.max(-1, True).values
    low_far = lo.abs() > hi.abs()
    edge = torch.where(low_far, lo, hi)
    scale = ((hi - lo) / 15).clamp(min=1e-7) * torch.where(low_far, 1.0, -1.0)
    steps = edge / scale
    steps = torch.sign(steps) * torch.floor(steps.abs() + 0.5)
    scale = torch.where(steps != 0, edge / steps, scale)
    bias = torch.where(steps != 0, edge, 0.0)
    code = torch.floor((x - bias) / scale + 0.5).clamp(0, 15)
    return (code * scale.half().double() + bias.half().double()).half().double()


def _exact_append(s):
    half = s["rope"] // 2
    out = []
    for name in "qkv":
        x = s[name].double()
        if name != "v" and s["norm"]:
            x = x / (x.pow(2).sum(-1, keepdim=True) / s["dim"] + EPS).sqrt() * s[name + "_norm"].double()
        if name != "v":
            y = x.clone()
            for i in range(half):
                t = s["pos"][s["axis_of"][i] if s["axis_of"] else 0].double()[:, None] / THETA ** (i / half)
                y[..., i] = x[..., i] * t.cos() - x[..., i + half] * t.sin()
                y[..., i + half] = x[..., i + half] * t.cos() + x[..., i] * t.sin()
            x = y
        out.append(x if name == "q" else _affine(x.float().half().double().unflatten(-1, (-1, GROUP))).flatten(-2))
    return out


def _exact_attend(s):
    dim, kv = s["dim"], s["kv_heads"]
    group = s["heads"] // kv
    out = torch.zeros(s["q"].shape, dtype=F64, device="cuda")
    starts, lens = s["q_start"].tolist(), s["kv_len"].tolist()
    for b, keys in enumerate(lens):
        lo, hi = starts[b], starts[b + 1]
        pages = s["table"][b, : -(-keys // s["page"])].long()
        at = torch.arange(keys, device="cuda")
        last = at.new_tensor(range(keys - (hi - lo), keys)) if s["causal"] else at.new_full((hi - lo,), keys)
        for h in range(kv):
            k, v = (_cell(s["cache"][pages, h], name).reshape(-1, dim)[:keys] for name in "kv")
            for g in range(group):
                score = s["q"][lo:hi, h * group + g].double() @ k.T / math.sqrt(dim)
                score = score.masked_fill(at[None] > last[:, None], -math.inf)
                out[lo:hi, h * group + g] = torch.softmax(score, 1) @ v
    return out * torch.sigmoid(s["g"].double()) if s["gate"] else out


def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] == "plan":
        return None
    return {"append": _exact_append, "read": _exact_read, "attend": _exact_attend}[s["op"]](s)

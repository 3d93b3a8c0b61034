"""The operators around the 4-bit KV cache against plain implementations in 64 bits.

Where the tolerances come from.  A value rounded to fp16 is off by at most 2^-11 of itself (2^-25 below the normal range).  Attention
rounds each weight p once more to fp16 on its way into the tensor cores, which moves an output by at most 2^-11 sum(p |v|) (p normalised),
and forms scores, exponentials and sums in 32 bits: 256 products of a score, the scale and the exponential's argument are each off by a
few 2^-24 of the largest partial sum, for scores below 2^6 an error of the exponent below 2^-14, of p below 2^-14 of itself, so of
an output below 2^-14 sum(p |v|).  A normed and rotated query is one rounding to fp16 of 32-bit arithmetic on two values (some ten
operations: 2^-20 of their sum of sizes)."""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu
F64, F16, I32, I64 = torch.float64, torch.float16, torch.int32, torch.int64


def ops():
    import qwisp_b200 as Q
    return Q.ops


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def ints(v, t=I32):
    return torch.tensor(v, dtype=t, device="cuda")


def codes_of(cache):
    """(codes [pages, kv, page, D], scales and biases [pages, kv, page, D / 64]) of K and of V, read by the layout's description."""
    pages, kv, blocks, size = cache.shape
    D = size // 18
    o = torch.arange(8 * D, device=cache.device)
    out = []
    for r in range(2):
        raw = cache[..., 8 * D * r: 8 * D * (r + 1)][..., o ^ (16 * (o // 128 % 8))]
        code = torch.stack([raw & 15, raw >> 4], -1).reshape(pages, kv, blocks * 16, D)
        sb = cache[..., 16 * D + r * D: 17 * D + r * D].contiguous().view(F16).view(pages, kv, blocks, D // 64, 2, 16)
        s, b = (sb[..., i, :].transpose(3, 4).reshape(pages, kv, blocks * 16, D // 64) for i in range(2))
        out.append((code, s, b))
    return out


def values_of(cache):
    """fp16 values of K and V [pages, kv, page, D]."""
    return [(c.to(F64) * s.to(F64).repeat_interleave(64, -1) + b.to(F64).repeat_interleave(64, -1)).float().to(F16) for c, s, b in codes_of(cache)]


def random_cache(pages, page, kv, D, seed, spread=1.0):
    """A cache of normally distributed K and V, put there through the append operator."""
    c = ops().kv4_cache(pages, page, kv, D)
    n, g = pages * page, gen(seed)
    for at in range(0, n, 8192):
        m = min(8192, n - at)
        k, v = (torch.randn((m, kv, D), generator=g, device="cuda").mul_(spread).to(F16) for _ in range(2))
        ops().kv4_append(c, torch.arange(at, at + m, device="cuda"), None, k, v)
    return c


# ---------------------------------------------------------------------------------------------- plan
def plan_reference(lens, news, table, free, count, page, max_rows):
    B, W = table.shape
    table, free = table.copy(), free.copy()
    bad = sum(1 for v, n in zip(lens, news) if v < 0 or -(-(v + max(0, n)) // page) > W)
    rows = sum(max(0, n) for v, n in zip(lens, news) if not (v < 0 or -(-(v + max(0, n)) // page) > W))
    have = [-(-v // page) for v in lens]
    back = sum(h for h, n in zip(have, news) if n < 0)
    grown = sum(-(-(v + n) // page) - h for v, n, h in zip(lens, news, have) if n >= 0)
    if not bad and count + back > len(free):
        bad = 1
    short = 0 if bad else max(0, grown - count - back)
    over = max(0, rows - max_rows)
    slots, pos = np.full(max_rows, -1, np.int64), np.zeros(max_rows, np.int32)
    if bad or short or over:
        return np.array(lens), np.zeros(B + 1, int), slots, pos, count, [short, bad, over], table, free
    for b in range(B):
        if news[b] < 0:
            for j in range(have[b]):
                free[count] = table[b, j]
                count += 1
    starts, kv_len = [0], []
    for b in range(B):
        kv_len.append(0 if news[b] < 0 else lens[b] + news[b])
        if news[b] >= 0:
            for j in range(have[b], -(-kv_len[b] // page)):
                count -= 1
                table[b, j] = free[count]
            for i in range(news[b]):
                p = lens[b] + i
                slots[starts[-1] + i], pos[starts[-1] + i] = int(table[b, p // page]) * page + p % page, p
        starts.append(starts[-1] + max(0, news[b]))
    return np.array(kv_len), np.array(starts), slots, pos, count, [0, 0, 0], table, free


def plan_inputs(B, page, past, new, seed, width=None, spare=0):
    r = np.random.default_rng(seed)
    lens = [int(v) for v in r.integers(0, past + 1, B)]
    news = [int(v) for v in r.integers(-1, new + 1, B)]
    have = [-(-v // page) for v in lens]
    need = [-(-(v + max(0, n)) // page) for v, n in zip(lens, news)]
    width = width or max(need + [1]) + 2
    grown = sum(max(0, n - h) for n, h in zip(need, have))
    order = r.permutation(sum(have) + grown + spare)
    table, at = r.integers(-5, 5, (B, width)).astype(np.int32), 0
    for b in range(B):
        table[b, :have[b]] = order[at: at + have[b]]
        at += have[b]
    free = np.full(len(order) + 3, -9, np.int32)
    free[: len(order) - at] = order[at:]
    return lens, news, table, free, len(order) - at


def check_plan(lens, news, table, free, count, page, max_rows, alias=False):
    want = plan_reference(lens, news, table, free, count, page, max_rows)
    B, W = table.shape
    wide = torch.full((B, W + 3), 77, dtype=I32, device="cuda")            # a table whose rows lie further apart
    wide[:, :W] = torch.from_numpy(table).cuda()
    lens_d, count_d, free_d = ints(lens), ints([count]), torch.from_numpy(free).cuda()
    out = None
    if alias:
        from qwisp_b200.ops import KvPlan
        out = KvPlan(lens_d, ints([5] * (B + 1)), torch.zeros(max_rows, dtype=I64, device="cuda"), ints([5] * max_rows), count_d, ints([5] * 3))
    p = ops().kv_plan(lens_d, ints(news), wide[:, :W], free_d, count_d, page, max_rows, out=out)
    got = [p.kv_len, p.q_start, p.slots, p.pos, p.free_count, p.status, wide[:, :W], free_d]
    for name, g, w in zip(("kv_len", "q_start", "slots", "pos", "free_count", "status", "table", "free"), got, want):
        assert np.array_equal(g.cpu().numpy().reshape(-1), np.asarray(w).reshape(-1)), name
    assert (wide[:, W:] == 77).all()
    return p


@pytest.mark.parametrize("B,page,past,new", [(1, 16, 0, 1), (1, 64, 64, 1), (2, 16, 15, 1), (7, 48, 300, 40), (64, 64, 2000, 1), (33, 16, 100, 0), (200, 32, 1, 3),
                                             (1023, 16, 90, 5), (1024, 32, 90, 5), (1025, 16, 200, 30), (3000, 64, 500, 2), (40, 16, 1000, 900), (3, 128, 5, 9000)])
@pytest.mark.parametrize("alias", [False, True])
def test_plan(B, page, past, new, alias):
    lens, news, table, free, count = plan_inputs(B, page, past, new, B + page)
    rows = sum(max(0, n) for n in news)
    check_plan(lens, news, table, free, count, page, rows + 5, alias)
    check_plan(lens, news, table, free, count, page, rows, alias)


def test_plan_that_does_not_fit_changes_nothing():
    lens, news, table, free, count = plan_inputs(60, 16, 100, 50, 3)
    rows = sum(max(0, n) for n in news)
    back = sum(-(-v // 16) for v, n in zip(lens, news) if n < 0)
    assert 0 < back < count                                                # (what the ended requests return covers as much)
    assert check_plan(lens, news, table, free, count - back, 16, rows).status.tolist() == [0, 0, 0]
    assert check_plan(lens, news, table, free, count - back - 1, 16, rows).status.tolist() == [1, 0, 0]
    assert check_plan(lens, news, table, free, count, 16, rows - 7).status.tolist() == [0, 0, 7]
    assert check_plan(lens, news, table[:, :5].copy(), free, count, 16, rows).status.tolist()[1] > 0
    assert check_plan([-1] + lens[1:], news, table, free, count, 16, rows).status.tolist()[1] == 1
    assert check_plan(lens, news, table, free[:count], count, 16, rows).status.tolist()[1] == 1       # no room for what comes back
    # numbers near the end of 31 bits are refused, not wrapped
    p = ops().kv_plan(ints([2147483647, 5]), ints([2147483647, 1]), ints([[0], [0]]), ints([1, 2]), ints([2]), 16, 4)
    assert p.status.tolist() == [0, 1, 0] and p.slots.tolist() == [-1] * 4 and p.kv_len.tolist() == [2147483647, 5]
    assert ops().kv_plan(ints([5]), ints([1]), ints([[0]]), ints([1]), ints([-3]), 16, 4).status.tolist()[1] == 1


def test_plan_without_requests_or_rows():
    p = ops().kv_plan(ints([]), ints([]), torch.zeros((0, 4), dtype=I32, device="cuda"), ints([3]), ints([1]), 16, 5)
    assert p.q_start.tolist() == [0] and p.slots.tolist() == [-1] * 5 and p.status.tolist() == [0, 0, 0] and p.free_count.tolist() == [1]
    p = ops().kv_plan(ints([0, 0]), ints([0, -1]), torch.zeros((2, 0), dtype=I32, device="cuda"), ints([]), ints([0]), 16, 0)
    assert p.q_start.tolist() == [0, 0, 0] and p.kv_len.tolist() == [0, 0] and p.status.tolist() == [0, 0, 0]


# ---------------------------------------------------------------------------------------------- append, read
def rotated(x, w, pos, rope, theta, axis_of, eps=1e-6):
    x = x.to(F64)
    if w is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w.to(F64)
    y, half = x.clone(), rope // 2
    size = x.abs().clone()
    for i in range(half):
        t = (pos if pos.dim() == 1 else pos[axis_of[i] if axis_of else 0]).to(F64)[:, None] * theta ** (-2.0 * i / rope)
        y[..., i] = x[..., i] * t.cos() - x[..., i + half] * t.sin()
        y[..., i + half] = x[..., i + half] * t.cos() + x[..., i] * t.sin()
        size[..., i] = size[..., i + half] = x[..., i].abs() + x[..., i + half].abs()
    return y, size


def near_half(got, want, size):
    err = (got.to(F64) - want).abs()
    bound = want.abs() * 2.0 ** -11 + size * 2.0 ** -20 + 2.0 ** -24
    assert (err <= bound).all(), float((err / bound).max())


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("rows,NH,KV,page", [(1, 16, 2, 64), (5, 3, 3, 16), (37, 7, 1, 48), (700, 12, 4, 32)])
def test_append_quantises_as_the_weights_quantiser(D, rows, NH, KV, page):
    """K (no norm, no rotation) and V at scattered slots: codes, scales and biases are those of the weights' quantiser on the same rows;
    every other byte of the cache stays."""
    g = gen(D + rows)
    pages = -(-rows // page) + 2
    cache = torch.randint(0, 256, (pages, KV, page // 16, 18 * D), generator=g, device="cuda", dtype=torch.uint8)
    before = [[t.clone() for t in part] for part in codes_of(cache)]
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:rows]
    k, v = (torch.randn((rows, KV, D), generator=g, device="cuda").to(F16) for _ in range(2))
    v[0, 0, :64] = 0.25                                                    # a constant group
    k[0, 0, :64] = 0                                                       # an all-zero group
    v[0, KV - 1, 0] = 60000.0                                              # an outlier
    k[-1] *= 1e-6                                                          # values at the end of fp16's range
    assert ops().kv4_append(cache, slots, None, k, v) is None
    for x, (code, s, b), (code0, s0, b0) in zip((k, v), codes_of(cache), before):
        pk, sw, bw = ops().quantize_q4(x.reshape(rows * KV, D).cpu().numpy())
        want = torch.from_numpy((pk[:, :, None] >> (4 * np.arange(8, dtype=np.uint32)) & 15).astype(np.uint8)).cuda().view(rows, KV, D)
        page_of, off = slots // page, slots % page
        assert torch.equal(code[page_of, :, off], want)
        bits = lambda t: t.contiguous().view(torch.int16)  # noqa: E731
        assert torch.equal(bits(s[page_of, :, off]), torch.from_numpy(sw).cuda().view(rows, KV, D // 64).view(torch.int16))
        assert torch.equal(bits(b[page_of, :, off]), torch.from_numpy(bw).cuda().view(rows, KV, D // 64).view(torch.int16))
        other = torch.ones((pages, page), dtype=torch.bool, device="cuda")
        other[page_of, off] = False
        for new, old in ((code, code0), (bits(s), bits(s0)), (bits(b), bits(b0))):
            assert torch.equal(new.transpose(1, 2)[other], old.transpose(1, 2)[other])


@pytest.mark.parametrize("D,rope,axes,norm", [(64, 64, 1, True), (64, 32, 3, True), (128, 128, 3, True), (128, 0, 0, True), (128, 96, 1, False), (256, 64, 1, True), (256, 256, 2, True),
                                              (256, 16, 1, True)])
@pytest.mark.parametrize("rows,NH,KV", [(1, 4, 1), (9, 5, 5), (801, 24, 8)])
def test_append_norm_and_rotation(D, rope, axes, norm, rows, NH, KV):
    g = gen(rows + D + rope)
    page, theta = 32, 1e6
    cache = ops().kv4_cache(rows // page + 1, page, KV, D)
    fused = torch.randn((rows, (NH + 2 * KV) * D + 8), generator=g, device="cuda").to(F16)             # rows of one projection
    q, k, v = (fused[:, a * D: b * D].view(rows, b - a, D) for a, b in ((0, NH), (NH, NH + KV), (NH + KV, NH + 2 * KV)))
    w = [(1 + 0.3 * torch.randn(D, generator=g, device="cuda")).to(F16) if norm else None for _ in range(2)]
    pos = torch.randint(0, 300000, (max(axes, 1), rows), generator=g, device="cuda", dtype=I32)
    pos[0, 0] = 2000000
    axis_of = None if axes < 2 else [i % axes for i in range(rope // 2)]
    slots = torch.randperm(rows, generator=g, device="cuda")
    got = ops().kv4_append(cache, slots, q, k, v, q_norm=w[0], k_norm=w[1], pos=pos[0] if axes == 1 else pos, rope_dims=rope, rope_theta=theta, axis_of=axis_of)
    want, size = rotated(q, w[0], pos, rope, theta, axis_of)
    near_half(got, want, size)
    # K: rounded to fp16 once, then the quantiser
    kh = rotated(k, w[1], pos, rope, theta, axis_of)[0].float().to(F16)
    pk, sw, bw = ops().quantize_q4(kh.reshape(rows * KV, D).cpu().numpy())
    code = codes_of(cache)[0][0][slots // page, :, slots % page]
    want = torch.from_numpy((pk[:, :, None] >> (4 * np.arange(8, dtype=np.uint32)) & 15).astype(np.uint8)).cuda().view(rows, KV, D)
    # (64-bit operations in another order: an angle of 2e6 radians is off by 2^-31, so one rounding to fp16 in 2^20 may differ)
    assert float((code != want).double().mean()) <= 1e-4
    # queries alone, in place, without a cache's slots: the same queries
    again = q.clone()
    assert ops().kv4_append(cache, None, again, q_norm=w[0], pos=pos[0] if axes == 1 else pos, rope_dims=rope, rope_theta=theta, axis_of=axis_of, q_out=again) is again
    assert torch.equal(again, got)
    # the read operator gives the values that the codes stand for
    for got, want in zip(ops().kv4_read(cache, slots), values_of(cache)):
        assert torch.equal(got, want[slots // page, :, slots % page])


def test_padding_rows_and_slots_of_no_page():
    g = gen(5)
    cache = random_cache(3, 16, 2, 64, 1)
    before = cache.clone()
    q, k, v = (torch.randn((6, h, 64), generator=g, device="cuda").to(F16) for h in (4, 2, 2))
    out = torch.full((6, 4, 64), 7.0, dtype=F16, device="cuda")
    slots = ints([-1, 48, 1 << 40, -(1 << 62), 5, 47], I64)
    ops().kv4_append(cache, slots, q, k, v, q_norm=torch.ones(64, dtype=F16, device="cuda"), q_out=out)
    assert (out[:4] == 7).all() and (out[4:] != 7).any()
    want = before.clone()
    ops().kv4_append(want, slots[4:], None, k[4:], v[4:])
    assert torch.equal(cache, want)
    kr, vr = (torch.full((6, 2, 64), 9.0, dtype=F16, device="cuda") for _ in range(2))
    ops().kv4_read(cache, slots, kr, vr)
    assert (kr[:4] == 9).all() and (vr[:4] == 9).all() and torch.equal(kr[5], values_of(cache)[0][2, :, 15])
    assert ops().kv4_read(cache, slots[:0])[0].shape == (0, 2, 64)
    assert ops().kv4_append(cache, slots[:0], q[:0], k[:0], v[:0]).shape == (0, 4, 64)


def test_a_group_with_an_infinity_or_nan_reads_back_as_nan():
    cache = ops().kv4_cache(1, 16, 1, 128)
    k, v = (torch.randn((4, 1, 128), generator=gen(3), device="cuda").to(F16) for _ in range(2))
    k[1, 0, 70], v[2, 0, 3], v[3, 0, 127] = math.nan, math.inf, -math.inf
    ops().kv4_append(cache, torch.arange(4, device="cuda"), None, k, v)
    kr, vr = ops().kv4_read(cache, torch.arange(4, device="cuda"))
    bad = lambda t: t.isnan().view(4, 2, 64)  # noqa: E731
    want = torch.zeros((2, 4, 2), dtype=torch.bool, device="cuda")
    want[0, 1, 1] = want[1, 2, 0] = want[1, 3, 1] = True
    for got, w in zip((kr, vr), want):
        assert torch.equal(bad(got).all(-1), w) and torch.equal(bad(got).any(-1), w)


def test_pages_of_an_arena_and_offsets_past_32_bits():
    """A layer's pages inside pages of several layers; a cache whose last page is 6 GB from the first."""
    arena = torch.empty((7000, 2, 2, 4, 18 * 64), dtype=torch.uint8, device="cuda")
    far = torch.empty((1300000, 1, 4, 18 * 64), dtype=torch.uint8, device="cuda")
    for cache in (arena[:, 1], far):
        pages, kv = cache.shape[:2]
        slots = ints([64 * (pages - 1) + 63, 64 * (pages // 2), 0], I64)
        k, v = (torch.randn((3, kv, 64), generator=gen(4), device="cuda").to(F16) for _ in range(2))
        small = ops().kv4_cache(1, 64, kv, 64)
        ops().kv4_append(small, torch.arange(3, device="cuda"), None, k, v)
        ops().kv4_append(cache, slots, None, k, v)
        for a, b in zip(ops().kv4_read(cache, slots), ops().kv4_read(small, torch.arange(3, device="cuda"))):
            assert torch.equal(a, b)
        q = torch.randn((1, kv, 64), generator=gen(5), device="cuda").to(F16)
        got = ops().kv4_attention(cache, ints([[pages - 1]]), ints([64]), q, ints([0, 1]), 1)
        tail = cache[pages - 1:].clone()
        assert torch.equal(got, ops().kv4_attention(tail, ints([[0]]), ints([64]), q, ints([0, 1]), 1))


# ---------------------------------------------------------------------------------------------- attention
def attention_reference(cache, table, kv_len, q, q_start, causal, scale, gate=None, max_q=1 << 30):
    """(outputs in 64 bits, sum of p |v|, whether the row belongs to a request)."""
    K, V = (t.to(F64) for t in values_of(cache))
    kv, D = K.shape[1], K.shape[3]
    page = K.shape[2]
    out = torch.zeros(q.shape, dtype=F64, device="cuda")
    size, live = torch.zeros_like(out), torch.zeros(q.shape[0], dtype=torch.bool, device="cuda")
    G = q.shape[1] // kv
    for b in range(len(kv_len)):
        lo, hi = q_start[b], q_start[b + 1]
        rows = min(hi - lo, max_q)
        if rows <= 0:
            continue
        live[lo: lo + rows] = True
        n = max(0, kv_len[b])
        pages = table[b][: -(-n // page)].long()
        there = ((pages >= 0) & (pages < K.shape[0])).repeat_interleave(page)[:n]
        pages = pages.clamp(0, K.shape[0] - 1)
        k, v = (t[pages].transpose(0, 1).reshape(kv, -1, D)[:, :n] for t in (K, V))
        at = torch.arange(n, device="cuda")
        sees = (n - (hi - lo) + torch.arange(rows, device="cuda") + 1) if causal else torch.full((rows,), n, device="cuda")
        mask = there[None] & (at[None] < sees[:, None])
        k, v = k.nan_to_num(0, 0, 0), torch.where(mask.any(0)[None, :, None], v, 0.0)                   # (what nobody sees does not count)
        for h in range(q.shape[1]):
            s = (q[lo: lo + rows, h].to(F64) @ k[h // G].T * scale).masked_fill(~mask, -math.inf)
            m = s.amax(1, keepdim=True) if n else s.new_zeros(rows, 1)
            p = (s - m.clamp(min=-1e300)).exp()
            p = p / p.sum(1, keepdim=True).clamp(min=1e-300)
            g = torch.sigmoid(gate[lo: lo + rows, h].to(F64)) if gate is not None else 1.0
            out[lo: lo + rows, h], size[lo: lo + rows, h] = p @ v[h // G] * g, p @ v[h // G].abs() * g
    return out, size, live


def near(got, want, size, live):
    err = (got.to(F64) - want).abs()[live]
    bound = (want.abs() * 2.0 ** -11 + size * (2.0 ** -11 + 2.0 ** -14) + 2.0 ** -24)[live]
    assert (err <= bound).all(), (float((err / bound).max()), err.argmax())


def attention_case(D, NH, KV, page, news, keys, seed=1, spread=1.0, spare=2):
    g = gen(seed)
    need = [-(-max(0, n) // page) for n in keys]
    pages = sum(need) + spare
    cache = random_cache(pages, page, KV, D, seed, spread)
    order = torch.randperm(pages, generator=g, device="cuda").to(I32)
    table = torch.full((len(keys), max(need + [1]) + 1), -1, dtype=I32, device="cuda")
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at: at + n]
        at += n
    starts = [0]
    for n in news:
        starts.append(starts[-1] + n)
    q = torch.randn((starts[-1], NH, D), generator=g, device="cuda").mul_(1.5).to(F16)
    return cache, table, q, starts


DECODE = [  # D, heads, kv heads, page, rows of the requests, their keys
    (128, 8, 1, 64, [1], [1]), (64, 8, 1, 16, [1], [2]), (256, 16, 2, 64, [1], [513]), (128, 32, 8, 64, [1] * 5, [17, 16, 15, 4000, 64]),
    (128, 4, 4, 32, [1] * 3, [100, 0, 33]), (64, 3, 1, 48, [1, 0, 1], [1000, 70, 49]), (256, 12, 4, 16, [2, 1, 2], [65, 1, 2]), (128, 32, 8, 48, [4] * 7, [2003] * 7),
    (128, 10, 2, 128, [3] * 2, [300, 2]), (64, 16, 1, 64, [1], [20000]), (256, 8, 1, 64, [1] * 2, [9000, 1]), (128, 14, 2, 16, [1] * 40, list(range(1, 800, 20))),
    (128, 20, 1, 64, [1, 1], [777, 8]), (64, 64, 1, 32, [1, 1], [77, 800])]
PROMPT = [
    (128, 32, 8, 16, [129], [129]), (256, 16, 2, 64, [200], [1200]), (64, 12, 12, 32, [77, 19, 64], [77, 19, 64]), (128, 8, 2, 48, [33, 1, 0, 250], [333, 500, 9, 250]),
    (128, 6, 2, 64, [100, 30], [100, 31]), (256, 7, 1, 16, [61], [61]), (64, 5, 5, 64, [300], [1001]), (256, 8, 8, 32, [40, 40], [40, 30]), (128, 128, 1, 64, [20], [70]),
    (64, 8, 1, 128, [130], [130]), (128, 4, 1, 64, [600], [600])]


@pytest.mark.parametrize("case", DECODE + PROMPT, ids=lambda c: "-".join(str(v) if not isinstance(v, list) else f"{len(v)}x{max(v)}" for v in c))
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("gated", [False, True])
def test_attention(case, causal, gated):
    D, NH, KV, page, news, keys = case
    cache, table, q, starts = attention_case(D, NH, KV, page, news, keys)
    gate = torch.randn(q.shape, generator=gen(9), device="cuda").mul_(2).to(F16) if gated else None
    got = ops().kv4_attention(cache, table, ints(keys), q, ints(starts), max(news), causal=causal, gate=gate)
    want = attention_reference(cache, table, keys, q, starts, causal, D ** -0.5, gate)
    near(got, *want)
    # the same with a table made for far longer caches, whose work is dealt out in another way
    wide = torch.nn.functional.pad(table, (0, 70000 // page - table.shape[1]), value=-1)
    near(ops().kv4_attention(cache, wide, ints(keys), q, ints(starts), max(news), causal=causal, gate=gate), *want)


@pytest.mark.parametrize("D,NH,KV,new", [(64, 32, 8, 1), (128, 32, 8, 1), (128, 32, 8, 3), (256, 16, 4, 1), (256, 32, 4, 2)])
def test_long_caches_of_many_requests(D, NH, KV, new):
    """So many key blocks that every warp walks its ring many times over, and the same bits again and again."""
    keys = [new + (i * 977) % 3301 for i in range(48)]
    news = [new] * len(keys)
    cache, table, q, starts = attention_case(D, NH, KV, 64, news, keys)
    first = ops().kv4_attention(cache, table, ints(keys), q, ints(starts), new)
    near(first, *attention_reference(cache, table, keys, q, starts, True, D ** -0.5))
    for _ in range(20):
        assert torch.equal(ops().kv4_attention(cache, table, ints(keys), q, ints(starts), new), first)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("news,keys", [([1, 1], [37, 5]), ([90, 3], [200, 3])])
def test_what_lies_behind_the_keys_does_not_count(D, news, keys):
    """Stale positions, scales of NaN and infinity in them, pages that nobody has, and table entries of no page."""
    cache, table, q, starts = attention_case(D, 8, 2, 32, news, keys)
    want = ops().kv4_attention(cache, table, ints(keys), q, ints(starts), max(news))
    dirty = cache.clone()
    halves = dirty.view(F16)                                               # [pages, kv, blocks, 9 D]
    seen = torch.zeros(cache.shape[0] * 32, dtype=torch.bool, device="cuda")
    for b, n in enumerate(keys):
        p = torch.arange(n, device="cuda")
        seen[table[b].long()[p // 32] * 32 + p % 32] = True
    hidden = ~seen.view(cache.shape[0], 1, 2, 1, 16)                       # [pages, kv, blocks, group and half, position]
    junk = torch.tensor([math.nan, math.inf, -math.inf, 65504.0], dtype=F16, device="cuda").repeat(4)
    sb = halves[..., 8 * D:].view(*cache.shape[:3], -1, 16)
    sb.copy_(torch.where(hidden, junk, sb))
    beyond = table.clone()
    for b, n in enumerate(keys):
        beyond[b, -(-n // 32):] = 2 ** 31 - 1 if b else -2 ** 31
    got = ops().kv4_attention(dirty, beyond, ints(keys), q, ints(starts), max(news))
    assert torch.equal(got, want)
    # a page in the middle that is not there holds no keys
    holes = table.clone()
    holes[0, 0], holes[1, 0] = cache.shape[0], -1
    got = ops().kv4_attention(cache, holes, ints(keys), q, ints(starts), max(news))
    near(got, *attention_reference(cache, holes, keys, q, starts, True, D ** -0.5))


@pytest.mark.parametrize("D,NH,KV,new,past", [(128, 32, 8, 300, 1800), (128, 16, 4, 90, 2500), (64, 16, 8, 200, 1900), (256, 16, 2, 140, 1700), (256, 16, 2, 300, 1000), (64, 8, 8, 600, 700),
                                              (128, 8, 8, 65, 3000), (256, 8, 8, 33, 2000)])
@pytest.mark.parametrize("causal", [True, False])
def test_keys_shared_out(D, NH, KV, new, past, causal):
    """Few tiles of rows over many keys: shares of every size, some of them without keys for a tile."""
    news, keys = [new, 20], [new + past, 21]
    cache, table, q, starts = attention_case(D, NH, KV, 16, news, keys)
    got = ops().kv4_attention(cache, table, ints(keys), q, ints(starts), new, causal=causal)
    near(got, *attention_reference(cache, table, keys, q, starts, causal, D ** -0.5))
    for _ in range(10):
        assert torch.equal(ops().kv4_attention(cache, table, ints(keys), q, ints(starts), new, causal=causal), got)


@pytest.mark.parametrize("D,NH,KV,batch,new", [(64, 8, 8, 150, 1), (128, 24, 8, 90, 2), (256, 8, 4, 200, 1), (128, 12, 4, 301, 4)])
def test_more_requests_than_the_device_holds(D, NH, KV, batch, new):
    """Few rows a request, each (request, kv head) whole in one place."""
    keys = [(i * 389) % 601 if i % 7 else i % 3 for i in range(batch)]
    news = [new if i % 5 else 0 for i in range(batch)]
    cache, table, q, starts = attention_case(D, NH, KV, 32, news, keys)
    got = ops().kv4_attention(cache, table, ints(keys), q, ints(starts), new)
    near(got, *attention_reference(cache, table, keys, q, starts, True, D ** -0.5))
    for _ in range(5):
        assert torch.equal(ops().kv4_attention(cache, table, ints(keys), q, ints(starts), new), got)


@pytest.mark.parametrize("D,NH,KV,batch,new,gated", [(64, 12, 12, 16, 77, False), (64, 32, 8, 30, 9, True), (64, 8, 8, 20, 50, False), (128, 32, 8, 12, 9, True),
                                                     (128, 16, 4, 40, 33, False), (256, 8, 8, 12, 60, True), (64, 8, 4, 30, 90, False)])
@pytest.mark.parametrize("width", [40, 400])
def test_many_requests_of_a_tile_of_rows(D, NH, KV, batch, new, gated, width):
    """More tiles than multiprocessors, or nearly; requests of one row, of none and without keys among them; tables of 640 and of 6400 positions."""
    keys = [(i * 389) % 601 for i in range(batch)]
    news = [[new, 1, new - 3, 0][i % 4] if i else new for i in range(batch)]
    cache, table, q, starts = attention_case(D, NH, KV, 16, news, keys)
    table = torch.nn.functional.pad(table, (0, width - table.shape[1]), value=-1)
    gate = torch.randn(q.shape, generator=gen(9), device="cuda").to(F16) if gated else None
    for causal in (True, False):
        got = ops().kv4_attention(cache, table, ints(keys), q, ints(starts), new, causal=causal, gate=gate)
        near(got, *attention_reference(cache, table, keys, q, starts, causal, D ** -0.5, gate))
        for _ in range(5):
            assert torch.equal(ops().kv4_attention(cache, table, ints(keys), q, ints(starts), new, causal=causal, gate=gate), got)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("n", [1, 3, 70])
@pytest.mark.parametrize("width", [0, 1, 5000])
def test_requests_without_positions(D, n, width):
    """No keys at all, in tables of no columns too: zeros, whatever the tables hold."""
    cache = random_cache(2, 16, 2, D, 3)
    table = torch.full((3, width), 1 << 30, dtype=I32, device="cuda")
    q = torch.randn((3 * n, 8, D), generator=gen(4), device="cuda").to(F16)
    for causal in (False, True):
        for lens in ([0, 0, 0], [-5, 0, 0]):
            out = torch.full_like(q, 7.0)
            ops().kv4_attention(cache, table, ints(lens), q, ints([0, n, 2 * n, 3 * n]), n, causal=causal, out=out)
            assert (out == 0).all()


@pytest.mark.parametrize("n", [1, 70])
def test_rows_that_belong_to_nobody_stay_as_they_were(n):
    cache, table, q, starts = attention_case(128, 8, 2, 64, [n, n + 4, n], [100, 200, 50])
    rows = q.shape[0]
    wide = torch.randn((rows + 9, 8, 128), generator=gen(2), device="cuda").to(F16)
    wide[:rows] = q
    out = torch.full_like(wide, 5.0)
    keys, q_start = [100, 200, -7], ints(starts)
    ops().kv4_attention(cache, table, ints(keys), wide, q_start, n, out=out)            # the middle request has four rows too many
    want, size, live = attention_reference(cache, table, keys, q, starts, True, 128 ** -0.5, None, n)
    near(out[:rows], want, size, live)
    assert (out[rows:] == 5).all() and (out[:rows][~live] == 5).all() and int(live.sum()) == 3 * n
    # more keys than the table has pages for: those of its pages
    long = ops().kv4_attention(cache, table[:, :1], ints([1000, 1000, 64]), q, q_start, n + 4, causal=False)
    near(long, *attention_reference(cache, table[:, :1], [64] * 3, q, starts, False, 128 ** -0.5))


@pytest.mark.parametrize("news,keys", [([1] * 4, [300, 1, 65, 2000]), ([3] * 4, [300, 3, 65, 2000]), ([50, 1, 9], [300, 60, 2000])])
def test_strides_places_and_streams(news, keys):
    """Queries, gates and outputs inside wider rows, out in place of q, a caller's workspace, another stream: the same bits."""
    NH, D = 8, 128
    cache, table, q, starts = attention_case(D, NH, 2, 64, news, keys)
    gate = torch.randn(q.shape, generator=gen(8), device="cuda").to(F16)
    want = ops().kv4_attention(cache, table, ints(keys), q, ints(starts), max(news), gate=gate)
    again = ops().kv4_attention(cache, table, ints(keys), q, ints(starts), max(news), gate=gate)
    assert torch.equal(want, again)
    fused = torch.zeros((q.shape[0], NH, 2 * D + 8), dtype=F16, device="cuda")           # a head's query and gate side by side
    fused[..., :D], fused[..., D: 2 * D] = q, gate
    out = torch.zeros((q.shape[0] + 1, NH + 1, D), dtype=F16, device="cuda")[1:, 1:]
    need = ops().kv4_attention_workspace(NH, 2, D, len(keys), max(news), q.shape[0])
    ws = torch.full((need,), 255, dtype=torch.uint8, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops().kv4_attention(cache, table, ints(keys), fused[..., :D], ints(starts), max(news), gate=fused[..., D: 2 * D], out=out, workspace=ws)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out, want)
    same = q.clone()
    assert torch.equal(ops().kv4_attention(cache, table, ints(keys), same, ints(starts), max(news), gate=gate, out=same, workspace=ws), want)
    with pytest.raises(Exception):
        ops().kv4_attention(cache, table, ints(keys), q, ints(starts), max(news), workspace=ws[: need - 1])


@pytest.mark.parametrize("D", [64, 256])
@pytest.mark.parametrize("news,keys", [([1, 1], [900, 300]), ([80], [300])])
def test_scores_far_apart(D, news, keys):
    """Scores of hundreds: one key takes all; and a scale of zero: all keys alike."""
    cache, table, q, starts = attention_case(D, 8, 2, 64, news, keys, spread=4.0)
    for scale in (1.0, 0.0, -0.25):
        got = ops().kv4_attention(cache, table, ints(keys), q, ints(starts), max(news), scale=scale)
        want, size, live = attention_reference(cache, table, keys, q, starts, True, scale)
        # (scores of up to 2^11 here: their 32-bit sums move the exponent by 2^-9 of a unit)
        err, bound = (got.to(F64) - want).abs(), want.abs() * 2.0 ** -11 + size * (2.0 ** -11 + 2.0 ** -8) + 2.0 ** -24
        assert (err <= bound).all(), float((err / bound).max())


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("news,keys", [([1, 1], [900, 300]), ([2] * 3, [700, 64, 333]), ([90, 70], [200, 400]), ([40], [1500])])
def test_maxima_that_rise_along_the_keys(D, news, keys):
    """Keys that get longer along the positions, so that rows raise their maxima, and rescale what they have, at tiles of their own; the
    same bits a hundred times."""
    cache, table, q, starts = attention_case(D, 8, 2, 32, news, keys)
    g = gen(6)
    for b, n in enumerate(keys):
        p = torch.arange(n, device="cuda")
        k, v = (torch.randn((n, 2, D), generator=g, device="cuda") for _ in range(2))
        k *= (1 + 4 * p.double() / n).float()[:, None, None] * (1 + (p % 7 == 3).float())[:, None, None]
        ops().kv4_append(cache, table[b].long()[p // 32] * 32 + p % 32, None, k.to(F16), v.to(F16))
    for t in (table, torch.nn.functional.pad(table, (0, 1000), value=-1)):
        call = lambda: ops().kv4_attention(cache, t, ints(keys), q, ints(starts), max(news))  # noqa: E731,B023
        first = call()
        near(first, *attention_reference(cache, t, keys, q, starts, True, D ** -0.5))
        for _ in range(100):
            assert torch.equal(call(), first)


def test_a_long_tail_of_small_weights_counts():
    """One key far ahead of 30000 others whose weights are 2^-17 each: together they are a fifth of the result."""
    D, page, n = 128, 64, 30000
    cache = ops().kv4_cache(-(-n // page), page, 1, D)
    k, v = torch.zeros((n, 1, D), dtype=F16, device="cuda"), torch.ones((n, 1, D), dtype=F16, device="cuda")
    k[4321], v[4321] = 1.0, -1.0
    v[:, :, ::2] *= 0.5
    ops().kv4_append(cache, torch.arange(n, device="cuda"), None, k, v)
    table = torch.arange(-(-n // page), dtype=I32, device="cuda")[None]
    q = torch.full((1, 8, D), 1.0, dtype=F16, device="cuda")
    for rows in (1, 40):
        qs = q.expand(rows, -1, -1).contiguous()
        got = ops().kv4_attention(cache, table, ints([n]), qs, ints([0, rows]), rows, causal=False, scale=17 * math.log(2) / D)
        near(got, *attention_reference(cache, table, [n], qs, [0, rows], False, 17 * math.log(2) / D))


# ---------------------------------------------------------------------------------------------- together


@pytest.mark.parametrize("graph", [False, True])
def test_serving_steps(graph):
    """Prompts, decode steps, a request that ends and a new one in its place: plan, append and attention as a server calls them, its
    decode steps as one replayed graph, against attention over the values that the rows left in the cache."""
    D, NH, KV, page, rope, theta = 128, 8, 2, 16, 64, 1e6
    B, pages, width = 4, 60, 24
    g = gen(11)
    w = [(1 + 0.2 * torch.randn(D, generator=g, device="cuda")).to(F16) for _ in range(2)]
    cache = ops().kv4_cache(pages, page, KV, D)
    cache.view(F16)[:] = math.nan                                          # nothing may be read before it is written
    table = torch.full((B, width), -1, dtype=I32, device="cuda")
    free, count = torch.randperm(pages, generator=g, device="cuda").to(I32), ints([pages])
    lens = ints([0] * B)
    held = [[] for _ in range(B)]                                          # the rows' (k, v) as appended, per request
    from qwisp_b200.ops import KvPlan

    def step(news_d, rows, max_q, fused, out):
        p = ops().kv_plan(lens, news_d, table, free, count, page, rows, out=KvPlan(lens, *bufs[rows][:3], count, bufs[rows][3]))
        q, k, v = fused[:, :NH], fused[:, NH: NH + KV], fused[:, NH + KV:]
        qr = ops().kv4_append(cache, p.slots, q, k, v, q_norm=w[0], k_norm=w[1], pos=p.pos, rope_dims=rope, rope_theta=theta)
        return qr, ops().kv4_attention(cache, table, p.kv_len, qr, p.q_start, max_q, out=out)

    bufs, captured = {}, {}

    def run(news):
        rows = -(-max(1, sum(max(0, n) for n in news)) // 4) * 4
        if rows not in bufs:
            bufs[rows] = [torch.zeros(B + 1, dtype=I32, device="cuda"), torch.zeros(rows, dtype=I64, device="cuda"), torch.zeros(rows, dtype=I32, device="cuda"), ints([0] * 3)]
        fused = torch.randn((rows, NH + 2 * KV, D), generator=g, device="cuda").to(F16)
        before = lens.tolist()
        decode = graph and max(news) <= 1
        if decode:
            if rows not in captured:
                f, n, out = torch.zeros_like(fused), ints(news), torch.zeros((rows, NH, D), dtype=F16, device="cuda")
                side = torch.cuda.Stream()
                side.wait_stream(torch.cuda.current_stream())
                cg = torch.cuda.CUDAGraph()
                with torch.cuda.graph(cg, stream=side):
                    qr, _ = step(n, rows, 1, f, out)
                captured[rows] = cg, f, n, qr, out
            cg, f, n, qr, out = captured[rows]
            f.copy_(fused)
            n.copy_(ints(news))
            out.fill_(3.0)
            cg.replay()
        else:
            out = torch.full((rows, NH, D), 3.0, dtype=F16, device="cuda")
            qr, _ = step(ints(news), rows, max(1, max(news)), fused, out)
        assert bufs[rows][3].tolist() == [0, 0, 0]
        at = 0
        for b, n in enumerate(news):
            if n < 0:
                held[b] = []
                assert lens[b] == 0
                continue
            for i in range(n):
                held[b].append((fused[at, NH: NH + KV], fused[at, NH + KV:], before[b] + i))
                at += 1
            assert int(lens[b]) == len(held[b])
        assert (out[at:] == 3).all()
        # what the requests' rows left in the cache, in order
        at = 0
        K, V = values_of(cache)
        for b, n in enumerate(news):
            if n < 1:
                continue
            size = len(held[b])
            p = torch.arange(size, device="cuda")
            pg = table[b].long()[p // page]
            k, v = K[pg, :, p % page].to(F64), V[pg, :, p % page].to(F64)
            raw = torch.stack([h[0] for h in held[b]])
            kn = rotated(raw, w[1], ints([h[2] for h in held[b]]), rope, theta, None)[0]
            vn = torch.stack([h[1] for h in held[b]]).to(F64)
            # Within a step, a fifteenth of the group's range, and the roundings of scale and bias to fp16: the quantiser moves its step so
            # that the edge is a whole number r' >= 8 of them, which takes up to 15 (1 - 7.5 / 8) = 0.94 steps off the other end.
            for x, y in ((k, kn), (v, vn)):
                grp = y.reshape(size, KV, 2, 64)
                assert ((x - y).abs().reshape(size, KV, 2, 64) <= (grp.amax(-1) - grp.amin(-1))[..., None] / 15 + 0.02).all()
            sees = size - n + torch.arange(n, device="cuda") + 1
            for h in range(NH):
                s = qr[at: at + n, h].to(F64) @ k[:, h // 4].T * D ** -0.5
                pr = s.masked_fill(p[None] >= sees[:, None], -math.inf).softmax(1)
                want, mass = pr @ v[:, h // 4], pr @ v[:, h // 4].abs()
                near(out[at: at + n, h], want, mass, torch.ones(n, dtype=torch.bool, device="cuda"))
            at += n
        own = [int(x) for b in range(B) for x in table[b][: -(-int(lens[b]) // page)]] + free[: int(count)].tolist()
        assert sorted(own) == list(range(pages))                           # every page has one owner

    run([37, 5, 0, 100])
    for _ in range(4):
        run([1, 1, 1, 1])
    run([1, -1, 1, 1])
    run([1, 60, 1, 1])
    for _ in range(18):
        run([1, 1, 1, 1])
    run([-1, -1, -1, -1])
    assert int(count) == pages

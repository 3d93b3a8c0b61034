"""Calls around the 4-bit KV cache that its documentation allows and that are out of the ordinary."""
import pytest

torch = pytest.importorskip("torch")

from test_gpu_kv4 import F16, F64, I32, attention_case, attention_reference, codes_of, gen, ints, near, ops, random_cache, rotated

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D,NH,KV,new,keys", [(128, 32, 8, 1, [100, 37, 101, 1]), (256, 16, 2, 2, [1500, 600, 1400, 2]), (64, 12, 12, 33, [70, 64, 33, 20]), (128, 8, 2, 70, [2000, 70, 1999, 1000])])
@pytest.mark.parametrize("more", [0, 3000])
def test_requests_that_share_a_row_of_the_table(D, NH, KV, new, keys, more):
    """One prefix, or one encoder's states, for all requests: the row expanded gives what its copies give."""
    cache, table, q, starts = attention_case(D, NH, KV, 32, [new] * len(keys), [max(keys)] + [0] * (len(keys) - 1))
    row = torch.nn.functional.pad(table[:1], (0, more), value=-1)
    shared = row.expand(len(keys), -1)
    assert shared.stride(0) == 0
    for causal in (True, False):
        got = ops().kv4_attention(cache, shared, ints(keys), q, ints(starts), new, causal=causal)
        assert torch.equal(got, ops().kv4_attention(cache, row.repeat(len(keys), 1), ints(keys), q, ints(starts), new, causal=causal))
        near(got, *attention_reference(cache, shared, keys, q, starts, causal, D ** -0.5))


def test_workspace_of_the_current_device():
    cache, table, q, starts = attention_case(128, 8, 2, 64, [1, 1], [100, 40])
    size = ops().kv4_attention_workspace(8, 2, 128, 2, 1, 2)
    assert size > 0 and size == ops().kv4_attention_workspace(8, 2, 128, 2, 1, 500)
    want = ops().kv4_attention(cache, table, ints([100, 40]), q, ints(starts), 1)
    assert torch.equal(want, ops().kv4_attention(cache, table, ints([100, 40]), q, ints(starts), 1, workspace=torch.empty(size, dtype=torch.uint8, device="cuda")))
    with pytest.raises(Exception):
        ops().kv4_attention_workspace(8, 2, 128, 2, 1, -1)


@pytest.mark.parametrize("D,rope,axes", [(64, 64, 1), (64, 32, 3), (128, 128, 3), (128, 0, 1), (256, 64, 1), (256, 256, 2)])
@pytest.mark.parametrize("rows,KV", [(3, 1), (801, 4)])
def test_appended_keys_have_their_size(D, rope, axes, rows, KV):
    """Normed and rotated keys: scales and biases are those that the weights' quantiser has for them (codes alone do not tell a key from its
    double), and what is read back is within a step of the key in 64 bits."""
    g, page, eps = gen(rows + D + rope), 32, 3e-2                          # (an eps that shows)
    cache = ops().kv4_cache(rows // page + 1, page, KV, D)
    k, v = (torch.randn((rows, KV, D), generator=g, device="cuda").mul_(torch.rand((rows, KV, 1), generator=g, device="cuda") * 2).to(F16) for _ in range(2))
    w = (1 + 0.3 * torch.randn(D, generator=g, device="cuda")).to(F16)
    pos = torch.randint(0, 300000, (axes, rows), generator=g, device="cuda", dtype=I32)
    axis_of = None if axes < 2 else [i % axes for i in range(rope // 2)]
    slots = torch.randperm(rows, generator=g, device="cuda")
    ops().kv4_append(cache, slots, None, k, v, k_norm=w, eps=eps, pos=pos, rope_dims=rope, rope_theta=1e6, axis_of=axis_of)
    want = rotated(k, w, pos, rope, 1e6, axis_of, eps)[0]
    _, sw, bw = ops().quantize_q4(want.float().to(F16).reshape(rows * KV, D).cpu().numpy())
    differ = 0
    for got, x in zip(codes_of(cache)[0][1:], (sw, bw)):
        differ += int((got[slots // page, :, slots % page].contiguous().view(torch.int16) != torch.from_numpy(x).cuda().view(rows, KV, D // 64).view(torch.int16)).sum())
    # A key's rounding to fp16 may differ where another order of 64-bit operations takes it over a border: one in 2^20, and of a group's 64
    # only its ends show, in its scale or its bias.  Of these at most 25632 numbers hardly one.
    assert differ <= (0 if rows < 100 else 2)
    back = ops().kv4_read(cache, slots)[0].to(F64)
    grp = want.reshape(rows, KV, D // 64, 64)
    # (the quantiser takes up to 0.94 of a step off one end, half a step off the others; the roundings of scale and bias to fp16 16 x 2^-11 of the edge)
    bound = (grp.amax(-1) - grp.amin(-1)) / 15 + grp.abs().amax(-1) * 16 * 2.0 ** -11 + 2.0 ** -20
    assert ((back - want).abs().reshape(grp.shape) <= bound[..., None]).all()


def test_a_full_page_far_from_the_first():
    """A last page of a layer in pages of several, and one 6 GB from the first, all of it written: values, and attention over them, as in a cache of one page."""
    arena = torch.empty((7000, 2, 2, 4, 18 * 64), dtype=torch.uint8, device="cuda")
    far = torch.empty((1300000, 1, 4, 18 * 64), dtype=torch.uint8, device="cuda")
    for cache in (arena[:, 1], far):
        pages, kv = cache.shape[:2]
        slots, small = torch.arange(64, device="cuda"), ops().kv4_cache(1, 64, kv, 64)
        k, v = (torch.randn((64, kv, 64), generator=gen(4), device="cuda").to(F16) for _ in range(2))
        ops().kv4_append(small, slots, None, k, v)
        ops().kv4_append(cache, slots + 64 * (pages - 1), None, k, v)
        for a, b in zip(ops().kv4_read(cache, slots + 64 * (pages - 1)), ops().kv4_read(small, slots)):
            assert torch.equal(a, b)
        for rows in (1, 40):
            q = torch.randn((rows, kv, 64), generator=gen(5), device="cuda").to(F16)
            got = ops().kv4_attention(cache, ints([[pages - 1]]), ints([64]), q, ints([0, rows]), rows)
            near(got, *attention_reference(small, ints([[0]]), [64], q, [0, rows], True, 64 ** -0.5))


@pytest.mark.parametrize("D,NH,KV,news,width", [(128, 32, 8, [1, 70, 2, 0], 2048), (64, 8, 8, [33, 1, 40], 1536), (64, 16, 4, [200, 3], 2048), (256, 16, 2, [1, 90, 5], 4096), (128, 20, 1, [3, 30], 1024)])
def test_steps_of_many_rows_replayed(D, NH, KV, news, width):
    """A step of prompts and decoding requests together as one replayed graph: the kernel for many rows, its keys shared out by clusters,
    starts ahead of the end of those for few.  Other lengths, rows and pages at each replay; the bits of eager calls."""
    page, B, rows = 64, len(news), sum(news)
    pages = B * width // page
    g = gen(7)
    cache = random_cache(pages, page, KV, D, 3)
    q, k, v = (torch.zeros((rows, h, D), dtype=F16, device="cuda") for h in (NH, KV, KV))
    gate = torch.randn((rows, NH, D), generator=g, device="cuda").to(F16)
    table = torch.zeros((B, width // page), dtype=I32, device="cuda")
    lens, new = ints([0] * B), ints(news)
    free, count = torch.zeros(pages, dtype=I32, device="cuda"), ints([0])

    def step(cache, table, free):
        p = ops().kv_plan(lens, new, table, free, count, page, rows + 3)
        ops().kv4_append(cache, p.slots[:rows], None, k, v)
        return p, ops().kv4_attention(cache, table, p.kv_len, q, p.q_start, max(news), gate=gate)

    def fill(i):
        past = [(i * 611 + b * 389) % (width - max(news) - page) for b in range(B)]
        have = [-(-n // page) for n in past]
        order = torch.randperm(pages, generator=g, device="cuda").to(I32)
        lens.copy_(ints(past))
        for b, n in enumerate(have):
            table[b, :n] = order[sum(have[:b]): sum(have[:b]) + n]
        free[: pages - sum(have)] = order[sum(have):]
        count.copy_(ints([pages - sum(have)]))
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, generator=g, device="cuda"))
        return past

    fill(0)
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        plan, out = step(cache, table, free)
    for i in range(6):
        past = fill(i)
        eager = [t.clone() for t in (cache, table, free)]
        want_plan, want = step(*eager)
        graph.replay()
        assert plan.status.tolist() == [0, 0, 0]
        for a, b in zip((*plan, out, cache, table, free), (*want_plan, want, *eager)):
            assert torch.equal(a, b)
        starts = want_plan.q_start.tolist()
        near(out, *attention_reference(cache, table, [p + n for p, n in zip(past, news)], q, starts, True, D ** -0.5, gate))


def test_calls_at_once():
    """Calls of every kernel on streams of their own, many in flight: clusters of one call and of others share the device.  The bits of one after
    another."""
    shapes = [(64, 8, 8, [33] * 3, 1600), (64, 16, 4, [200, 90], 2100), (128, 8, 2, [70], 3000), (256, 16, 2, [90], 2000), (64, 8, 1, [1] * 4, 900), (128, 32, 8, [2] * 20, 3000), (64, 12, 12, [77] * 16, 600)]
    made = []
    for D, NH, KV, news, n in shapes:
        keys = [n - i for i in range(len(news))]
        cache, table, q, starts = attention_case(D, NH, KV, 64, news, keys)
        args = (cache, table, ints(keys), q, ints(starts), max(news))
        made.append((args, ops().kv4_attention(*args), torch.cuda.Stream()))
    torch.cuda.synchronize()
    outs = []
    for _ in range(30):
        for args, _, stream in made:
            with torch.cuda.stream(stream):
                outs.append(ops().kv4_attention(*args))
    torch.cuda.synchronize()
    for i, out in enumerate(outs):
        assert torch.equal(out, made[i % len(made)][1])

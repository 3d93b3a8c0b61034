"""Values at the edges of the attention over the 4-bit KV cache: gates and queries that are no numbers, lengths past
the table.  The kernels' tolerances are those of test_gpu_kv4.py, whose references these tests use."""
import math

import pytest

torch = pytest.importorskip("torch")

from test_gpu_kv4 import F16, attention_case, attention_reference, gen, ints, near, ops

pytestmark = pytest.mark.gpu

ENDS = [  # D, heads, kv heads, rows of the requests, their keys, columns that the table has more: each of the kernels' ends
    (128, 8, 2, [1, 1], [37, 5], 0),               # decode, clusters
    (256, 16, 2, [1, 1], [40, 2100], 3000),        # decode, dealt out: whole in a CTA, and joined
    (64, 8, 2, [3, 2], [50, 700], 5000),           # the same, two tiles of rows
    (128, 16, 2, [40, 3], [90, 3], 0),             # prompt, a tile of rows and two
    (256, 8, 2, [40], [30], 0),                    # prompt, rows that see nothing
    (64, 4, 4, [20] * 9, [100] * 9, 0),            # prompt, tiles of 64 dims by themselves
    (128, 8, 2, [70], [2100], 0),                  # prompt, keys shared out by a cluster
    (64, 4, 4, [33], [1500], 0),
]
each_end = pytest.mark.parametrize("case", ENDS, ids=lambda c: "-".join(str(v) if not isinstance(v, list) else f"{len(v)}x{max(v)}" for v in c))


def inputs(case):
    D, NH, KV, news, keys, more = case
    cache, table, q, starts = attention_case(D, NH, KV, 32, news, keys)
    return cache, torch.nn.functional.pad(table, (0, more), value=-1), q, starts


def alike(got, want, size, live):
    """NaN where it has to be and nowhere else, the rest near."""
    assert torch.equal(got.isnan()[live], want.isnan()[live])
    near(got.nan_to_num(0.0), want.nan_to_num(0.0), size.nan_to_num(0.0), live)


@each_end
@pytest.mark.parametrize("causal", [True, False])
def test_gates_that_are_no_numbers(case, causal):
    """A gate of NaN gives NaN, one of minus infinity zero, one of infinity the attention itself, each in its own place."""
    D, news, keys = case[0], case[3], case[4]
    cache, table, q, starts = inputs(case)
    gate = torch.randn(q.shape, generator=gen(3), device="cuda").mul_(2).to(F16)
    odd = torch.rand(q.shape, generator=gen(4), device="cuda")
    for lo, v in enumerate((math.nan, -math.nan, math.inf, -math.inf, 65504.0, -65504.0)):
        gate[(odd >= lo * 0.02) & (odd < lo * 0.02 + 0.02)] = v
    gate[0, 0, :9] = math.nan
    got = ops().kv4_attention(cache, table, ints(keys), q, ints(starts), max(news), causal=causal, gate=gate)
    want = attention_reference(cache, table, keys, q, starts, causal, D ** -0.5, gate)
    assert want[0].isnan().any()
    alike(got, *want)


@each_end
@pytest.mark.parametrize("scale", [None, -0.05, 0.0])
def test_queries_that_are_no_numbers(case, scale):
    """An infinity or a NaN among a row's queries makes its scores infinities and NaN, and so, whatever their signs, its outputs NaN: with
    one key as with many.  Heads and rows beside it keep their values; a row that sees nothing stays zero."""
    D, NH, _, news, keys, _ = case
    cache, table, q, starts = inputs(case)
    g, rows = gen(5), q.shape[0]
    clean = q.clone()
    bad = torch.rand((rows, NH), generator=g, device="cuda") < 0.3
    bad[0, 0] = True
    at = torch.randint(0, D, (rows, NH, 1), generator=g, device="cuda")
    what = torch.tensor([math.nan, math.inf, -math.inf], dtype=F16, device="cuda")[torch.randint(0, 3, (rows, NH, 1), generator=g, device="cuda")]
    q.scatter_(2, at, torch.where(bad[..., None], what, q.gather(2, at)))
    for causal in (True, False):
        want, size, live = attention_reference(cache, table, keys, clean, starts, causal, D ** -0.5 if scale is None else scale)
        sees = torch.zeros(rows, dtype=torch.bool, device="cuda")
        for b, n in enumerate(keys):
            lo, hi = starts[b], starts[b + 1]
            sees[lo:hi] = (n - (hi - lo) + torch.arange(hi - lo, device="cuda") + 1 if causal else torch.full((hi - lo,), n, device="cuda")) > 0
        want[bad & sees[:, None]] = math.nan
        alike(ops().kv4_attention(cache, table, ints(keys), q, ints(starts), max(news), causal=causal, scale=scale), want, size, live)


@pytest.mark.parametrize("D,NH,KV,news,keys,pages", [(128, 8, 2, [1, 1, 1], [1000, 64, 129], 2), (64, 8, 2, [3, 5], [140, 131], 2), (256, 16, 2, [2], [900], 9), (128, 16, 4, [40, 70], [140, 150], 2),
                                                     (64, 4, 4, [30] * 5, [70, 64, 80, 94, 93], 1), (128, 8, 2, [65, 3], [2100, 70], 30), (256, 8, 8, [33], [100], 1)])
@pytest.mark.parametrize("more", [0, 3000])
def test_lengths_past_the_table(D, NH, KV, news, keys, pages, more):
    """Positions that the table has no page for hold no keys, like those of entries of no page: a causal row's place goes by the
    request's length all the same."""
    cache, table, q, starts = attention_case(D, NH, KV, 64, news, keys)
    cut = table[:, :pages].contiguous()
    gone = table.clone()
    gone[:, pages:] = -1
    for causal in (True, False):
        want = attention_reference(cache, gone, keys, q, starts, causal, D ** -0.5)
        near(ops().kv4_attention(cache, cut, ints(keys), q, ints(starts), max(news), causal=causal), *want)
        near(ops().kv4_attention(cache, torch.nn.functional.pad(gone, (0, more), value=-1), ints(keys), q, ints(starts), max(news), causal=causal), *want)
    # the longest length that there is
    far = ops().kv4_attention(cache, cut, ints([2 ** 31 - 1] * len(keys)), q, ints(starts), max(news))
    assert torch.equal(far, ops().kv4_attention(cache, cut, ints([pages * 64] * len(keys)), q, ints(starts), max(news), causal=False))

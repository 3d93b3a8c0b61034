"""Calls around the 4-bit KV cache that its documentation allows and that are out of the ordinary."""
import pytest

torch = pytest.importorskip("torch")

from test_gpu_kv4 import attention_case, attention_reference, ints, near, ops

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

"""Refusals of the operators around the 4-bit KV cache: arguments are looked at before a device is, so these run anywhere.  The pointers
are never followed: every call here is refused, or ends with "no device" where there is none."""
import ctypes as C

import pytest

from conftest import has_gpu
from qwisp_b200 import _lib

P = 1 << 20                                            # a 16-byte aligned address that nothing follows
INVALID, CAPACITY, NO_DEVICE = _lib.SL_ERR_INVALID, _lib.SL_ERR_CAPACITY, _lib.SL_ERR_NO_DEVICE


def cache(**kw):
    d = dict(data=P, page_stride=2 * 4 * 18 * 128, pages=8, page_size=64, kv_heads=2, head_dim=128)
    return _lib.SlKv4Cache(**{**d, **kw})


def plan(**kw):
    d = dict(lens=P, new_rows=P, batch=4, page_size=64, table=P, table_stride=8, table_width=8, free_pages=P, free_capacity=32, free_count=P,
             kv_len=P, q_start=P, slots=P, pos=P, max_rows=16, free_count_out=P, status=P)
    return _lib.SlKvPlan(**{**d, **kw})


def append(**kw):
    d = dict(q=P, k=P, v=P, q_row=2048, q_head=128, k_row=2048, k_head=128, v_row=2048, v_head=128, q_out=P, q_out_row=2048, q_out_head=128,
             rows=3, q_heads=8, q_norm=P, k_norm=P, eps=1e-6, pos=P, pos_axis=3, axes=1, rope_dims=64, rope_theta=1e4, axis_of=None, slots=P)
    return _lib.SlKv4Append(**{**d, **kw})


def read(**kw):
    d = dict(slots=P, rows=3, k=P, v=P, k_row=256, k_head=128, v_row=256, v_head=128)
    return _lib.SlKv4Read(**{**d, **kw})


def attention(**kw):
    d = dict(q=P, q_row=1024, q_head=128, gate=None, gate_row=0, gate_head=0, out=P, out_row=1024, out_head=128, rows=3, q_heads=8, q_start=P, kv_len=P,
             batch=2, max_q=2, table=P, table_stride=8, table_width=8, causal=1, scale=0.1, workspace=P, workspace_bytes=1 << 40)
    return _lib.SlKv4Attention(**{**d, **kw})


def call(name, *structs):
    return getattr(_lib.lib(), name)(*[C.byref(s) if s is not None else None for s in structs], None)


@pytest.mark.parametrize("kw", [dict(data=None), dict(data=P + 8), dict(pages=0), dict(pages=-1), dict(page_size=0), dict(page_size=24), dict(kv_heads=0),
                                dict(head_dim=96), dict(kv_heads=65536, page_stride=65536 * 4 * 18 * 128), dict(page_stride=2 * 4 * 18 * 128 - 16), dict(page_stride=2 * 4 * 18 * 128 + 8)])
def test_caches_that_cannot_be_addressed_are_refused(kw):
    c = cache(**kw)
    assert call("sl_op_kv4_append_device", c, append()) == INVALID
    assert call("sl_op_kv4_read_device", c, read()) == INVALID
    assert call("sl_op_kv4_attention_device", c, attention()) == INVALID


@pytest.mark.parametrize("kw", [dict(batch=-1), dict(page_size=0), dict(max_rows=-1), dict(table_width=-1), dict(free_capacity=-1), dict(lens=None), dict(new_rows=None),
                                dict(table=None), dict(table_stride=7), dict(free_pages=None), dict(free_count=None), dict(kv_len=None), dict(q_start=None),
                                dict(slots=None), dict(pos=None), dict(free_count_out=None), dict(status=None)])
def test_plan_refusals(kw):
    assert call("sl_op_kv_plan_device", plan(**kw)) == INVALID


@pytest.mark.parametrize("kw", [dict(q=None, k=None, v=None), dict(v=None), dict(k=None), dict(q_out=None), dict(q_heads=0), dict(q_heads=-1), dict(q_heads=65536), dict(rows=-1), dict(q=P + 2),
                                dict(q_row=2044), dict(k_head=100), dict(v_row=12), dict(q_out_head=4), dict(q_norm=P + 8), dict(eps=-1.0), dict(eps=float("nan")),
                                dict(slots=None), dict(pos=None), dict(rope_dims=24), dict(rope_dims=144), dict(rope_dims=-16), dict(axes=0),
                                dict(rope_theta=0.5), dict(rope_theta=float("inf")), dict(rope_theta=float("nan")), dict(axis_of=bytes([1] * 32))])
def test_append_refusals(kw):
    assert call("sl_op_kv4_append_device", cache(), append(**kw)) == INVALID


@pytest.mark.parametrize("kw", [dict(slots=None), dict(k=None), dict(v=None), dict(rows=-1), dict(k=P + 4), dict(v_head=3)])
def test_read_refusals(kw):
    assert call("sl_op_kv4_read_device", cache(), read(**kw)) == INVALID


@pytest.mark.parametrize("kw", [dict(q=None), dict(out=None), dict(q_start=None), dict(kv_len=None), dict(table=None), dict(rows=-1), dict(batch=-1), dict(max_q=0),
                                dict(q_heads=0), dict(q_heads=7), dict(q=P + 8), dict(q_row=4), dict(out_head=2), dict(gate=P + 8), dict(gate=P, gate_row=3),
                                dict(table_width=-1), dict(table_stride=7), dict(scale=float("nan")), dict(scale=float("inf")), dict(workspace=None), dict(workspace=P + 4)])
def test_attention_refusals(kw):
    assert call("sl_op_kv4_attention_device", cache(), attention(**kw)) == INVALID


def test_sizes_beyond_the_kernels_are_refused():
    assert call("sl_op_kv4_attention_device", cache(), attention(q_heads=2 * 129)) == CAPACITY
    assert call("sl_op_kv4_attention_device", cache(), attention(table_width=1 << 25, table_stride=1 << 25)) == CAPACITY      # positions past 31 bits
    assert call("sl_op_kv4_attention_device", cache(), attention(batch=4097)) == CAPACITY
    assert call("sl_op_kv4_attention_device", cache(), attention(batch=4096, table_width=1 << 17, table_stride=1 << 17)) == CAPACITY      # key blocks
    assert call("sl_op_kv_plan_device", plan(batch=1 << 16, table_width=1 << 16, table_stride=1 << 16)) == CAPACITY
    assert _lib.lib().sl_kv4_attention_workspace(2 * 129, 2, 128, 1, 1, 1) == CAPACITY
    for args in ((7, 2, 128, 1, 1, 1), (8, 0, 128, 1, 1, 1), (8, 2, 96, 1, 1, 1), (8, 2, 128, -1, 1, 1), (8, 2, 128, 1, 0, 1), (8, 2, 128, 1, 1, -1)):
        assert _lib.lib().sl_kv4_attention_workspace(*args) == INVALID


def test_workspace_of_a_span():
    """Never more than for tables of any width, nothing where the kernels take the work whole, refusals as there."""
    any_width, of = _lib.lib().sl_kv4_attention_workspace, _lib.lib().sl_kv4_attention_workspace_span
    for heads, kv, dim, batch, max_q in ((8, 2, 128, 1, 1), (16, 2, 256, 64, 1), (64, 2, 64, 3, 5), (32, 8, 128, 4096, 4), (16, 1, 256, 2, 900)):
        most = any_width(heads, kv, dim, batch, max_q, 7)
        assert most > 0
        assert all(of(heads, kv, dim, batch, max_q, span) in (0, most) for span in (0, 1, 512, 8192, 1 << 30, 1 << 40))
        assert of(heads, kv, dim, batch, max_q, 1 << 40) == (0 if heads // kv > 16 else most)
    assert of(8, 2, 128, 1, 1, 512) == 0
    for args in ((7, 2, 128, 1, 1, 1), (8, 2, 96, 1, 1, 1), (8, 2, 128, -1, 1, 1), (8, 2, 128, 1, 0, 1), (8, 2, 128, 1, 1, -1)):
        assert of(*args) == INVALID
    assert of(2 * 129, 2, 128, 1, 1, 1) == CAPACITY


def test_page_bytes():
    f = _lib.lib().sl_kv4_page_bytes
    assert f(2, 256, 64) == 2 * 64 * 256 * 9 // 8 and f(8, 128, 16) == 8 * 16 * 144
    assert f(2, 96, 64) == f(0, 128, 64) == f(2, 128, 40) == f(2, 128, 0) == INVALID


def test_null_blocks_are_refused():
    for name in ("sl_op_kv4_append_device", "sl_op_kv4_read_device", "sl_op_kv4_attention_device"):
        assert call(name, cache(), None) == INVALID
        assert getattr(_lib.lib(), name)(None, None, None) == INVALID
    assert call("sl_op_kv_plan_device", None) == INVALID


@pytest.mark.skipif(has_gpu(), reason="checks the no-device error path")
def test_without_a_device_the_calls_say_so():
    assert call("sl_op_kv_plan_device", plan()) == NO_DEVICE
    assert call("sl_op_kv4_append_device", cache(), append()) == NO_DEVICE
    assert call("sl_op_kv4_read_device", cache(), read()) == NO_DEVICE
    assert call("sl_op_kv4_attention_device", cache(), attention()) == NO_DEVICE


def test_struct_layouts():
    """The sizes of the header's argument blocks (pointers and 64-bit numbers on 8-byte boundaries)."""
    for s, n in ((_lib.SlKv4Cache, 32), (_lib.SlKvPlan, 128), (_lib.SlKv4Append, 176), (_lib.SlKv4Read, 64), (_lib.SlKv4Attention, 152)):
        assert C.sizeof(s) == n, (s, C.sizeof(s))


def test_tensors_on_the_host_are_refused():
    torch = pytest.importorskip("torch")
    import qwisp_b200 as Q
    host = torch.zeros((2, 1, 4, 18 * 64), dtype=torch.uint8)
    i = lambda *v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    for f in (lambda: Q.ops.kv4_read(host, torch.zeros(1, dtype=torch.int64)),
              lambda: Q.ops.kv4_append(host, torch.zeros(1, dtype=torch.int64), torch.zeros(1, 1, 64).half()),
              lambda: Q.ops.kv4_attention(host, i(0).view(1, 1), i(1), torch.zeros(1, 1, 64).half(), i(0, 1), 1),
              lambda: Q.ops.kv_plan(i(0), i(1), i(0).view(1, 1), i(0), i(1), 64, 8),
              lambda: Q.ops.kv4_cache(4, 24, 1, 64)):
        with pytest.raises(Q.SeedlessError) as e:
            f()
        assert e.value.code == INVALID


def test_packed_argument_blocks_are_the_structures():
    """The wrappers pack an argument block's bytes in one go: every field lands where the structure has it."""
    from qwisp_b200 import ops
    for fmt, s in ((ops._CACHE, _lib.SlKv4Cache), (ops._PLAN, _lib.SlKvPlan), (ops._APPEND, _lib.SlKv4Append), (ops._READ, _lib.SlKv4Read),
                   (ops._ATTENTION, _lib.SlKv4Attention)):
        assert fmt.size == C.sizeof(s)
        values = [0.5 * i if t is C.c_float else i + 1 for i, (_, t) in enumerate(s._fields_)]
        got = s.from_buffer_copy(fmt.pack(*values))
        for (name, t), v in zip(s._fields_, values):
            w = C.c_void_p.from_buffer(got, getattr(s, name).offset).value if t is C.c_char_p else getattr(got, name)
            assert w == v, (s, name)

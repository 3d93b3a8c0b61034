"""What the wrappers around the 4-bit KV cache hand to the library.  They take host tensors here that say they are on a device, and the
library's entry points are not called: the argument blocks are looked at."""
import ctypes as C

import pytest

torch = pytest.importorskip("torch")

import qwisp_b200 as Q
from qwisp_b200 import _lib, ops

F16, I32, I64 = torch.float16, torch.int32, torch.int64


class OnDevice(torch.Tensor):
    index = 0

    def get_device(self):
        return self.index


class OnAnother(OnDevice):
    index = 1


def on(t, device=OnDevice):
    return t.as_subclass(device)


def ints(*v):
    return on(torch.tensor(v, dtype=I32))


@pytest.fixture
def blocks(monkeypatch):
    """The argument blocks of the calls that would have been made."""
    made = []
    monkeypatch.setattr(ops, "_cuda", lambda: (lambda: 0, lambda index: 0))
    monkeypatch.setattr(ops, "_call", lambda fn, index, where, *b: made.append((where, b)))
    return made


def refused(f):
    with pytest.raises(Q.SeedlessError) as e:
        f()
    assert e.value.code == _lib.SL_ERR_INVALID


def attention(table, B=3, **kw):
    cache = on(torch.zeros((4, 1, 4, 18 * 64), dtype=torch.uint8))
    return ops.kv4_attention(cache, table, ints(*[5] * B), on(torch.zeros((B, 2, 64), dtype=F16)), ints(*range(B + 1)), 1, **kw)


def plan(table, B=3):
    return ops.kv_plan(ints(*[5] * B), ints(*[1] * B), table, ints(*range(9)), ints(9), 16, 8)


def test_rows_of_the_table(blocks):
    """The stride that the table has: of rows inside wider ones, of one row for all requests; a single row's does not count."""
    wide, one = on(torch.zeros((3, 7), dtype=I32)), on(torch.zeros((1, 5), dtype=I32))
    for table, B, stride in ((wide, 3, 7), (wide[:, :5], 3, 7), (one.expand(3, -1), 3, 0), (one, 1, 5), (one.as_strided((1, 5), (0, 1)), 1, 5), (one.as_strided((1, 5), (2, 1)), 1, 5)):
        attention(table, B)
        got = _lib.SlKv4Attention.from_buffer_copy(blocks[-1][1][1])
        assert (got.table_stride, got.table_width, got.table) == (stride, table.shape[1], table.data_ptr())
        if stride:
            plan(table, B)
            got = _lib.SlKvPlan.from_buffer_copy(blocks[-1][1][0])
            assert (got.table_stride, got.table_width, got.table) == (stride, table.shape[1], table.data_ptr())


def test_a_table_that_grows_in_place_has_rows_of_its_own(blocks):
    one = on(torch.zeros((1, 5), dtype=I32))
    for table in (one.expand(3, -1), on(torch.zeros(9, dtype=I32)).as_strided((3, 5), (2, 1))):
        refused(lambda: plan(table))  # noqa: B023
    assert not blocks


def test_results_have_places_of_their_own(blocks):
    """Outputs that are one row, or one head, expanded are refused; expanded inputs are not, nor is a stride of zero where there is one row."""
    cache = on(torch.zeros((4, 2, 4, 18 * 64), dtype=torch.uint8))
    full, slots = on(torch.zeros((3, 2, 64), dtype=F16)), on(torch.zeros(3, dtype=I64))
    rows, heads = full[:1].expand(3, -1, -1), full[:, :1].expand(-1, 2, -1)
    table, lens, starts = on(torch.zeros((3, 5), dtype=I32)), ints(5, 5, 5), ints(0, 1, 2, 3)
    for bad in (rows, heads):
        refused(lambda: ops.kv4_append(cache, slots, full, q_out=bad))  # noqa: B023
        refused(lambda: ops.kv4_read(cache, slots, k=bad, v=full))  # noqa: B023
        refused(lambda: ops.kv4_read(cache, slots, k=full, v=bad))  # noqa: B023
        refused(lambda: ops.kv4_attention(cache, table, lens, full, starts, 1, out=bad))  # noqa: B023
        assert not blocks
        ops.kv4_append(cache, slots, bad, bad, bad, q_out=full)
        ops.kv4_attention(cache, table, lens, bad, starts, 1, gate=bad, out=full)
        assert len(blocks) == 2
        blocks.clear()
    one = full.as_strided((1, 2, 64), (0, 64, 1))
    ops.kv4_attention(cache, table[:1], ints(5), one, ints(0, 1), 1, out=one)
    assert blocks


def test_the_library_refuses_rows_that_overlap_in_part():
    """One row for all requests, but not rows that begin inside one another.  (Pointers that nothing follows: without a device the call
    that is in order ends there, with one it has no rows.)"""
    P = 1 << 20
    cache = _lib.SlKv4Cache(data=P, page_stride=2 * 4 * 18 * 128, pages=8, page_size=64, kv_heads=2, head_dim=128)
    for stride, width, want in ((0, 8, (0, _lib.SL_ERR_NO_DEVICE)), (0, 0, (0, _lib.SL_ERR_NO_DEVICE)), (8, 8, (0, _lib.SL_ERR_NO_DEVICE)),
                                (1, 8, (_lib.SL_ERR_INVALID,)), (-1, 8, (_lib.SL_ERR_INVALID,)), (-1, 0, (_lib.SL_ERR_INVALID,))):
        call = _lib.SlKv4Attention(q=P, q_row=1024, q_head=128, out=P, out_row=1024, out_head=128, rows=0, q_heads=8, q_start=P, kv_len=P, batch=2, max_q=2, table=P,
                                   table_stride=stride, table_width=width, causal=1, scale=0.1, workspace=P, workspace_bytes=1 << 40)
        assert _lib.lib().sl_op_kv4_attention_device(C.byref(cache), C.byref(call), None) in want


def test_the_workspace_is_that_of_the_tensors_device(monkeypatch):
    """Devices of different numbers of multiprocessors: the size is asked for with the call's device current, and kept for each."""
    import contextlib
    current, calls = [0], []

    class Lib:
        sl_kv4_attention_workspace = staticmethod(lambda *a: 1000 * (current[0] + 1))
        sl_kv4_attention_workspace_span = staticmethod(lambda *a: 10 * (current[0] + 1))

        @staticmethod
        def sl_op_kv4_attention_device(cache, block, stream):
            calls.append((current[0], _lib.SlKv4Attention.from_buffer_copy(block).workspace_bytes))
            return 0

    @contextlib.contextmanager
    def device(index):
        before, current[0] = current[0], index
        yield
        current[0] = before

    monkeypatch.setattr(ops, "lib", Lib)
    monkeypatch.setattr(ops, "_cuda", lambda: (lambda: current[0], lambda index: 0))
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(torch.cuda, "is_available", lambda: True)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: current[0])
    ops._workspace.cache_clear()

    def attend(kind, **kw):
        z = lambda *shape, dtype=I32: on(torch.zeros(shape, dtype=dtype), kind)  # noqa: E731
        ops.kv4_attention(z(4, 1, 4, 18 * 64, dtype=torch.uint8), z(3, 5), z(3), z(3, 2, 64, dtype=F16), z(4), 1, **{k: on(v, kind) for k, v in kw.items()})

    try:
        for now in (0, 1, 0):
            current[0] = now
            for kind in (OnDevice, OnAnother, OnDevice):
                attend(kind)
                assert calls.pop() == (kind.index, 10 * (kind.index + 1)) and current[0] == now
                attend(kind, workspace=torch.zeros(1000 * (kind.index + 1), dtype=torch.uint8))
                assert calls.pop() == (kind.index, 1000 * (kind.index + 1))
                refused(lambda: attend(kind, workspace=torch.zeros(1000 * (kind.index + 1) - 1, dtype=torch.uint8)))  # noqa: B023
            assert ops.kv4_attention_workspace(2, 1, 64, 3, 1, 3) == 1000 * (now + 1)
    finally:
        ops._workspace.cache_clear()

"""Single operators over the C ABI -- the counterparts of the reference's per-op wrappers
its kernel tests call (SeedlessMetalForward.qmm, routeTop8Rows, moeBlockRows, gdnLayerRows,
attnLayerRows: swift/Sources/QwispCore/SeedlessMetalForward.swift:222,
SeedlessVerifyForward.swift:37-248)."""
import collections
import ctypes as C
import functools
import struct

import numpy as np

from ._lib import SL_ERR_INVALID, SeedlessError, lib


def _p(a):
    return a.ctypes.data_as(C.c_void_p) if a is not None else None


def qmm4(x, packed, scales, biases):
    x = np.ascontiguousarray(x, dtype=np.float16)
    packed = np.ascontiguousarray(packed, dtype=np.uint32)
    scales = np.ascontiguousarray(scales, dtype=np.float16)
    biases = np.ascontiguousarray(biases, dtype=np.float16)
    M, K = x.shape
    N = packed.shape[0]
    y = np.empty((M, N), dtype=np.float16)
    rc = lib().sl_op_qmm4(_p(x), _p(packed), _p(scales), _p(biases), M, K, N, _p(y))
    if rc != 0:
        raise SeedlessError(rc, "sl_op_qmm4")
    return y


def quantize_q4(w):
    w = np.ascontiguousarray(w, dtype=np.float16)
    N, K = w.shape
    packed = np.empty((N, K // 8), dtype=np.uint32)
    s = np.empty((N, K // 64), dtype=np.float16)
    b = np.empty((N, K // 64), dtype=np.float16)
    rc = lib().sl_op_quantize_q4(_p(w), N, K, _p(packed), _p(s), _p(b))
    if rc != 0:
        raise SeedlessError(rc, "sl_op_quantize_q4")
    return packed, s, b


def moe_block(engine, layer, x):
    x = np.ascontiguousarray(x, dtype=np.float16)
    M = x.shape[0]
    out = np.empty_like(x)
    inds = np.empty((M, engine.cfg.top_k), dtype=np.int32)
    scores = np.empty((M, engine.cfg.top_k), dtype=np.float16)
    engine._check(lib().sl_op_moe_block(engine._h, layer, _p(x), M, _p(out), _p(inds), _p(scores)), "sl_op_moe_block")
    return out, inds, scores


def mixer(stream, layer, x, pos0):
    x = np.ascontiguousarray(x, dtype=np.float16)
    out = np.empty_like(x)
    stream.engine._check(lib().sl_op_mixer(stream._h, layer, _p(x), x.shape[0], pos0, _p(out)), "sl_op_mixer")
    return out


def read_kv(stream, layer_index, pos0, n):
    """Cached K (post-RoPE) and V of an attention layer at positions pos0..pos0+n-1: two fp16 [kv_heads, n, 256]."""
    cfg = stream.engine.cfg
    k = np.empty((cfg.attn_kv_heads, n, 256), dtype=np.float16)
    v = np.empty_like(k)
    stream.engine._check(lib().sl_op_read_kv(stream._h, layer_index, pos0, n, _p(k), _p(v)), "sl_op_read_kv")
    return k, v


def layer(stream, layer_index, h_in, pos0):
    h_in = np.ascontiguousarray(h_in, dtype=np.float16)
    out = np.empty_like(h_in)
    stream.engine._check(lib().sl_op_layer(stream._h, layer_index, _p(h_in), h_in.shape[0], pos0, _p(out)), "sl_op_layer")
    return out


def head(engine, h_rows, want_logits=True):
    h_rows = np.ascontiguousarray(h_rows, dtype=np.float16)
    M = h_rows.shape[0]
    logits = np.empty((M, engine.cfg.vocab), dtype=np.float16) if want_logits else None
    toks = np.empty(M, dtype=np.int32)
    engine._check(lib().sl_op_head(engine._h, _p(h_rows), M, _p(logits), _p(toks)), "sl_op_head")
    return logits, toks


def lm_head(engine, normed, want_logits=True):
    normed = np.ascontiguousarray(normed, dtype=np.float16)
    M = normed.shape[0]
    logits = np.empty((M, engine.cfg.vocab), dtype=np.float16) if want_logits else None
    toks = np.empty(M, dtype=np.int32)
    engine._check(lib().sl_op_lm_head(engine._h, _p(normed), M, _p(logits), _p(toks)), "sl_op_lm_head")
    return logits, toks


def synth_tokens(seed, name, n, vocab):
    out = np.empty(n, dtype=np.int32)
    rc = lib().sl_synth_tokens(seed, name.encode(), n, vocab, _p(out))
    if rc != 0:
        raise SeedlessError(rc, "sl_synth_tokens")
    return out


def synth_f16(seed, name, n, mean=0.0, std=1.0):
    out = np.empty(n, dtype=np.float16)
    rc = lib().sl_synth_f16(seed, name.encode(), n, mean, std, _p(out))
    if rc != 0:
        raise SeedlessError(rc, "sl_synth_f16")
    return out


def sample_rows(engine, logits, draft, inv_t, top_p, seed_lo, seed_hi, base_pos, logit_adj=None):
    """The sampling kernel on host logits [M, vocab] fp16 -> (full, resid, accept) int32 [M].
    logit_adj: optional f32 [vocab] added to every row first (penalties + bias)."""
    logits = np.ascontiguousarray(logits, dtype=np.float16)
    M = logits.shape[0]
    d = None if draft is None else np.ascontiguousarray(draft, dtype=np.int32)
    adj = None if logit_adj is None else np.ascontiguousarray(logit_adj, dtype=np.float32)
    full, resid, acc = (np.empty(M, dtype=np.int32) for _ in range(3))
    engine._check(lib().sl_op_sample_rows(engine._h, _p(logits), M, _p(d) if d is not None else None,
                                          _p(adj) if adj is not None else None, float(inv_t), float(top_p),
                                          int(seed_lo), int(seed_hi), int(base_pos), _p(full), _p(resid), _p(acc)), "sl_op_sample_rows")
    return full, resid, acc


# ---------------------------------------------------------------------------------------------- a KV cache held in 4 bits
# These take CUDA tensors and run on their device's current stream; nothing is synchronised.  A cache is a uint8 tensor
# [pages, kv heads, page size / 16, 18 * head dim] (include/seedless_b200.h has the layout); its pages may lie further apart than one
# page is long (a layer of an arena whose pages hold several).  A decode step calls three of them per layer, so they are lean: one look
# at each tensor's type, shape and device here, alignment and ranges in the library, argument blocks packed in one go.
KvPlan = collections.namedtuple("KvPlan", "kv_len q_start slots pos free_count status")
_CACHE, _PLAN = struct.Struct("@Pqiiii"), struct.Struct("@PPiiPqiPiPPPPPiPP0q")
_APPEND, _READ = struct.Struct("@PPPqqqqqqPqqiiPPfPqiifPP0q"), struct.Struct("@PiPPqqqq0q")
_ATTENTION = struct.Struct("@PqqPqqPqqiiPPiiPqiifPQ0q")


def _no(where, what):
    return SeedlessError(SL_ERR_INVALID, where, what)


@functools.lru_cache(maxsize=1)
def _cuda():
    """(current device, current stream of a device) as numbers.  (torch's own accessors where it has them: a Stream object is 1.5 us.)"""
    import torch
    return (getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device),
            getattr(torch._C, "_cuda_getCurrentRawStream", lambda index: torch.cuda.current_stream(index).cuda_stream))


def _on(index, fn, *args):
    """fn's result with that device current."""
    if _cuda()[0]() == index:
        return fn(*args)
    import torch
    with torch.cuda.device(index):
        return fn(*args)


def _call(fn, index, where, *blocks):
    """The call on the device's current stream."""
    rc = _on(index, fn, *blocks, _cuda()[1](index))
    if rc != 0:
        raise SeedlessError(rc, where)


def _heads(where, name, t, shape, index):
    """(pointer, row stride, head stride) of fp16 [rows, heads, dim] on that device."""
    import torch
    by = t.stride()
    if t.dtype is not torch.float16 or t.shape != shape or by[2] != 1 or t.get_device() != index:
        raise _no(where, f"{name} has to be fp16 {list(shape)} on the cache's device, a head's dims contiguous")
    return t.data_ptr(), by[0], by[1]


def _heads_out(where, name, t, shape, index):
    """The same of one that is written: an expanded one has one place for many results."""
    at = _heads(where, name, t, shape, index)
    if (at[1] == 0 and shape[0] > 1) or (at[2] == 0 and shape[1] > 1):
        raise _no(where, f"{name} is written: its rows and heads must not overlap")
    return at


def _flat(where, name, t, dtype, n, index):
    """The pointer of a contiguous tensor of n values (None: any number) on that device."""
    if t.dtype is not dtype or (n is not None and t.shape != (n,)) or not t.is_contiguous() or t.get_device() != index:
        raise _no(where, f"{name} has to be contiguous {dtype}{'' if n is None else ' [%d]' % n} on the call's device")
    return t.data_ptr()


def _cache(where, cache):
    """(argument block, page size, kv heads, head dim, device index) of a cache."""
    import torch
    shape, by, index = cache.shape, cache.stride(), cache.get_device()
    if len(shape) != 4 or cache.dtype is not torch.uint8 or index < 0 or shape[3] not in (18 * 64, 18 * 128, 18 * 256) or not cache.numel() or \
            by[3] != 1 or (by[2] != shape[3] and shape[2] > 1) or (by[1] != shape[2] * shape[3] and shape[1] > 1):
        raise _no(where, "a cache is a CUDA tensor uint8 [pages, kv heads, page size / 16, 18 * head dim] of whole pages")
    pages, kv, blocks, size = shape
    return _CACHE.pack(cache.data_ptr(), by[0] if pages > 1 else kv * blocks * size, pages, blocks * 16, kv, size // 18), blocks * 16, kv, size // 18, index


def kv4_cache(pages, page_size, kv_heads, head_dim, device="cuda"):
    """An empty cache for one layer."""
    import torch
    if lib().sl_kv4_page_bytes(kv_heads, head_dim, page_size) < 0 or pages < 1:
        raise _no("kv4_cache", "page_size is a multiple of 16, head_dim 64, 128 or 256")
    return torch.zeros((pages, kv_heads, page_size // 16, 18 * head_dim), dtype=torch.uint8, device=device)


def kv_plan(lens, new_rows, table, free_pages, free_count, page_size, max_rows, out=None):
    """Page tables, slot map, positions and row offsets of a step from the requests' lengths: KvPlan(kv_len [B], q_start [B + 1],
    slots int64 [max_rows], pos [max_rows], free_count [1], status [3]).  table [B, width] grows in place by pages off the top of the
    stack free_pages[: free_count]; new_rows[b] < 0 gives an ended request's pages back.  status other than zeros (pages short,
    requests out of range, rows beyond max_rows): nothing was planned.  out: a KvPlan to write into, whose kv_len may be lens and
    whose free_count may be free_count."""
    import torch
    where, i32, index = "sl_op_kv_plan_device", torch.int32, lens.get_device()
    if index < 0 or lens.dim() != 1 or table.dim() != 2 or max_rows < 0:
        raise _no(where, "lens and new_rows are CUDA int32 [B], table int32 [B, pages]")
    B, (rows, width), by = lens.shape[0], table.shape, table.stride()
    if rows != B or table.dtype is not i32 or (by[1] != 1 and width > 1) or table.get_device() != index:
        raise _no(where, f"table has to be int32 [{B}, pages] on the call's device")
    if B > 1 and by[0] < width:                                            # (an expanded one: its requests would write each other's pages)
        raise _no(where, "the table's rows must not overlap")
    at = [_flat(where, "lens", lens, i32, B, index), _flat(where, "new_rows", new_rows, i32, B, index), _flat(where, "free_pages", free_pages, i32, None, index),
          _flat(where, "free_count", free_count, i32, 1, index)]
    if out is None:                                                        # one allocation
        buf = lens.new_empty(3 * max_rows + 2 * B + 5)
        slots, kv_len, q_start, pos, count, status = torch.split_with_sizes(buf, (2 * max_rows, B, B + 1, max_rows, 1, 3))
        out, p, n = KvPlan(kv_len, q_start, slots.view(torch.int64), pos, count, status), buf.data_ptr(), 8 * max_rows
        to = (p + n, p + n + 4 * B, p, p + n + 8 * B + 4, p + n + 8 * B + 4 + 4 * max_rows, p + n + 8 * B + 8 + 4 * max_rows)
    else:
        to = [_flat(where, name + " out", t, torch.int64 if name == "slots" else i32, n, index) for name, t, n in zip(KvPlan._fields, out, (B, B + 1, max_rows, max_rows, 1, 3))]
    _call(lib().sl_op_kv_plan_device, index, where, _PLAN.pack(at[0], at[1], B, page_size, table.data_ptr(), by[0] if B > 1 else width, width, at[2], free_pages.shape[0], at[3], *to[:4], max_rows, *to[4:]))
    return out


def kv4_append(cache, slots, q=None, k=None, v=None, *, q_norm=None, k_norm=None, eps=1e-6, pos=None, rope_dims=0, rope_theta=1e7,
               axis_of=None, q_out=None):
    """Norms of queries and keys, rotation, and K and V into the cache at slots int64 [rows].  q [rows, heads, dim], k and v [rows, kv
    heads, dim] fp16; pos int32 [rows] or [axes, rows], axis_of: the position axis of each of the rope_dims / 2 frequencies (None: the
    first).  Returns the rotated queries (q_out, which may be q; None without q).  Rows whose slot is not one of the cache's are padding:
    nothing of them is written, so that without q_out they hold anything."""
    import torch
    where = "sl_op_kv4_append_device"
    block, _, kv, dim, index = _cache(where, cache)
    if (k is None) != (v is None) or (q is None and k is None):
        raise _no(where, "k and v come together, or queries alone")
    qa = oa = ka = va = (0, 0, 0)
    heads, axes, pa, apart, table, sa, qn, kn = 0, 0, 0, 0, 0, 0, 0, 0
    rows = (k if q is None else q).shape[0]
    if q is not None:
        heads = q.shape[1] if q.dim() == 3 else 0
        qa = _heads(where, "q", q, (rows, heads, dim), index)
        if q_out is None:
            q_out = torch.empty_like(q) if q.is_contiguous() else q.new_empty((rows, heads, dim))
            oa = (q_out.data_ptr(), heads * dim, dim)
        else:
            oa = _heads_out(where, "q_out", q_out, (rows, heads, dim), index)
    if k is not None:
        ka, va = _heads(where, "k", k, (rows, kv, dim), index), _heads(where, "v", v, (rows, kv, dim), index)
        if slots is None:
            raise _no(where, "k and v need slots")
    if q_norm is not None:
        qn = _flat(where, "q_norm", q_norm, torch.float16, dim, index)
    if k_norm is not None:
        kn = _flat(where, "k_norm", k_norm, torch.float16, dim, index)
    if slots is not None:
        sa = _flat(where, "slots", slots, torch.int64, rows, index)
    if rope_dims:
        if pos is None or pos.dtype is not torch.int32 or pos.dim() not in (1, 2) or pos.shape[-1] != rows or (pos.stride(-1) != 1 and rows > 1) or pos.get_device() != index:
            raise _no(where, f"pos has to be int32 [{rows}] or [axes, {rows}] on the call's device")
        axes, apart = (1, 0) if pos.dim() == 1 else (pos.shape[0], pos.stride(0))
        pa = pos.data_ptr()
        if axis_of is not None:
            try:
                table = bytes(axis_of)
            except (TypeError, ValueError):
                table = b""
            if len(table) != rope_dims // 2:
                raise _no(where, f"axis_of has one of {axes} axes for each of {rope_dims // 2} frequencies")
            table = C.create_string_buffer(table, max(1, len(table)))      # (lives until the call returns)
    if rows:
        _call(lib().sl_op_kv4_append_device, index, where, block, _APPEND.pack(qa[0], ka[0], va[0], qa[1], qa[2], ka[1], ka[2], va[1], va[2], *oa, rows, heads, qn, kn, eps,
                                                                             pa, apart, axes, rope_dims, rope_theta, C.addressof(table) if table else 0, sa))
    return q_out


def kv4_read(cache, slots, k=None, v=None):
    """K and V at slots int64 [rows] as fp16 [rows, kv heads, dim] (into k and v if given).  Rows whose slot is not one of the
    cache's stay as they were: in new tensors, anything."""
    import torch
    where = "sl_op_kv4_read_device"
    block, _, kv, dim, index = _cache(where, cache)
    rows = slots.shape[0] if slots.dim() == 1 else -1
    sa = _flat(where, "slots", slots, torch.int64, rows, index)
    shape = (rows, kv, dim)
    if k is None:
        k = cache.new_empty(shape, dtype=torch.float16)
        kp, kr, kh = k.data_ptr(), kv * dim, dim
    else:
        kp, kr, kh = _heads_out(where, "k", k, shape, index)
    if v is None:
        v = torch.empty_like(k) if k.is_contiguous() else cache.new_empty(shape, dtype=torch.float16)
        vp, vr, vh = v.data_ptr(), kv * dim, dim
    else:
        vp, vr, vh = _heads_out(where, "v", v, shape, index)
    if rows:
        _call(lib().sl_op_kv4_read_device, index, where, block, _READ.pack(sa, rows, kp, vp, kr, kh, vr, vh))
    return k, v


@functools.lru_cache(maxsize=256)
def _workspace(index, q_heads, kv_heads, head_dim, batch, max_q, span):
    """Bytes of workspace of such a call on that device (-1: whichever is current), by its number of multiprocessors; span None: tables of any width."""
    call = (q_heads, kv_heads, head_dim, batch, max_q)
    fn, where, more = (lib().sl_kv4_attention_workspace, "sl_kv4_attention_workspace", 0) if span is None else \
        (lib().sl_kv4_attention_workspace_span, "sl_kv4_attention_workspace_span", span)
    n = fn(*call, more) if index < 0 else _on(index, fn, *call, more)
    if n < 0:
        raise SeedlessError(n, where)
    return n


def kv4_attention_workspace(q_heads, kv_heads, head_dim, batch, max_q, rows):
    """Bytes of workspace of such a call of kv4_attention on the current device."""
    import torch
    if rows < 0:
        raise _no("sl_kv4_attention_workspace", "rows is not negative")
    return _workspace(torch.cuda.current_device() if torch.cuda.is_available() else -1, q_heads, kv_heads, head_dim, batch, max_q, None)


def kv4_attention(cache, table, kv_len, q, q_start, max_q, *, causal=True, scale=None, gate=None, out=None, workspace=None):
    """softmax(scale q K^T) V [* sigmoid(gate)] over the cache: q [rows, heads, dim] fp16, request b's rows q_start[b] .. q_start[b + 1] - 1 (at most
    max_q) over its positions 0 .. kv_len[b] - 1 in the pages table[b] (one row expanded to all requests will do where they share them);
    causal: its rows are its last positions.  scale: dim ** -0.5 if None.  A row that sees no position is zero; rows of no request stay as they
    were: without out, anything.  The kernels take the table's width for the longest request's length, so cut a wide table to the step's
    (table[:, :n]) where that is known: one row over 513 positions takes the GPU 8.2 us, and 14.4 with a table for 32768.  workspace: a uint8
    tensor of kv4_attention_workspace() bytes, allocated for the call if None; calls that may run at the same time need one each."""
    import torch
    where, i32 = "sl_op_kv4_attention_device", torch.int32
    block, page, kv, dim, index = _cache(where, cache)
    if q.dim() != 3 or table.dim() != 2 or kv_len.dim() != 1 or max_q < 1:
        raise _no(where, "q is [rows, heads, dim], table int32 [B, pages], kv_len int32 [B], q_start int32 [B + 1]")
    shape, B, by = q.shape, kv_len.shape[0], table.stride()
    rows, heads = shape[0], shape[1]
    width = table.shape[1]
    if table.shape[0] != B or table.dtype is not i32 or (by[1] != 1 and width > 1) or table.get_device() != index:
        raise _no(where, f"table has to be int32 [{B}, pages] on the call's device")
    qa = _heads(where, "q", q, (rows, heads, dim), index)
    if out is None:
        out = torch.empty_like(q) if q.is_contiguous() else q.new_empty(shape)
        oa = (out.data_ptr(), heads * dim, dim)
    else:
        oa = _heads_out(where, "out", out, shape, index)
    ga = (0, 0, 0) if gate is None else _heads(where, "gate", gate, shape, index)
    la, ra = _flat(where, "kv_len", kv_len, i32, B, index), _flat(where, "q_start", q_start, i32, B + 1, index)
    if workspace is None:
        size = _workspace(index, heads, kv, dim, B, max_q, width * page)
        if size:
            workspace = torch.empty(size, dtype=torch.uint8, device=q.device)
        wa = workspace.data_ptr() if size else qa[0]
    else:
        need, size = _workspace(index, heads, kv, dim, B, max_q, None), workspace.numel()
        if size < need:
            raise _no(where, f"workspace has to have {need} bytes")
        wa = _flat(where, "workspace", workspace, torch.uint8, None, index)
    if rows:
        _call(lib().sl_op_kv4_attention_device, index, where, block,
              _ATTENTION.pack(*qa, *ga, *oa, rows, heads, ra, la, B, max_q, table.data_ptr(), by[0] if B > 1 else width, width, 1 if causal else 0,
                              dim ** -0.5 if scale is None else scale, wa, size))
    return out

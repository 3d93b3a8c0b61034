"""Single operators over the C ABI -- the counterparts of the reference's per-op wrappers
its kernel tests call (SeedlessMetalForward.qmm, routeTop8Rows, moeBlockRows, gdnLayerRows,
attnLayerRows: swift/Sources/QwispCore/SeedlessMetalForward.swift:222,
SeedlessVerifyForward.swift:37-248)."""
import collections
import ctypes as C

import numpy as np

from ._lib import SL_ERR_INVALID, SeedlessError, SlKv4Append, SlKv4Attention, SlKv4Cache, SlKv4Read, SlKvPlan, lib


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
# page is long (a layer of an arena whose pages hold several).
KvPlan = collections.namedtuple("KvPlan", "kv_len q_start slots pos free_count status")


def _no(where, what):
    return SeedlessError(SL_ERR_INVALID, where, what)


def _call(fn, device, where, *structs):
    import torch
    if device.index == torch.cuda.current_device():
        rc = fn(*[C.byref(s) for s in structs], torch.cuda.current_stream(device).cuda_stream)
    else:
        with torch.cuda.device(device):
            rc = fn(*[C.byref(s) for s in structs], torch.cuda.current_stream(device).cuda_stream)
    if rc != 0:
        raise SeedlessError(rc, where)


def _same(where, device, **tensors):
    for name, t in tensors.items():
        if t is not None and t.device != device:
            raise _no(where, f"{name} is on {t.device}, the call on {device}")


def _whole(where, dtype, **tensors):
    for name, t in tensors.items():
        if t.dtype != dtype or not t.is_contiguous():
            raise _no(where, f"{name} has to be contiguous and {dtype}")


def _heads(where, name, t, rows, heads, dim):
    """A tensor [rows, heads, dim] of halves whose heads the kernels can address; None passes."""
    if t is not None and (str(t.dtype) != "torch.float16" or tuple(t.shape) != (rows, heads, dim) or t.stride(2) != 1 or
                          t.stride(0) % 8 or t.stride(1) % 8 or t.data_ptr() % 16):
        raise _no(where, f"{name} has to be fp16 [{rows}, {heads}, {dim}], a head's dims contiguous and on a 16-byte boundary")


def _cache(where, cache):
    pages, kv, blocks, size = cache.shape if cache.dim() == 4 else (0, 0, 0, 0)
    if str(cache.dtype) != "torch.uint8" or not cache.is_cuda or size not in (18 * 64, 18 * 128, 18 * 256) or not pages * kv * blocks or \
            cache.stride(3) != 1 or (blocks > 1 and cache.stride(2) != size) or (kv > 1 and cache.stride(1) != blocks * size):
        raise _no(where, "a cache is a CUDA tensor uint8 [pages, kv heads, page size / 16, 18 * head dim] of whole pages")
    stride = cache.stride(0) if pages > 1 else kv * blocks * size
    return SlKv4Cache(cache.data_ptr(), stride, pages, blocks * 16, kv, size // 18)


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
    where, dev, B = "sl_op_kv_plan_device", lens.device, lens.numel()
    if not lens.is_cuda or new_rows.shape != (B,) or table.dim() != 2 or table.shape[0] != B or table.dtype != torch.int32 or \
            (table.numel() and table.stride(1) != 1) or max_rows < 0:
        raise _no(where, "lens and new_rows are CUDA int32 [B], table int32 [B, pages]")
    if out is None:
        i32 = lambda n: torch.empty(n, dtype=torch.int32, device=dev)  # noqa: E731
        out = KvPlan(i32(B), i32(B + 1), torch.empty(max_rows, dtype=torch.int64, device=dev), i32(max_rows), i32(1), i32(3))
    elif [t.numel() for t in out] != [B, B + 1, max_rows, max_rows, 1, 3]:
        raise _no(where, "out has other sizes")
    _same(where, dev, new_rows=new_rows, table=table, free_pages=free_pages, free_count_in=free_count, **out._asdict())
    _whole(where, torch.int32, lens=lens, new_rows=new_rows, free_pages=free_pages, free_count_in=free_count, kv_len=out.kv_len, q_start=out.q_start,
           pos=out.pos, free_count=out.free_count, status=out.status)
    _whole(where, torch.int64, slots=out.slots)
    if free_count.numel() != 1:
        raise _no(where, "free_count is one number")
    p = SlKvPlan(lens.data_ptr(), new_rows.data_ptr(), B, page_size, table.data_ptr(), max(table.stride(0), table.shape[1]), table.shape[1],
                 free_pages.data_ptr(), free_pages.numel(), free_count.data_ptr(), out.kv_len.data_ptr(), out.q_start.data_ptr(),
                 out.slots.data_ptr(), out.pos.data_ptr(), max_rows, out.free_count.data_ptr(), out.status.data_ptr())
    _call(lib().sl_op_kv_plan_device, dev, where, p)
    return out


def kv4_append(cache, slots, q=None, k=None, v=None, *, q_norm=None, k_norm=None, eps=1e-6, pos=None, rope_dims=0, rope_theta=1e7,
               axis_of=None, q_out=None):
    """Norms of queries and keys, rotation, and K and V into the cache at slots int64 [rows].  q [rows, heads, dim], k and v [rows, kv
    heads, dim] fp16; pos int32 [rows] or [axes, rows], axis_of: the position axis of each of the rope_dims / 2 frequencies (None: the
    first).  Returns the rotated queries (q_out, which may be q; None without q).  Rows whose slot is not one of the cache's are padding."""
    import torch
    where, c = "sl_op_kv4_append_device", _cache("sl_op_kv4_append_device", cache)
    dev, dim = cache.device, c.head_dim
    if (k is None) != (v is None) or (q is None and k is None):
        raise _no(where, "k and v come together, or queries alone")
    rows, heads = (q if q is not None else k).shape[0], 0 if q is None else q.shape[1]
    if q is not None and q_out is None:
        q_out = torch.empty((rows, heads, dim), dtype=torch.float16, device=dev)
    for name, t, n in (("q", q, heads), ("q_out", q_out, heads), ("k", k, c.kv_heads), ("v", v, c.kv_heads)):
        _heads(where, name, t, rows, n, dim)
    for name, t in (("q_norm", q_norm), ("k_norm", k_norm)):
        if t is not None and (t.dtype != torch.float16 or tuple(t.shape) != (dim,) or not t.is_contiguous() or t.data_ptr() % 16):
            raise _no(where, f"{name} has to be fp16 [{dim}]")
    if slots is None and k is not None:
        raise _no(where, "k and v need slots")
    if slots is not None and (slots.dtype != torch.int64 or tuple(slots.shape) != (rows,) or not slots.is_contiguous()):
        raise _no(where, f"slots has to be contiguous int64 [{rows}]")
    axes, table = 0, None
    if rope_dims:
        if pos is None or pos.dtype != torch.int32 or pos.shape[-1] != rows or pos.dim() not in (1, 2) or (rows > 1 and pos.stride(-1) != 1):
            raise _no(where, f"pos has to be int32 [{rows}] or [axes, {rows}]")
        axes = 1 if pos.dim() == 1 else pos.shape[0]
        if axis_of is not None:
            if len(axis_of) != rope_dims // 2 or not all(0 <= i < min(axes, 256) for i in axis_of):
                raise _no(where, f"axis_of has one of {axes} axes for each of {rope_dims // 2} frequencies")
            table = bytes(axis_of)
    _same(where, dev, q=q, k=k, v=v, q_out=q_out, q_norm=q_norm, k_norm=k_norm, pos=pos, slots=slots)
    at = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    by = lambda t: (0, 0) if t is None else (t.stride(0), t.stride(1))  # noqa: E731
    p = SlKv4Append(at(q), at(k), at(v), *by(q), *by(k), *by(v), at(q_out), *by(q_out), rows, heads, at(q_norm), at(k_norm), eps,
                    at(pos) if rope_dims else None, pos.stride(0) if rope_dims and pos.dim() == 2 else 0, axes, rope_dims, rope_theta, table, at(slots))
    if rows:
        _call(lib().sl_op_kv4_append_device, dev, where, c, p)
    return q_out


def kv4_read(cache, slots, k=None, v=None):
    """K and V at slots int64 [rows] as fp16 [rows, kv heads, dim] (into k and v if given).  Rows whose slot is not one of the
    cache's stay as they were."""
    import torch
    where, c = "sl_op_kv4_read_device", _cache("sl_op_kv4_read_device", cache)
    if slots.dtype != torch.int64 or slots.dim() != 1 or not slots.is_contiguous():
        raise _no(where, "slots has to be contiguous int64 [rows]")
    shape = (slots.numel(), c.kv_heads, c.head_dim)
    k, v = (torch.empty(shape, dtype=torch.float16, device=cache.device) if t is None else t for t in (k, v))
    _heads(where, "k", k, *shape)
    _heads(where, "v", v, *shape)
    _same(where, cache.device, slots=slots, k=k, v=v)
    p = SlKv4Read(slots.data_ptr(), shape[0], k.data_ptr(), v.data_ptr(), k.stride(0), k.stride(1), v.stride(0), v.stride(1))
    if shape[0]:
        _call(lib().sl_op_kv4_read_device, cache.device, where, c, p)
    return k, v


def kv4_attention_workspace(q_heads, kv_heads, head_dim, batch, max_q, rows):
    """Bytes of workspace of such a call of kv4_attention."""
    n = lib().sl_kv4_attention_workspace(q_heads, kv_heads, head_dim, batch, max_q, rows)
    if n < 0:
        raise SeedlessError(n, "sl_kv4_attention_workspace")
    return n


def kv4_attention(cache, table, kv_len, q, q_start, max_q, *, causal=True, scale=None, gate=None, out=None, workspace=None):
    """softmax(scale q K^T) V [* sigmoid(gate)] over the cache: q [rows, heads, dim] fp16, request b's rows q_start[b] .. q_start[b + 1] - 1 (at most
    max_q) over its positions 0 .. kv_len[b] - 1 in the pages table[b]; causal: its rows are its last positions.  scale: dim ** -0.5 if
    None.  A row that sees no position is zero.  workspace: a uint8 tensor of kv4_attention_workspace() bytes, allocated for the call
    if None; calls that may run at the same time need one each."""
    import torch
    where, c = "sl_op_kv4_attention_device", _cache("sl_op_kv4_attention_device", cache)
    dev, dim, B = cache.device, c.head_dim, kv_len.numel()
    if q.dim() != 3 or table.dim() != 2 or table.shape[0] != B or table.dtype != torch.int32 or (table.numel() and table.stride(1) != 1) or \
            q_start.numel() != B + 1 or max_q < 1:
        raise _no(where, "q is [rows, heads, dim], table int32 [B, pages], kv_len int32 [B], q_start int32 [B + 1]")
    rows, heads = q.shape[:2]
    if out is None:
        out = torch.empty((rows, heads, dim), dtype=torch.float16, device=dev)
    for name, t in (("q", q), ("gate", gate), ("out", out)):
        _heads(where, name, t, rows, heads, dim)
    _whole(where, torch.int32, kv_len=kv_len, q_start=q_start)
    need = kv4_attention_workspace(heads, c.kv_heads, dim, B, max_q, rows)
    if workspace is None:
        workspace = torch.empty(need, dtype=torch.uint8, device=dev)
    elif workspace.dtype != torch.uint8 or not workspace.is_contiguous() or workspace.numel() < need:
        raise _no(where, f"workspace has to be contiguous uint8 of {need} bytes")
    _same(where, dev, table=table, kv_len=kv_len, q=q, q_start=q_start, gate=gate, out=out, workspace=workspace)
    g = (None, 0, 0) if gate is None else (gate.data_ptr(), gate.stride(0), gate.stride(1))
    p = SlKv4Attention(q.data_ptr(), q.stride(0), q.stride(1), *g, out.data_ptr(), out.stride(0), out.stride(1), rows, heads,
                       q_start.data_ptr(), kv_len.data_ptr(), B, max_q, table.data_ptr(), max(table.stride(0), table.shape[1]), table.shape[1],
                       1 if causal else 0, dim ** -0.5 if scale is None else scale, workspace.data_ptr(), workspace.numel())
    if rows:
        _call(lib().sl_op_kv4_attention_device, dev, where, c, p)
    return out

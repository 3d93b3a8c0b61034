// kv4_api.cu -- C entry points of the operators around the cache held in 4 bits: arguments checked, then the kernel enqueued.
#include "../../include/seedless_b200.h"
#include "kv4.cuh"
#include <algorithm>
#include <cmath>
#include <cstdio>

using namespace sl;

namespace {
constexpr int KV4_HEADS = 65535;                             // (a grid's second axis)
bool aligned(const void* p, int64_t row, int64_t head) { return ((uintptr_t)p & 15) == 0 && row % 8 == 0 && head % 8 == 0; }
// a cache that the kernels can address; its geometry as they take it
bool cache_of(const sl_kv4_cache* c, Kv4Cache& o) {
    if (!c || !c->data || ((uintptr_t)c->data & 15) || c->pages <= 0 || c->kv_heads <= 0 || c->kv_heads > KV4_HEADS || c->page_size <= 0 || c->page_size % KV4_B) return false;
    if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256) return false;
    if (c->page_stride % 16 || c->page_stride < sl_kv4_page_bytes(c->kv_heads, c->head_dim, c->page_size)) return false;
    o = Kv4Cache{(unsigned char*)c->data, c->page_stride, c->pages, c->page_size, c->kv_heads, c->head_dim};
    return true;
}
// The status of a call's launches, which report their own errors: one that another call has left behind is not looked at, and none is left.
int32_t launched(int err, const char* what) {
    if (err == 0) return SL_OK;
    cudaGetLastError();
    fprintf(stderr, "%s: CUDA error %d (%s)\n", what, err, cudaGetErrorString((cudaError_t)err));
    return SL_ERR_CUDA;
}
}  // namespace

extern "C" {

int64_t sl_kv4_page_bytes(int32_t kv_heads, int32_t head_dim, int32_t page_size) {
    if (kv_heads <= 0 || page_size <= 0 || page_size % KV4_B || (head_dim != 64 && head_dim != 128 && head_dim != 256)) return SL_ERR_INVALID;
    return (int64_t)kv_heads * (page_size / KV4_B) * kv4_block_bytes(head_dim);
}
int32_t sl_op_kv_plan_device(const sl_kv_plan* p, void* cuda_stream) try {
    if (!p || p->batch < 0 || p->max_rows < 0 || p->page_size <= 0 || p->table_width < 0 || p->free_capacity < 0) return SL_ERR_INVALID;
    if (!p->q_start || !p->free_count || !p->free_count_out || !p->status || (p->max_rows && (!p->slots || !p->pos))) return SL_ERR_INVALID;
    if (p->batch && (!p->lens || !p->new_rows || !p->kv_len || (!p->table && p->table_width) || (!p->free_pages && p->free_capacity) || p->table_stride < p->table_width)) return SL_ERR_INVALID;
    if ((int64_t)p->batch * p->table_width > 0x7fffffffll) return SL_ERR_CAPACITY;
    if (!device_ok()) return SL_ERR_NO_DEVICE;
    KvPlanArgs a{p->lens, p->new_rows, p->batch, p->page_size, p->table, p->table_stride, p->table_width, p->free_pages, p->free_capacity, p->free_count,
                 p->kv_len, p->q_start, p->slots, p->pos, p->max_rows, p->free_count_out, p->status};
    return launched(launch_kv_plan(a, (cudaStream_t)cuda_stream), "sl_op_kv_plan_device");
} catch (...) {
    return SL_ERR_CAPACITY;                                   // no host memory
}
int32_t sl_op_kv4_append_device(const sl_kv4_cache* cache, const sl_kv4_append* p, void* cuda_stream) try {
    Kv4Cache c{};
    if (!p || !cache_of(cache, c) || p->rows < 0 || p->q_heads < 0 || p->q_heads > KV4_HEADS || (!p->q && !p->k) || !p->k != !p->v) return SL_ERR_INVALID;
    if (p->q && (!p->q_out || p->q_heads == 0 || !aligned(p->q, p->q_row, p->q_head) || !aligned(p->q_out, p->q_out_row, p->q_out_head))) return SL_ERR_INVALID;
    if (p->k && (!p->slots || !aligned(p->k, p->k_row, p->k_head) || !aligned(p->v, p->v_row, p->v_head))) return SL_ERR_INVALID;
    if (!aligned(p->q_norm, 0, 0) || !aligned(p->k_norm, 0, 0) || !(p->eps >= 0.f)) return SL_ERR_INVALID;
    if (p->rope_dims < 0 || p->rope_dims > c.D || p->rope_dims % 16 || p->axes < 0) return SL_ERR_INVALID;
    Kv4AppendArgs a{};
    if (p->rope_dims) {
        if (!p->pos || p->axes < 1 || !(p->rope_theta >= 1.f) || !std::isfinite(p->rope_theta)) return SL_ERR_INVALID;
        for (int i = 0; i < p->rope_dims / 2; ++i) {
            a.axis[i] = p->axis_of ? p->axis_of[i] : 0;
            if (a.axis[i] >= p->axes) return SL_ERR_INVALID;
            // theta^(-2 i / dims) radians a position, as a 64-bit fraction of a turn
            a.turn[i] = (uint64_t)std::ldexp(std::pow((double)p->rope_theta, -2.0 * i / p->rope_dims) * 0.15915494309189533577, 64);
        }
    }
    if (!device_ok()) return SL_ERR_NO_DEVICE;
    if (p->rows == 0) return SL_OK;
    a.q = (const __half*)p->q; a.q_row = p->q_row; a.q_head = p->q_head;
    a.k = (const __half*)p->k; a.k_row = p->k_row; a.k_head = p->k_head;
    a.v = (const __half*)p->v; a.v_row = p->v_row; a.v_head = p->v_head;
    a.q_out = (__half*)p->q_out; a.o_row = p->q_out_row; a.o_head = p->q_out_head;
    a.rows = p->rows; a.NH = p->q_heads; a.q_norm = (const __half*)p->q_norm; a.k_norm = (const __half*)p->k_norm; a.eps = p->eps;
    a.pos = p->pos; a.pos_axis = p->pos_axis; a.rope = p->rope_dims; a.slots = p->slots;
    return launched(launch_kv4_append(c, a, (cudaStream_t)cuda_stream), "sl_op_kv4_append_device");
} catch (...) {
    return SL_ERR_CAPACITY;                                   // no host memory
}
int32_t sl_op_kv4_read_device(const sl_kv4_cache* cache, const sl_kv4_read* p, void* cuda_stream) try {
    Kv4Cache c{};
    if (!p || !cache_of(cache, c) || p->rows < 0 || !p->slots || !p->k || !p->v) return SL_ERR_INVALID;
    if (!aligned(p->k, p->k_row, p->k_head) || !aligned(p->v, p->v_row, p->v_head)) return SL_ERR_INVALID;
    if (!device_ok()) return SL_ERR_NO_DEVICE;
    if (p->rows == 0) return SL_OK;
    Kv4ReadArgs a{p->slots, p->rows, (__half*)p->k, (__half*)p->v, p->k_row, p->k_head, p->v_row, p->v_head};
    return launched(launch_kv4_read(c, a, (cudaStream_t)cuda_stream), "sl_op_kv4_read_device");
} catch (...) {
    return SL_ERR_CAPACITY;                                   // no host memory
}
int64_t sl_kv4_attention_workspace(int32_t q_heads, int32_t kv_heads, int32_t head_dim, int32_t batch, int32_t max_q, int32_t rows) {
    if (kv_heads <= 0 || q_heads <= 0 || q_heads % kv_heads || batch < 0 || max_q < 1 || rows < 0 || (head_dim != 64 && head_dim != 128 && head_dim != 256)) return SL_ERR_INVALID;
    if (q_heads / kv_heads > 128) return SL_ERR_CAPACITY;
    return (int64_t)kv4_attn_workspace(head_dim, q_heads / kv_heads, kv_heads, batch, max_q, -1);
}
int64_t sl_kv4_attention_workspace_span(int32_t q_heads, int32_t kv_heads, int32_t head_dim, int32_t batch, int32_t max_q, int64_t span) {
    const int64_t most = sl_kv4_attention_workspace(q_heads, kv_heads, head_dim, batch, max_q, 0);
    return most < 0 ? most : span < 0 ? SL_ERR_INVALID : (int64_t)kv4_attn_workspace(head_dim, q_heads / kv_heads, kv_heads, batch, max_q, std::min<int64_t>(span, 0x7fffffff));
}
int32_t sl_op_kv4_attention_device(const sl_kv4_cache* cache, const sl_kv4_attention* p, void* cuda_stream) try {
    Kv4Cache c{};
    if (!p || !cache_of(cache, c) || p->rows < 0 || p->batch < 0 || p->max_q < 1 || p->table_width < 0) return SL_ERR_INVALID;
    if (p->q_heads <= 0 || p->q_heads % c.KV || !std::isfinite(p->scale)) return SL_ERR_INVALID;
    if (!p->q || !p->out || !p->q_start || !p->workspace || ((uintptr_t)p->workspace & 15)) return SL_ERR_INVALID;
    if (p->batch && (!p->kv_len || (!p->table && p->table_width) || (p->table_stride && p->table_stride < p->table_width))) return SL_ERR_INVALID;
    if (!aligned(p->q, p->q_row, p->q_head) || !aligned(p->out, p->out_row, p->out_head) || (p->gate && !aligned(p->gate, p->gate_row, p->gate_head))) return SL_ERR_INVALID;
    // (positions and key blocks are counted in 31 bits)
    const int64_t span = (int64_t)p->table_width * c.page_size;
    if (p->q_heads / c.KV > 128 || p->batch > 4096 || span > 0x7fffffffll - 65536 || (span / KV4_B + 1) * p->batch * c.KV > 0x7fffffffll - 65536) return SL_ERR_CAPACITY;
    if (!device_ok()) return SL_ERR_NO_DEVICE;
    if (p->rows == 0 || p->batch == 0) return SL_OK;
    if (p->workspace_bytes < kv4_attn_workspace(c.D, p->q_heads / c.KV, c.KV, p->batch, p->max_q, span)) return SL_ERR_CAPACITY;
    Kv4AttnArgs a{(const __half*)p->q, p->q_row, p->q_head, (const __half*)p->gate, p->gate_row, p->gate_head, (__half*)p->out, p->out_row, p->out_head,
                  p->rows, p->q_heads, p->q_heads / c.KV, p->q_start, p->kv_len, p->batch, p->max_q, p->table, p->table_stride, p->table_width,
                  p->causal ? 1 : 0, p->scale, p->workspace, (size_t)p->workspace_bytes};
    return launched(launch_kv4_attn(c, a, (cudaStream_t)cuda_stream), "sl_op_kv4_attention_device");
} catch (...) {
    return SL_ERR_CAPACITY;                                   // no host memory
}

}  // extern "C"

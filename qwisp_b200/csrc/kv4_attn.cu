// kv4_attn.cu -- attention of a ragged batch of query rows over the cache held in 4 bits (kv4.cuh):
//   out = softmax(scale * q K^T) V, optionally times sigmoid(gate), K and V the fp16 values that the codes stand for.
// Request b's rows are q_start[b] .. q_start[b + 1] - 1, its keys positions 0 .. kv_len[b] - 1; causal: its row i of n sees
// kv_len - n + i + 1 keys.  A row that sees none is zero.  A page that the cache does not have holds no keys.
#include "kv4.cuh"

namespace sl {

// a warp a (row, head), D / 32 dims a lane, one key at a time
template <int D>
__global__ void __launch_bounds__(256) k_kv4_attn(Kv4Cache c, Kv4AttnArgs a) {
    constexpr int V = D / 32;
    const int lane = threadIdx.x & 31, row = blockIdx.x, h = blockIdx.y * 8 + (threadIdx.x >> 5);
    if (h >= a.NH) return;
    int lo = 0, hi = a.batch - 1;
    while (lo < hi) { const int mid = (lo + hi + 1) >> 1; if (a.q_start[mid] <= row) lo = mid; else hi = mid - 1; }
    const int b = lo, q0 = a.q_start[b], qn = a.q_start[b + 1] - q0, i = row - q0;
    if (i < 0 || i >= qn || i >= a.max_q) return;
    const int keys = min(max(a.kv_len[b], 0), a.table_width * c.page_size), n = a.causal ? keys - qn + i + 1 : keys;
    float q[V], o[V] = {}, m = -INFINITY, l = 0.f;
#pragma unroll
    for (int j = 0; j < V; ++j) q[j] = h2f(a.q[row * a.q_row + h * a.q_head + lane * V + j]) * a.scale;
    for (int k = 0; k < n; ++k) {
        const int page = a.table[(int64_t)b * a.table_stride + k / c.page_size];
        if (page < 0 || page >= c.pages) continue;
        const int off = k % c.page_size, at = off % KV4_B;
        const unsigned char* blk = kv4_block(c, page, h / a.G, off / KV4_B);
        float x[2][V];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const __half* sb = reinterpret_cast<const __half*>(blk + (16 + r) * D) + (lane * V >> 6) * 2 * KV4_B + at;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const int d = lane * V + j;
                const unsigned char byte = blk[r * 8 * D + kv4_swz((uint32_t)(at * (D / 2) + (d >> 1)))];
                x[r][j] = h2f(f2h(fmaf((float)((d & 1) ? byte >> 4 : byte & 15), h2f(sb[0]), h2f(sb[KV4_B]))));
            }
        }
        float s = 0.f;
#pragma unroll
        for (int j = 0; j < V; ++j) s = fmaf(q[j], x[0][j], s);
        s = warp_sum(s);
        const float nm = fmaxf(m, s), f = __expf(m - nm), e = __expf(s - nm);
        m = nm; l = l * f + e;
#pragma unroll
        for (int j = 0; j < V; ++j) o[j] = o[j] * f + e * x[1][j];
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
        float v = l == 0.f ? 0.f : o[j] / l;
        if (a.gate) v *= sigmoid_f(h2f(a.gate[row * a.g_row + h * a.g_head + lane * V + j]));
        a.out[row * a.o_row + h * a.o_head + lane * V + j] = f2h(v);
    }
}

size_t kv4_attn_workspace(int, int, int, int, int, int) { return 16; }
int launch_kv4_attn(const Kv4Cache& c, const Kv4AttnArgs& a, cudaStream_t st) {
    const dim3 grid((unsigned)a.rows, (unsigned)((a.NH + 7) / 8));
    int rc = 0;
    profile_launch("k_kv4_attn", st, [&] {
        if (c.D == 64) return rc = launch_pdl(false, k_kv4_attn<64>, grid, 256, 0, st, c, a);
        if (c.D == 128) return rc = launch_pdl(false, k_kv4_attn<128>, grid, 256, 0, st, c, a);
        return rc = launch_pdl(false, k_kv4_attn<256>, grid, 256, 0, st, c, a);
    });
    return rc;
}

}  // namespace sl

// kv4_attn.cu -- attention of a ragged batch of query rows over the cache held in 4 bits (kv4.cuh):
//   out = softmax(scale * q K^T) V, optionally times sigmoid(gate), K and V the fp16 values that the codes stand for.
// Request b's rows are q_start[b] .. q_start[b + 1] - 1, its keys positions 0 .. kv_len[b] - 1; causal: its row i of n sees
// kv_len - n + i + 1 keys.  A row that sees none is zero.  A page that the cache does not have, or the table no column for, holds no keys.
//
// Requests of up to 16 rows a kv head (tokens x query heads of the head) take k_kv4_decode, the others k_kv4_prompt.
#include "kv4.cuh"
#include "kv4_mma.cuh"

namespace sl {

// ================================================================================ few rows a request
// The work is the requests' key blocks: request b has ceil(keys / 16) units for each of its kv heads, and every CTA takes an equal
// run of them, whatever the lengths are: a run may hold the end of one (request, head), several whole ones and the start of another.
// Whole ones are finished by their CTA, the others leave partial sums that k_kv4_join adds up.
// A CTA's four warps take the blocks of a run in turn, each through a ring of its own that cp.async fills (a warp waits for nobody
// inside an item).  Per block: S^T = K Q^T and O^T += V^T P^T on m16n8k16 with 16 keys (16 dims) as M and up to eight rows as N, so that
// decode rows fill the tensor cores' narrow side.  ldmatrix brings a lane words of eight dims of a key for K and, transposed, words of
// four dims of two neighbouring keys for V; both expand to operand registers as they are, and the order of dims inside a step is
// the queries' (the outputs') to follow.  The running maximum is raised only when a score exceeds it by 2^6; the weights are
// carried times 2^8, so that fp16 holds them from 2^-32 of the largest on.
//
// CL: a cluster of 8, 4, 2 or 1 CTAs takes a (request, kv head), a share of its blocks a CTA, and adds the sums up through one another's shared
// memory: no look at the other requests, no second kernel; for tables so narrow that no CTA's share gets long (KD_CL_SPAN).
//
// What bounds it, 64 requests of up to 8192 positions, 32/8 heads of 128: 102 us, 3.8 TB/s = 0.58 of the measured copy rate (floor 60 us).  The memory
// alone, expansion left out, took 74 us; the expansion alone 100: a word of eight codes is 4 LOP3, 4 subtractions and 4 multiply-adds in half
// precision, all pipes of half rate, about 25 cycles of a scheduler with the scores' and weights' share.  Requests of up to 30000: 308 us, 0.71.
// 16 warps a multiprocessor (registers), two blocks a step, so that one block's MMAs cover the other one's expansion; more warps, deeper rings and
// expansion by integer shifts alone were no faster.  One request of 513 positions, 16/2 heads of 256: 8.2 us, latency: the launch, five dependent loads
// (lengths, table, codes), 5 key blocks a warp, two meetings of the cluster.
constexpr int KD_WARPS = 4, KD_MAX_BATCH = 4096;
template <int D, int NT> constexpr int kd_step = D == 256 || NT == 2 ? 1 : 2;                              // blocks a warp takes at a time
template <int D> constexpr int kd_stages = D == 256 ? 3 : D == 128 ? 4 : 6;                               // blocks of a warp's ring
template <int D, int NT> constexpr int kd_ctas = D == 256 ? 2 : NT == 1 ? 4 : 3;                          // CTAs of a multiprocessor
template <int D> constexpr size_t kd_ring = (size_t)KD_WARPS * kd_stages<D> * kv4_block_bytes(D);
template <int D> constexpr size_t kd_smem(int batch) { return kd_ring<D> + (size_t)(batch + 1) * 4; }
constexpr float KD_UP = 8.0f, KD_SLACK = 6.0f;

// rows of request b (0: none, or more than `most` rows a kv head), its keys in the table, keys before the first row's own (as many as the
// table's, if more), and the units of one of its kv heads
struct KdSeq { int q0, rows, keys, past, units; };
__device__ __forceinline__ KdSeq kd_seq(const Kv4Cache& c, const Kv4AttnArgs& a, int b, int most) {
    KdSeq s;
    s.q0 = a.q_start[b];
    const int n = a.q_start[b + 1] - s.q0;
    s.rows = min(min(n, a.max_q), a.rows - s.q0);
    const int len = max(a.kv_len[b], 0);
    s.keys = min(len, a.table_width * c.page_size);
    s.past = min(len - n, s.keys);
    if (s.q0 < 0 || s.rows <= 0 || s.rows > most / a.G) { s.rows = 0; s.units = 0; return s; }
    const int sees = a.causal ? min(s.keys, max(0, s.past + s.rows)) : s.keys;                            // (rows behind max_q see more)
    s.units = max(1, (sees + KV4_B - 1) / KV4_B);
    return s;
}
// exclusive sums of all requests' units in pre[0 .. batch]; by all threads (128)
__device__ __forceinline__ void kd_prefix(const Kv4Cache& c, const Kv4AttnArgs& a, int most, int* pre, int* ws) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    int base = 0;
    for (int b0 = 0; b0 < a.batch; b0 += KD_WARPS * 32) {
        const int b = b0 + tid;
        int x = b < a.batch ? kd_seq(c, a, b, most).units * c.KV : 0;
        const int own = x;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) { const int u = __shfl_up_sync(0xffffffffu, x, d); if (lane >= d) x += u; }
        if (lane == 31) ws[warp] = x;
        __syncthreads();
        int before = base, all = 0;
#pragma unroll
        for (int w = 0; w < KD_WARPS; ++w) { if (w < warp) before += ws[w]; all += ws[w]; }
        if (b < a.batch) pre[b] = before + x - own;
        base += all;
        __syncthreads();
    }
    if (tid == 0) pre[a.batch] = base;
    __syncthreads();
}
__device__ __forceinline__ int kd_find(const int* pre, int n, int u) {        // the last b with pre[b] <= u
    int lo = 0, hi = n - 1;
    while (lo < hi) { const int mid = (lo + hi + 1) >> 1; if (pre[mid] <= u) lo = mid; else hi = mid - 1; }
    return lo;
}
__device__ __forceinline__ int kd_run(int total, int ctas, int least) {       // units of a CTA
    const int per = max(least, (total + ctas - 1) / ctas);
    return (per + 2 * KD_WARPS - 1) / (2 * KD_WARPS) * (2 * KD_WARPS);
}
// a finished row's four dims, gated and rounded once
__device__ __forceinline__ void kd_finish(const Kv4AttnArgs& a, int row, int h, int d, float4 o, float l) {
    const float inv = l == 0.f ? 0.f : 1.0f / l;
    o.x *= inv; o.y *= inv; o.z *= inv; o.w *= inv;
    if (a.gate) {
        const uint2 g = *reinterpret_cast<const uint2*>(a.gate + row * a.g_row + h * a.g_head + d);
        const float2 g0 = __half22float2(*reinterpret_cast<const __half2*>(&g.x)), g1 = __half22float2(*reinterpret_cast<const __half2*>(&g.y));
        o.x *= kv4_sigmoid(g0.x); o.y *= kv4_sigmoid(g0.y); o.z *= kv4_sigmoid(g1.x); o.w *= kv4_sigmoid(g1.y);
    }
    const __half2 r0 = __floats2half2_rn(o.x, o.y), r1 = __floats2half2_rn(o.z, o.w);
    uint2 r; r.x = *reinterpret_cast<const uint32_t*>(&r0); r.y = *reinterpret_cast<const uint32_t*>(&r1);
    *reinterpret_cast<uint2*>(a.out + row * a.o_row + h * a.o_head + d) = r;
}
// The workspace: the exclusive sums of the units, then the partial sums of a CTA: two places (the item that began before its run, the one that goes on behind it), each [R][D] sums and [R] (max, norm).
template <int D, int R> __device__ __forceinline__ float* kd_part(const Kv4AttnArgs& a, int cta, int place) {
    return (float*)a.ws + (a.batch + 4) / 4 * 4 + ((size_t)cta * 2 + place) * R * (D + 2);
}

template <int D, int NT, int CL>
__global__ void __launch_bounds__(KD_WARPS * 32, kd_ctas<D, NT>) k_kv4_decode(Kv4Cache c, Kv4AttnArgs a, int most, int least) {
    constexpr int R = 8 * NT, U = kd_step<D, NT>, S = kd_stages<D> / U, CH = D / 32, BB = kv4_block_bytes(D), PIECES = BB / 16;
    extern __shared__ __align__(128) unsigned char smem[];
    float* s_o = reinterpret_cast<float*>(smem);                            // [warps][8 rows][D + 4], where the rings were
    int* s_pre = reinterpret_cast<int*>(smem + kd_ring<D>);
    float* s_c = s_o + KD_WARPS * 8 * (D + 4);                               // CL: [R][D], the CTA's sums
    static_assert(kd_ring<D> >= (size_t)(KD_WARPS * 8 * (D + 4) + R * D) * 4, "");
    __shared__ float2 s_ml[CL ? R : 1];                                       // CL: their (max, norm)
    __shared__ float s_m[KD_WARPS][R], s_l[KD_WARPS][R];
    __shared__ int s_ws[KD_WARPS];
    __shared__ uint4 s_q[NT * CH][32];
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31, g = lane >> 2, t = lane & 3;
    pdl_launch_dependents();
    int u = 0, u1 = 0, b = blockIdx.y;
    KdSeq sq;
    if (CL) {
        sq = kd_seq(c, a, b, most);
        if (!sq.units) return;                                                // (the whole cluster)
    } else {
        kd_prefix(c, a, most, s_pre, s_ws);
        if (blockIdx.x == 0) for (int x = tid; x <= a.batch; x += KD_WARPS * 32) ((int*)a.ws)[x] = s_pre[x];      // (for k_kv4_join)
        const int total = s_pre[a.batch], per = kd_run(total, gridDim.x, least);
        u = min((long long)blockIdx.x * per, (long long)total);
        u1 = min(u + per, total);
        if (u >= u1) return;
        b = kd_find(s_pre, a.batch, u);
        sq = kd_seq(c, a, b, most);
    }
    unsigned char* ring = smem + warp * S * U * BB;
    const uint32_t ring_u = smem_u32(ring);
    // ldmatrix: lanes 0-7 the rows of keys 0-7, 8-15 of keys 8-15, 16-31 the same of the next piece
    uint32_t lm[CH / 2];
#pragma unroll
    for (int i = 0; i < CH / 2; ++i) lm[i] = kv4_swz((uint32_t)((lane & 15) * (D / 2) + (2 * i + (lane >> 4)) * 16));
    const int page_blocks = c.page_size / KV4_B;
    while (CL || u < u1) {
        int head, j0, j1;                                                     // blocks j0 .. of a head
        if constexpr (CL != 0) {
            const int per = ((sq.units + CL - 1) / CL + U - 1) / U * U;
            head = blockIdx.x / CL;
            j0 = min((int)(blockIdx.x % CL) * per, sq.units); j1 = min(j0 + per, sq.units);
        } else {
            const int rel = u - s_pre[b];
            head = rel / sq.units; j0 = rel % sq.units; j1 = min(sq.units, j0 + (u1 - u));
        }
        const bool whole = j0 == 0 && j1 == sq.units;
        const int live = sq.rows * a.G;                                       // rows of the tile that exist
        // ---- the warp's steps of U blocks: warp, + 4, .. of the item's; 32 blocks looked up at a time, a lane each
        const int mine = max(0, ((j1 - j0 + U - 1) / U - warp + KD_WARPS - 1) / KD_WARPS);
        const int* table = a.table + (int64_t)b * a.table_stride;
        auto look = [&](int it) {                                             // the page of the lane's block of the 32 from step `it` on
            const int j = j0 + (warp + (it + lane / U) * KD_WARPS) * U + lane % U;
            return j < j1 && j * KV4_B < sq.keys ? table[j / page_blocks] : -1;      // (an item without keys has a block that is none)
        };
        unsigned long long addr = 0;
        int ahead = look(0);
        unsigned absent = 0;                                                  // blocks of the ring that there are none of
        auto issue = [&](int it) {
            if (it < mine) {
                if (it % (32 / U) == 0) {
                    const int j = j0 + (warp + (it + lane / U) * KD_WARPS) * U + lane % U;
                    addr = ahead >= 0 && ahead < c.pages ? (unsigned long long)kv4_block(c, ahead, head, j % page_blocks) : 0;
                } else if (it % (32 / U) == 32 / U / 2) ahead = look(it + 32 / U / 2);
#pragma unroll
                for (int x = 0; x < U; ++x) {
                    const unsigned char* src = (const unsigned char*)__shfl_sync(0xffffffffu, addr, it % (32 / U) * U + x);
                    const int st = it % S * U + x;
                    absent &= ~(1u << st);
                    if (src) {
                        const uint32_t dst = ring_u + st * BB + lane * 16;
                        src += lane * 16;
#pragma unroll
                        for (int i = 0; i < (PIECES + 31) / 32; ++i) if (i < PIECES / 32 || lane < PIECES % 32) kv4_cp16(dst + i * 512, src + i * 512);
                    } else absent |= 1u << st;
                }
            }
            kv4_commit();
        };
#pragma unroll
        for (int it = 0; it < S - 1; ++it) issue(it);
        // ---- queries: B operands, row g of each N tile; dims 32 i + 8 t .. of piece i in the order that the codes expand in
        for (int x = warp; x < NT * CH; x += KD_WARPS) {
            const int nt = x / CH, ch = x % CH, r = nt * 8 + g, i = r / a.G;
            uint4 v = make_uint4(0, 0, 0, 0);
            if (r < live) v = *reinterpret_cast<const uint4*>(a.q + (int64_t)(sq.q0 + i) * a.q_row + (int64_t)(head * a.G + r % a.G) * a.q_head + 8 * t + 32 * ch);
            s_q[x][lane] = make_uint4(__byte_perm(v.x, v.z, 0x5410), __byte_perm(v.x, v.z, 0x7632), __byte_perm(v.y, v.w, 0x5410), __byte_perm(v.y, v.w, 0x7632));
        }
        __syncthreads();
        // keys that the lane's columns (rows 2 t, 2 t + 1 of each tile) see, and what all rows see
        int sees[NT][2], all = sq.keys;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) sees[nt][e] = a.causal ? sq.past + (nt * 8 + 2 * t + e) / a.G + 1 : sq.keys;
        if (a.causal) all = min(all, sq.past + 1);
        float o[NT][CH][2][4], base[NT][2], l[NT][2];                        // base: KD_UP - the maximum
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int ch = 0; ch < CH; ++ch)
#pragma unroll
                for (int i = 0; i < 8; ++i) o[nt][ch][i >> 2][i & 3] = 0.f;
            base[nt][0] = base[nt][1] = INFINITY; l[nt][0] = l[nt][1] = 0.f;
        }
#pragma unroll 1
        for (int it = 0; it < mine; ++it) {
            kv4_wait<S - 2>();
            __syncwarp();
            issue(it + S - 1);                                                // (into the stage that the step before has left)
            const int st = it % S * U, key0 = (j0 + (warp + it * KD_WARPS) * U) * KV4_B;
            const unsigned gone = absent >> st & ((1u << U) - 1);
            if (gone == (1u << U) - 1) continue;
            const uint32_t blk = ring_u + st * BB;
            // ---- S^T: 16 U keys x 8 rows
            float s[U][NT][4];
#pragma unroll
            for (int x = 0; x < U; ++x)
#pragma unroll
                for (int i = 0; i < NT * 4; ++i) s[x][i >> 2][i & 3] = 0.f;
#pragma unroll
            for (int i = 0; i < CH / 2; ++i) {                                // a 64-dim group: two pieces
                uint32_t w[U][4], sb[U][4];
#pragma unroll
                for (int x = 0; x < U; ++x) {
                    kv4_ldsm(w[x], blk + x * BB + lm[i]);
                    kv4_ldsm_t(sb[x], blk + x * BB + 16 * D + i * 64 + (lane >> 3) * 16);      // (eight equal rows, transposed: scales of keys g, g + 8, biases, each twice)
                }
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    uint4 qf[NT];
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) qf[nt] = s_q[nt * CH + 2 * i + e][lane];
#pragma unroll
                    for (int x = 0; x < U; ++x) {
                        uint32_t k0[4], k8[4];
                        kv4_expand(w[x][2 * e], kv4_h2(sb[x][0]), kv4_h2(sb[x][2]), k0); kv4_expand(w[x][2 * e + 1], kv4_h2(sb[x][1]), kv4_h2(sb[x][3]), k8);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            kv4_mma(s[x][nt], k0[0], k8[0], k0[1], k8[1], qf[nt].x, qf[nt].y);
                            kv4_mma(s[x][nt], k0[2], k8[2], k0[3], k8[3], qf[nt].z, qf[nt].w);
                        }
                    }
                }
            }
            const bool edge = key0 + U * KV4_B > all || gone;
            float p[U][NT][4], high = -INFINITY;
            auto hidden = [&](int x, int nt, int e) { return key0 + x * KV4_B + g + 8 * (e >> 1) >= sees[nt][e & 1] || (gone >> x & 1); };
            auto weigh = [&] {                                                // exponents of the weights; above KD_UP + KD_SLACK: the maximum has to be raised
#pragma unroll
                for (int x = 0; x < U; ++x)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int e = 0; e < 4; ++e) p[x][nt][e] = fmaf(s[x][nt][e], a.scale, base[nt][e & 1]);      // (scale: times log2 e, by the host)
                if (edge) {
#pragma unroll
                    for (int x = 0; x < U; ++x)
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int e = 0; e < 4; ++e) if (hidden(x, nt, e)) p[x][nt][e] = -INFINITY;
                }
            };
            weigh();
#pragma unroll
            for (int x = 0; x < U; ++x)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) high = fmaxf(high, fmaxf(fmaxf(p[x][nt][0], p[x][nt][1]), fmaxf(p[x][nt][2], p[x][nt][3])));
            if (__any_sync(0xffffffffu, high > KD_UP + KD_SLACK)) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float y = -INFINITY;
#pragma unroll
                        for (int x = 0; x < U; ++x) {
                            if (!edge || !hidden(x, nt, e)) y = fmaxf(y, s[x][nt][e] * a.scale);
                            if (!edge || !hidden(x, nt, e + 2)) y = fmaxf(y, s[x][nt][e + 2] * a.scale);
                        }
                        y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, 4)); y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, 8)); y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, 16));
                        const float old = KD_UP - base[nt][e], top = fmaxf(y, old), f = top == -INFINITY ? 1.f : kv4_exp2(old - top);
                        base[nt][e] = KD_UP - top; l[nt][e] *= f;
#pragma unroll
                        for (int ch = 0; ch < CH; ++ch)
#pragma unroll
                            for (int k = 0; k < 2; ++k) { o[nt][ch][k][e] *= f; o[nt][ch][k][e + 2] *= f; }
                    }
                weigh();
            }
            uint32_t pb[U][NT][2];
#pragma unroll
            for (int x = 0; x < U; ++x)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) { p[x][nt][e] = kv4_exp2(p[x][nt][e]); l[nt][e & 1] += p[x][nt][e]; }
                    pb[x][nt][0] = kv4_transpose(kv4_pack(p[x][nt][0], p[x][nt][1])); pb[x][nt][1] = kv4_transpose(kv4_pack(p[x][nt][2], p[x][nt][3]));
                }
            // ---- O^T: dims x 8 rows; a lane's registers: dims 32 ch + 4 g + (0 .. 3) of rows 2 t, 2 t + 1
            const bool tail = key0 + U * KV4_B > sq.keys || gone;
#pragma unroll
            for (int i = 0; i < CH / 2; ++i) {
                uint32_t w[U][4], sv[U][4];
#pragma unroll
                for (int x = 0; x < U; ++x) {
                    kv4_ldsm_t(w[x], blk + x * BB + 8 * D + lm[i]);
                    kv4_ldsm(sv[x], blk + x * BB + 17 * D + i * 64 + (lane >> 3) * 16);        // (scales of keys 2 t, 2 t + 1; of 2 t + 8, + 9; biases)
                }
                if (tail) {                                                   // positions that nobody has: their weights are 0, their scales anything
#pragma unroll
                    for (int x = 0; x < U; ++x)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int k = key0 + x * KV4_B + 2 * t + 8 * (e & 1);
                            if (k >= sq.keys || (gone >> x & 1)) sv[x][e] = 0; else if (k + 1 >= sq.keys) sv[x][e] &= 0xffffu;
                        }
                }
#pragma unroll
                for (int x = 0; x < U; ++x)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        uint32_t v0[4], v8[4];
                        kv4_expand(w[x][2 * e], kv4_h2(sv[x][0]), kv4_h2(sv[x][2]), v0); kv4_expand(w[x][2 * e + 1], kv4_h2(sv[x][1]), kv4_h2(sv[x][3]), v8);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            kv4_mma(o[nt][2 * i + e][0], v0[0], v0[1], v8[0], v8[1], pb[x][nt][0], pb[x][nt][1]);
                            kv4_mma(o[nt][2 * i + e][1], v0[2], v0[3], v8[2], v8[3], pb[x][nt][0], pb[x][nt][1]);
                        }
                    }
            }
        }
        kv4_wait<0>();
        // ---- the warps' sums together
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], 4); l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], 8); l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], 16);
                if (g == 0) { s_m[warp][nt * 8 + 2 * t + e] = KD_UP - base[nt][e]; s_l[warp][nt * 8 + 2 * t + e] = l[nt][e]; }
            }
        float* part = kd_part<D, R>(a, blockIdx.x, j0 > 0 ? 0 : 1);
        __syncthreads();                                                      // (the rings are done with)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int ch = 0; ch < CH; ++ch)
#pragma unroll
                for (int e = 0; e < 2; ++e)
                    *reinterpret_cast<float4*>(s_o + (warp * 8 + 2 * t + e) * (D + 4) + 32 * ch + 4 * g) =
                        make_float4(o[nt][ch][0][e], o[nt][ch][0][e + 2], o[nt][ch][1][e], o[nt][ch][1][e + 2]);
            __syncthreads();
            for (int x = tid; x < 8 * D / 4; x += KD_WARPS * 32) {
                const int r = x / (D / 4), d = x % (D / 4) * 4, rr = nt * 8 + r;
                if (rr >= live) continue;
                float top = -INFINITY, sum = 0.f;
#pragma unroll
                for (int w = 0; w < KD_WARPS; ++w) top = fmaxf(top, s_m[w][rr]);
                float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int w = 0; w < KD_WARPS; ++w) {
                    const float f = s_m[w][rr] == -INFINITY ? 0.f : kv4_exp2(s_m[w][rr] - top);
                    const float4 y = *reinterpret_cast<const float4*>(s_o + (w * 8 + r) * (D + 4) + d);
                    sum = fmaf(s_l[w][rr], f, sum);
                    v.x = fmaf(y.x, f, v.x); v.y = fmaf(y.y, f, v.y); v.z = fmaf(y.z, f, v.z); v.w = fmaf(y.w, f, v.w);
                }
                if (CL) {
                    *reinterpret_cast<float4*>(s_c + rr * D + d) = v;
                    if (d == 0) s_ml[rr] = make_float2(top, sum);
                } else if (whole) kd_finish(a, sq.q0 + rr / a.G, head * a.G + rr % a.G, d, v, sum);
                else {
                    *reinterpret_cast<float4*>(part + (size_t)rr * D + d) = v;
                    if (d == 0) *reinterpret_cast<float2*>(part + (size_t)R * D + 2 * rr) = make_float2(top, sum);
                }
            }
            __syncthreads();
        }
        if constexpr (CL != 0) {
            kv4_cluster_sync();
            for (int x = (int)(blockIdx.x % CL) * (KD_WARPS * 32) + tid; x < live * (D / 4); x += CL * KD_WARPS * 32) {      // four dims a thread
                const int r = x / (D / 4), d = x % (D / 4) * 4;
                float2 ml[CL]; float4 y[CL];
#pragma unroll
                for (int i = 0; i < CL; ++i) {
                    ml[i] = kv4_peer2(kv4_peer(smem_u32(&s_ml[r]), i));
                    y[i] = kv4_peer4(kv4_peer(smem_u32(s_c + r * D + d), i));
                }
                float top = -INFINITY, sum = 0.f;
                float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int i = 0; i < CL; ++i) top = fmaxf(top, ml[i].x);
#pragma unroll
                for (int i = 0; i < CL; ++i) {
                    const float f = ml[i].x == -INFINITY ? 0.f : kv4_exp2(ml[i].x - top);
                    sum = fmaf(ml[i].y, f, sum);
                    v.x = fmaf(y[i].x, f, v.x); v.y = fmaf(y[i].y, f, v.y); v.z = fmaf(y[i].z, f, v.z); v.w = fmaf(y[i].w, f, v.w);
                }
                kd_finish(a, sq.q0 + r / a.G, head * a.G + r % a.G, d, v, sum);
            }
            __syncwarp();
            kv4_cluster_sync();                                                // (nobody leaves while its shared memory is read)
            return;
        }
        u += j1 - j0;
        if (u < u1 && u >= s_pre[b + 1]) { b = kd_find(s_pre, a.batch, u); sq = kd_seq(c, a, b, most); }
    }
}
// grid (rows, kv heads, requests): adds up the partial sums of a row whose (request, kv head) more than one CTA had.  A warp takes every
// fourth of them, eight in flight, behind one look at all their maxima.
template <int D, int NT>
__global__ void __launch_bounds__(KD_WARPS * 32) k_kv4_join(Kv4Cache c, Kv4AttnArgs a, int most, int least, int ctas) {
    constexpr int R = 8 * NT, V = D / 32;
    __shared__ __align__(16) float s_o[KD_WARPS][D];
    const int r = blockIdx.x, head = blockIdx.y, b = blockIdx.z, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    pdl_launch_dependents();
    const KdSeq sq = kd_seq(c, a, b, most);
    pdl_wait();                              // (every CTA: what follows this kernel in the stream also follows the one before)
    if (r >= sq.rows * a.G) return;
    const int* pre = (const int*)a.ws;
    const int per = kd_run(pre[a.batch], ctas, least), u0 = pre[b] + head * sq.units, c0 = u0 / per, n = (u0 + sq.units - 1) / per - c0 + 1;
    if (n == 1) return;
    // piece i: the first CTA's item goes on behind its run, the others' began before theirs
    auto part = [&](int i) { return kd_part<D, R>(a, c0 + i, i > 0 ? 0 : 1); };
    auto ml_of = [&](int i) { return i < n ? *reinterpret_cast<const float2*>(part(i) + (size_t)R * D + 2 * r) : make_float2(-INFINITY, 0.f); };
    float y[8][V];
    auto sums = [&](int i0) {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const int i = i0 + warp + 4 * k;
            const float* src = part(i) + (size_t)r * D + lane * V;
#pragma unroll
            for (int x = 0; x < V; x += 2) {
                float2 t = make_float2(0.f, 0.f);
                if (i < n) t = *reinterpret_cast<const float2*>(src + x);
                y[k][x] = t.x; y[k][x + 1] = t.y;
            }
        }
    };
    float2 ml = ml_of(lane);
    sums(0);
    float top = ml.x;
    for (int i = 32; i < n; i += 32) top = fmaxf(top, ml_of(i + lane).x);
    top = warp_max(top);
    float v[V] = {}, sum = 0.f;
    for (int i0 = 0; i0 < n; i0 += 32) {
        if (i0) { ml = ml_of(i0 + lane); sums(i0); }
        const float f = ml.x == -INFINITY ? 0.f : kv4_exp2(ml.x - top);
        sum = fmaf(ml.y, f, sum);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const float fk = __shfl_sync(0xffffffffu, f, warp + 4 * k);
#pragma unroll
            for (int x = 0; x < V; ++x) v[x] = fmaf(y[k][x], fk, v[x]);
        }
    }
    sum = warp_sum(sum);
#pragma unroll
    for (int x = 0; x < V; ++x) s_o[warp][lane * V + x] = v[x];
    __syncthreads();
    const int d = threadIdx.x * 4;
    if (d >= D) return;
    float4 o = *reinterpret_cast<const float4*>(&s_o[0][d]);
#pragma unroll
    for (int w = 1; w < KD_WARPS; ++w) {
        const float4 y = *reinterpret_cast<const float4*>(&s_o[w][d]);
        o.x += y.x; o.y += y.y; o.z += y.z; o.w += y.w;
    }
    kd_finish(a, sq.q0 + r / a.G, head * a.G + r % a.G, d, o, sum);
}
constexpr int KD_LEAST = 8;              // units a CTA takes at least
// Positions x dims of a table's row for each CTA of a cluster, at most: 1024 positions of 128.  GPU time of a call by clusters | evenly dealt out, us
// (the call as a program waits for it, launches and all, in brackets).  Heads of 128, 32/8: 1 x 1001 positions 8.2 | 12.3, 1 x 4001 10.3 | 13.3, 1 x 8101
// 14.4 | 16.4, 7 x (2000 + 4) 14.4 | 20.3, 16 x 1001 12.2 | 16.4, 64 x up to 1001 22.9 | 32.2.  16/2 of 256: 1 x 513 8.2 | 14.3, 1 x 2048 10.3 | 11.3, 1 x 4096
// 14.4 | 12.3 [14.7 | 17.5], 1 x 8101 20.5 | 16.4.  8/1 of 64: 1 x 16001 16.4 | 13.6 [16.5 | 18.9].  The bound is that of the call in brackets: the second
// launch costs the host more there than it saves the GPU.  In a graph dealing out would be 2 to 3 us ahead at those two.  Four CTAs for 16 x up to 8101 of 128: 36.9 | 35.4.
constexpr long long KD_CL_SPAN = 1024 * 128;
// CTAs of a cluster for that many (request, kv head) pairs with tables of `span` positions; 0: the work is dealt out evenly.  One CTA a pair may have the
// longer spans the more pairs there are, beside which a long one does not show.  By single CTAs | dealt out, us, heads of 128, 32/8: 128 x up to 301 18.7 | 30.8,
// 128 x up to 2001 60 | 70, 300 x up to 3001 160 | 184, 40 x (up to 1500 + 4) 33 | 39; 300 x up to 1501, 16/2 of 256: 61 | 80; 64 x up to 2001 (span of
// 2 x 1024): 39 | 41, of 256, 16/2 (span of 4 x): 35 | 29.
template <int D, int NT>
static int decode_cluster(long long pairs, long long span) {
    const long long room = (long long)sm_count() * kd_ctas<D, NT>;
    for (int cl = 8; cl > 1; cl >>= 1) if (pairs * cl <= room && span * D <= cl * KD_CL_SPAN) return cl;
    return span * D <= KD_CL_SPAN * (1 + 2 * pairs / room) ? 1 : 0;
}
template <int D, int NT, int CL>
static int decode_ready(int smem) {      // shared memory, once for each device
    static std::atomic<unsigned long long> configured{0};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 64 && configured.load(std::memory_order_relaxed) >> dev & 1) return 0;
    const cudaError_t err = cudaFuncSetAttribute(k_kv4_decode<D, NT, CL>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (err == cudaSuccess && dev < 64) configured.fetch_or(1ull << dev);
    return (int)err;
}
template <int D, int NT, int CL>
static int launch_cluster(const Kv4Cache& c, const Kv4AttnArgs& a, int most, cudaStream_t st) {
    int rc = decode_ready<D, NT, CL>((int)kd_ring<D>);
    if (rc) return rc;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(c.KV * CL), (unsigned)a.batch); cfg.blockDim = dim3(KD_WARPS * 32); cfg.dynamicSmemBytes = kd_ring<D>; cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = CL; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr; cfg.numAttrs = 1;
    profile_launch("k_kv4_decode", st, [&] { return rc = (int)cudaLaunchKernelEx(&cfg, k_kv4_decode<D, NT, CL>, c, a, most, 0); });
    return rc;
}
template <int D, int NT>
static int launch_decode(const Kv4Cache& c, Kv4AttnArgs a, int most, cudaStream_t st) {
    a.scale *= 1.4426950408889634f;
    switch (decode_cluster<D, NT>((long long)a.batch * c.KV, (long long)a.table_width * c.page_size)) {
        case 8: return launch_cluster<D, NT, 8>(c, a, most, st);
        case 4: return launch_cluster<D, NT, 4>(c, a, most, st);
        case 2: return launch_cluster<D, NT, 2>(c, a, most, st);
        case 1: return launch_cluster<D, NT, 1>(c, a, most, st);
    }
    const int ctas = sm_count() * kd_ctas<D, NT>;
    int rc = 0;
    if ((rc = decode_ready<D, NT, 0>((int)kd_smem<D>(KD_MAX_BATCH)))) return rc;
    profile_launch("k_kv4_decode", st, [&] { return rc = launch_pdl(false, k_kv4_decode<D, NT, 0>, dim3((unsigned)ctas), KD_WARPS * 32, kd_smem<D>(a.batch), st, c, a, most, KD_LEAST); });
    if (rc) return rc;
    profile_launch("k_kv4_join", st, [&] { return rc = launch_pdl(true, k_kv4_join<D, NT>, dim3((unsigned)(a.G * (a.max_q < most / a.G ? a.max_q : most / a.G)), (unsigned)c.KV, (unsigned)a.batch), KD_WARPS * 32, 0, st, c, a, most, KD_LEAST, ctas); });
    return rc;
}

template <int D, int NT>
static size_t decode_workspace(int KV, int batch, long long span) {
    if (span >= 0 && decode_cluster<D, NT>((long long)batch * KV, span)) return 0;
    return (size_t)(batch + 4) / 4 * 16 + (size_t)sm_count() * kd_ctas<D, NT> * 2 * 8 * NT * (D + 2) * 4;
}
template <int D>
static size_t attn_workspace(int G, int KV, int batch, int max_q, long long span) {
    if (G > 16 && span >= 0) return 0;                                        // (all requests are k_kv4_prompt's)
    return max_q > 8 / G ? decode_workspace<D, 2>(KV, batch, span) : decode_workspace<D, 1>(KV, batch, span);
}
size_t kv4_attn_workspace(int D, int G, int KV, int batch, int max_q, long long span) {
    return D == 64 ? attn_workspace<64>(G, KV, batch, max_q, span) : D == 128 ? attn_workspace<128>(G, KV, batch, max_q, span) : attn_workspace<256>(G, KV, batch, max_q, span);
}
template <int D>
static int launch_attn(const Kv4Cache& c, const Kv4AttnArgs& a, cudaStream_t st) {
    int rc = 0;
    const bool many = a.max_q > 16 / a.G;
    if (a.G <= 16) rc = a.max_q > 8 / a.G ? launch_decode<D, 2>(c, a, 16, st) : launch_decode<D, 1>(c, a, 8, st);
    if (rc || !many) return rc;
    return launch_kv4_prompt(c, a, a.G <= 16 ? 16 : 0, st, a.G <= 16);
}
int launch_kv4_attn(const Kv4Cache& c, const Kv4AttnArgs& a, cudaStream_t st) {
    return c.D == 64 ? launch_attn<64>(c, a, st) : c.D == 128 ? launch_attn<128>(c, a, st) : launch_attn<256>(c, a, st);
}

}  // namespace sl

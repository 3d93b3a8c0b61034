// kv4_rows.cu -- rows of queries, keys and values on their way into the cache held in 4 bits (kv4.cuh), and back out of it.
//
// k_kv4_append: y = rope(x * rsqrt(mean(x^2) + eps) * w) for every query and key head of a row; queries leave as fp16, keys are rounded to
// fp16 and, like the values, quantised 64 dims at a time (lo, hi: the group's extremes):
//   scale = max((hi - lo) / 15, 1e-7), signed so that the extreme further from zero is the edge;  q0 = round(edge / scale)
//   scale = edge / q0, bias = edge  (q0 == 0: bias = 0);  code = round((x - bias) / scale) in 0 .. 15
// the arithmetic of the weights' quantiser (synth.cu), in 32 bits with every operation rounded once.  A group that holds an infinity or
// a NaN gets a NaN scale: all of it reads back as NaN.
// k_kv4_read: fp16(code * scale + bias) of K and V at given slots.
//
// What bounds them.  Append, 4093 rows of 32/8 heads of 128 with norms and three axes, at scattered slots: 34 us, 2.6 TB/s with what it reads
// and writes.  No unit is full: issue slots 64 %, 5.9 warps a scheduler, which wait for results in flight and for shared memory.  The quantiser (two divisions
// for a group, eight rounded quotients a word, exact) is some 200 instructions a lane's word; keys in 64 bits are about 4 us.  One row: 4 us, latency.
// Read, 30001 rows of 8 heads of 128: 45 us, 3.5 TB/s: 123 MB of writes, which a fill alone needs 35 us for (floor at the copy rate: 24).  Larger CTAs, more CTAs a row, streaming stores, eight words in flight: no faster.
#include "kv4.cuh"
#include "kv4_mma.cuh"

namespace sl {

constexpr int KA_WARPS = 4;

// a / s, rounded to nearest, where r is 1 / s rounded to nearest: the quotient's remainder by one fused multiply-add, and a second one
// that adds what it is worth (Markstein, "Computation of elementary functions on the IBM RISC System/6000", 1990).  For the sizes
// of a group's values: nothing here under- or overflows.
__device__ __forceinline__ float kv4_div(float a, float s, float r) {
    const float q = __fmul_rn(a, r);
    return __fmaf_rn(__fmaf_rn(-q, s, a), r, q);
}
// Eight dims of a head a lane as halves, eight lanes a group: stores the lane's word of codes and the group's scale and bias.  By whole
// warps; `store`: the lane has a head.  region: 0 = K, 1 = V.
template <int D>
__device__ __forceinline__ void kv4_store(unsigned char* blk, int at, int region, int hl, const uint4& raw, bool store) {
    const __half2* h = reinterpret_cast<const __half2*>(&raw);
    // (lowest, negated highest) of the group; a NaN stays one
    const __half2 lo2 = __hmin2_nan(__hmin2_nan(h[0], h[1]), __hmin2_nan(h[2], h[3])), hi2 = __hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3]));
    __half2 ends = __hmin2_nan(__lows2half2(lo2, __hneg2(hi2)), __highs2half2(lo2, __hneg2(hi2)));
#pragma unroll
    for (int d = 1; d < 8; d <<= 1) ends = __hmin2_nan(ends, __shfl_xor_sync(0xffffffffu, ends, d));
    const float lo = __low2float(ends), hi = -__high2float(ends);
    float scale = fmaxf(kv4_div(__fsub_rn(hi, lo), 15.0f, 0x1.111112p-4f), 1e-7f);
    const bool side = fabsf(lo) > fabsf(hi), bad = !(fabsf(lo) <= 65504.0f && fabsf(hi) <= 65504.0f);
    scale = side ? scale : -scale;
    const float edge = side ? lo : hi, q0 = roundf(__fdiv_rn(edge, scale));
    const bool zero = q0 == 0.0f;
    scale = zero ? scale : __fdiv_rn(edge, q0);
    const float bias = zero ? 0.0f : edge, r = __frcp_rn(scale);
    // Rounded to the nearest code, halves up: with the addition rounded towards zero, adding a half and 2^23 truncates into the lowest bits
    // of 0x4b000000.  (A quotient is never below zero: the bias is the end that the scale leads away from.)
    uint32_t word = 0;
#pragma unroll
    for (int i = 3; i >= 0; --i) {
        const float2 f = __half22float2(h[i]);
        const float u = fminf(kv4_div(__fsub_rn(f.x, bias), scale, r), 15.0f), v = fminf(kv4_div(__fsub_rn(f.y, bias), scale, r), 15.0f);
        word = word * 16u + __float_as_uint(__fadd_rz(__fadd_rz(v, 0.5f), 8388608.0f));
        word = word * 16u + __float_as_uint(__fadd_rz(__fadd_rz(u, 0.5f), 8388608.0f));
    }
    word -= 0x4b000000u + 0xb0000000u;                        // (the first's, and the second's times 16; the others' have left the word)
    if (!store) return;
    *reinterpret_cast<uint32_t*>(blk + region * 8 * D + kv4_swz((uint32_t)(at * (D / 2) + hl * 4))) = word;
    if ((hl & 7) == 0) {
        __half* sb = reinterpret_cast<__half*>(blk + (16 + region) * D) + (hl >> 3) * 2 * KV4_B + at;
        sb[0] = bad ? __ushort_as_half(0x7fff) : f2h(scale);
        sb[KV4_B] = f2h(bias);
    }
}

// A row's angles once per CTA: turns = position * frequency as a 64-bit fraction of a turn, exact for every position, then cos and
// sin in 64 bits.  Keys stay in 64 bits up to their rounding, to fp32 and then fp16 (a code next to a border then does not go by the order of a sum or
// by the shape of the launch); queries take 32.
// RPC rows at a time, KA_WARPS / RPC warps each; grid (row groups, parts).  A warp's task: 32 / (D / 8) heads of one kind, eight dims a lane,
// the next task's halves on their way.  Many rows: CTAs that stay, so that frequencies and weights are fetched once (from the parameters a
// lane's own frequency costs a constant-cache access for every lane).  Few: a task a warp.
template <int D, int RPC>
__global__ void __launch_bounds__(KA_WARPS * 32, 7) k_kv4_append(Kv4Cache c, Kv4AppendArgs a) {
    constexpr int LPH = D / 8, HPW = 32 / LPH, WPR = KA_WARPS / RPC;      // lanes of a head, heads of a warp, warps of a row
    __shared__ __align__(16) double2 s_d[RPC][8][LPH];        // (cos, sin with the sign that dim takes it with) of dim 8 hl + i at [i][hl]
    __shared__ __align__(16) float2 s_f[RPC][4][LPH][2];      // the same in 32 bits, of dims 8 hl + 2 j, + 1
    __shared__ uint64_t s_turn[D / 2];
    __shared__ unsigned char s_axis[D / 2];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, hl = lane % LPH, hs = lane / LPH, rr = warp / WPR;
    const int half = a.rope >> 1;
    for (int f = tid; f < half; f += KA_WARPS * 32) { s_turn[f] = a.turn[f]; s_axis[f] = a.axis[f]; }
    for (int i = tid; i < RPC * (D - a.rope); i += KA_WARPS * 32) {      // dims that are not rotated
        const int d = a.rope + i / RPC, r = i % RPC;
        s_d[r][d & 7][d >> 3] = make_double2(1.0, 0.0);
        s_f[r][(d & 7) >> 1][d >> 3][d & 1] = make_float2(1.f, 0.f);
    }
    const int partner = hl * 8 >= a.rope ? lane : hl * 8 < half ? lane + a.rope / 16 : lane - a.rope / 16;      // has the dims these are rotated with
    // tasks: nk of K, nk of V, then the queries'; this warp's are g0, g0 + stride, ..
    const int nk = a.k ? (c.KV + HPW - 1) / HPW : 0, nq = a.q ? (a.NH + HPW - 1) / HPW : 0, stride = gridDim.y * WPR, g0 = blockIdx.y * WPR + warp % WPR;
    auto from = [&](int first) { return first <= g0 ? g0 - first : (stride - (first - g0) % stride) % stride; };      // the warp's first of a kind
    const int k0 = from(0), v0 = from(nk), q0 = from(2 * nk);
    auto halves = [](const uint4& v, float x[8]) {
        const __half2* h = reinterpret_cast<const __half2*>(&v);
#pragma unroll
        for (int k = 0; k < 4; ++k) { const float2 f = __half22float2(h[k]); x[2 * k] = f.x; x[2 * k + 1] = f.y; }
    };
    auto weight = [&](const __half* w) { return w ? reinterpret_cast<const uint4*>(w)[hl] : make_uint4(0, 0, 0, 0); };
    const uint4 kw = weight(a.k_norm), qw = weight(a.q_norm);
    for (int row0 = blockIdx.x * RPC; row0 < a.rows; row0 += gridDim.x * RPC) {
        const int row = row0 + rr;
        const int64_t slot = row >= a.rows ? -1 : a.slots ? a.slots[row] : 0;
        const bool live = row < a.rows && (!a.slots || (slot >= 0 && slot < c.pages * (int64_t)c.page_size));        // (else: padding)
        auto load = [&](const __half* src, int64_t by_head, int task, int heads) {
            const int head = task * HPW + hs;
            return live && head < heads ? reinterpret_cast<const uint4*>(src + head * by_head)[hl] : make_uint4(0, 0, 0, 0);
        };
        const __half *ksrc = a.k + row * a.k_row, *vsrc = a.v + row * a.v_row, *qsrc = a.q + row * a.q_row;
        uint4 kraw = load(ksrc, a.k_head, k0, a.k ? c.KV : 0), vraw = load(vsrc, a.v_head, v0, a.k ? c.KV : 0), qraw = load(qsrc, a.q_head, q0, a.q ? a.NH : 0);
        __syncthreads();
        for (int i = tid; i < RPC * half; i += KA_WARPS * 32) {
            const int r = i / half, f = i - r * half, at = min(row0 + r, a.rows - 1);
            const uint64_t t = (uint64_t)(int64_t)a.pos[(int64_t)s_axis[f] * a.pos_axis + at] * s_turn[f];      // (modulo 2^64: a whole turn)
            double sn, cs;
            sincospi((double)(int64_t)t * 0x1p-63, &sn, &cs);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int d = f + e * half;
                s_d[r][d & 7][d >> 3] = make_double2(cs, e ? sn : -sn);
                s_f[r][(d & 7) >> 1][d >> 3][d & 1] = make_float2((float)cs, (float)(e ? sn : -sn));
            }
        }
        __syncthreads();
        if (!live) continue;
        if (nk) {
            int pg, off;
            kv4_place(c, slot, pg, off);
            const int at = off % KV4_B;
            unsigned char* blk = kv4_block(c, pg, 0, off / KV4_B);               // (head 0's)
            const int64_t head_bytes = (int64_t)(c.page_size / KV4_B) * kv4_block_bytes(D);
            for (int t = k0; t < nk; t += stride) {
                const int head = t * HPW + hs;
                uint4 cur = kraw;
                kraw = load(ksrc, a.k_head, t + stride, c.KV);
                if (a.k_norm || a.rope) {
                    float x[8];
                    double y[8];
                    halves(cur, x);
#pragma unroll
                    for (int k = 0; k < 8; ++k) y[k] = (double)x[k];
                    if (a.k_norm) {
                        float w[8];
                        halves(kw, w);
                        double ss = 0.0;
#pragma unroll
                        for (int k = 0; k < 8; ++k) ss = fma(y[k], y[k], ss);
#pragma unroll
                        for (int d = 1; d < LPH; d <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, d);
                        const double inv = rsqrt(fma(ss, 1.0 / D, (double)a.eps));
#pragma unroll
                        for (int k = 0; k < 8; ++k) y[k] = (double)(x[k] * w[k]) * inv;      // (two halves' product: exact in 32 bits)
                    }
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const double2 cs = s_d[rr][k][hl];
                        const double other = __shfl_sync(0xffffffffu, y[k], partner);
                        x[k] = (float)fma(other, cs.y, y[k] * cs.x);
                    }
                    uint32_t* cw = reinterpret_cast<uint32_t*>(&cur);
#pragma unroll
                    for (int j = 0; j < 4; ++j) { const __half2 y2 = __floats2half2_rn(x[2 * j], x[2 * j + 1]); cw[j] = *reinterpret_cast<const uint32_t*>(&y2); }
                }
                kv4_store<D>(blk + head * head_bytes, at, 0, hl, cur, head < c.KV);
            }
            for (int t = v0; t < nk; t += stride) {
                const int head = t * HPW + hs;
                const uint4 cur = vraw;
                vraw = load(vsrc, a.v_head, t + stride, c.KV);
                kv4_store<D>(blk + head * head_bytes, at, 1, hl, cur, head < c.KV);
            }
        }
        if (q0 >= nq) continue;
        float w[8], cs[8], sn[8];
        halves(qw, w);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float4 f = *reinterpret_cast<const float4*>(s_f[rr][j][hl]);
            cs[2 * j] = f.x; sn[2 * j] = f.y; cs[2 * j + 1] = f.z; sn[2 * j + 1] = f.w;
        }
        __half* dst = a.q_out + row * a.o_row;
        for (int t = q0; t < nq; t += stride) {
            const int head = t * HPW + hs;
            float x[8];
            halves(qraw, x);
            qraw = load(qsrc, a.q_head, t + stride, a.NH);
            if (a.q_norm) {
                float ss = 0.f;
#pragma unroll
                for (int k = 0; k < 8; ++k) ss = fmaf(x[k], x[k], ss);
#pragma unroll
                for (int d = 1; d < LPH; d <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, d);
                const float inv = rsqrtf(fmaf(ss, 1.0f / D, a.eps));
#pragma unroll
                for (int k = 0; k < 8; ++k) x[k] = x[k] * w[k] * inv;
            }
            uint4 o; uint32_t* ow = reinterpret_cast<uint32_t*>(&o);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float u = __shfl_sync(0xffffffffu, x[2 * j], partner), v = __shfl_sync(0xffffffffu, x[2 * j + 1], partner);
                const __half2 y = __floats2half2_rn(fmaf(u, sn[2 * j], x[2 * j] * cs[2 * j]), fmaf(v, sn[2 * j + 1], x[2 * j + 1] * cs[2 * j + 1]));
                ow[j] = *reinterpret_cast<const uint32_t*>(&y);
            }
            if (head < a.NH) reinterpret_cast<uint4*>(dst + head * a.o_head)[hl] = o;
        }
    }
}

// a warp a row, a lane a word of codes: eight dims of K or V of a head
template <int D>
__global__ void __launch_bounds__(256) k_kv4_read(Kv4Cache c, Kv4ReadArgs a) {
    constexpr int LPH = D / 8;
    const int lane = threadIdx.x & 31, n = c.KV * 2 * LPH, parts = gridDim.y * 32;
    const int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (row >= a.rows) return;
    const int64_t slot = a.slots[row];
    if (slot < 0 || slot >= c.pages * (int64_t)c.page_size) return;
    int page, off;
    kv4_place(c, slot, page, off);
    const int at = off % KV4_B;
    const unsigned char* base = kv4_block(c, page, 0, off / KV4_B);
    const int64_t head_bytes = (int64_t)(c.page_size / KV4_B) * kv4_block_bytes(D);
#pragma unroll 4
    for (int i = blockIdx.y * 32 + lane; i < n; i += parts) {
        const int hl = i % LPH, region = i / LPH & 1, head = i / (2 * LPH);
        const unsigned char* blk = base + head * head_bytes;
        const uint32_t w = __ldg(reinterpret_cast<const uint32_t*>(blk + region * 8 * D + kv4_swz((uint32_t)(at * (D / 2) + hl * 4))));
        const __half* sb = reinterpret_cast<const __half*>(blk + (16 + region) * D) + (hl >> 3) * 2 * KV4_B + at;
        const __half2 s = __half2half2(__ldg(sb)), b = __half2half2(__ldg(sb + KV4_B));
        uint32_t x[4];
        kv4_expand(w, s, b, x);                                               // (dims 0 4, 1 5, 2 6, 3 7)
        const uint4 o = make_uint4(__byte_perm(x[0], x[1], 0x5410), __byte_perm(x[2], x[3], 0x5410), __byte_perm(x[0], x[1], 0x7632), __byte_perm(x[2], x[3], 0x7632));
        __half* dst = region ? a.v + row * a.v_row + head * a.v_head : a.k + row * a.k_row + head * a.k_head;
        reinterpret_cast<uint4*>(dst)[hl] = o;
    }
}

template <int D>
static int launch_append(const Kv4Cache& c, const Kv4AppendArgs& a, cudaStream_t st) {
    constexpr int HPW = 32 / (D / 8);
    const int tasks = (a.q ? (a.NH + HPW - 1) / HPW : 0) + (a.k ? 2 * ((c.KV + HPW - 1) / HPW) : 0), most = sm_count() * 7;
    if (a.rows < 4 * sm_count()) return launch_pdl(false, k_kv4_append<D, 1>, dim3((unsigned)a.rows, (unsigned)((tasks + KA_WARPS - 1) / KA_WARPS)), KA_WARPS * 32, 0, st, c, a);
    return launch_pdl(false, k_kv4_append<D, 2>, dim3((unsigned)((a.rows + 1) / 2 < most ? (a.rows + 1) / 2 : most)), KA_WARPS * 32, 0, st, c, a);
}
int launch_kv4_append(const Kv4Cache& c, const Kv4AppendArgs& a, cudaStream_t st) {
    int rc = 0;
    profile_launch("k_kv4_append", st, [&] { return rc = c.D == 64 ? launch_append<64>(c, a, st) : c.D == 128 ? launch_append<128>(c, a, st) : launch_append<256>(c, a, st); });
    return rc;
}
int launch_kv4_read(const Kv4Cache& c, const Kv4ReadArgs& a, cudaStream_t st) {
    const int words = c.KV * 2 * (c.D / 8) / 32 + 1;
    const dim3 grid((unsigned)((a.rows + 7) / 8), (unsigned)(a.rows < 8 * sm_count() ? (words + 3) / 4 : 1));
    int rc = 0;
    profile_launch("k_kv4_read", st, [&] {
        if (c.D == 64) return rc = launch_pdl(false, k_kv4_read<64>, grid, 256, 0, st, c, a);
        if (c.D == 128) return rc = launch_pdl(false, k_kv4_read<128>, grid, 256, 0, st, c, a);
        return rc = launch_pdl(false, k_kv4_read<256>, grid, 256, 0, st, c, a);
    });
    return rc;
}

}  // namespace sl

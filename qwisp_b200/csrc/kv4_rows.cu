// kv4_rows.cu -- rows of queries, keys and values on their way into the cache held in 4 bits (kv4.cuh), and back out of it.
//
// k_kv4_append: y = rope(x * rsqrt(mean(x^2) + eps) * w) for every query and key head of a row; queries leave as fp16, keys are rounded to
// fp16 and, like the values, quantised 64 dims at a time (lo, hi: the group's extremes):
//   scale = max((hi - lo) / 15, 1e-7), signed so that the extreme further from zero is the edge;  q0 = round(edge / scale)
//   scale = edge / q0, bias = edge  (q0 == 0: bias = 0);  code = round((x - bias) / scale) in 0 .. 15
// the arithmetic of the weights' quantiser (synth.cu), in 32 bits with every operation rounded once.  A group that holds an infinity or
// a NaN gets a NaN scale: all of it reads back as NaN.
// k_kv4_read: fp16(code * scale + bias) of K and V at given slots.
#include "kv4.cuh"

namespace sl {

constexpr int KA_WARPS = 4;

// a / s, rounded to nearest, where r is 1 / s rounded to nearest: the quotient's remainder by one fused multiply-add, and a second one
// that adds what it is worth (Markstein, "Computation of elementary functions on the IBM RISC System/6000", 1990).  For the sizes
// of a group's values: nothing here under- or overflows.
__device__ __forceinline__ float kv4_div(float a, float s, float r) {
    const float q = __fmul_rn(a, r);
    return __fmaf_rn(__fmaf_rn(-q, s, a), r, q);
}
// Eight dims of a head a lane, eight lanes a group: stores the lane's word of codes and the group's scale and bias.  By whole warps;
// `store`: the lane has a head.  region: 0 = K, 1 = V.
__device__ __forceinline__ void kv4_store(const Kv4Cache& c, unsigned char* blk, int at, int region, int hl, const float x[8], bool store) {
    float lo = x[0], hi = x[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) { lo = fminf(lo, x[i]); hi = fmaxf(hi, x[i]); }
    // fmin and fmax pass a NaN over, so the sum of 0 * x tells of one (and of an infinity)
    float odd = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) odd = fmaf(x[i], 0.f, odd);
#pragma unroll
    for (int d = 1; d < 8; d <<= 1) { lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, d)); hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, d)); }
    const bool bad = (__ballot_sync(0xffffffffu, odd != 0.f) >> (threadIdx.x & 24) & 0xffu) != 0;
    float scale = fmaxf(kv4_div(__fsub_rn(hi, lo), 15.0f, 0x1.111112p-4f), 1e-7f);
    const bool side = fabsf(lo) > fabsf(hi);
    scale = side ? scale : -scale;
    const float edge = side ? lo : hi, q0 = roundf(__fdiv_rn(edge, scale));
    const bool zero = q0 == 0.0f;
    scale = zero ? scale : __fdiv_rn(edge, q0);
    const float bias = zero ? 0.0f : edge, r = __frcp_rn(scale);
    // rounded to the nearest code, halves up: with the addition rounded towards zero, adding a half and 2^23 truncates to the lowest bits
    float w[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 7; i >= 0; --i) {
        const float q = fminf(fmaxf(kv4_div(__fsub_rn(x[i], bias), scale, r), 0.0f), 15.0f);
        w[i >> 2] = fmaf(w[i >> 2], 16.0f, __fadd_rn(__fadd_rz(__fadd_rz(q, 0.5f), 8388608.0f), -8388608.0f));        // (four codes: below 2^16, exact)
    }
    const uint32_t word = __byte_perm(__float_as_uint(w[0] + 8388608.0f), __float_as_uint(w[1] + 8388608.0f), 0x5410);
    if (!store) return;
    *reinterpret_cast<uint32_t*>(blk + region * 8 * c.D + kv4_swz((uint32_t)(at * (c.D / 2) + hl * 4))) = word;
    if ((hl & 7) == 0) {
        __half* sb = reinterpret_cast<__half*>(blk + (16 + region) * c.D) + (hl >> 3) * 2 * KV4_B + at;
        sb[0] = bad ? __ushort_as_half(0x7fff) : f2h(scale);
        sb[KV4_B] = f2h(bias);
    }
}

// A row's angles once per CTA: turns = position * frequency as a 64-bit fraction of a turn, exact for every position, then cos and
// sin in 64 bits.  Keys stay in 64 bits up to the one rounding to fp16 (a code next to a border then does not go by the order of a sum or
// by the shape of the launch); queries take 32.
// grid (rows, parts), a warp a task: 32 / (D / 8) heads of one kind, eight dims a lane, the next task's halves on their way.
template <int D>
__global__ void __launch_bounds__(KA_WARPS * 32, 8) k_kv4_append(Kv4Cache c, Kv4AppendArgs a) {
    constexpr int LPH = D / 8, HPW = 32 / LPH;                // lanes of a head, heads of a warp
    __shared__ __align__(16) double2 s_d[8][LPH];             // (cos, sin with the sign that dim takes it with) of dim 8 hl + i at [i][hl]
    __shared__ __align__(16) float2 s_f[4][LPH][2];           // the same in 32 bits, of dims 8 hl + 2 j, + 1
    const int row = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, hl = lane % LPH, hs = lane / LPH;
    const int64_t slot = a.slots ? a.slots[row] : 0;
    if (a.slots && (slot < 0 || slot >= c.pages * (int64_t)c.page_size)) return;         // padding
    // tasks: nk of K, nk of V, then the queries'; this warp's are g0, g0 + stride, ..
    const int nk = a.k ? (c.KV + HPW - 1) / HPW : 0, nq = a.q ? (a.NH + HPW - 1) / HPW : 0, stride = gridDim.y * KA_WARPS, g0 = blockIdx.y * KA_WARPS + warp;
    auto from = [&](int first) { return first <= g0 ? g0 - first : (stride - (first - g0) % stride) % stride; };      // the warp's first of a kind
    const int k0 = from(0), v0 = from(nk), q0 = from(2 * nk);
    auto load = [&](const __half* src, int64_t by_head, int task, int heads) {
        const int head = task * HPW + hs;
        return head < heads ? reinterpret_cast<const uint4*>(src + head * by_head)[hl] : make_uint4(0, 0, 0, 0);
    };
    const __half *ksrc = a.k + row * a.k_row, *vsrc = a.v + row * a.v_row, *qsrc = a.q + row * a.q_row;
    uint4 kraw = load(ksrc, a.k_head, k0, a.k ? c.KV : 0), vraw = load(vsrc, a.v_head, v0, a.k ? c.KV : 0), qraw = load(qsrc, a.q_head, q0, a.q ? a.NH : 0);
    const int half = a.rope >> 1;
    auto put = [&](int d, double cs, double sn) {
        s_d[d & 7][d >> 3] = make_double2(cs, sn);
        s_f[(d & 7) >> 1][d >> 3][d & 1] = make_float2((float)cs, (float)sn);
    };
    for (int f = tid; f < half; f += KA_WARPS * 32) {
        const uint64_t t = (uint64_t)(int64_t)a.pos[(int64_t)a.axis[f] * a.pos_axis + row] * a.turn[f];      // (modulo 2^64: a whole turn)
        double sn, cs;
        sincospi((double)(int64_t)t * 0x1p-63, &sn, &cs);
        put(f, cs, -sn); put(f + half, cs, sn);
    }
    for (int d = a.rope + tid; d < D; d += KA_WARPS * 32) put(d, 1.0, 0.0);
    __syncthreads();
    const int partner = hl * 8 >= a.rope ? lane : hl * 8 < half ? lane + a.rope / 16 : lane - a.rope / 16;      // has the dims these are rotated with
    auto halves = [](const uint4& v, float x[8]) {
        const __half2* h = reinterpret_cast<const __half2*>(&v);
#pragma unroll
        for (int k = 0; k < 4; ++k) { const float2 f = __half22float2(h[k]); x[2 * k] = f.x; x[2 * k + 1] = f.y; }
    };
    auto weight = [&](const __half* w, float x[8]) { halves(w ? reinterpret_cast<const uint4*>(w)[hl] : make_uint4(0, 0, 0, 0), x); };
    if (nk) {
        int pg, off;
        kv4_place(c, slot, pg, off);
        const int at = off % KV4_B;
        unsigned char* blk = kv4_block(c, pg, 0, off / KV4_B);               // (head 0's)
        const int64_t head_bytes = (int64_t)(c.page_size / KV4_B) * kv4_block_bytes(D);
        for (int t = k0; t < nk; t += stride) {
            const int head = t * HPW + hs;
            float x[8];
            halves(kraw, x);
            kraw = load(ksrc, a.k_head, t + stride, c.KV);
            if (a.k_norm || a.rope) {
                double y[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) y[k] = (double)x[k];
                if (a.k_norm) {
                    float w[8];
                    weight(a.k_norm, w);
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
                    const double2 cs = s_d[k][hl];
                    const double other = __shfl_sync(0xffffffffu, y[k], partner);
                    x[k] = h2f(f2h((float)fma(other, cs.y, y[k] * cs.x)));
                }
            }
            kv4_store(c, blk + head * head_bytes, at, 0, hl, x, head < c.KV);
        }
        for (int t = v0; t < nk; t += stride) {
            const int head = t * HPW + hs;
            float x[8];
            halves(vraw, x);
            vraw = load(vsrc, a.v_head, t + stride, c.KV);
            kv4_store(c, blk + head * head_bytes, at, 1, hl, x, head < c.KV);
        }
    }
    if (q0 >= nq) return;
    float w[8], cs[8], sn[8];
    weight(a.q_norm, w);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float4 f = *reinterpret_cast<const float4*>(s_f[j][hl]);
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
        const float s = h2f(__ldg(sb)), b = h2f(__ldg(sb + KV4_B));
        uint4 o; __half* oh = reinterpret_cast<__half*>(&o);
#pragma unroll
        for (int j = 0; j < 8; ++j) oh[j] = f2h(fmaf((float)(w >> (4 * j) & 15u), s, b));
        __half* dst = region ? a.v + row * a.v_row + head * a.v_head : a.k + row * a.k_row + head * a.k_head;
        reinterpret_cast<uint4*>(dst)[hl] = o;
    }
}

int launch_kv4_append(const Kv4Cache& c, const Kv4AppendArgs& a, cudaStream_t st) {
    const int hpw = 32 / (c.D / 8), tasks = (a.q ? (a.NH + hpw - 1) / hpw : 0) + (a.k ? 2 * ((c.KV + hpw - 1) / hpw) : 0);
    // few rows: every task a warp of its own
    const int parts = a.rows < 4 * sm_count() ? (tasks + KA_WARPS - 1) / KA_WARPS : 1;
    const dim3 grid((unsigned)a.rows, (unsigned)parts);
    int rc = 0;
    profile_launch("k_kv4_append", st, [&] {
        if (c.D == 64) return rc = launch_pdl(false, k_kv4_append<64>, grid, KA_WARPS * 32, 0, st, c, a);
        if (c.D == 128) return rc = launch_pdl(false, k_kv4_append<128>, grid, KA_WARPS * 32, 0, st, c, a);
        return rc = launch_pdl(false, k_kv4_append<256>, grid, KA_WARPS * 32, 0, st, c, a);
    });
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

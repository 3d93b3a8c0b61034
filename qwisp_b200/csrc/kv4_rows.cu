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

constexpr int KA_WARPS = 8;

__device__ __forceinline__ uint32_t kv4_code(float x, float bias, float scale) {
    return (uint32_t)fminf(fmaxf(roundf(__fdiv_rn(__fsub_rn(x, bias), scale)), 0.0f), 15.0f);
}
// Eight dims of a head a lane, eight lanes a group: stores the lane's word of codes and the group's scale and bias.  By whole warps;
// `store`: the lane has a head.  region: 0 = K, 1 = V.
__device__ __forceinline__ void kv4_store(const Kv4Cache& c, unsigned char* blk, int at, int region, int hl, const float x[8], bool store) {
    float lo = x[0], hi = x[0];
    bool odd = !(fabsf(x[0]) <= 65504.0f);
#pragma unroll
    for (int i = 1; i < 8; ++i) { lo = fminf(lo, x[i]); hi = fmaxf(hi, x[i]); odd |= !(fabsf(x[i]) <= 65504.0f); }
#pragma unroll
    for (int d = 1; d < 8; d <<= 1) { lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, d)); hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, d)); }
    odd = (__ballot_sync(0xffffffffu, odd) >> (threadIdx.x & 24) & 0xffu) != 0;
    float scale = fmaxf(__fdiv_rn(__fsub_rn(hi, lo), 15.0f), 1e-7f);
    const bool side = fabsf(lo) > fabsf(hi);
    scale = side ? scale : -scale;
    const float edge = side ? lo : hi, q0 = roundf(__fdiv_rn(edge, scale));
    const bool zero = q0 == 0.0f;
    scale = zero ? scale : __fdiv_rn(edge, q0);
    const float bias = zero ? 0.0f : edge;
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) w |= kv4_code(x[i], bias, scale) << (4 * i);
    if (!store) return;
    *reinterpret_cast<uint32_t*>(blk + region * 8 * c.D + kv4_swz((uint32_t)(at * (c.D / 2) + hl * 4))) = w;
    if ((hl & 7) == 0) {
        __half* sb = reinterpret_cast<__half*>(blk + (16 + region) * c.D) + (hl >> 3) * 2 * KV4_B + at;
        sb[0] = odd ? __ushort_as_half(0x7fff) : f2h(scale);
        sb[KV4_B] = f2h(bias);
    }
}

// A row's angles once per CTA: turns = position * frequency as a 64-bit fraction of a turn, exact for every position, then cos and
// sin in 64 bits.  Keys stay in 64 bits up to the one rounding to fp16 (a code next to a border then does not go by the order of a sum or
// by the shape of the launch); queries take 32.
// grid (rows, parts), a warp a task: 32 / (D / 8) heads of one kind, eight dims a lane.
template <int D>
__global__ void __launch_bounds__(KA_WARPS * 32) k_kv4_append(Kv4Cache c, Kv4AppendArgs a) {
    constexpr int LPH = D / 8, HPW = 32 / LPH;                // lanes of a head, heads of a warp
    __shared__ double2 s_cs[D / 2];
    const int row = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, hl = lane % LPH, hs = lane / LPH;
    const int64_t slot = a.slots ? a.slots[row] : 0;
    if (a.slots && (slot < 0 || slot >= c.pages * (int64_t)c.page_size)) return;         // padding
    const int half = a.rope >> 1;
    for (int i = tid; i < half; i += KA_WARPS * 32) {
        const uint64_t t = (uint64_t)(int64_t)a.pos[(int64_t)a.axis[i] * a.pos_axis + row] * a.turn[i];      // (modulo 2^64: a whole turn)
        double sn, cs;
        sincospi((double)(int64_t)t * 0x1p-63, &sn, &cs);
        s_cs[i] = make_double2(cs, sn);
    }
    __syncthreads();
    const int nq = a.q ? (a.NH + HPW - 1) / HPW : 0, nk = a.k ? (c.KV + HPW - 1) / HPW : 0;
    unsigned char* page = nullptr; int blk = 0, at = 0;
    if (nk) {
        const int off = (int)(slot % c.page_size);
        page = kv4_block(c, (int)(slot / c.page_size), 0, 0); blk = off / KV4_B; at = off % KV4_B;
    }
    const int64_t head_bytes = (int64_t)(c.page_size / KV4_B) * kv4_block_bytes(D);
    const int src_lane = hl < a.rope / 16 ? lane + a.rope / 16 : lane - a.rope / 16;     // has the dims these are rotated with
    const bool turned = hl * 8 < a.rope, first = hl * 8 < half;
    for (int task = blockIdx.y * KA_WARPS + warp; task < nq + 2 * nk; task += gridDim.y * KA_WARPS) {
        const int kind = task < nq ? 0 : task < nq + nk ? 1 : 2, head = (task - (kind ? nq + (kind - 1) * nk : 0)) * HPW + hs;
        const bool have = head < (kind ? c.KV : a.NH);
        const __half* src = kind == 0 ? a.q + row * a.q_row + head * a.q_head : kind == 1 ? a.k + row * a.k_row + head * a.k_head : a.v + row * a.v_row + head * a.v_head;
        uint4 raw = make_uint4(0, 0, 0, 0);
        if (have) raw = reinterpret_cast<const uint4*>(src)[hl];
        const __half* h = reinterpret_cast<const __half*>(&raw);
        unsigned char* dst = page + head * head_bytes + (int64_t)blk * kv4_block_bytes(D);
        if (kind == 2) {
            float x[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = h2f(h[i]);
            kv4_store(c, dst, at, 1, hl, x, have);
            continue;
        }
        const __half* w = kind ? a.k_norm : a.q_norm;
        uint4 wraw = make_uint4(0, 0, 0, 0);
        if (w) wraw = reinterpret_cast<const uint4*>(w)[hl];
        const __half* wh = reinterpret_cast<const __half*>(&wraw);
        if (kind == 0) {
            float x[8], ss = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) { x[i] = h2f(h[i]); ss = fmaf(x[i], x[i], ss); }
            if (w) {
#pragma unroll
                for (int d = 1; d < LPH; d <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, d);
                const float inv = 1.0f / sqrtf(ss * (1.0f / D) + a.eps);
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] = x[i] * inv * h2f(wh[i]);
            }
            uint4 o; __half* oh = reinterpret_cast<__half*>(&o);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float other = __shfl_sync(0xffffffffu, x[i], src_lane);
                if (turned) {
                    const double2 cs = s_cs[first ? hl * 8 + i : hl * 8 + i - half];
                    x[i] = first ? x[i] * (float)cs.x - other * (float)cs.y : x[i] * (float)cs.x + other * (float)cs.y;
                }
                oh[i] = f2h(x[i]);
            }
            if (have) reinterpret_cast<uint4*>(a.q_out + row * a.o_row + head * a.o_head)[hl] = o;
        } else {
            double x[8], ss = 0.0;
#pragma unroll
            for (int i = 0; i < 8; ++i) { x[i] = (double)h2f(h[i]); ss = fma(x[i], x[i], ss); }
            if (w) {
#pragma unroll
                for (int d = 1; d < LPH; d <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, d);
                const double inv = 1.0 / sqrt(ss * (1.0 / D) + (double)a.eps);
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] = x[i] * inv * (double)h2f(wh[i]);
            }
            float y[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const double other = __shfl_sync(0xffffffffu, x[i], src_lane);
                if (turned) {
                    const double2 cs = s_cs[first ? hl * 8 + i : hl * 8 + i - half];
                    x[i] = first ? x[i] * cs.x - other * cs.y : x[i] * cs.x + other * cs.y;
                }
                y[i] = h2f(f2h((float)x[i]));
            }
            kv4_store(c, dst, at, 0, hl, y, have);
        }
    }
}

// a lane a word of codes: eight dims of K or V of a (row, head)
template <int D>
__global__ void __launch_bounds__(256) k_kv4_read(Kv4Cache c, Kv4ReadArgs a) {
    constexpr int LPH = D / 8;
    const int64_t n = (int64_t)a.rows * c.KV * 2 * LPH;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        const int hl = (int)(i % LPH), region = (int)(i / LPH & 1), head = (int)(i / (2 * LPH) % c.KV);
        const int64_t row = i / ((int64_t)2 * LPH * c.KV), slot = a.slots[row];
        if (slot < 0 || slot >= c.pages * (int64_t)c.page_size) continue;
        const int off = (int)(slot % c.page_size), at = off % KV4_B;
        const unsigned char* blk = kv4_block(c, (int)(slot / c.page_size), head, off / KV4_B);
        const uint32_t w = *reinterpret_cast<const uint32_t*>(blk + region * 8 * D + kv4_swz((uint32_t)(at * (D / 2) + hl * 4)));
        const __half* sb = reinterpret_cast<const __half*>(blk + (16 + region) * D) + (hl >> 3) * 2 * KV4_B + at;
        const float s = h2f(sb[0]), b = h2f(sb[KV4_B]);
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
    const int64_t n = (int64_t)a.rows * c.KV * 2 * (c.D / 8), want = (n + 255) / 256, most = (int64_t)sm_count() * 64;
    const dim3 grid((unsigned)(want < most ? want : most));
    int rc = 0;
    profile_launch("k_kv4_read", st, [&] {
        if (c.D == 64) return rc = launch_pdl(false, k_kv4_read<64>, grid, 256, 0, st, c, a);
        if (c.D == 128) return rc = launch_pdl(false, k_kv4_read<128>, grid, 256, 0, st, c, a);
        return rc = launch_pdl(false, k_kv4_read<256>, grid, 256, 0, st, c, a);
    });
    return rc;
}

}  // namespace sl

// kv4_mma.cuh -- pieces of the attention kernels over the cache held in 4 bits.
#pragma once
#include "common.cuh"
#include <atomic>

namespace sl {

__device__ __forceinline__ void kv4_cp16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void kv4_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void kv4_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void kv4_ldsm(uint32_t r[4], uint32_t p) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(p) : "memory");
}
__device__ __forceinline__ void kv4_ldsm_t(uint32_t r[4], uint32_t p) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(p) : "memory");
}
__device__ __forceinline__ void kv4_mma(float c[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// an 8 x 8 matrix of halves, two of a row a lane, transposed
__device__ __forceinline__ uint32_t kv4_transpose(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ float kv4_exp2(float x) { float r; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x)); return r; }
// Pairs of f32 values in one 64-bit register (one instruction, the bits of two), and the larger of three
typedef unsigned long long kv4_f2;
__device__ __forceinline__ kv4_f2 kv4_pair(float x, float y) { kv4_f2 r; asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y)); return r; }
__device__ __forceinline__ float2 kv4_unpair(kv4_f2 v) { float2 r; asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v)); return r; }
__device__ __forceinline__ kv4_f2 kv4_fma2(kv4_f2 a, kv4_f2 b, kv4_f2 c) { kv4_f2 r; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c)); return r; }
__device__ __forceinline__ kv4_f2 kv4_add2(kv4_f2 a, kv4_f2 b) { kv4_f2 r; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
__device__ __forceinline__ float kv4_max3(float a, float b, float c) { float r; asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c)); return r; }
__device__ __forceinline__ float kv4_min_nan(float a, float b) { float r; asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b)); return r; }      // (fminf drops a NaN)
// 1 / (1 + e^-x), some 2^-21 of itself off: an infinite power makes it 0, a NaN stays one
__device__ __forceinline__ float kv4_sigmoid(float x) { return __fdividef(1.0f, 1.0f + kv4_min_nan(kv4_exp2(x * -1.4426950408889634f), 0x1p126f)); }
__device__ __forceinline__ uint32_t kv4_pack(float a, float b) { const __half2 h = __floats2half2_rn(a, b); return *reinterpret_cast<const uint32_t*>(&h); }
__device__ __forceinline__ __half2 kv4_h2(uint32_t v) { return *reinterpret_cast<const __half2*>(&v); }
__device__ __forceinline__ uint32_t kv4_u(__half2 v) { return *reinterpret_cast<const uint32_t*>(&v); }
// Eight codes of a word -> halves code * s + b in pairs (0, 4), (1, 5), (2, 6), (3, 7).  A code in the low bits of a half whose exponent says
// 1024 is 1024 + code, four bits further up under an exponent of 64 it is 64 + code: one masking instruction a pair, an exact
// subtraction and one multiply-add with one rounding.  (Mask and exponent written in C took two instructions.)
template <uint32_t MASK, uint32_t EXP> __device__ __forceinline__ __half2 kv4_codes(uint32_t w) {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(w), "n"(MASK), "r"(EXP));       // (w & MASK) | EXP
    return __hsub2(kv4_h2(r), kv4_h2(EXP));
}
__device__ __forceinline__ void kv4_expand(uint32_t w, __half2 s, __half2 b, uint32_t o[4]) {
    const uint32_t v = w >> 8;
    o[0] = kv4_u(__hfma2(kv4_codes<0x000f000fu, 0x64006400u>(w), s, b));
    o[1] = kv4_u(__hfma2(kv4_codes<0x00f000f0u, 0x54005400u>(w), s, b));
    o[2] = kv4_u(__hfma2(kv4_codes<0x000f000fu, 0x64006400u>(v), s, b));
    o[3] = kv4_u(__hfma2(kv4_codes<0x00f000f0u, 0x54005400u>(v), s, b));
}

// ---- the other CTAs of a cluster: a meeting of all of their threads, and places in their shared memory
__device__ __forceinline__ void kv4_cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t kv4_peer(uint32_t own, int rank) {        // where CTA `rank` has what this one has at `own`
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(own), "r"(rank));
    return r;
}
__device__ __forceinline__ float2 kv4_peer2(uint32_t p) {
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(p) : "memory");
    return v;
}
__device__ __forceinline__ float4 kv4_peer4(uint32_t p) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(p) : "memory");
    return v;
}

}  // namespace sl

// kv4_prompt.cu -- attention of many query rows of a request over the cache held in 4 bits (kv4.cuh), on the 5th-generation tensor cores.
//
// A CTA takes NQ tiles of 128 rows (tokens x query heads of one kv head, so that the codes are expanded once for all of a kv head's
// query heads) and walks the keys 64 at a time.  Warps have roles and meet only at mbarriers:
//   mma       1 warp: S = Q K^T (queries as the A operand, in tensor memory where there is room for them, keys in shared memory) and O += P V
//             (weights in tensor memory where the scores were, values in shared memory).  Scores are double buffered, so those of the next
//             64 keys are ready before the weights of these are: with one buffer a tile's softmax waited for its own MMAs each time;
//   expand    4 or 8 warps: a block of 16 keys or half of one each, codes from global memory a tile ahead, to fp16 (one multiply-add a pair),
//             into 128-byte swizzled tiles: rows of 64 dims, K-major for the scores and, the same bytes, MN-major for the values.  A word
//             expands to its dims in the order 0 4 1 5 2 6 3 7; the queries are loaded and the outputs stored in that order;
//   softmax   4 warps a tile, a thread a row: scores in, running maximum and sum in registers, weights out.  The maximum is raised (and the
//             outputs rescaled) only when a score exceeds it by 2^6; the weights are carried times 2^8, so that fp16 holds them from 2^-32 of the
//             largest on.
// NQ = 2 (D 64, 128): the expansion serves two tiles.  NQ = 1 (D 256): the outputs of one take half of tensor memory; (D 64) requests of one tile.
// SPLIT: where there are fewer tiles than multiprocessors a cluster of up to eight CTAs takes each, a run of the keys a CTA, and adds up its sums through shared
// memory.  17 rows over 4017 positions, 32/8 heads of 128: 55 us with one CTA, 18.5 with eight.
//
// What bounds it: 1024 rows over 8192 positions, 16/2 heads of 256: 134 us, 0.96 PFLOP/s = 0.57 of the measured cuBLAS rate; four prompts of up to
// 2900, 32/8 heads of 128: 227 us, 0.75 PFLOP/s = 0.45.  No unit is full (tensor pipe 39 %, MUFU 40 %, ALU 33 %, issue slots 43 % of the second): each tile of
// 64 keys is a chain scores -> exponents -> weights -> outputs over barriers, which two tiles of rows overlap only in part, and every CTA begins
// and ends alone (about 10 of 29 us there).  Leaving out the exponentials gave 12 %, the expansion 5 %, half of the MMAs nothing.  Tried, and no faster:
// tiles of 128 keys with one score buffer (7 % slower), two CTAs of one tile each (1.8 times the time: twice the expansion, 96 registers), more expanding
// warps with registers moved between the roles, a polynomial in place of some MUFU exponentials.
#include "kv4.cuh"
#include "kv4_mma.cuh"

namespace sl {

constexpr int KP_M = 128, KP_N = 64, KP_ST = 3;
// (D, NQ): two tiles a CTA; D 256: one, whose outputs alone take half of tensor memory
template <int D, int NQ> constexpr int kp_ctas = D == 64 && NQ == 1 ? 2 : 1;   // CTAs of a multiprocessor
template <int D> constexpr int kp_exp = D == 256 ? 8 : 4;                     // expanding warps
template <int D, int NQ> constexpr int kp_threads = (1 + kp_exp<D> + 4 * NQ) * 32;
template <int D> constexpr int kp_tile = KP_N * D * 2;                        // bytes of a tile of keys or values
template <int D> constexpr bool kp_qt = D != 128;                            // queries in tensor memory (128 dims: outputs and scores fill it)
template <int D, int NQ> constexpr int kp_io = 4 * NQ * 4096;      // where a softmax warp turns 32 rows of 64 dims
template <int D, int NQ> constexpr int kp_bytes = 2 * KP_ST * kp_tile<D> + kp_io<D, NQ> + (kp_qt<D> ? 0 : NQ * KP_M * D * 2);
// So much that no more of these kernels' CTAs, calls on other streams included, come to a multiprocessor than there is tensor memory for.
// tcgen05.alloc and the meetings of a cluster wait without a limit: two clusters, each with a CTA that has its tensor memory and one that waits
// for the other cluster's, would wait for ever.
template <int D, int NQ> constexpr int kp_least = (kp_ctas<D, NQ> == 2 ? 80 : 148) * 1024;
template <int D, int NQ> constexpr int kp_smem = (kp_bytes<D, NQ> > kp_least<D, NQ> ? kp_bytes<D, NQ> : kp_least<D, NQ>) + 1024;
constexpr int KP_SM = 228 * 1024;                                            // of a multiprocessor; a CTA takes 1 KB more than it asks for
static_assert(3 * (kp_smem<64, 1> + 1024) > KP_SM && kp_smem<64, 1> + kp_smem<64, 2> + 2048 > KP_SM && kp_smem<64, 1> + kp_smem<128, 2> + 2048 > KP_SM &&
              kp_smem<64, 1> + kp_smem<256, 1> + 2048 > KP_SM && 2 * (kp_smem<64, 2> + 1024) > KP_SM && kp_smem<64, 2> + kp_smem<128, 2> + 2048 > KP_SM &&
              kp_smem<64, 2> + kp_smem<256, 1> + 2048 > KP_SM && 2 * (kp_smem<128, 2> + 1024) > KP_SM && kp_smem<128, 2> + kp_smem<256, 1> + 2048 > KP_SM &&
              2 * (kp_smem<256, 1> + 1024) > KP_SM, "tensor memory of a multiprocessor");
constexpr int KP_LIMIT = 1 << 22;                                            // polls of a wait (up to 4 us each)
constexpr float KP_UP = 8.0f, KP_SLACK = 6.0f;

__device__ __forceinline__ uint64_t kp_desc(uint32_t addr, uint32_t lbo, uint32_t sbo) {      // version 1, 128-byte swizzle
    return (uint64_t)((addr >> 4) & 0x3FFFu) | ((uint64_t)(lbo >> 4) << 16) | ((uint64_t)(sbo >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
// D (tensor memory) (+)= A (tensor memory) B (shared memory)
__device__ __forceinline__ void kp_mma(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
                 ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void kp_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {      // both operands in shared memory
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void kp_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void kp_ld32(uint32_t t, uint32_t* r) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
                 "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]),
                   "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]),
                   "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]) : "r"(t) : "memory");
}
__device__ __forceinline__ void kp_st32(uint32_t t, const uint32_t* r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
                 "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
                 ::"r"(t), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
                   "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]),
                   "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]) : "memory");
}
__device__ __forceinline__ void kp_st16(uint32_t t, const uint32_t* r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
                 ::"r"(t), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
                   "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]) : "memory");
}
__device__ __forceinline__ void kp_sts(uint32_t p, const uint4& v) { asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(p), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory"); }
__device__ __forceinline__ uint4 kp_lds(uint32_t p) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(p) : "memory");
    return v;
}
__device__ __forceinline__ void kp_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void kp_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void kp_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void kp_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void kp_arrive(uint64_t* b) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(b)) : "memory"); }
__device__ __forceinline__ bool kp_elect() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}
// Bounded wait of a whole warp.  The first that runs out raises the CTA's abort word, and every later one gives up soon; a role then leaves
// its loop (nothing in the CTA waits for it unboundedly) and the rows come out as NaN.
__device__ __forceinline__ bool kp_wait_one(uint64_t* b, uint32_t parity, volatile int* abort_word) {      // by one thread
    if (mbar_try_wait(b, parity)) return true;
    for (int i = 0; i < KP_LIMIT; ++i) {
        if (mbar_try_wait(b, parity)) return true;
        if ((i & 255) == 255 && *abort_word) break;
    }
    *abort_word = 1;
    return false;
}
__device__ __forceinline__ bool kp_wait(uint64_t* b, uint32_t parity, volatile int* abort_word) {          // by a whole warp
    return __all_sync(0xffffffffu, kp_wait_one(b, parity, abort_word));
}

// CTAs (clusters) of a kv head at most: one a request where its rows are one CTA's, else its last tile may be short
template <int D, int NQ> static bool kp_one(const Kv4AttnArgs& a) { return a.max_q <= KP_M / a.G * NQ; }
template <int D, int NQ> static long long kp_items(const Kv4AttnArgs& a) { return kp_one<D, NQ>(a) ? a.batch : (long long)a.rows / (KP_M / a.G * NQ) + a.batch; }
constexpr int KP_PARTS = 8;                                                   // CTAs of a cluster at most
constexpr int KP_SPLIT = 256;                                                // keys a CTA of a cluster has at least, of a table's span
struct KpSeq { int q0, rows, keys, past; };                                   // past: keys before the first row's own (as many as the table's, if more)

template <int D, int NQ, bool SPLIT>
__global__ void __launch_bounds__(kp_threads<D, NQ>, kp_ctas<D, NQ>) k_kv4_prompt(Kv4Cache c, Kv4AttnArgs a, int least, uint32_t q_and, uint32_t q_xor, int parts) {
    constexpr int TILE = kp_tile<D>, NT = kp_threads<D, NQ>, W = NT / 32, SW0 = 4;      // softmax warps start at SW0
    constexpr bool QT = kp_qt<D>;
    constexpr uint32_t S0 = NQ * D, Q0 = S0 + NQ * 2 * KP_N, COLUMNS = 512 / kp_ctas<D, NQ>;      // of tensor memory: outputs, scores (two of each tile), queries
    static_assert(Q0 + (QT ? NQ * D / 2 : 0) <= COLUMNS, "tensor memory");
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    __shared__ __align__(8) uint64_t full[KP_ST], empty[KP_ST], s_full[2 * NQ], p_full[2 * NQ], q_full, o_done[2 * NQ];
    __shared__ uint32_t s_tmem;
    __shared__ float2 s_ml[SPLIT ? NQ * KP_M : 1];                            // SPLIT: the rows' (maximum, sum)
    static_assert(!SPLIT || NQ * KP_M * D * 4 <= kp_smem<D, NQ> - 1024, "");
    __shared__ KpSeq s_seq;
    __shared__ int s_abort, s_b, s_tile, s_sum[W];
    __shared__ __align__(4) uint8_t s_have[8][4];                             // whether a tile's blocks of 16 keys exist (softmax is up to four tiles behind)
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    const int tokens = KP_M / a.G, per_cta = tokens * NQ, CL = SPLIT ? parts : 1, rank = SPLIT ? (int)blockIdx.x % CL : 0;
    const int head = (int)blockIdx.x / CL % c.KV, item = (int)blockIdx.x / CL / c.KV;
    // ---- which request, and which of its tiles: the longest of a request first, of all kv heads (head by head, each head's shortest before the next
    // one's longest: 4 prompts of up to 2900, 238 us for 218; one of 4096: 177 for 148)
    if (tid == 0) { s_b = -1; s_abort = 0; }
    __syncthreads();
    for (int b0 = 0, base = 0; b0 < a.batch; b0 += NT) {
        const int b = b0 + tid;
        int x = 0;
        KpSeq one{0, 0, 0, 0};
        if (b < a.batch) {
            one.q0 = a.q_start[b];
            const int n = a.q_start[b + 1] - one.q0, len = max(a.kv_len[b], 0);
            one.rows = min(min(n, a.max_q), a.rows - one.q0);
            one.keys = min(len, a.table_width * c.page_size);
            one.past = min(len - n, one.keys);
            if (one.q0 >= 0 && one.rows > least / a.G) x = (one.rows + per_cta - 1) / per_cta;
        }
        const int own = x;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) { const int u = __shfl_up_sync(0xffffffffu, x, d); if (lane >= d) x += u; }
        if (lane == 31) s_sum[warp] = x;
        __syncthreads();
        int all = 0;
        x += base;
        for (int w = 0; w < W; ++w) { if (w < warp) x += s_sum[w]; all += s_sum[w]; }
        if (item < x && item >= x - own) { s_b = b; s_tile = x - 1 - item; s_seq = one; }
        base += all;
        __syncthreads();
        if (s_b >= 0) break;
    }
    // (Launched ahead of the end of the kernels for few rows, with whose requests it shares nothing.  Every thread waits for them before it
    // leaves, so that what follows this kernel in the stream follows those too.)
    const int b = s_b;
    if (b < 0) { pdl_wait(); return; }
    const KpSeq sq = s_seq;
    const int t0 = s_tile * per_cta;                                          // first token
    const int nq = NQ == 1 || t0 + tokens >= sq.rows ? 1 : 2;                 // tiles that have rows
    const int last = min(t0 + per_cta, sq.rows) - 1;
    const int span = a.causal ? min(sq.keys, max(0, sq.past + last + 1)) : sq.keys;
    // keys KP_N j0 .. : all of them, or the cluster's CTAs share them out
    const int all_tiles = (span + KP_N - 1) / KP_N, per = (all_tiles + CL - 1) / CL, j0 = min(rank * per, all_tiles);
    const int tiles = min(per, all_tiles - j0);
    if (tid == 0) {
        for (int i = 0; i < KP_ST; ++i) { mbar_init(&full[i], kp_exp<D>); mbar_init(&empty[i], 1); }
        for (int i = 0; i < 2 * NQ; ++i) { mbar_init(&s_full[i], 1); mbar_init(&p_full[i], 4); mbar_init(&o_done[i], 1); }
        mbar_init(&q_full, 4 * nq);
        mbar_fence_init();
    }
    if (warp == 0) {
        __syncwarp();
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)), "r"(COLUMNS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    kp_before();
    __syncthreads();
    kp_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, s_tmem, 0), smem0 = smem_u32(smem), io0 = smem0 + 2 * KP_ST * TILE, qs0 = io0 + kp_io<D, NQ>;
    bool ok = true;
    if (warp == 0) {
        // ------------------------------------------------------------ mma
        if (tiles > 0) {
            constexpr uint32_t ID_S = (1u << 4) | ((uint32_t)(KP_N >> 3) << 17) | ((uint32_t)(KP_M >> 4) << 24);                  // f32 += f16 x f16, K-major B
            constexpr uint32_t ID_O = (1u << 4) | (1u << 16) | ((uint32_t)(D >> 3) << 17) | ((uint32_t)(KP_M >> 4) << 24);       // MN-major B
            const uint64_t dk = kp_desc(smem0, 16, 1024), dv = kp_desc(smem0 + KP_ST * TILE, KP_N * 128, 1024);
            // One lane, elected once, does all of it: MMAs are ordered, and their commits count, by thread.  (With the whole warp walking the
            // tiles, votes and meetings around each wait cost more than the addresses that uniform registers saved.)
            if (kp_elect()) {
            const uint64_t dq = kp_desc(qs0, 16, 1024);
            auto scores = [&](int q, int slot, uint64_t keys) {
                {
                    const uint32_t d = tmem + S0 + (2 * q + slot) * KP_N, x = tmem + Q0 + q * (D / 2);
                    const uint64_t y = dq + (uint32_t)(q * (KP_M * D * 2 >> 4));
#pragma unroll
                    for (int i = 0; i < D / 16; ++i) {
                        const uint64_t k = keys + (uint32_t)((i >> 2) * (KP_N * 128 >> 4) + (i & 3) * 2);
                        if (QT) kp_mma(d, x + i * 8, k, ID_S, i > 0 ? 1u : 0u);
                        else kp_mma_ss(d, y + (uint32_t)((i >> 2) * (KP_M * 128 >> 4) + (i & 3) * 2), k, ID_S, i > 0 ? 1u : 0u);
                    }
                    kp_commit(&s_full[2 * q + slot]);
                }
            };
            ok = kp_wait_one(&q_full, 0, &s_abort) && kp_wait_one(&full[0], 0, &s_abort);
            kp_after();
            if (ok) for (int q = 0; q < nq; ++q) scores(q, 0, dk);
            int st = 0, nst = 1; uint32_t nph = 0;                            // stage of tile j and of the next, phase of the next one's
            for (int j = 0; j < tiles && ok; ++j) {
                const bool more = j + 1 < tiles;
                if (more) ok = kp_wait_one(&full[nst], nph, &s_abort) && ok;
                kp_after();
                const uint64_t kn = dk + (uint32_t)(nst * (TILE >> 4)), v = dv + (uint32_t)(st * (TILE >> 4));
                if (more && ok) {
                    scores(0, (j + 1) & 1, kn);
                    if (NQ == 2 && nq == 2) scores(NQ - 1, (j + 1) & 1, kn);
                }
#pragma unroll
                for (int q = 0; q < NQ; ++q) {
                    if (q >= nq || !ok) break;
                    ok = kp_wait_one(&p_full[2 * q + (j & 1)], (uint32_t)(j >> 1) & 1u, &s_abort);
                    if (!ok) break;
                    kp_after();
                    {
                        const uint32_t d = tmem + q * D, x = tmem + S0 + (2 * q + (j & 1)) * KP_N;
                        kp_mma(d, x, v, ID_O, j > 0 ? 1u : 0u);
#pragma unroll
                        for (int i = 1; i < KP_N / 16; ++i) kp_mma(d, x + i * 8, v + (uint32_t)(i * (2048 >> 4)), ID_O, 1u);
                        if (q == nq - 1) kp_commit(&empty[st]);
                        kp_commit(&o_done[2 * q + (j & 1)]);
                    }
                }
                st = nst;
                if (++nst == KP_ST) { nst = 0; nph ^= 1u; }
            }
            }
        }
    } else if (warp < SW0 || warp >= SW0 + 4 * NQ) {
        // ------------------------------------------------------------ expand: keys PER e .. of every tile
        // Pieces of 32 dims of a key, NC of K and of V a lane, half of the head apart.  Where a lane's pieces lie in a block and in a tile does
        // not change: a pointer for each, and constants from there.
        constexpr int CH = D / 32, PER = KP_N / kp_exp<D>, NC = CH * PER / 32, HALF = CH / 2;      // HALF: pieces of half a head
        const int e = warp < SW0 ? warp - 1 : warp - (SW0 + 4 * NQ) + SW0 - 1, key = lane & (PER - 1), at = (e * PER + key) % KV4_B;      // at: position in its block of 16
        const int page_blocks = c.page_size / KV4_B, ch = lane / PER;
        const int* table = a.table + (int64_t)b * a.table_stride;
        const int code_at = (int)kv4_swz((uint32_t)(at * (D / 2) + ch * 16)), sb_at = 16 * D + ((ch >> 1) * 32 + at) * 2;
        uint32_t to[4];                                                       // (a row of 64 dims: 128 bytes, its 16-byte pieces XORed with the key)
#pragma unroll
        for (int x = 0; x < 4; ++x) to[x] = (ch >> 1) * (KP_N * 128) + (e * PER + key) * 128 + (((((ch & 1) << 2) + x) ^ (key & 7)) << 4);
        unsigned long long page_at = 0;                                       // the block of tile (j & ~31) + lane, 0: there is none
        auto block_of = [&](int j) -> const unsigned char* {
            if ((j & 31) == 0) {
                const int blk = (j0 + j + lane) * (KP_N / KV4_B) + e * PER / KV4_B, pg = blk / page_blocks;
                page_at = 0;
                if (j + lane < tiles && blk * KV4_B < sq.keys) {
                    const int page = table[pg];
                    if (page >= 0 && page < c.pages) page_at = (unsigned long long)kv4_block(c, page, head, blk - pg * page_blocks);
                }
            }
            return (const unsigned char*)__shfl_sync(0xffffffffu, page_at, j & 31);
        };
        struct Raw { uint4 code[2][NC]; __half s[2][NC], b[2][NC]; bool have; };
        auto fetch = [&](int j, Raw& r) {
            const unsigned char* p = j < tiles ? block_of(j) : nullptr;
            r.have = p != nullptr;
            auto load = [&] {
                const unsigned char *code = p + code_at, *other = p + (code_at ^ (HALF * 16)), *sb = p + sb_at;
#pragma unroll
                for (int v = 0; v < 2; ++v)
#pragma unroll
                    for (int k = 0; k < NC; ++k) {
                        r.code[v][k] = *reinterpret_cast<const uint4*>((k ? other : code) + v * 8 * D);
                        const __half* h = reinterpret_cast<const __half*>(sb + v * D + k * (HALF / 2) * 64);
                        r.s[v][k] = h[0]; r.b[v][k] = h[16];
                    }
            };
            if (p && (j0 + j + 1) * KP_N <= sq.keys) load();
            else {                                                            // the last tile, or no page: what lies behind the keys is zero
#pragma unroll
                for (int v = 0; v < 2; ++v)
#pragma unroll
                    for (int k = 0; k < NC; ++k) { r.code[v][k] = make_uint4(0, 0, 0, 0); r.s[v][k] = r.b[v][k] = __ushort_as_half(0); }
                if (p && (j0 + j) * KP_N + e * PER + key < sq.keys) load();
                __syncwarp();
            }
        };
        int st = 0; uint32_t ph = 1;                                          // (a fresh barrier passes at 1)
        auto work = [&](int j, const Raw& now) {
            ok = kp_wait(&empty[st], ph, &s_abort);
            if (!ok) return;
            uint32_t at_x[4];
#pragma unroll
            for (int x = 0; x < 4; ++x) at_x[x] = to[x] + st * TILE;
#pragma unroll
            for (int v = 0; v < 2; ++v)
#pragma unroll
                for (int k = 0; k < NC; ++k) {
                    const __half2 s = __half2half2(now.s[v][k]), bi = __half2half2(now.b[v][k]);
                    const uint32_t w[4] = {now.code[v][k].x, now.code[v][k].y, now.code[v][k].z, now.code[v][k].w};
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        uint32_t o[4];
                        kv4_expand(w[x], s, bi, o);
                        *reinterpret_cast<uint4*>(smem + at_x[x] + (v * KP_ST * TILE + k * (HALF / 2) * (KP_N * 128))) = make_uint4(o[0], o[1], o[2], o[3]);
                    }
                }
            if (e * PER % KV4_B == 0 && lane == 0) s_have[j & 7][e * PER / KV4_B] = now.have;      // (read by softmax behind the scores, which wait for this)
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) kp_arrive(&full[st]);
            if (++st == KP_ST) { st = 0; ph ^= 1u; }
        };
        Raw one, two;
        fetch(0, one);
        for (int j = 0; j < tiles && ok; j += 2) {
            fetch(j + 1, two);
            work(j, one);
            if (j + 1 >= tiles || !ok) break;
            fetch(j + 2, one);
            work(j + 1, two);
        }
    } else {
        // ------------------------------------------------------------ softmax: a thread a row
        const int q = (warp - SW0) >> 2, row = (warp & 3) * 32 + lane;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        if (q < nq) {
            const int tok = t0 + q * tokens + row / a.G, h = head * a.G + row % a.G;
            const bool live = row < tokens * a.G && tok < sq.rows;
            const uint32_t io = io0 + (warp - SW0) * 4096, own = io + lane * 128;                // 32 rows of 128 bytes, 16-byte pieces XORed with the row
            auto place = [&](int64_t by_row, int64_t by_head) { return live ? (int64_t)(sq.q0 + tok) * by_row + (int64_t)h * by_head : (int64_t)-1; };
            // 64 dims of the warp's rows, eight lanes a row: 128 bytes at a time
            auto rows_in = [&](const __half* src, int64_t mine, int d, uint4 v[8]) {
                // (a row that there is none of reads the first, so that no load is behind a branch: eight in flight, not one)
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = __ldcg(reinterpret_cast<const uint4*>(src + max(__shfl_sync(0xffffffffu, mine, i * 4 + (lane >> 3)), (int64_t)0) + d + (lane & 7) * 8));
#pragma unroll
                for (int i = 0; i < 8; ++i) if (__shfl_sync(0xffffffffu, mine, i * 4 + (lane >> 3)) < 0) v[i] = make_uint4(0, 0, 0, 0);
            };
            auto turn = [&](int i) { const int r = i * 4 + (lane >> 3); return (uint32_t)(r * 128 + (((lane & 7) ^ (r & 7)) << 4)); };
            if (tiles > 0) {
                const int64_t mine = place(a.q_row, a.q_head);
#pragma unroll 1
                for (int d0 = 0; d0 < D; d0 += 128) {                         // (128 dims in flight)
                    constexpr int AT_ONCE = D == 64 ? 1 : 2;
                    uint4 v[AT_ONCE][8];
#pragma unroll
                    for (int k = 0; k < AT_ONCE; ++k) rows_in(a.q, mine, d0 + 64 * k, v[k]);
#pragma unroll
                    for (int k = 0; k < AT_ONCE; ++k) {
                        const int d = d0 + 64 * k;
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            // (x * 0 + x: an infinity, whose scores are infinities or NaN for every key, makes the row NaN whatever their signs, also where
                            // the scale is zero; anything finite is itself)
                            auto put = [&](uint32_t h) { return kv4_u(__hfma2(kv4_h2(h), kv4_h2(0u), kv4_h2(h & q_and))) ^ q_xor; };
                            const uint4 y = v[k][i], x = make_uint4(put(__byte_perm(y.x, y.z, 0x5410)), put(__byte_perm(y.x, y.z, 0x7632)), put(__byte_perm(y.y, y.w, 0x5410)), put(__byte_perm(y.y, y.w, 0x7632)));
                            kp_sts(QT ? io + turn(i) : qs0 + q * (KP_M * D * 2) + (d >> 6) * (KP_M * 128) + (warp & 3) * 4096 + turn(i), x);
                        }
                        if (QT) {
                            __syncwarp();
                            uint32_t r[32];
#pragma unroll
                            for (int i = 0; i < 8; ++i) *reinterpret_cast<uint4*>(r + 4 * i) = kp_lds(own + ((i ^ (lane & 7)) << 4));
                            kp_st32(tmem + lanes + Q0 + q * (D / 2) + d / 2, r);
                            __syncwarp();
                        }
                    }
                }
                if (QT) { kp_wait_st(); kp_before(); }
                else asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) kp_arrive(&q_full);
            }
            const int sees = !live ? 0 : a.causal ? sq.past + tok + 1 : sq.keys;
            // keys that all of the tile's rows see
            const int all = a.causal ? min(sq.keys, sq.past + t0 + q * tokens + 1) : sq.keys;
            float m = -INFINITY, l = 0.f;
            for (int j = 0; j < tiles && ok; ++j) {
                const int slot = 2 * q + (j & 1), k0 = (j0 + j) * KP_N;
                ok = kp_wait(&s_full[slot], (uint32_t)(j >> 1) & 1u, &s_abort);
                if (!ok) break;
                kp_after();
                const uint32_t have = *reinterpret_cast<const uint32_t*>(s_have[j & 7]);
                // (two CTAs a multiprocessor: half of the scores at a time, read twice, so that a thread's registers suffice)
                constexpr int PART = kp_ctas<D, NQ> == 2 ? 32 : 64;
                uint32_t r[PART];
                float* s = reinterpret_cast<float*>(r);
                const bool edge = k0 + KP_N > all || have != 0x01010101u;
                auto load = [&](int c0) {
#pragma unroll
                    for (int i = 0; i < PART; i += 32) kp_ld32(tmem + lanes + S0 + slot * KP_N + c0 + i, r + i);
                    kp_wait_ld();
                    if (edge) {
#pragma unroll
                        for (int i = 0; i < PART; ++i) if (k0 + c0 + i >= sees || !(have >> ((c0 + i) >> 4) * 8 & 1)) s[i] = -INFINITY;
                    }
                };
                float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int c0 = 0; c0 < KP_N; c0 += PART) {
                    load(c0);
                    if (PART == KP_N) {
#pragma unroll
                        for (int k = 0; k < 4; ++k) mx[k] = s[k];
#pragma unroll
                        for (int i = 4; i < PART - 4; i += 8)
#pragma unroll
                            for (int k = 0; k < 4; ++k) mx[k] = kv4_max3(mx[k], s[i + k], s[i + 4 + k]);
#pragma unroll
                        for (int k = 0; k < 4; ++k) mx[k] = fmaxf(mx[k], s[PART - 4 + k]);
                    } else {
#pragma unroll
                        for (int i = 0; i < PART; i += 8)
#pragma unroll
                            for (int k = 0; k < 4; ++k) mx[k] = kv4_max3(mx[k], s[i + k], s[i + 4 + k]);
                    }
                }
                const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * a.scale;
                if (__any_sync(0xffffffffu, top > m + KP_SLACK)) {
                    const float nm = fmaxf(m, top), f = nm == -INFINITY ? 1.f : kv4_exp2(m - nm);
                    m = nm; l *= f;
                    if (j > 0) {                                              // the outputs so far
                        // (a parity does not tell a phase from the one two before.  Even and odd tiles have a barrier each, and these scores'
                        // MMAs were issued, and so are done, behind O += P V of tile j - 2)
                        ok = kp_wait(&o_done[2 * q + ((j - 1) & 1)], (uint32_t)((j - 1) >> 1) & 1u, &s_abort);
                        if (!ok) break;
                        kp_after();
#pragma unroll 1
                        for (int c0 = 0; c0 < D; c0 += 32) {
                            uint32_t o[32];
                            kp_ld32(tmem + lanes + q * D + c0, o);
                            kp_wait_ld();
#pragma unroll
                            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                            kp_st32(tmem + lanes + q * D + c0, o);
                        }
                    }
                }
                const float base = KP_UP - (m == -INFINITY ? 0.f : m);
                kv4_f2 sum[2] = {0, 0};
                const kv4_f2 scale2 = kv4_pair(a.scale, a.scale), base2 = kv4_pair(base, base);
#pragma unroll
                for (int c0 = 0; c0 < KP_N; c0 += PART) {
                    if (PART < KP_N) load(c0);
#pragma unroll
                    for (int i0 = 0; i0 < PART / 2; i0 += 16) {
                        uint32_t p[16];
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            const float2 t = kv4_unpair(kv4_fma2(kv4_pair(s[2 * (i0 + i)], s[2 * (i0 + i) + 1]), scale2, base2));
                            const float2 e = make_float2(kv4_exp2(t.x), kv4_exp2(t.y));
                            sum[i & 1] = kv4_add2(sum[i & 1], kv4_pair(e.x, e.y));
                            p[i] = kv4_pack(e.x, e.y);
                        }
                        kp_st16(tmem + lanes + S0 + slot * KP_N + c0 / 2 + i0, p);
                    }
                }
                const float2 sums = kv4_unpair(kv4_add2(sum[0], sum[1]));
                l += sums.x + sums.y;
                kp_wait_st();
                kp_before();
                __syncwarp();
                if (lane == 0) kp_arrive(&p_full[slot]);
            }
            if constexpr (SPLIT) {
                // ---- the sums as they are, 16-byte pieces XORed with the row, over the ring and the queries (whose last readers were these MMAs)
                for (int i = 0; i < nq; ++i) if (tiles > 0 && ok) ok = kp_wait(&o_done[2 * i + ((tiles - 1) & 1)], (uint32_t)((tiles - 1) >> 1) & 1u, &s_abort);
                kp_after();
                s_ml[q * KP_M + row] = make_float2(m, ok ? l : __int_as_float(0x7fffffff));
                const uint32_t mine = smem0 + (q * KP_M + row) * (D * 4);
#pragma unroll 1
                for (int d = 0; d < D; d += 32) {
                    uint32_t o[32];
                    if (tiles > 0) { kp_ld32(tmem + lanes + q * D + d, o); kp_wait_ld(); }
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        kp_sts(mine + (((d / 4 + i) ^ (row & 7)) << 4), tiles > 0 && ok ? make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]) : make_uint4(0, 0, 0, 0));
                }
            } else {
            // ---- normalise, gate, round once; eight columns are the dims 0 4 1 5 2 6 3 7 of a word
            const int64_t to = place(a.o_row, a.o_head), gates = place(a.g_row, a.g_head);
            uint4 gate[8];
            if (a.gate) rows_in(a.gate, gates, 0, gate);
            if (tiles > 0 && ok) ok = kp_wait(&o_done[2 * q + ((tiles - 1) & 1)], (uint32_t)((tiles - 1) >> 1) & 1u, &s_abort);
            kp_after();
            const float inv = l == 0.f ? 0.f : 1.0f / l;
#pragma unroll 1
            for (int d = 0; d < D; d += 64) {
                if (a.gate) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) kp_sts(io + turn(i), gate[i]);
                    if (d + 64 < D) rows_in(a.gate, gates, d + 64, gate);     // (the next dims' on their way)
                }
                __syncwarp();
#pragma unroll
                for (int c0 = 0; c0 < 64; c0 += 32) {
                    uint32_t o[32];
                    if (tiles > 0) { kp_ld32(tmem + lanes + q * D + d + c0, o); kp_wait_ld(); }
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint32_t at = own + (((c0 / 8 + i) ^ (lane & 7)) << 4);
                        float x[8];
#pragma unroll
                        for (int k = 0; k < 8; ++k) x[(k & 1) * 4 + (k >> 1)] = !ok ? __int_as_float(0x7fffffff) : l == 0.f ? 0.f : __uint_as_float(o[8 * i + k]) * inv;
                        if (a.gate) {
                            const uint4 g = kp_lds(at);
                            const __half* gh = reinterpret_cast<const __half*>(&g);
#pragma unroll
                            for (int k = 0; k < 8; ++k) x[k] *= kv4_sigmoid(h2f(gh[k]));
                        }
                        kp_sts(at, make_uint4(kv4_pack(x[0], x[1]), kv4_pack(x[2], x[3]), kv4_pack(x[4], x[5]), kv4_pack(x[6], x[7])));
                    }
                }
                __syncwarp();
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int64_t at = __shfl_sync(0xffffffffu, to, i * 4 + (lane >> 3));
                    if (at >= 0) *reinterpret_cast<uint4*>(a.out + at + d + (lane & 7) * 8) = kp_lds(io + turn(i));
                }
                __syncwarp();
            }
            }
        }
    }
    if (!ok) {                                 // MMAs of this CTA may still be running: outlast them before tensor memory is given back
        const long long c0 = clock64();
        while (clock64() - c0 < 200000ll) { }
    }
    kp_before();
    __syncthreads();
    if constexpr (SPLIT) {
        // ---- each CTA adds up every CL-th row, eight columns a thread
        __syncwarp();
        kv4_cluster_sync();
        for (int x = tid; x < (NQ * KP_M + CL - 1) / CL * (D / 8); x += NT) {
            const int r = x / (D / 8) * CL + rank, d = x % (D / 8) * 8, q = r / KP_M, row = r % KP_M, tok = t0 + q * tokens + row / a.G, h = head * a.G + row % a.G;
            if (q >= nq || row >= tokens * a.G || tok >= sq.rows) continue;
            const int64_t at_row = sq.q0 + tok;
            uint4 g = make_uint4(0, 0, 0, 0);
            if (a.gate) g = __ldcg(reinterpret_cast<const uint4*>(a.gate + at_row * a.g_row + h * a.g_head + d));
            const uint32_t p0 = smem0 + r * (D * 4) + (((d / 4) ^ (r & 7)) << 4), p1 = smem0 + r * (D * 4) + (((d / 4 + 1) ^ (r & 7)) << 4);
            float2 ml[KP_PARTS];
            float top = -INFINITY, l = 0.f, v[8] = {};
            // (ranks from CL on: the last one's place, for nothing, so that no load is behind a branch)
#pragma unroll
            for (int i0 = 0; i0 < KP_PARTS; i0 += 4) {
                if (i0 >= CL) break;
#pragma unroll
                for (int i = i0; i < i0 + 4; ++i) ml[i] = kv4_peer2(kv4_peer(smem_u32(&s_ml[SPLIT ? r : 0]), min(i, CL - 1)));
#pragma unroll
                for (int i = i0; i < i0 + 4; ++i) top = fmaxf(top, ml[i].x);
            }
#pragma unroll
            for (int i0 = 0; i0 < KP_PARTS; i0 += 4) {
                if (i0 >= CL) break;
                float4 y0[4], y1[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) { y0[i] = kv4_peer4(kv4_peer(p0, min(i0 + i, CL - 1))); y1[i] = kv4_peer4(kv4_peer(p1, min(i0 + i, CL - 1))); }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 x = ml[i0 + i];
                    const float f = i0 + i >= CL || x.x == -INFINITY ? 0.f : kv4_exp2(x.x - top);
                    l = fmaf(x.y, f, l);
                    v[0] = fmaf(y0[i].x, f, v[0]); v[1] = fmaf(y0[i].y, f, v[1]); v[2] = fmaf(y0[i].z, f, v[2]); v[3] = fmaf(y0[i].w, f, v[3]);
                    v[4] = fmaf(y1[i].x, f, v[4]); v[5] = fmaf(y1[i].y, f, v[5]); v[6] = fmaf(y1[i].z, f, v[6]); v[7] = fmaf(y1[i].w, f, v[7]);
                }
            }
            const float inv = l == 0.f ? 0.f : 1.0f / l;
            float y[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) y[(k & 1) * 4 + (k >> 1)] = v[k] * inv;
            if (a.gate) {
                const __half* gh = reinterpret_cast<const __half*>(&g);
#pragma unroll
                for (int k = 0; k < 8; ++k) y[k] *= kv4_sigmoid(h2f(gh[k]));
            }
            *reinterpret_cast<uint4*>(a.out + at_row * a.o_row + h * a.o_head + d) = make_uint4(kv4_pack(y[0], y[1]), kv4_pack(y[2], y[3]), kv4_pack(y[4], y[5]), kv4_pack(y[6], y[7]));
        }
        __syncwarp();
        kv4_cluster_sync();                                                   // (nobody leaves while its shared memory is read)
    }
    __syncwarp();
    if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(COLUMNS) : "memory");
    pdl_wait();
}

// shared memory, once for each device
template <int D, int NQ, bool SPLIT>
static int prompt_ready() {
    static std::atomic<unsigned long long> configured{0};                     // devices
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 64 && (configured.load(std::memory_order_relaxed) >> dev & 1)) return 0;
    const cudaError_t err = cudaFuncSetAttribute(k_kv4_prompt<D, NQ, SPLIT>, cudaFuncAttributeMaxDynamicSharedMemorySize, kp_smem<D, NQ>);
    if (err == cudaSuccess && dev < 64) configured.fetch_or(1ull << dev);
    return (int)err;
}
// a launch of clusters of cl CTAs; attr: room for two attributes
template <int D, int NQ>
static cudaLaunchConfig_t prompt_config(long long ctas, int cl, bool pdl, cudaStream_t st, cudaLaunchAttribute* attr) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)ctas); cfg.blockDim = dim3(kp_threads<D, NQ>); cfg.dynamicSmemBytes = kp_smem<D, NQ>; cfg.stream = st; cfg.attrs = attr;
    if (pdl) { attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization; attr[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1; }
    if (cl > 1) { attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension; attr[cfg.numAttrs].val.clusterDim.x = (unsigned)cl; attr[cfg.numAttrs].val.clusterDim.y = 1; attr[cfg.numAttrs++].val.clusterDim.z = 1; }
    return cfg;
}
template <int D, int NQ>
static int launch_prompt_t(const Kv4Cache& c, Kv4AttnArgs a, int least, cudaStream_t st, bool pdl, int cl) {
    // a scale below zero, or zero, goes into the queries: the maximum of the scores is that of the scaled ones then
    const uint32_t q_and = a.scale == 0.f ? 0u : 0xffffffffu, q_xor = a.scale < 0.f ? 0x80008000u : 0u;
    a.scale = a.scale == 0.f ? 1.f : fabsf(a.scale) * 1.4426950408889634f;
    int rc = cl > 1 ? prompt_ready<D, NQ, true>() : prompt_ready<D, NQ, false>();
    if (rc) return rc;
    cudaLaunchAttribute attr[2];
    const cudaLaunchConfig_t cfg = prompt_config<D, NQ>(kp_items<D, NQ>(a) * c.KV * cl, cl, pdl, st, attr);
    profile_launch("k_kv4_prompt", st, [&] {
        return rc = (int)(cl > 1 ? cudaLaunchKernelEx(&cfg, k_kv4_prompt<D, NQ, true>, c, a, least, q_and, q_xor, cl) : cudaLaunchKernelEx(&cfg, k_kv4_prompt<D, NQ, false>, c, a, least, q_and, q_xor, 1));
    });
    return rc;
}
// clusters of cl CTAs that the device holds at once (they do not fill every part of it)
template <int D, int NQ>
static int prompt_room(int cl) {
    static std::atomic<int> known[64][KP_PARTS + 1] = {};                     // (+ 1)
    int dev = 0, n = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) { cudaGetLastError(); return 0; }
    if ((n = known[dev][cl].load(std::memory_order_relaxed))) return n - 1;
    cudaLaunchAttribute attr[2];
    const cudaLaunchConfig_t cfg = prompt_config<D, NQ>(cl * 1024, cl, false, nullptr, attr);
    if (prompt_ready<D, NQ, true>() || cudaOccupancyMaxActiveClusters(&n, k_kv4_prompt<D, NQ, true>, &cfg) != cudaSuccess || n < 0) { n = 0; cudaGetLastError(); }
    known[dev][cl].store(n + 1, std::memory_order_relaxed);
    return n;
}
// CTAs of a cluster.  So many that all run at once; of requests of one CTA each, half as many again, as they are seldom alike (12 x 9 rows, 32/8 heads of 128,
// up to 2809 keys: 51 -> 39 us for two CTAs; 20 x 50, 8/8 of 64, up to 4350: 69 -> 57; but 24 x 9, 32/8 of 128: 64 -> 65.5, 40 x 77, 12 of 64, up to 1500: 63 -> 67).
template <int D, int NQ>
static int prompt_cluster(const Kv4Cache& c, const Kv4AttnArgs& a) {
    const long long ctas = kp_items<D, NQ>(a) * c.KV, span = (long long)a.table_width * c.page_size, room = (long long)sm_count() * kp_ctas<D, NQ>;
    auto keys = [&](int cl) { return span >= KP_SPLIT * cl; };
    if (keys(8) && ctas * 8 <= room * 7 / 8 && ctas <= prompt_room<D, NQ>(8)) return 8;
    if (keys(6) && ctas * 6 <= room && ctas <= prompt_room<D, NQ>(6) * 7 / 8) return 6;      // (three in a part of the device: where the kernels before still leave room)
    if (keys(4) && ctas * 4 <= room) return 4;
    if (keys(3) && ctas * 3 <= room && ctas <= prompt_room<D, NQ>(3)) return 3;      // 300 rows over 30300, 32/8 heads of 128: 260 -> 183 us against two, over 9300, 16/2 of 256: 83 -> 67
    if (keys(2) && ctas * 2 <= room) return 2;
    return kp_one<D, NQ>(a) && ctas * 4 <= room * 3 && span >= KP_SPLIT * 8 ? 2 : 1;
}
template <int D, int NQ>
static int launch_prompt_d(const Kv4Cache& c, const Kv4AttnArgs& a, int least, cudaStream_t st, bool pdl) {
    const int cl = prompt_cluster<D, NQ>(c, a);
    // 64 dims, requests of one tile: two CTAs a multiprocessor where there are more of them than multiprocessors.  16 x 77 rows, 12 heads, up to 1500 keys:
    // 37 -> 34 us, all of 1500: 46 -> 35, 40 x 77: 74 -> 63; 30 x 9, 32/8 heads, up to 809: 28.7 -> 24.2; 20 x 50, 8/4 heads, up to 3050, a
    // cluster of two each: 41 -> 34
    if constexpr (D == 64) {
        if (cl <= 2 && kp_one<64, 1>(a)) {
            const int pairs = prompt_cluster<64, 1>(c, a);
            if (cl < pairs || (long long)a.batch * c.KV * cl > sm_count()) return launch_prompt_t<64, 1>(c, a, least, st, pdl, pairs);
        }
    }
    return launch_prompt_t<D, NQ>(c, a, least, st, pdl, cl);
}
int launch_kv4_prompt(const Kv4Cache& c, const Kv4AttnArgs& a, int least, cudaStream_t st, bool pdl) {
    return c.D == 64 ? launch_prompt_d<64, 2>(c, a, least, st, pdl) : c.D == 128 ? launch_prompt_d<128, 2>(c, a, least, st, pdl) : launch_prompt_d<256, 1>(c, a, least, st, pdl);
}

}  // namespace sl

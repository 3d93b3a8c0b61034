// kv_plan.cu -- page tables, slot map, positions and row offsets of a step, on the device, from the requests' lengths.
//
// Request b has lens[b] positions cached and news[b] rows to come (negative: it has ended and gives its pages back).  With
// have = ceil(lens / P) and need = ceil((lens + news) / P) its table grows by need - have pages, taken from the top of the stack of
// free pages; the rows' offsets, the pages returned and the pages taken are prefix sums over the requests, so the result does not
// depend on the order in which threads run.  All of it or nothing: where pages, table columns or rows are short, the tables and the
// stack stay as they are and the status says what was short.
//
// A few hundred requests are bound by latency alone (three dependent loads and the launch), so one CTA does everything: sums, pages and,
// up to PLAN_ROWS of them, the rows.  More rows get a kernel of their own over the whole device.
// 64 requests of a row each: 6.2 us (256 threads; 1024 take longer to start and to meet).  700 requests of up to 4001 positions and 509 rows in pages of
// 16: 18.5 us, two kernels that take 14.5 and 8.7 by themselves; the first is the chain lengths -> sums -> pages -> offsets, with a bisection for each page.
#include "kv4.cuh"

namespace sl {

constexpr int PLAN_ROWS = 8192, PLAN_FIND = 2048;      // rows that one CTA does; requests whose offsets the rows' kernel keeps in shared memory

struct PlanOne { long long len; int rows, have, need; bool ended, bad; };

__device__ __forceinline__ PlanOne plan_one(const KvPlanArgs& a, int b) {
    PlanOne r{0, 0, 0, 0, false, false};
    if (b >= a.batch) return r;
    const int len = a.lens[b], n = a.news[b];
    r.len = len; r.ended = n < 0; r.rows = n < 0 ? 0 : n;
    const long long have = (r.len + a.page_size - 1) / a.page_size, need = (r.len + r.rows + a.page_size - 1) / a.page_size;
    r.bad = len < 0 || need > a.table_width || r.len + r.rows > 0x7fffffffll;
    if (r.bad) r.rows = 0;
    else { r.have = (int)have; r.need = r.ended ? 0 : (int)need; }
    return r;
}
// inclusive sums over the CTA of two values, the totals in ws[.][last warp]; all threads call it
template <int T>
__device__ __forceinline__ void plan_scan(int& x, int& y, int (*ws)[32]) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, x, d), v = __shfl_up_sync(0xffffffffu, y, d);
        if (lane >= d) { x += u; y += v; }
    }
    __syncthreads();
    if (lane == 31) { ws[0][warp] = x; ws[1][warp] = y; }
    __syncthreads();
    if (warp == 0) {
        int u = lane < T / 32 ? ws[0][lane] : 0, v = lane < T / 32 ? ws[1][lane] : 0;
#pragma unroll
        for (int d = 1; d < T / 32; d <<= 1) {
            const int p = __shfl_up_sync(0xffffffffu, u, d), q = __shfl_up_sync(0xffffffffu, v, d);
            if (lane >= d) { u += p; v += q; }
        }
        ws[0][lane] = u; ws[1][lane] = v;
    }
    __syncthreads();
    if (warp) { x += ws[0][warp - 1]; y += ws[1][warp - 1]; }
}
// the last i of [0, n) with start[i] <= v (start[0] <= v); of entries that start alike the last is the one that is not empty
__device__ __forceinline__ int plan_find(const int* start, int n, int v) {
    int lo = 0, hi = n - 1;
    while (lo < hi) { const int mid = (lo + hi + 1) >> 1; if (start[mid] <= v) lo = mid; else hi = mid - 1; }
    return lo;
}
__device__ __forceinline__ void plan_row(const KvPlanArgs& a, int r, int b, int pos) {
    a.slots[r] = (int64_t)a.table[(int64_t)b * a.table_stride + pos / a.page_size] * a.page_size + pos % a.page_size;
    a.pos[r] = pos;
}

// T: threads, and requests of a chunk
template <int T>
__global__ void __launch_bounds__(T) k_kv_plan(KvPlanArgs a, int rows_here) {
    __shared__ int ws[2][32], s_a[T], s_b[T], s_c[T], s_tot[3];
    __shared__ unsigned long long s_rows;
    constexpr int TOP = T / 32 - 1;
    const int tid = threadIdx.x, lane = tid & 31;
    pdl_launch_dependents();
    if (tid == 0) { s_rows = 0; s_tot[0] = s_tot[1] = s_tot[2] = 0; }
    // ---- what the whole step needs (warps' sums first: a thousand atomic additions of one word took 18 us)
    const int F = *a.free_count;
    const PlanOne mine = plan_one(a, tid);
    long long rows = 0; int back = 0, grown = 0, bad = 0;
    for (int b = tid; b < a.batch; b += T) {
        const PlanOne r = b == tid ? mine : plan_one(a, b);
        rows += r.rows; bad += r.bad;
        if (r.ended) back += r.have; else grown += r.need - r.have;
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) rows += __shfl_xor_sync(0xffffffffu, rows, d);
    back = __reduce_add_sync(0xffffffffu, back); grown = __reduce_add_sync(0xffffffffu, grown); bad = __reduce_add_sync(0xffffffffu, bad);
    __syncthreads();
    if (lane == 0) {                     // (pages number below 2^31 in all: the host has looked)
        atomicAdd(&s_rows, (unsigned long long)rows);
        atomicAdd(&s_tot[0], back); atomicAdd(&s_tot[1], grown); atomicAdd(&s_tot[2], bad);
    }
    __syncthreads();
    rows = (long long)s_rows; back = s_tot[0]; grown = s_tot[1];
    const bool stack_bad = F < 0 || (long long)F + back > a.free_cap;
    const long long top = (long long)F + back;
    bad = s_tot[2] + (stack_bad ? 1 : 0);
    const long long shrt = stack_bad || grown <= top ? 0 : grown - top, over = rows > a.max_rows ? rows - a.max_rows : 0;
    const bool fine = !bad && !shrt && !over;
    if (tid == 0) {
        a.status[0] = (int)shrt; a.status[1] = bad; a.status[2] = (int)(over > 0x7fffffffll ? 0x7fffffffll : over);
        *a.free_count_out = fine ? (int)(top - grown) : F;
        a.q_start[a.batch] = fine ? (int)rows : 0;
    }
    if (!fine) {
        for (int b = tid; b < a.batch; b += T) { const int len = a.lens[b]; a.q_start[b] = 0; a.kv_len[b] = len; }
        for (int r = tid; rows_here && r < a.max_rows; r += T) { a.slots[r] = -1; a.pos[r] = 0; }
        return;
    }
    // ---- pages of ended requests onto the stack
    if (back) {
        int base = F;
        for (int b0 = 0; b0 < a.batch; b0 += T) {
            const PlanOne r = b0 ? plan_one(a, b0 + tid) : mine;
            const int own = r.ended ? r.have : 0;
            int x = own, y = 0;
            plan_scan<T>(x, y, ws);
            s_a[tid] = x - own;
            __syncthreads();
            const int n = ws[0][TOP];
#pragma unroll 4
            for (int i = tid; i < n; i += T) {
                const int j = plan_find(s_a, T, i);
                a.free_pages[base + i] = a.table[(int64_t)(b0 + j) * a.table_stride + i - s_a[j]];
            }
            base += n;
        }
        __syncthreads();
    }
    // ---- row offsets, new lengths, pages off the stack, and the rows
    int row0 = 0, taken = 0;
    for (int b0 = 0; b0 < a.batch; b0 += T) {
        const PlanOne r = b0 ? plan_one(a, b0 + tid) : mine;
        const int own = r.ended ? 0 : r.need - r.have;
        int x = r.rows, y = own;
        plan_scan<T>(x, y, ws);
        s_a[tid] = y - own; s_b[tid] = r.have;
        if (b0 + tid < a.batch) {
            a.q_start[b0 + tid] = row0 + x - r.rows;
            a.kv_len[b0 + tid] = r.ended ? 0 : (int)r.len + r.rows;           // (may be the array of lengths: its reader was this thread)
        }
        __syncthreads();
        const int n = ws[1][TOP], m = ws[0][TOP];
#pragma unroll 4
        for (int i = tid; i < n; i += T) {
            const int j = plan_find(s_a, T, i);
            a.table[(int64_t)(b0 + j) * a.table_stride + s_b[j] + i - s_a[j]] = a.free_pages[top - 1 - taken - i];
        }
        if (rows_here) {
            s_c[tid] = x - r.rows;
            __syncthreads();                                                  // (also: the table's new pages are there, s_b is read)
            s_b[tid] = (int)r.len;
            __syncthreads();
#pragma unroll 4
            for (int i = tid; i < m; i += T) {
                const int j = plan_find(s_c, T, i);
                plan_row(a, row0 + i, b0 + j, s_b[j] + i - s_c[j]);
            }
        }
        row0 += m; taken += n;
        __syncthreads();
    }
    if (rows_here) for (int r = (int)rows + tid; r < a.max_rows; r += T) { a.slots[r] = -1; a.pos[r] = 0; }
}
// the rows, four a thread: which request a row is of by bisection of the offsets
__global__ void __launch_bounds__(256) k_kv_plan_rows(KvPlanArgs a) {
    __shared__ int s_start[PLAN_FIND];
    pdl_wait();
    const int rows = a.q_start[a.batch];
    const bool near = a.batch <= PLAN_FIND;
    if (near) for (int b = threadIdx.x; b < a.batch; b += 256) s_start[b] = a.q_start[b];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = blockIdx.x * 1024 + i * 256 + threadIdx.x;
        if (r >= a.max_rows) return;
        if (r >= rows) { a.slots[r] = -1; a.pos[r] = 0; continue; }
        const int b = near ? plan_find(s_start, a.batch, r) : plan_find(a.q_start, a.batch, r);
        plan_row(a, r, b, a.kv_len[b] - (a.q_start[b + 1] - r));
    }
}

int launch_kv_plan(const KvPlanArgs& a, cudaStream_t st) {
    const bool here = a.max_rows <= PLAN_ROWS, small = a.batch <= 256 && a.max_rows <= 1024;
    int rc = 0;
    profile_launch("k_kv_plan", st, [&] {
        return rc = small ? launch_pdl(false, k_kv_plan<256>, dim3(1), 256, 0, st, a, 1) : launch_pdl(false, k_kv_plan<1024>, dim3(1), 1024, 0, st, a, here ? 1 : 0);
    });
    if (rc == 0 && !here) profile_launch("k_kv_plan_rows", st, [&] { return rc = launch_pdl(true, k_kv_plan_rows, dim3((unsigned)((a.max_rows + 1023) / 1024)), 256, 0, st, a); });
    return rc;
}

}  // namespace sl

// kv4.cuh -- the KV cache held in 4 bits: its layout, and the argument blocks of the kernels that fill and read it.
//
// A page of one layer holds page_size positions of every kv head in blocks of 16 positions of one head:
//   [page][kv head][page_size / 16][18 * D bytes]
//   block:  K codes, 8 D bytes | V codes, 8 D bytes | K scales and biases, D bytes | V scales and biases, D bytes
// A position's codes are D / 2 bytes, eight dims to a 32-bit word, the first in the lowest nibble; the 16-byte piece at byte o of a
// code region stands at o ^ (16 * (o / 128 mod 8)), so that eight positions' pieces of the same dims lie in different banks of shared
// memory once a block has been copied there as it is (ldmatrix reads them so).  Scales and biases are fp16, [64-dim group][16 scales |
// 16 biases].  An element is worth fp16(code * scale + bias), one rounding: the affine group-64 scheme of the weights
// (swift/Sources/QwispCore/SeedlessMetalForward.swift:82-87, 219-221).  A block is self-contained: any run of blocks of a head's page is
// one contiguous piece of memory, of 1.125 bytes a dim for K and V together.
#pragma once
#include "kernels.h"

namespace sl {

constexpr int KV4_B = 16;                                     // positions of a block

__host__ __device__ constexpr int kv4_block_bytes(int D) { return 18 * D; }
__host__ __device__ constexpr uint32_t kv4_swz(uint32_t o) { return o ^ (((o >> 7) & 7u) << 4); }

struct Kv4Cache {
    unsigned char* data; int64_t page_stride;                 // bytes from a page to the next
    int pages, page_size, KV, D;
    int64_t slots() const { return (int64_t)pages * page_size; }
};
__device__ __forceinline__ unsigned char* kv4_block(const Kv4Cache& c, int page, int head, int block) {
    return c.data + (int64_t)page * c.page_stride + ((int64_t)head * (c.page_size / KV4_B) + block) * kv4_block_bytes(c.D);
}
// (page, offset in it) of a slot of the cache.  (A 64-bit division is some hundred instructions: only where the slot needs it.)
__device__ __forceinline__ void kv4_place(const Kv4Cache& c, int64_t slot, int& page, int& off) {
    if (slot >> 31 == 0) { page = (int)((uint32_t)slot / (uint32_t)c.page_size); off = (int)slot - page * c.page_size; }
    else { page = (int)(slot / c.page_size); off = (int)(slot - (int64_t)page * c.page_size); }
}

struct KvPlanArgs {
    const int *lens, *news; int batch, page_size;
    int* table; int64_t table_stride; int table_width;
    int* free_pages; int free_cap; const int* free_count;
    int *kv_len, *q_start; int64_t* slots; int* pos; int max_rows;
    int *free_count_out, *status;
};
struct Kv4AppendArgs {
    const __half *q, *k, *v; int64_t q_row, q_head, k_row, k_head, v_row, v_head;      // nullptr: none (k and v together)
    __half* q_out; int64_t o_row, o_head;
    int rows, NH;
    const __half *q_norm, *k_norm; float eps;                 // nullptr: no norm
    const int* pos; int64_t pos_axis;                         // [axes][rows]
    int rope;                                                 // rotated dims
    const int64_t* slots;
    uint64_t turn[128]; unsigned char axis[128];              // a frequency as turns a position (64-bit fraction), and its axis
};
struct Kv4ReadArgs { const int64_t* slots; int rows; __half *k, *v; int64_t k_row, k_head, v_row, v_head; };
struct Kv4AttnArgs {
    const __half* q; int64_t q_row, q_head;
    const __half* gate; int64_t g_row, g_head;                // nullptr: no gate
    __half* out; int64_t o_row, o_head;
    int rows, NH, G;                                          // query heads, of them for a kv head
    const int *q_start, *kv_len; int batch, max_q;
    const int* table; int64_t table_stride; int table_width;
    int causal; float scale;
    void* ws; size_t ws_bytes;
};

int launch_kv_plan(const KvPlanArgs& a, cudaStream_t st);
int launch_kv4_append(const Kv4Cache& c, const Kv4AppendArgs& a, cudaStream_t st);
int launch_kv4_read(const Kv4Cache& c, const Kv4ReadArgs& a, cudaStream_t st);
size_t kv4_attn_workspace(int D, int G, int KV, int batch, int max_q, long long span);      // span: positions of a table's row, -1: any
// requests of more than `least` rows a kv head; pdl: the kernel before it in the stream is one of this call's
int launch_kv4_prompt(const Kv4Cache& c, const Kv4AttnArgs& a, int least, cudaStream_t st, bool pdl);
int launch_kv4_attn(const Kv4Cache& c, const Kv4AttnArgs& a, cudaStream_t st);

}  // namespace sl

// A paged cache of keys and values in 8 bits (kv8.cu) and attention over it (kv8_attn.cu, kv8_prefix.cu).
#pragma once
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace hm {

constexpr int KV8_PAGE = 64;        // tokens per page
constexpr int KV8_MAX_DIM = 256;    // elements of a key or a value
constexpr int KV8_MAX_ROWS = 8192;  // rows of one attention call
constexpr int KV8_PAIRS = 8;        // (row, head) pairs of one item of kv8_attn.cu

// A page holds one block per key/value head, in two halves of 32 tokens: the 32 scales of its keys (f32) and their codes, one signed byte each, then the same of its values.
// Codes stand in the order in which the lanes of warp-level MMAs want them:
//   keys    slabs of 32 elements, [pad / 32][32 rows][32]; row r holds the token t with kv8_key_row(t) = r
//   values  [pad][32 tokens]
struct Kv8Pool {
    unsigned char* pages;
    const int32_t* page_table;  // [n_seq][max_pages]
    int n_pages, n_seq, max_pages;
    int kv_heads, dim, vdim;
};
__host__ __device__ __forceinline__ int kv8_pad(int d) { return (d + 31) & ~31; }
constexpr int KV8_HALF = 32;  // tokens of a half
__host__ __device__ __forceinline__ int kv8_part_bytes(int d) { return KV8_HALF * (4 + kv8_pad(d)); }  // keys or values of a half
__host__ __device__ __forceinline__ size_t kv8_half_bytes(int dim, int vdim) { return (size_t)kv8_part_bytes(dim) + kv8_part_bytes(vdim); }
__host__ __device__ __forceinline__ size_t kv8_block_bytes(int dim, int vdim) { return 2 * kv8_half_bytes(dim, vdim); }
// Token 8 i + 2 j + e of a half (i, j < 4) is column 2 i + e of the scores' tile j: the lane with columns 2 i and 2 i + 1 of all tiles has eight tokens that follow one another.
__host__ __device__ __forceinline__ int kv8_key_row(int t) { return (((t >> 1) & 3) << 3) | ((t >> 3) << 1) | (t & 1); }
// Places in their part of a half of token t's codes of element d.
__host__ __device__ __forceinline__ int kv8_key_at(int t, int d) { return KV8_HALF * 4 + ((d >> 5) * KV8_HALF + kv8_key_row(t)) * 32 + (d & 31); }
__host__ __device__ __forceinline__ int kv8_value_at(int t, int d) { return KV8_HALF * 4 + d * KV8_HALF + t; }

// Page of a position, or -1 where there is none (a sequence, a position or a page that is out of range).
__device__ __forceinline__ int kv8_page(const Kv8Pool& p, int seq, int pos) {
    if ((unsigned)seq >= (unsigned)p.n_seq || pos < 0 || pos / KV8_PAGE >= p.max_pages) return -1;
    const int page = __ldg(p.page_table + (size_t)seq * p.max_pages + pos / KV8_PAGE);
    return (unsigned)page < (unsigned)p.n_pages ? page : -1;
}

struct Kv8RowsArgs {
    Kv8Pool pool;
    void *k, *v;             // [M] rows of kv_heads * dim and kv_heads * vdim elements, ldk and ldv apart
    size_t ldk, ldv;
    int bf16;
    int M;
    const int32_t *row_seq, *row_pos;
};
cudaError_t launch_kv8_write(const Kv8RowsArgs& a, int sm_count, cudaStream_t st);
cudaError_t launch_kv8_read(const Kv8RowsArgs& a, int sm_count, cudaStream_t st);

struct Kv8AttnArgs {
    Kv8Pool pool;
    const void* q;           // [M] rows of heads * dim elements
    void* out;               // [M] rows of heads * vdim elements
    size_t ldq, ldo;
    int bf16;
    int M, heads;
    const int32_t *row_seq, *row_pos;
    float scale;
    const int32_t* shared;   // the first n_shared pages of every row's sequence
    int n_shared;
    void* work;
    int* err_flag;
    // filled in by the launcher
    int solo, team;          // items of at most so many pieces belong to so many warps
    int whole;               // a CTA takes an item as a whole, and there are no more items than CTAs
    int direct;              // kv8_prefix.cu writes the rows that have nothing but the prefix
    int own_from;            // the rows' own pieces (halves of pages) begin here: what stands in front is in `prefix`
    const float* prefix;     // [prefix_n parts][kv_heads][M * heads / kv_heads][padded vdim + 4]: reference and sum of a pair, then from the fifth on its elements
    int prefix_n;
};
// How the shared pages are taken on their own (kv8_prefix.cu): tiles of 128 (row, head) pairs, or of 256, times splits of the pages.
struct Kv8Prefix {
    int paired, groups, splits, cluster;
    int parts;               // splits / cluster; 0: they are taken with the rows' own
    size_t sums;             // floats of the sums that CTAs with many blocks keep in memory
};
Kv8Prefix kv8_prefix_plan(int kv_heads, int dim, int vdim, int bf16, int M, int heads, int n_shared, int sm_count);
int kv8_prefix_most_parts(int kv_heads, int M, int heads, int n_shared, int sm_count);  // of any plan
cudaError_t launch_kv8_prefix(const Kv8AttnArgs& a, const Kv8Prefix& p, float* parts, float* sums, cudaStream_t st);
cudaError_t launch_kv8_attn(const Kv8AttnArgs& a, int sm_count, cudaStream_t st);
size_t kv8_attn_bytes(int kv_heads, int dim, int vdim, int M, int heads, int n_shared, int sm_count);

}  // namespace hm

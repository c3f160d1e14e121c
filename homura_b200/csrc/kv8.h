// A paged cache of keys and values in 8 bits (kv8.cu) and attention over it (kv8_attn.cu).
#pragma once
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace hm {

constexpr int KV8_PAGE = 64;        // tokens per page
constexpr int KV8_MAX_DIM = 256;    // elements of a key or a value
constexpr int KV8_MAX_ROWS = 8192;  // rows of one attention call

// A page holds one block per key/value head: 64 scales of keys, 64 of values (f32), then the codes of keys and of values (value + 128, one byte), in slabs
// of 32 elements, [pad / 32][64 rows][32].  Row r of a slab is token r of the values; of the keys it is token key_token(r): within every eight tokens
// 0 4 1 5 2 6 3 7, the order in which the lanes of a warp-level MMA want them.
struct Kv8Pool {
    unsigned char* pages;
    const int32_t* page_table;  // [n_seq][max_pages]
    int n_pages, n_seq, max_pages;
    int kv_heads, dim, vdim;
};
__host__ __device__ __forceinline__ int kv8_pad(int d) { return (d + 31) & ~31; }
__host__ __device__ __forceinline__ size_t kv8_block_bytes(int dim, int vdim) { return (size_t)KV8_PAGE * (8 + kv8_pad(dim) + kv8_pad(vdim)); }
__host__ __device__ __forceinline__ int kv8_key_row(int t) { return (t & ~7) | ((t & 3) << 1) | ((t >> 2) & 1); }

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
cudaError_t launch_kv8_write(const Kv8RowsArgs& a, cudaStream_t st);
cudaError_t launch_kv8_read(const Kv8RowsArgs& a, cudaStream_t st);

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
};
cudaError_t launch_kv8_attn(const Kv8AttnArgs& a, int sm_count, cudaStream_t st);
size_t kv8_attn_bytes(int kv_heads, int vdim, int M, int heads, int n_shared, int sm_count);

}  // namespace hm

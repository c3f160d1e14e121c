// What both kernels of attention over the 8-bit cache do with rows.
#pragma once
#include "kv8.h"
#include "rows.cuh"

namespace hm {

// Tokens that a row sees, of those that its page table has room for; 0 for a row without a sequence.
__device__ __forceinline__ int kv8_row_len(const Kv8AttnArgs& a, int m) {
    const int seq = __ldg(a.row_seq + m);
    return (unsigned)seq < (unsigned)a.pool.n_seq ? min(__ldg(a.row_pos + m), a.pool.max_pages * KV8_PAGE - 1) + 1 : 0;
}
// Of halves of pages, behind those that are taken as a prefix.
__device__ __forceinline__ int kv8_row_pieces(const Kv8AttnArgs& a, int m) { return max(0, (kv8_row_len(a, m) + KV8_HALF - 1) / KV8_HALF - a.own_from); }

// Two results of a row: elements d and d + 1 of a head.
template <bool BF16>
__device__ __forceinline__ void kv8_store2(const Kv8AttnArgs& a, int m, int head, int d, float x, float y, bool wide) {
    const size_t at = (size_t)m * a.ldo + (size_t)head * a.pool.vdim + d;
    if (wide) {  // an even number of elements, pairs aligned
        if (d >= a.pool.vdim) return;
        if (BF16) *reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(a.out) + at) = bf16x2_rne(x, y);
        else *reinterpret_cast<float2*>(static_cast<float*>(a.out) + at) = make_float2(x, y);
        return;
    }
    const float v[2][1] = {{x}, {y}};
    if (d < a.pool.vdim) store_row<BF16, 1>(a.out, at, v[0]);
    if (d + 1 < a.pool.vdim) store_row<BF16, 1>(a.out, at + 1, v[1]);
}

// bit 0 of `wide`: results in pairs, bit 1: queries in groups of four
inline int kv8_wide(const Kv8AttnArgs& a) {
    const int size = a.bf16 ? 2 : 4;
    return (a.pool.vdim % 2 == 0 && (((uintptr_t)a.out | a.ldo * size) & (2 * size - 1)) == 0 ? 1 : 0) | (a.pool.dim % 8 == 0 && (((uintptr_t)a.q | a.ldq * size) & (4 * size - 1)) == 0 ? 2 : 0);
}

}  // namespace hm

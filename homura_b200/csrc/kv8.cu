// Keys and values into a paged cache of 8 bits, and back.
//
// A row's key (or value) of one head is quantised as a whole: m = max |x|, code = rint(x * (127 / m)), scale = m / 127, every step rounded to f32, so that
// each implementation gives the same bits; m < 2^-100 leaves zeros with the scale 0, an infinity or a NaN makes the scale NaN and with it the whole vector.
// The maximum is taken over the bits of |x|, among which those of infinities and NaN are the largest.
//
// A CTA takes `rows` consecutive rows of the call and one head.  LANES lanes share a vector, four elements at a time.  Codes of keys stand by token and go straight
// to their places; codes of values stand by element, 32 tokens side by side, so they pass through shared memory: four rows that follow one another in a page (rows of a
// prompt) become words of four tokens, others single bytes.  What bounds both directions is bytes.
#include "kv8.h"
#include "rows.cuh"

#include <type_traits>

namespace hm {
namespace {

constexpr int WT = 256;
constexpr int MOST_ROWS = 32;                   // of a CTA
constexpr float TINY = 7.888609052210118e-31f;  // 2^-100
constexpr int LDV = KV8_MAX_DIM + 4;            // bytes from row to row in shared memory

template <bool BF16, bool VEC>
__device__ __forceinline__ void load_quad(const void* base, size_t at, int n, float (&x)[4]) {
    if constexpr (VEC) {
        load_row<BF16, 4>(base, at, x);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            float one[1] = {0.f};
            if (e < n) load_row<BF16, 1>(base, at + e, one);
            x[e] = one[0];
        }
    }
}
template <bool BF16, bool VEC>
__device__ __forceinline__ void store_quad(void* base, size_t at, int n, const float (&x)[4]) {
    if constexpr (VEC) {
        store_row<BF16, 4>(base, at, x);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float one[1] = {x[e]};
            if (e < n) store_row<BF16, 1>(base, at + e, one);
        }
    }
}

// Where a CTA's rows belong.
struct Places {
    unsigned char* key[MOST_ROWS];    // its half of this head's block, which begins with the keys; null: no place
    int token[MOST_ROWS];             // within the half
    uint8_t four[MOST_ROWS / 4];      // rows 4 i .. 4 i + 3 are four tokens that begin at a multiple of four
};
__device__ __forceinline__ void find_places(const Kv8RowsArgs& a, int m0, int rows, int h, Places& s) {
    const int r = threadIdx.x;
    if (r < rows) {
        const int pos = m0 + r < a.M ? __ldg(a.row_pos + m0 + r) : -1, page = pos < 0 ? -1 : kv8_page(a.pool, __ldg(a.row_seq + m0 + r), pos);
        s.key[r] = page < 0 ? nullptr : a.pool.pages + ((size_t)page * a.pool.kv_heads + h) * kv8_block_bytes(a.pool.dim, a.pool.vdim) + ((pos & (KV8_PAGE - 1)) / KV8_HALF) * kv8_half_bytes(a.pool.dim, a.pool.vdim);
        s.token[r] = pos & (KV8_HALF - 1);
    }
    __syncthreads();
    if (r < rows / 4) {
        const int t = s.token[4 * r];
        bool four = s.key[4 * r] && (t & 3) == 0;
        for (int i = 1; i < 4; ++i) four = four && s.key[4 * r + i] == s.key[4 * r] && s.token[4 * r + i] == t + i;
        s.four[r] = four;
    }
    __syncthreads();
}
// Four words [row][element] to four words [element][row], and back.
__device__ __forceinline__ void transpose4(uint32_t (&x)[4]) {
    const uint32_t a = __byte_perm(x[0], x[1], 0x5140), b = __byte_perm(x[2], x[3], 0x5140), c = __byte_perm(x[0], x[1], 0x7362), d = __byte_perm(x[2], x[3], 0x7362);
    x[0] = __byte_perm(a, b, 0x5410);
    x[1] = __byte_perm(a, b, 0x7632);
    x[2] = __byte_perm(c, d, 0x5410);
    x[3] = __byte_perm(c, d, 0x7632);
}

template <bool BF16, bool VEC, int LANES>
__global__ void __launch_bounds__(WT) kv8_write_kernel(const Kv8RowsArgs a, int rows) {
    constexpr int QUADS = LANES == 32 ? 2 : 1, GROUPS = WT / LANES;  // a lane's quads; vectors at a time
    __shared__ Places s;
    __shared__ __align__(16) unsigned char vbuf[MOST_ROWS][LDV];
    const int h = blockIdx.y, m0 = blockIdx.x * rows, lane = threadIdx.x % LANES, group = threadIdx.x / LANES, dim = a.pool.dim, vdim = a.pool.vdim;
    find_places(a, m0, rows, h, s);
    const unsigned mask = LANES == 32 ? 0xffffffffu : ((1u << LANES % 32) - 1u) << (threadIdx.x & 31 & ~(LANES - 1));
    for (int i = group; i < 2 * rows; i += GROUPS) {  // keys of all rows, then values
        const bool value = i >= rows;
        const int r = value ? i - rows : i, n = value ? vdim : dim;
        if (!s.key[r]) continue;
        unsigned char* part = s.key[r] + (value ? kv8_part_bytes(dim) : 0);
        const void* src = value ? a.v : a.k;
        const size_t at = (size_t)(m0 + r) * (value ? a.ldv : a.ldk) + (size_t)h * n;
        float x[QUADS][4];
        uint32_t top = 0;
#pragma unroll
        for (int j = 0; j < QUADS; ++j) {
            const int d = 4 * (lane + j * LANES);
            x[j][0] = x[j][1] = x[j][2] = x[j][3] = 0.f;
            if (d < n) load_quad<BF16, VEC>(src, at + d, n - d, x[j]);
#pragma unroll
            for (int e = 0; e < 4; ++e) top = max(top, __float_as_uint(x[j][e]) & 0x7FFFFFFFu);
        }
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(mask, top, o));
        const float most = __uint_as_float(top);
        const bool finite = top < 0x7F800000u, some = finite && most >= TINY;
        const float up = some ? __fdiv_rn(127.f, most) : 0.f;
        if (lane == 0) reinterpret_cast<float*>(part)[s.token[r]] = !finite ? __uint_as_float(0x7FC00000u) : some ? __fdiv_rn(most, 127.f) : 0.f;
#pragma unroll
        for (int j = 0; j < QUADS; ++j) {
            const int d = 4 * (lane + j * LANES);
            if (d >= n) continue;
            uint32_t c[4];  // codes in the last byte: of 1.5 * 2^23 + code
#pragma unroll
            for (int e = 0; e < 4; ++e) c[e] = some ? __float_as_uint(__fadd_rn(__fmul_rn(x[j][e], up), 12582912.f)) : 0u;
            const uint32_t w = __byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410);
            if (value) *reinterpret_cast<uint32_t*>(&vbuf[r][d]) = w;
            else *reinterpret_cast<uint32_t*>(part + kv8_key_at(s.token[r], d)) = w;
        }
    }
    __syncthreads();
    // values: eight lanes take the groups of four rows of a quad of elements, so that a word's neighbours are written with it
    const int quads = (vdim + 3) / 4, fours = rows / 4, values = kv8_part_bytes(dim);
    for (int i = threadIdx.x; i < quads * fours; i += WT) {
        const int f = i % fours, d = i / fours * 4;
        uint32_t x[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) x[r] = *reinterpret_cast<const uint32_t*>(&vbuf[4 * f + r][d]);
        if (s.four[f]) {
            transpose4(x);
            unsigned char* to = s.key[4 * f] + values;
#pragma unroll
            for (int e = 0; e < 4; ++e) *reinterpret_cast<uint32_t*>(to + kv8_value_at(s.token[4 * f], d + e)) = x[e];  // elements behind the last are padding
        } else {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                unsigned char* to = s.key[4 * f + r];
                if (!to) continue;
#pragma unroll
                for (int e = 0; e < 4; ++e) to[values + kv8_value_at(s.token[4 * f + r], d + e)] = (unsigned char)(x[r] >> (8 * e));
            }
        }
    }
}

template <bool BF16, bool VEC, int LANES>
__global__ void __launch_bounds__(WT) kv8_read_kernel(const Kv8RowsArgs a, int rows) {
    constexpr int QUADS = LANES == 32 ? 2 : 1, GROUPS = WT / LANES;
    __shared__ Places s;
    __shared__ __align__(16) unsigned char vbuf[MOST_ROWS][LDV];
    const int h = blockIdx.y, m0 = blockIdx.x * rows, lane = threadIdx.x % LANES, group = threadIdx.x / LANES, dim = a.pool.dim, vdim = a.pool.vdim;
    find_places(a, m0, rows, h, s);
    const int quads = (vdim + 3) / 4, fours = rows / 4, values = kv8_part_bytes(dim);
    for (int i = threadIdx.x; i < quads * fours; i += WT) {
        const int f = i % fours, d = i / fours * 4;
        uint32_t x[4];
        if (s.four[f]) {
            const unsigned char* from = s.key[4 * f] + values;
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = *reinterpret_cast<const uint32_t*>(from + kv8_value_at(s.token[4 * f], d + e));
            transpose4(x);
        } else {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const unsigned char* from = s.key[4 * f + r];
                x[r] = 0;
                if (!from) continue;
#pragma unroll
                for (int e = 0; e < 4; ++e) x[r] |= (uint32_t)from[values + kv8_value_at(s.token[4 * f + r], d + e)] << (8 * e);
            }
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) *reinterpret_cast<uint32_t*>(&vbuf[4 * f + r][d]) = x[r];
    }
    __syncthreads();
    for (int i = group; i < 2 * rows; i += GROUPS) {
        const bool value = i >= rows;
        const int r = value ? i - rows : i, n = value ? vdim : dim;
        if (!s.key[r]) continue;
        const unsigned char* part = s.key[r] + (value ? kv8_part_bytes(dim) : 0);
        const size_t at = (size_t)(m0 + r) * (value ? a.ldv : a.ldk) + (size_t)h * n;
        const float scale = reinterpret_cast<const float*>(part)[s.token[r]];
#pragma unroll
        for (int j = 0; j < QUADS; ++j) {
            const int d = 4 * (lane + j * LANES);
            if (d >= n) continue;
            const uint32_t w = value ? *reinterpret_cast<const uint32_t*>(&vbuf[r][d]) : *reinterpret_cast<const uint32_t*>(part + kv8_key_at(s.token[r], d));
            float x[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = (float)(int8_t)(w >> (8 * e)) * scale;
            store_quad<BF16, VEC>(value ? a.v : a.k, at + d, n - d, x);
        }
    }
}

template <bool BF16, bool VEC, int LANES>
cudaError_t launch_rows(const Kv8RowsArgs& a, bool write, int sm_count, cudaStream_t st) {
    // as many rows to a CTA as leave every SM two of them: 8 (one vector of a key and of a value per warp) to 32 (whole sectors of values)
    int rows = MOST_ROWS;
    while (rows > 8 && (long)((a.M + rows - 1) / rows) * a.pool.kv_heads < 2 * sm_count) rows /= 2;
    const dim3 grid((unsigned)((a.M + rows - 1) / rows), (unsigned)a.pool.kv_heads);
    if (write) kv8_write_kernel<BF16, VEC, LANES><<<grid, WT, 0, st>>>(a, rows);
    else kv8_read_kernel<BF16, VEC, LANES><<<grid, WT, 0, st>>>(a, rows);
    return cudaGetLastError();
}

template <bool BF16>
cudaError_t launch_typed(const Kv8RowsArgs& a, bool write, int sm_count, cudaStream_t st) {
    const int size = BF16 ? 2 : 4, most = a.pool.dim > a.pool.vdim ? a.pool.dim : a.pool.vdim;
    const bool vec = (((uintptr_t)a.k | (uintptr_t)a.v | (a.ldk * size) | (a.ldv * size)) & (4 * size - 1)) == 0 && ((a.pool.dim | a.pool.vdim) & 3) == 0;
    auto go = [&](auto lanes) { return vec ? launch_rows<BF16, true, decltype(lanes)::value>(a, write, sm_count, st) : launch_rows<BF16, false, decltype(lanes)::value>(a, write, sm_count, st); };
    if (most <= 32) return go(std::integral_constant<int, 8>{});
    if (most <= 64) return go(std::integral_constant<int, 16>{});
    return go(std::integral_constant<int, 32>{});
}

}  // namespace

cudaError_t launch_kv8_write(const Kv8RowsArgs& a, int sm_count, cudaStream_t st) { return a.bf16 ? launch_typed<true>(a, true, sm_count, st) : launch_typed<false>(a, true, sm_count, st); }
cudaError_t launch_kv8_read(const Kv8RowsArgs& a, int sm_count, cudaStream_t st) { return a.bf16 ? launch_typed<true>(a, false, sm_count, st) : launch_typed<false>(a, false, sm_count, st); }

}  // namespace hm

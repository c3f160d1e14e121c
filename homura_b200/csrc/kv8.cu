// Keys and values into a paged cache of 8 bits, and back.
//
// A row's key (or value) of one head is quantised as a whole: m = max |x|, code = rint(x * (127 * (1 / m))), scale = m * (1 / 127), every step rounded to f32, so that each implementation
// gives the same bits (those of the elementary operations of torch on a GPU, where a quotient with a number is a product with a reciprocal); m < 2^-100 leaves zeros with the scale 0, an infinity or a NaN makes the scale NaN and with it the whole vector.
// The maximum is taken over the bits of |x|, among which those of infinities and NaN are the largest.
//
// A CTA takes `rows` consecutive rows of the call and one head.  LANES lanes share a vector, eight elements each, and have several vectors on their way before they look for the rows' places.
// Codes of keys stand by token and go straight to their places; codes of values stand by element, 32 tokens side by side, so they pass through shared memory: four rows that follow one
// another in a page (rows of a prompt) become words of four tokens, others single bytes.
// 8191 rows of 8 heads of 128 in bf16, written and read back: 27 us (102 MB, 3.8 TB/s), where bytes alone take 15.5: the write's instructions, some 85 for 256 elements, are in the way (the schedulers
// issue in 6 of 10 cycles).  Blocks of 256 and 512 threads: 29 and 49 us; 16 rows to a block instead of 32: 44 us; four elements a lane, one vector of a group at a time: 47 us.
#include "kv8.h"
#include "rows.cuh"

#include <type_traits>

namespace hm {
namespace {

constexpr int WT = 128;
constexpr int MOST_ROWS = 32;                   // of a CTA
constexpr float TINY = 7.888609052210118e-31f;  // 2^-100
constexpr int LDV = KV8_MAX_DIM + 4;            // bytes from row to row in shared memory: an odd number of words

// n of eight elements, as they stand in memory where they are taken as one (VEC: all eight, 16-byte aligned), else as f32.
template <bool BF16, bool VEC>
struct Eight {
    static constexpr bool PACKED = BF16 && VEC;
    uint32_t w[PACKED ? 4 : 8];
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < (PACKED ? 4 : 8); ++i) w[i] = 0u;
    }
    __device__ __forceinline__ void load(const void* base, size_t at, int n) {
        if constexpr (PACKED) {
            const uint4 u = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(base) + at);
            w[0] = u.x; w[1] = u.y; w[2] = u.z; w[3] = u.w;
        } else if constexpr (VEC) {
            const uint4 u = *reinterpret_cast<const uint4*>(static_cast<const float*>(base) + at), v = *reinterpret_cast<const uint4*>(static_cast<const float*>(base) + at + 4);
            w[0] = u.x; w[1] = u.y; w[2] = u.z; w[3] = u.w;
            w[4] = v.x; w[5] = v.y; w[6] = v.z; w[7] = v.w;
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                float one[1] = {0.f};
                if (e < n) load_row<BF16, 1>(base, at + e, one);
                w[e] = __float_as_uint(one[0]);
            }
        }
    }
    // bits of the largest magnitude
    __device__ __forceinline__ uint32_t top() const {
        if constexpr (PACKED) {
            const uint32_t m = __vmaxu2(__vmaxu2(w[0] & 0x7FFF7FFFu, w[1] & 0x7FFF7FFFu), __vmaxu2(w[2] & 0x7FFF7FFFu, w[3] & 0x7FFF7FFFu));
            return max(m << 16, m & 0xFFFF0000u);
        } else {
            uint32_t m = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) m = max(m, w[e] & 0x7FFFFFFFu);
            return m;
        }
    }
    __device__ __forceinline__ float at(int e) const { return __uint_as_float(PACKED ? (e & 1 ? w[e / 2] & 0xFFFF0000u : w[e / 2] << 16) : w[PACKED ? 0 : e]); }
};
template <bool BF16, bool VEC>
__device__ __forceinline__ void store8(void* base, size_t at, int n, const float (&x)[8]) {
    if constexpr (VEC && BF16) {
        store_row<true, 8>(base, at, x);
    } else if constexpr (VEC) {
        const float y[2][4] = {{x[0], x[1], x[2], x[3]}, {x[4], x[5], x[6], x[7]}};
        store_row<false, 4>(base, at, y[0]);
        store_row<false, 4>(base, at + 4, y[1]);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
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
        const int pos = m0 + r < a.M ? __ldg(a.row_pos + m0 + r) : -1, seq = m0 + r < a.M ? __ldg(a.row_seq + m0 + r) : -1, page = kv8_page(a.pool, seq, pos);
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
    constexpr int GROUPS = WT / LANES, AHEAD = 4;  // vectors at a time; of a group that are on their way
    __shared__ Places s;
    __shared__ __align__(16) unsigned char vbuf[MOST_ROWS][LDV];
    const int h = blockIdx.y, m0 = blockIdx.x * rows, lane = threadIdx.x % LANES, group = threadIdx.x / LANES, dim = a.pool.dim, vdim = a.pool.vdim, d = 8 * lane;
    const unsigned mask = LANES == 32 ? 0xffffffffu : ((1u << LANES % 32) - 1u) << (threadIdx.x & 31 & ~(LANES - 1));
    for (int base = 0; base < 2 * rows; base += AHEAD * GROUPS) {  // keys of all rows, then values
        Eight<BF16, VEC> x[AHEAD];
        uint32_t top = 0;  // lane k of a group: of its vector k
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
            const int i = base + group + k * GROUPS, r = i >= rows ? i - rows : i, n = i >= rows ? vdim : dim;
            x[k].zero();
            if (i < 2 * rows && m0 + r < a.M && d < n) x[k].load(i >= rows ? a.v : a.k, (size_t)(m0 + r) * (i >= rows ? a.ldv : a.ldk) + (size_t)h * n + d, n - d);
        }
        if (base == 0) find_places(a, m0, rows, h, s);
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
            uint32_t t = x[k].top();
#pragma unroll
            for (int o = LANES / 2; o > 0; o >>= 1) t = max(t, __shfl_xor_sync(mask, t, o));
            if (lane == k) top = t;
        }
        // the first lanes find the factors for all
        const float most = __uint_as_float(top);
        const bool finite = top < 0x7F800000u, some = finite && most >= TINY;
        const float up = some ? __fmul_rn(__frcp_rn(most), 127.f) : 0.f;
        {
            const int i = base + group + lane * GROUPS, r = i >= rows ? i - rows : i;
            if (lane < AHEAD && i < 2 * rows && s.key[r])
                reinterpret_cast<float*>(s.key[r] + (i >= rows ? kv8_part_bytes(dim) : 0))[s.token[r]] = !finite ? __uint_as_float(0x7FC00000u) : some ? __fmul_rn(most, 1.0f / 127.0f) : 0.f;
        }
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
            const int i = base + group + k * GROUPS;
            const float f = __shfl_sync(mask, up, k, LANES);
            if (!__shfl_sync(mask, (int)finite, k, LANES)) x[k].zero();
            const bool value = i >= rows;
            const int r = value ? i - rows : i, n = value ? vdim : dim;
            if (i >= 2 * rows || d >= n) continue;
            unsigned char* key = s.key[r];
            if (!key) continue;
            uint32_t c[8];  // codes in the last byte: of 1.5 * 2^23 + code.  One by one: of two packed operations, product and sum, the compiler makes one that rounds once
#pragma unroll
            for (int e = 0; e < 8; ++e) c[e] = __float_as_uint(__fadd_rn(__fmul_rn(x[k].at(e), f), 12582912.f));
            const uint2 w = make_uint2(__byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410), __byte_perm(__byte_perm(c[4], c[5], 0x0040), __byte_perm(c[6], c[7], 0x0040), 0x5410));
            if (value) {
                *reinterpret_cast<uint32_t*>(&vbuf[r][d]) = w.x;
                *reinterpret_cast<uint32_t*>(&vbuf[r][d + 4]) = w.y;
            } else {
                *reinterpret_cast<uint2*>(key + kv8_key_at(s.token[r], d)) = w;  // elements behind the last are padding
            }
        }
    }
    __syncthreads();
    // values: eight lanes take the groups of four rows of a quad of elements, so that a word's neighbours are written with it
    const int quads = (vdim + 3) / 4, fours = rows / 4, shift = 31 - __clz(fours), values = kv8_part_bytes(dim);  // rows is a power of two
    for (int i = threadIdx.x; i < quads * fours; i += WT) {
        const int f = i & (fours - 1), d = (i >> shift) * 4;
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
    constexpr int GROUPS = WT / LANES, AHEAD = 4;
    __shared__ Places s;
    __shared__ __align__(16) unsigned char vbuf[MOST_ROWS][LDV];
    const int h = blockIdx.y, m0 = blockIdx.x * rows, lane = threadIdx.x % LANES, group = threadIdx.x / LANES, dim = a.pool.dim, vdim = a.pool.vdim, d = 8 * lane;
    find_places(a, m0, rows, h, s);
    const int quads = (vdim + 3) / 4, fours = rows / 4, shift = 31 - __clz(fours), values = kv8_part_bytes(dim);  // rows is a power of two
    for (int i = threadIdx.x; i < quads * fours; i += WT) {
        const int f = i & (fours - 1), d = (i >> shift) * 4;
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
    // keys, while the values are on their way; then these
    for (int value = 0; value < 2; ++value) {
        const int n = value ? vdim : dim;
        if (value) __syncthreads();
        for (int r0 = group; r0 < rows && d < n; r0 += AHEAD * GROUPS) {
            uint2 w[AHEAD];
            float scale[AHEAD];
#pragma unroll
            for (int k = 0; k < AHEAD; ++k) {
                const int r = r0 + k * GROUPS;
                w[k] = make_uint2(0u, 0u);
                scale[k] = 0.f;
                if (r >= rows || !s.key[r]) continue;
                const unsigned char* part = s.key[r] + (value ? values : 0);
                scale[k] = reinterpret_cast<const float*>(part)[s.token[r]];
                if (value) w[k] = make_uint2(*reinterpret_cast<const uint32_t*>(&vbuf[r][d]), *reinterpret_cast<const uint32_t*>(&vbuf[r][d + 4]));
                else w[k] = *reinterpret_cast<const uint2*>(part + kv8_key_at(s.token[r], d));
            }
#pragma unroll
            for (int k = 0; k < AHEAD; ++k) {
                const int r = r0 + k * GROUPS;
                if (r >= rows || !s.key[r]) continue;
                float x[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = (float)(int8_t)((e < 4 ? w[k].x : w[k].y) >> (8 * (e & 3))) * scale[k];
                store8<BF16, VEC>(value ? a.v : a.k, (size_t)(m0 + r) * (value ? a.ldv : a.ldk) + (size_t)h * n + d, n - d, x);
            }
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
    // eight elements at a time where all of them begin at a multiple of 16 bytes, else one by one
    const int size = BF16 ? 2 : 4, most = a.pool.dim > a.pool.vdim ? a.pool.dim : a.pool.vdim;
    const bool vec = (((uintptr_t)a.k | (uintptr_t)a.v | (a.ldk * size) | (a.ldv * size)) & 15) == 0 && ((a.pool.dim | a.pool.vdim) & 7) == 0;
    auto go = [&](auto lanes) { return vec ? launch_rows<BF16, true, decltype(lanes)::value>(a, write, sm_count, st) : launch_rows<BF16, false, decltype(lanes)::value>(a, write, sm_count, st); };
    if (most <= 32) return go(std::integral_constant<int, 4>{});
    if (most <= 64) return go(std::integral_constant<int, 8>{});
    if (most <= 128) return go(std::integral_constant<int, 16>{});
    return go(std::integral_constant<int, 32>{});
}

}  // namespace

cudaError_t launch_kv8_write(const Kv8RowsArgs& a, int sm_count, cudaStream_t st) { return a.bf16 ? launch_typed<true>(a, true, sm_count, st) : launch_typed<false>(a, true, sm_count, st); }
cudaError_t launch_kv8_read(const Kv8RowsArgs& a, int sm_count, cudaStream_t st) { return a.bf16 ? launch_typed<true>(a, false, sm_count, st) : launch_typed<false>(a, false, sm_count, st); }

}  // namespace hm

// Keys and values into a paged cache of 8 bits, and back.
//
// A row's key (or value) of one head is quantised as a whole: m = max |x|, code = rint(x * (127 / m)), scale = m / 127, every step rounded to f32, so that
// each implementation gives the same bits; m < 2^-100 leaves zeros with the scale 0, an infinity or a NaN makes the scale NaN and with it the whole vector.
// The maximum is taken over the bits of |x|, among which those of infinities and NaN are the largest.
//
// What bounds both: bytes.  LANES lanes share a vector, four elements at a time.
#include "kv8.h"
#include "rows.cuh"

#include <type_traits>

namespace hm {
namespace {

constexpr int WT = 256;
constexpr float TINY = 7.888609052210118e-31f;  // 2^-100

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

struct Slot {
    unsigned char* block;
    int token, d;
    bool value;
};
// Vector `i` of the call: row i / (2 kv_heads), keys first.  Its block is null where the row has no place.
__device__ __forceinline__ Slot slot_of(const Kv8RowsArgs& a, int m, int h, bool value) {
    const int pos = __ldg(a.row_pos + m), page = kv8_page(a.pool, __ldg(a.row_seq + m), pos);
    Slot s;
    s.block = page < 0 ? nullptr : a.pool.pages + ((size_t)page * a.pool.kv_heads + h) * kv8_block_bytes(a.pool.dim, a.pool.vdim);
    s.token = pos & (KV8_PAGE - 1);
    s.value = value;
    s.d = value ? a.pool.vdim : a.pool.dim;
    return s;
}
__device__ __forceinline__ float* scale_at(const Kv8Pool& p, const Slot& s) { return reinterpret_cast<float*>(s.block) + (s.value ? KV8_PAGE : 0) + s.token; }
__device__ __forceinline__ unsigned char* codes_at(const Kv8Pool& p, const Slot& s, int d) {
    const int row = s.value ? s.token : kv8_key_row(s.token);
    return s.block + 8 * KV8_PAGE + (s.value ? KV8_PAGE * kv8_pad(p.dim) : 0) + (d >> 5) * (KV8_PAGE * 32) + row * 32 + (d & 31);
}

template <bool BF16, bool VEC, int LANES>
__global__ void __launch_bounds__(WT) kv8_write_kernel(const Kv8RowsArgs a) {
    constexpr int QUADS = LANES == 32 ? 2 : 1;  // a lane's quads: KV8_MAX_DIM / 4 / 32
    const int lane = threadIdx.x % LANES;
    const long vectors = 2l * a.M * a.pool.kv_heads, i = (blockIdx.x * (long)WT + threadIdx.x) / LANES;
    if (i >= vectors) return;  // whole groups of LANES
    const int m = (int)(i / (2 * a.pool.kv_heads)), r = (int)(i - (long)m * 2 * a.pool.kv_heads), h = r >> 1;
    const Slot s = slot_of(a, m, h, r & 1);
    if (!s.block) return;
    const void* src = s.value ? a.v : a.k;
    const size_t at = (size_t)m * (s.value ? a.ldv : a.ldk) + (size_t)h * s.d;
    float x[QUADS][4];
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < QUADS; ++j) {
        const int d = 4 * (lane + j * LANES);
        x[j][0] = x[j][1] = x[j][2] = x[j][3] = 0.f;
        if (d < s.d) load_quad<BF16, VEC>(src, at + d, s.d - d, x[j]);
#pragma unroll
        for (int e = 0; e < 4; ++e) top = max(top, __float_as_uint(x[j][e]) & 0x7FFFFFFFu);
    }
    const unsigned group = LANES == 32 ? 0xffffffffu : ((1u << LANES % 32) - 1u) << (threadIdx.x & 31 & ~(LANES - 1));
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(group, top, o));
    const float most = __uint_as_float(top);
    const bool finite = top < 0x7F800000u, some = finite && most >= TINY;
    const float up = some ? __fdiv_rn(127.f, most) : 0.f;
    if (lane == 0) *scale_at(a.pool, s) = !finite ? __uint_as_float(0x7FC00000u) : some ? __fdiv_rn(most, 127.f) : 0.f;
#pragma unroll
    for (int j = 0; j < QUADS; ++j) {
        const int d = 4 * (lane + j * LANES);
        if (d >= s.d) continue;
        uint32_t w = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) w |= (uint32_t)(some ? __float2int_rn(__fmul_rn(x[j][e], up)) + 128 : 128) << (8 * e);
        *reinterpret_cast<uint32_t*>(codes_at(a.pool, s, d)) = w;
    }
}

template <bool BF16, bool VEC, int LANES>
__global__ void __launch_bounds__(WT) kv8_read_kernel(const Kv8RowsArgs a) {
    constexpr int QUADS = LANES == 32 ? 2 : 1;
    const int lane = threadIdx.x % LANES;
    const long vectors = 2l * a.M * a.pool.kv_heads, i = (blockIdx.x * (long)WT + threadIdx.x) / LANES;
    if (i >= vectors) return;
    const int m = (int)(i / (2 * a.pool.kv_heads)), r = (int)(i - (long)m * 2 * a.pool.kv_heads), h = r >> 1;
    const Slot s = slot_of(a, m, h, r & 1);
    if (!s.block) return;
    void* dst = s.value ? a.v : a.k;
    const size_t at = (size_t)m * (s.value ? a.ldv : a.ldk) + (size_t)h * s.d;
    const float scale = *scale_at(a.pool, s);
#pragma unroll
    for (int j = 0; j < QUADS; ++j) {
        const int d = 4 * (lane + j * LANES);
        if (d >= s.d) continue;
        const uint32_t w = *reinterpret_cast<const uint32_t*>(codes_at(a.pool, s, d));
        float x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = (float)((int)((w >> (8 * e)) & 0xFFu) - 128) * scale;
        if constexpr (VEC) {
            store_row<BF16, 4>(dst, at + d, x);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float one[1] = {x[e]};
                if (d + e < s.d) store_row<BF16, 1>(dst, at + d + e, one);
            }
        }
    }
}

template <bool BF16, bool VEC, int LANES>
cudaError_t launch_rows(const Kv8RowsArgs& a, bool write, cudaStream_t st) {
    const long blocks = (2l * a.M * a.pool.kv_heads * LANES + WT - 1) / WT;
    if (write) kv8_write_kernel<BF16, VEC, LANES><<<(unsigned)blocks, WT, 0, st>>>(a);
    else kv8_read_kernel<BF16, VEC, LANES><<<(unsigned)blocks, WT, 0, st>>>(a);
    return cudaGetLastError();
}

template <bool BF16>
cudaError_t launch_typed(const Kv8RowsArgs& a, bool write, cudaStream_t st) {
    const int size = BF16 ? 2 : 4, most = a.pool.dim > a.pool.vdim ? a.pool.dim : a.pool.vdim;
    const bool vec = (((uintptr_t)a.k | (uintptr_t)a.v | (a.ldk * size) | (a.ldv * size)) & (4 * size - 1)) == 0 && ((a.pool.dim | a.pool.vdim) & 3) == 0;
    auto go = [&](auto lanes) { return vec ? launch_rows<BF16, true, decltype(lanes)::value>(a, write, st) : launch_rows<BF16, false, decltype(lanes)::value>(a, write, st); };
    if (most <= 32) return go(std::integral_constant<int, 8>{});
    if (most <= 64) return go(std::integral_constant<int, 16>{});
    return go(std::integral_constant<int, 32>{});
}

}  // namespace

cudaError_t launch_kv8_write(const Kv8RowsArgs& a, cudaStream_t st) { return a.bf16 ? launch_typed<true>(a, true, st) : launch_typed<false>(a, true, st); }
cudaError_t launch_kv8_read(const Kv8RowsArgs& a, cudaStream_t st) { return a.bf16 ? launch_typed<true>(a, false, st) : launch_typed<false>(a, false, st); }

}  // namespace hm

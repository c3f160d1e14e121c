// Rows into operand images and back, the plan that groups rows by expert, and the weighted sum of the experts' results.
//
//   pack_kernel     a warp per row and one or three k-blocks (128 bytes of the image each: one line): a lane has 4 bytes of codes (eight values) or 4 bytes of
//                   bf16 (two).  Bound by the bytes of x: 1999 x 8960 bf16 8.3 us (45 MB, 0.83 of the measured copy bandwidth).
//   unpack_kernel   the way back; f32 rows leave in whole sectors: the same rows 11.8 us (81 MB, 1.05 of it, most of them writes)
//   blocks_kernel   GGUF blocks into the image
//   plan_kernel     stable counting sort of the pairs by expert: a CTA per expert reads all ids (they stay in the L2), so that neither order nor
//                   result depends on atomics' order and nothing is kept between calls.  512 pairs 2.5 us, 16384 pairs 7.3 us: bound by latency
//   sum_kernel      y = resid + sum of the chosen experts' rows times their weights, in the order of the choice; bound by the rows' bytes
#include "image.h"

#include <algorithm>
#include <type_traits>

namespace hm {
namespace {

constexpr int THREADS = 256, WARPS = THREADS / 32;

__device__ __forceinline__ float load1(const void* x, int bf16, size_t i) { return bf16 ? bf16_bits_to_f32(__ldg(static_cast<const uint16_t*>(x) + i)) : __ldg(static_cast<const float*>(x) + i); }

// silu(g) u from e^-|g|: gates below -87 keep what a large u makes of them, and the divisor is from 1 to 2, where the fast quotient is good to 2 ulp (the full one:
// 11.7 us for 4136 x 1120 f32 pairs, 4-bit).
__device__ __forceinline__ float gated(float g, float u) {
    const float t = expf(-fabsf(g));
    return __fdividef(g < 0.f ? g * t : g, 1.0f + t) * u;
}

// Eight codes of a lane, and the scales of its four blocks (the same in sixteen lanes).  Block of 32 values over four lanes (eight each): e = floor(log2 max) - 2, at least -127, as byte e + 127; codes x 2^-e to nearest even, saturated at 6.
// The largest exponent field is 255 where a value is infinite or no number: the whole block is then no number.
__device__ __forceinline__ uint32_t mx_block(int lane, float (&v)[8], uint32_t& scales) {
    float most = 0.f;  // keeps a NaN
#pragma unroll
    for (int e = 0; e < 8; ++e) asm("max.NaN.f32 %0, %0, %1;" : "+f"(most) : "f"(fabsf(v[e])));
    uint32_t top = __float_as_uint(most) & 0x7FFFFFFFu;
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const uint32_t field = top >> 23, s = field == 255u ? 255u : field > 2u ? field - 2u : 0u;
    const float up = __uint_as_float((254u - s) << 23);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = field == 255u ? 0.f : v[e] * up;
    scales = s << (8 * (lane >> 2 & 3));
    scales |= __shfl_xor_sync(0xffffffffu, scales, 4);
    scales |= __shfl_xor_sync(0xffffffffu, scales, 8);
    return mx_codes(v);
}

// CTA: eight rows of x, a warp each (grid x); U k-blocks of a row per warp (grid y).  With a plan a row is read and rounded once for all its pairs.  Everything a warp loads is asked for before it works on the first.
template <bool MX, bool BF16, bool GLU, bool PLAN, int U>
__global__ void __launch_bounds__(THREADS) pack_kernel(const PackArgs a, int kblocks) {
    constexpr int V = MX ? 8 : 2;  // values of a lane and k-block
    using Word = typename Words<V * (BF16 ? 2 : 4)>::type;
    constexpr int NW = V * (BF16 ? 2 : 4) / sizeof(Word);
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31, row = blockIdx.x * WARPS + (threadIdx.x >> 5), kb0 = blockIdx.y * U;
    if (row >= a.rows) return;
    const size_t es = BF16 ? 2 : 4;
    const char* x = static_cast<const char*>(a.x) + (size_t)row * a.ldx * es;
    const int k0 = kb0 * (MX ? MX_K : BF_K) + lane * V;
    const bool aligned = ((uintptr_t)x & (sizeof(Word) - 1)) == 0 && (!GLU || (a.K * es & (sizeof(Word) - 1)) == 0);
    const int copies = PLAN ? a.top : 1;
    int place = row;  // lane c: where copy c of the row goes
    if (PLAN) place = lane < copies ? __ldg(a.place + (size_t)row * a.top + lane) : -1;
    Word w[U][NW], g[GLU ? U : 1][NW];
#pragma unroll
    for (int i = 0; i < U; ++i) {
        const int k = k0 + i * (MX ? MX_K : BF_K);
        if (aligned && k + V <= a.K) {
#pragma unroll
            for (int e = 0; e < NW; ++e) {
                w[i][e] = __ldg(reinterpret_cast<const Word*>(x + k * es) + e);
                if (GLU) g[GLU ? i : 0][e] = __ldg(reinterpret_cast<const Word*>(x + ((size_t)a.K + k) * es) + e);
            }
        } else {
            load_ragged<V, BF16>(x, k, a.K, w[i]);
            if (GLU) load_ragged<V, BF16>(x + (size_t)a.K * es, k, a.K, g[GLU ? i : 0]);
        }
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
        if (kb0 + i >= kblocks) return;
        float v[V];
        widen<V, BF16>(w[i], v);
        if constexpr (GLU) {
            float u[V];
            widen<V, BF16>(g[i], u);
#pragma unroll
            for (int e = 0; e < V; ++e) v[e] = gated(v[e], u[e]);
        }
        uint32_t codes, scales = 0;
        if constexpr (MX) codes = mx_block(lane, v, scales);
        else codes = bf16x2_rne(v[0], v[1]);
        // to the row's own place, or to those of its pairs
        if (PLAN && copies > 32 && i) place = __ldg(a.place + (size_t)row * a.top + lane);
        for (int c = 0; c < copies; ++c) {
            if (PLAN && c && (c & 31) == 0) place = c + lane < copies ? __ldg(a.place + (size_t)row * a.top + c + lane) : -1;
            const int to = PLAN ? __shfl_sync(0xffffffffu, place, c & 31) : row;
            if (PLAN && (to < 0 || to >= a.image_rows)) continue;
            const int r = to % IMG_ROWS;
            unsigned char* tile = a.image + ((size_t)(to / IMG_ROWS) * kblocks + kb0 + i) * (MX ? MX_TILE : IMG_CODES);
            *reinterpret_cast<uint32_t*>(tile + (MX ? MX_SCALES : 0) + r * 128 + (((lane >> 2) ^ (r & 7)) << 4) + (lane & 3) * 4) = codes;
            if (MX && (lane & 15) == 0) *reinterpret_cast<uint32_t*>(tile + mx_scale_at(r, lane >> 2)) = scales;
        }
    }
}

template <bool MX, bool BF16, int U>
__global__ void __launch_bounds__(THREADS) unpack_kernel(const unsigned char* image, int rows, int K, int kblocks, void* out, size_t ld) {
    constexpr int V = MX ? 8 : 2;
    using Word = typename Words<V * (BF16 ? 2 : 4)>::type;
    constexpr int NW = V * (BF16 ? 2 : 4) / sizeof(Word);
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31, row = blockIdx.x * WARPS + (threadIdx.x >> 5), kb0 = blockIdx.y * U;
    if (row >= rows) return;
    const size_t es = BF16 ? 2 : 4;
    char* y = static_cast<char*>(out) + (size_t)row * ld * es;
    const bool aligned = ((uintptr_t)y & (sizeof(Word) - 1)) == 0;
    const int r = row % IMG_ROWS, piece = lane >> 2, k0 = kb0 * (MX ? MX_K : BF_K) + lane * V;
    const unsigned char* tile = image + ((size_t)(row / IMG_ROWS) * kblocks + kb0) * (MX ? MX_TILE : IMG_CODES);
    uint32_t w[U], s[U];
#pragma unroll
    for (int i = 0; i < U; ++i)
        if (kb0 + i < kblocks) {
            const unsigned char* t = tile + (size_t)i * (MX ? MX_TILE : IMG_CODES);
            w[i] = __ldg(reinterpret_cast<const uint32_t*>(t + (MX ? MX_SCALES : 0) + r * 128 + ((piece ^ (r & 7)) << 4) + (lane & 3) * 4));
            if (MX) s[i] = __ldg(t + mx_scale_at(r, piece));
        }
#pragma unroll
    for (int i = 0; i < U; ++i) {
        if (kb0 + i >= kblocks) return;
        const int k = k0 + i * (MX ? MX_K : BF_K), n = K - k;
        float v[V];
        if constexpr (MX) {
            uint32_t h[4];
            mx_halves(w[i], h);
            const float f = mx_scale(s[i]);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                v[2 * e] = f16_bits_to_f32((uint16_t)h[e]) * f;
                v[2 * e + 1] = f16_bits_to_f32((uint16_t)(h[e] >> 16)) * f;
            }
        } else {
            v[0] = bf16_lo(w[i]);
            v[1] = bf16_hi(w[i]);
        }
        uint32_t p[V * (BF16 ? 2 : 4) / 4];
#pragma unroll
        for (int e = 0; e < V; ++e) {
            if (!BF16) p[e] = __float_as_uint(v[e]);
            else if ((e & 1) == 0) p[e / 2] = bf16x2_rne(v[e], v[e + 1]);
        }
        if (MX && !BF16 && aligned && __all_sync(0xffffffffu, n >= V)) {
            // lanes in pairs swap halves, so that a store fills whole sectors of 32 bytes
            const bool odd = lane & 1;
            uint32_t q[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) q[e] = __shfl_xor_sync(0xffffffffu, odd ? p[e] : p[4 % V + e], 1);
            char* o = y + (k - (odd ? V : 0)) * es + (odd ? 16 : 0);
            *reinterpret_cast<uint4*>(o) = odd ? make_uint4(q[0], q[1], q[2], q[3]) : make_uint4(p[0], p[1], p[2 % V], p[3 % V]);
            *reinterpret_cast<uint4*>(o + 32) = odd ? make_uint4(p[4 % V], p[5 % V], p[6 % V], p[7 % V]) : make_uint4(q[0], q[1], q[2], q[3]);
        } else if (aligned && n >= V) {
#pragma unroll
            for (int e = 0; e < NW; ++e) {
                Word o;
#pragma unroll
                for (int q = 0; q < (int)sizeof(Word) / 4; ++q) reinterpret_cast<uint32_t*>(&o)[q] = p[e * (sizeof(Word) / 4) + q];
                reinterpret_cast<Word*>(y + k * es)[e] = o;
            }
        } else {
#pragma unroll
            for (int e = 0; e < V; ++e)
                if (e < n) {
                    if (BF16) reinterpret_cast<uint16_t*>(y)[k + e] = (uint16_t)(p[e / 2] >> (16 * (e & 1)));
                    else reinterpret_cast<uint32_t*>(y)[k + e] = p[e];
                }
        }
    }
}

// A warp per row and k-block of 256 values: eight blocks of 17 bytes; four lanes share a block, each with eight values.
__global__ void __launch_bounds__(THREADS) blocks_kernel(const uint8_t* blocks, int K, int kblocks, long long units, unsigned char* image) {
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31;
    const long long u = (long long)blockIdx.x * WARPS + (threadIdx.x >> 5);
    if (u >= units) return;
    const int row = (int)(u / kblocks), kb = (int)(u - (long long)row * kblocks), r = row % IMG_ROWS, piece = lane >> 2, q = lane & 3, b = kb * 8 + piece;
    uint32_t w = 0, s = 0;
    if (b < K / 32) {
        const uint8_t* src = blocks + ((size_t)row * (K / 32) + b) * 17;
        s = __ldg(src);
#pragma unroll
        for (int e = 0; e < 8; ++e) {  // values 8 q + e: low halves hold values 0 .. 15 of the block, high halves 16 .. 31
            const uint32_t byte = __ldg(src + 1 + (q & 1) * 8 + e);
            w |= (q < 2 ? byte & 15u : byte >> 4) << (4 * e);
        }
    }
    unsigned char* tile = image + ((size_t)(row / IMG_ROWS) * kblocks + kb) * MX_TILE;
    *reinterpret_cast<uint32_t*>(tile + MX_SCALES + r * 128 + ((piece ^ (r & 7)) << 4) + q * 4) = w;
    if (q == 0) tile[mx_scale_at(r, piece)] = (unsigned char)s;
}

// CTA e: the expert's rows.  A warp looks at a run of up to 32 * PLAN_IDS ids of a round, 32 at a time, so that votes and sums in front of a warp keep the pairs'
// order; one round (16384 pairs) stays in registers between the two passes.  First the counts of all experts, in copies per lane so that neither a bank nor an
// address is hit twice by a warp.
constexpr int PLAN_THREADS = 512, PLAN_WARPS = PLAN_THREADS / 32, PLAN_IDS = 32;
inline int plan_copies(int experts) { return experts <= 256 ? 32 : 8; }
__global__ void __launch_bounds__(PLAN_THREADS) plan_kernel(const int32_t* __restrict__ ids, const Plan p, int copies) {
    extern __shared__ int hist[];  // [experts][copies], then the sums in the first copy
    __shared__ int warp_sums[PLAN_WARPS], first_s[2];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, e = blockIdx.x;
    for (int i = tid; i < p.experts * copies; i += PLAN_THREADS) hist[i] = 0;
    __syncthreads();
    pdl_wait();
    int id[PLAN_IDS];
    const int per = min(PLAN_IDS, max((p.pairs + PLAN_THREADS - 1) / PLAN_THREADS, 1)), round = per * PLAN_THREADS;  // ids of a thread, of all threads
    auto fetch = [&](int i0) {
#pragma unroll
        for (int k = 0; k < PLAN_IDS; ++k) {
            if (k >= per) break;
            id[k] = i0 + k * 32 < p.pairs ? __ldg(ids + i0 + k * 32) : -1;
        }
    };
    const int at = warp * per * 32 + lane;
    for (int c0 = 0; c0 < p.pairs; c0 += round) {
        fetch(c0 + at);
#pragma unroll
        for (int k = 0; k < PLAN_IDS; ++k) {
            if (k >= per) break;
            if (id[k] >= 0 && id[k] < p.experts) atomicAdd(&hist[id[k] * copies + (lane & (copies - 1))], 1);  // counts: the same in any order
            else if (e == 0 && c0 + at + k * 32 < p.pairs) p.place[c0 + at + k * 32] = -1;
        }
    }
    __syncthreads();
    for (int i = warp; i < p.experts; i += PLAN_WARPS) {
        const int n = __reduce_add_sync(0xffffffffu, lane < copies ? hist[i * copies + lane] : 0);
        if (lane == 0) hist[i * copies] = n;
    }
    __syncthreads();
    const int n = hist[e * copies];
    if (warp == 0) {  // blocks in front of the expert, and of all experts
        int before = 0, all = 0;
        for (int i = lane; i < p.experts; i += 32) {
            const int b = (hist[i * copies] + IMG_ROWS - 1) / IMG_ROWS;
            all += b;
            if (i < e) before += b;
        }
        before = __reduce_add_sync(0xffffffffu, before);
        all = __reduce_add_sync(0xffffffffu, all);
        if (lane == 0) {
            first_s[0] = before;
            first_s[1] = all;
            p.first[e] = before;
            p.count[e] = n;
            if (e == 0) p.first[p.experts] = all;
        }
    }
    __syncthreads();
    const int row0 = first_s[0] * IMG_ROWS;
    int base = row0;
    for (int c0 = 0; c0 < p.pairs && base < row0 + n; c0 += round) {
        if (p.pairs > round) fetch(c0 + at);
        int mine = 0;
#pragma unroll
        for (int k = 0; k < PLAN_IDS; ++k) {
            if (k >= per) break;
            mine += id[k] == e;
        }
        mine = __reduce_add_sync(0xffffffffu, mine);
        if (lane == 0) warp_sums[warp] = mine;
        __syncthreads();
        int r = base;
#pragma unroll
        for (int w = 0; w < PLAN_WARPS; ++w) {
            if (w < warp) r += warp_sums[w];
            base += warp_sums[w];
        }
#pragma unroll
        for (int k = 0; k < PLAN_IDS; ++k) {
            if (k >= per) break;
            const uint32_t votes = __ballot_sync(0xffffffffu, id[k] == e);
            if (id[k] == e) {
                const int to = r + __popc(votes & ((1u << lane) - 1u));
                p.place[c0 + at + k * 32] = to;
                p.row[to] = c0 + at + k * 32;
            }
            r += __popc(votes);
        }
        __syncthreads();
    }
    // rows behind the expert's last, and behind the last expert's
    for (int r = row0 + n + tid; r < row0 + (n + IMG_ROWS - 1) / IMG_ROWS * IMG_ROWS; r += PLAN_THREADS) p.row[r] = -1;
    for (int r = first_s[1] * IMG_ROWS + e * PLAN_THREADS + tid; r < p.rows; r += p.experts * PLAN_THREADS) p.row[r] = -1;
}

template <bool RB, bool YB>
__global__ void __launch_bounds__(THREADS) sum_kernel(const SumArgs a, int v4) {
    pdl_launch_dependents();
    pdl_wait();
    const int t = blockIdx.y;
    const int per = v4 ? 4 : 1;
    const int i = (blockIdx.x * THREADS + threadIdx.x) * per;
    if (i >= a.W) return;
    float s[4] = {0.f, 0.f, 0.f, 0.f};
    const size_t at = (size_t)t * a.W + i;
    for (int j0 = 0; j0 < a.top; j0 += 4) {  // four rows are asked for at a time
        float w[4], v[4][4];
        bool on[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const size_t j = (size_t)t * a.top + j0 + q;
            const int id = j0 + q < a.top ? __ldg(a.ids + j) : -1;
            on[q] = id >= 0 && id < a.experts;
            if (!on[q]) continue;
            w[q] = __ldg(a.weights + j);
            const size_t p = j * a.W + i;
            if (v4 && RB) {
                const uint2 u = __ldg(reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(a.rows) + p));
                v[q][0] = bf16_lo(u.x), v[q][1] = bf16_hi(u.x), v[q][2] = bf16_lo(u.y), v[q][3] = bf16_hi(u.y);
            } else if (v4) {
                const float4 u = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(a.rows) + p));
                v[q][0] = u.x, v[q][1] = u.y, v[q][2] = u.z, v[q][3] = u.w;
            } else
                v[q][0] = load1(a.rows, RB, p);
        }
#pragma unroll
        for (int q = 0; q < 4; ++q)
            if (on[q])
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    if (c < per) s[c] = fmaf(w[q], v[q][c], s[c]);
    }
    if (a.resid) {
        const float* x = static_cast<const float*>(a.resid) + at;
        for (int c = 0; c < per; ++c) s[c] += x[c];  // (may be y itself)
    }
    if (YB) {
        uint16_t* y = static_cast<uint16_t*>(a.y) + at;
        if (v4) *reinterpret_cast<uint2*>(y) = make_uint2(bf16x2_rne(s[0], s[1]), bf16x2_rne(s[2], s[3]));
        else *y = (uint16_t)bf16x2_rne(s[0], 0.f);
    } else {
        float* y = static_cast<float*>(a.y) + at;
        if (v4) *reinterpret_cast<float4*>(y) = make_float4(s[0], s[1], s[2], s[3]);
        else *y = s[0];
    }
}

inline cudaError_t grid_of(long long units, int per, unsigned* g) {
    const long long n = (units + per - 1) / per;
    *g = (unsigned)n;
    return n > 0x7FFFFFFFLL ? cudaErrorInvalidValue : cudaSuccess;
}

}  // namespace

// k-blocks of a warp: three, or one where that gives too few warps (two rounds of 148 SMs with 64 warps each).
static int pack_units(long long rows, int kblocks) { return kblocks < 3 || rows * kblocks < 2 * 148 * 64 ? 1 : 3; }

cudaError_t launch_image_pack(const PackArgs& a, bool mx, cudaStream_t st) {
    const int kblocks = img_kblocks(mx, a.K), U = pack_units(a.rows, kblocks);
    const dim3 g((a.rows + WARPS - 1) / WARPS, (kblocks + U - 1) / U);
    if (g.y > 65535) return cudaErrorInvalidValue;
    auto launch = [&](auto MX, auto B, auto G, auto P) {
        if (U == 1) return launch_after(pack_kernel<MX.value, B.value, G.value, P.value, 1>, g, THREADS, 0, 1, st, a, kblocks);
        return launch_after(pack_kernel<MX.value, B.value, G.value, P.value, 3>, g, THREADS, 0, 1, st, a, kblocks);
    };
    const std::true_type yes;
    const std::false_type no;
    auto with_glu = [&](auto MX, auto B, auto G) { return a.place ? launch(MX, B, G, yes) : launch(MX, B, G, no); };
    auto with = [&](auto MX, auto B) { return a.glu ? with_glu(MX, B, yes) : with_glu(MX, B, no); };
    if (mx) return a.bf16 ? with(yes, yes) : with(yes, no);
    return a.bf16 ? with(no, yes) : with(no, no);
}

cudaError_t launch_image_unpack(const unsigned char* image, bool mx, int rows, int K, void* out, bool bf16, size_t ld, cudaStream_t st) {
    const int kblocks = img_kblocks(mx, K), U = pack_units(rows, kblocks);
    const dim3 g((rows + WARPS - 1) / WARPS, (kblocks + U - 1) / U);
    if (g.y > 65535) return cudaErrorInvalidValue;
    auto with = [&](auto MX, auto B) {
        if (U == 1) return launch_after(unpack_kernel<MX.value, B.value, 1>, g, THREADS, 0, 1, st, image, rows, K, kblocks, out, ld);
        return launch_after(unpack_kernel<MX.value, B.value, 3>, g, THREADS, 0, 1, st, image, rows, K, kblocks, out, ld);
    };
    if (mx) return bf16 ? with(std::true_type{}, std::true_type{}) : with(std::true_type{}, std::false_type{});
    return bf16 ? with(std::false_type{}, std::true_type{}) : with(std::false_type{}, std::false_type{});
}

cudaError_t launch_image_blocks(const uint8_t* blocks, int rows, int K, unsigned char* image, cudaStream_t st) {
    const int kblocks = img_kblocks(true, K);
    const long long units = (long long)rows * kblocks;
    unsigned g;
    if (const cudaError_t e = grid_of(units, WARPS, &g)) return e;
    return launch_after(blocks_kernel, dim3(g), THREADS, 0, 1, st, blocks, K, kblocks, units, image);
}

cudaError_t launch_plan(const int32_t* ids, const Plan& p, cudaStream_t st) {
    const int copies = plan_copies(p.experts);
    return launch_after(plan_kernel, dim3(p.experts), PLAN_THREADS, (size_t)p.experts * copies * 4, 1, st, ids, p, copies);
}

cudaError_t launch_expert_sum(const SumArgs& a, cudaStream_t st) {
    const int rs = a.rows_bf16 ? 8 : 16, ys = a.y_bf16 ? 8 : 16;
    const int v4 = a.W % 4 == 0 && (uintptr_t)a.rows % rs == 0 && (uintptr_t)a.y % ys == 0;
    if (a.tokens > 65535) {  // the grid's second dimension
        SumArgs b = a, c = a;
        b.tokens = 65535;
        c.tokens = a.tokens - 65535;
        const size_t n = 65535;
        c.rows = static_cast<const char*>(a.rows) + n * a.top * a.W * (a.rows_bf16 ? 2 : 4);
        c.ids = a.ids + n * a.top;
        c.weights = a.weights + n * a.top;
        if (a.resid) c.resid = static_cast<const float*>(a.resid) + n * a.W;
        c.y = static_cast<char*>(a.y) + n * a.W * (a.y_bf16 ? 2 : 4);
        if (const cudaError_t e = launch_expert_sum(b, st)) return e;
        return launch_expert_sum(c, st);
    }
    const dim3 g((a.W / (v4 ? 4 : 1) + THREADS - 1) / THREADS, a.tokens);
    void (*const kernels[2][2])(SumArgs, int) = {{sum_kernel<false, false>, sum_kernel<false, true>}, {sum_kernel<true, false>, sum_kernel<true, true>}};
    return launch_after(kernels[a.rows_bf16 != 0][a.y_bf16 != 0], g, THREADS, 0, 1, st, a, v4);
}

}  // namespace hm

// Rows into operand images and back, the plan that groups rows by expert, and the weighted sum of the experts' results.
//
//   pack_kernel     a warp per row and k-block (128 bytes of the image: one line): a lane has 4 bytes of codes (eight values) or 4 bytes of bf16 (two).
//                   Bound by the bytes of x: each warp asks for PACK_UNITS units before it works on the first.
//   unpack_kernel   the way back
//   blocks_kernel   GGUF blocks into the image
//   plan_kernel     stable counting sort of the pairs by expert: a CTA per expert reads all ids (they stay in the L2), so that neither order nor
//                   result depends on atomics' order and nothing is kept between calls
//   sum_kernel      y = resid + sum of the chosen experts' rows times their weights, in the order of the choice
#include "image.h"

#include <algorithm>

namespace hm {
namespace {

constexpr int THREADS = 256, WARPS = THREADS / 32;
constexpr int PACK_UNITS = 4;

__device__ __forceinline__ float load1(const void* x, int bf16, size_t i) { return bf16 ? bf16_bits_to_f32(__ldg(static_cast<const uint16_t*>(x) + i)) : __ldg(static_cast<const float*>(x) + i); }

// Eight values from element i on (16-byte aligned), or fewer: n exist, the others are zero.
template <bool BF16>
__device__ __forceinline__ void load8(const void* x, size_t i, int n, bool aligned, float (&v)[8]) {
    if (aligned && n >= 8) {
        if (BF16) {
            const uint4 u = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(x) + i));
            const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                v[2 * e] = bf16_lo(w[e]);
                v[2 * e + 1] = bf16_hi(w[e]);
            }
        } else {
            const float4 a = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(x) + i)), b = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(x) + i) + 1);
            v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = e < n ? load1(x, BF16, i + e) : 0.f;
    }
}
__device__ __forceinline__ float gated(float g, float u) { return g / (1.0f + expf(-g)) * u; }

// Row of x that image row r comes from; -1: none.
__device__ __forceinline__ long long source_row(const PackArgs& a, int r) {
    if (!a.src) return r;
    const int s = __ldg(a.src + r);
    if (s < 0) return -1;
    const int q = s / a.div;
    return q < a.src_rows ? q : -1;
}

// Block of 32 values over four lanes (eight each): e = floor(log2 max) - 2, at least -127, as byte e + 127; codes x 2^-e to nearest even, saturated at 6.
// The largest exponent field is 255 where a value is infinite or no number: the whole block is then no number.
__device__ __forceinline__ void store_mx(unsigned char* tile, int r, int lane, float (&v)[8]) {
    uint32_t top = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(v[e]) & 0x7FFFFFFFu);
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const uint32_t field = top >> 23, s = field == 255u ? 255u : field > 2u ? field - 2u : 0u;
    const float up = __uint_as_float((254u - s) << 23);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = field == 255u ? 0.f : v[e] * up;
    const int piece = lane >> 2;
    *reinterpret_cast<uint32_t*>(tile + MX_SCALES + r * 128 + ((piece ^ (r & 7)) << 4) + (lane & 3) * 4) = mx_codes(v);
    uint32_t w = s << (8 * (piece & 3));
    w |= __shfl_xor_sync(0xffffffffu, w, 4);
    w |= __shfl_xor_sync(0xffffffffu, w, 8);
    if ((lane & 15) == 0) *reinterpret_cast<uint32_t*>(tile + mx_scale_at(r, piece)) = w;
}

template <bool MX, bool BF16, bool GLU>
__global__ void __launch_bounds__(THREADS) pack_kernel(const PackArgs a, int kblocks, long long units) {
    const int lane = threadIdx.x & 31;
    const long long u0 = ((long long)blockIdx.x * WARPS + (threadIdx.x >> 5)) * PACK_UNITS;
    // values of a lane: eight codes; two bf16, of which four units make the same eight loads
    constexpr int V = MX ? 8 : 2;
    const size_t es = BF16 ? 2 : 4;
    const bool aligned = MX ? ((uintptr_t)a.x & 15) == 0 && (a.ldx * es & 15) == 0 && (!GLU || (a.K * es & 15) == 0)
                            : ((uintptr_t)a.x & (2 * es - 1)) == 0 && (a.ldx & 1) == 0 && (!GLU || (a.K & 1) == 0);
    float v[PACK_UNITS][V], g[GLU ? PACK_UNITS : 1][V];
    long long from[PACK_UNITS];
    int row[PACK_UNITS], kb[PACK_UNITS];
#pragma unroll
    for (int i = 0; i < PACK_UNITS; ++i) {
        const long long u = u0 + i;
        row[i] = u < units ? (int)(u / kblocks) : 0;
        kb[i] = u < units ? (int)(u - (long long)row[i] * kblocks) : 0;
        from[i] = u < units ? source_row(a, row[i]) : -1;
    }
#pragma unroll
    for (int i = 0; i < PACK_UNITS; ++i) {
        if (from[i] < 0) continue;
        const int k = kb[i] * (MX ? MX_K : BF_K) + lane * V, n = max(0, a.K - k);
        const size_t at = (size_t)from[i] * a.ldx + k;
        if constexpr (MX) {
            load8<BF16>(a.x, at, n, aligned, v[i]);
            if constexpr (GLU) load8<BF16>(a.x, at + a.K, n, aligned, g[i]);
        } else {
            auto load2 = [&](size_t p, float (&d)[V]) {
                if (aligned && n >= 2) {
                    if (BF16) {
                        const uint32_t w = __ldg(reinterpret_cast<const uint32_t*>(static_cast<const uint16_t*>(a.x) + p));
                        d[0] = bf16_lo(w), d[1] = bf16_hi(w);
                    } else {
                        const float2 w = __ldg(reinterpret_cast<const float2*>(static_cast<const float*>(a.x) + p));
                        d[0] = w.x, d[1] = w.y;
                    }
                } else {
                    d[0] = n > 0 ? load1(a.x, BF16, p) : 0.f;
                    d[1] = n > 1 ? load1(a.x, BF16, p + 1) : 0.f;
                }
            };
            load2(at, v[i]);
            if constexpr (GLU) load2(at + a.K, g[i]);
        }
    }
#pragma unroll
    for (int i = 0; i < PACK_UNITS; ++i) {
        if (from[i] < 0) continue;  // the same for the whole warp
        if constexpr (GLU)
#pragma unroll
            for (int e = 0; e < V; ++e) v[i][e] = gated(v[i][e], g[i][e]);
        unsigned char* tile = a.image + ((size_t)(row[i] / IMG_ROWS) * kblocks + kb[i]) * (MX ? MX_TILE : IMG_CODES);
        const int r = row[i] % IMG_ROWS;
        if constexpr (MX)
            store_mx(tile, r, lane, v[i]);
        else
            *reinterpret_cast<uint32_t*>(tile + r * 128 + (((lane >> 2) ^ (r & 7)) << 4) + (lane & 3) * 4) = bf16x2_rne(v[i][0], v[i][1]);
    }
}

template <bool MX, bool BF16>
__global__ void __launch_bounds__(THREADS) unpack_kernel(const unsigned char* image, int K, int kblocks, long long units, void* out, size_t ld) {
    const int lane = threadIdx.x & 31;
    const long long u0 = ((long long)blockIdx.x * WARPS + (threadIdx.x >> 5)) * PACK_UNITS;
    constexpr int V = MX ? 8 : 2;
    const size_t es = BF16 ? 2 : 4;
    const bool aligned = ((uintptr_t)out & (V * es >= 16 ? 15 : V * es - 1)) == 0 && (ld * es & (V * es >= 16 ? 15 : V * es - 1)) == 0;
    uint32_t w[PACK_UNITS], s[PACK_UNITS];
#pragma unroll
    for (int i = 0; i < PACK_UNITS; ++i) {
        const long long u = u0 + i;
        if (u >= units) continue;
        const int row = (int)(u / kblocks), kb = (int)(u - (long long)row * kblocks), r = row % IMG_ROWS, piece = lane >> 2;
        const unsigned char* tile = image + ((size_t)(row / IMG_ROWS) * kblocks + kb) * (MX ? MX_TILE : IMG_CODES);
        w[i] = __ldg(reinterpret_cast<const uint32_t*>(tile + (MX ? MX_SCALES : 0) + r * 128 + ((piece ^ (r & 7)) << 4) + (lane & 3) * 4));
        if (MX) s[i] = __ldg(tile + mx_scale_at(r, piece));
    }
#pragma unroll
    for (int i = 0; i < PACK_UNITS; ++i) {
        const long long u = u0 + i;
        if (u >= units) continue;
        const int row = (int)(u / kblocks), kb = (int)(u - (long long)row * kblocks);
        const int k = kb * (MX ? MX_K : BF_K) + lane * V, n = K - k;
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
        const size_t at = (size_t)row * ld + k;
        if (aligned && n >= V) {
            if constexpr (BF16) {
                uint32_t p[V / 2];
#pragma unroll
                for (int e = 0; e < V / 2; ++e) p[e] = bf16x2_rne(v[2 * e], v[2 * e + 1]);
                if constexpr (MX) *reinterpret_cast<uint4*>(static_cast<uint16_t*>(out) + at) = make_uint4(p[0], p[1], p[2], p[3]);
                else *reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(out) + at) = p[0];
            } else {
                float* o = static_cast<float*>(out) + at;
                if constexpr (MX) {
                    reinterpret_cast<float4*>(o)[0] = make_float4(v[0], v[1], v[2], v[3]);
                    reinterpret_cast<float4*>(o)[1] = make_float4(v[4], v[5], v[6], v[7]);
                } else
                    *reinterpret_cast<float2*>(o) = make_float2(v[0], v[1]);
            }
        } else {
#pragma unroll
            for (int e = 0; e < V; ++e)
                if (e < n) {
                    if (BF16) static_cast<uint16_t*>(out)[at + e] = (uint16_t)bf16x2_rne(v[e], 0.f);
                    else static_cast<float*>(out)[at + e] = v[e];
                }
        }
    }
}

// A warp per row and k-block of 256 values: eight blocks of 17 bytes; four lanes share a block, each with eight values.
__global__ void __launch_bounds__(THREADS) blocks_kernel(const uint8_t* blocks, int K, int kblocks, long long units, unsigned char* image) {
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

// CTA e: the expert's rows.  A thread looks at a run of consecutive ids, so that prefix sums over the threads keep the pairs' order.
constexpr int PLAN_THREADS = 512;
__global__ void __launch_bounds__(PLAN_THREADS) plan_kernel(const int32_t* __restrict__ ids, const Plan p) {
    __shared__ int hist[PLAN_EXPERTS], warp_sums[PLAN_THREADS / 32], first_s[2];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, e = blockIdx.x;
    for (int i = tid; i < p.experts; i += PLAN_THREADS) hist[i] = 0;
    __syncthreads();
    for (int i = tid; i < p.pairs; i += PLAN_THREADS) {
        const int id = __ldg(ids + i);
        if (id >= 0 && id < p.experts) atomicAdd(&hist[id], 1);  // counts: the same in any order
        else if (e == 0) p.place[i] = -1;
    }
    __syncthreads();
    if (warp == 0) {  // blocks in front of the expert, and of all experts
        int before = 0, all = 0;
        for (int i = lane; i < p.experts; i += 32) {
            const int b = (hist[i] + IMG_ROWS - 1) / IMG_ROWS;
            all += b;
            if (i < e) before += b;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            before += __shfl_xor_sync(0xffffffffu, before, o);
            all += __shfl_xor_sync(0xffffffffu, all, o);
        }
        if (lane == 0) {
            first_s[0] = before;
            first_s[1] = all;
            p.first[e] = before;
            p.count[e] = hist[e];
            if (e == 0) p.first[p.experts] = all;
        }
    }
    __syncthreads();
    const int row0 = first_s[0] * IMG_ROWS, n = hist[e];
    int base = 0;
    for (int c0 = 0; c0 < p.pairs && base < n; c0 += PLAN_THREADS) {
        const int i = c0 + tid;
        const bool mine = i < p.pairs && __ldg(ids + i) == e;
        const uint32_t votes = __ballot_sync(0xffffffffu, mine);
        if (lane == 0) warp_sums[warp] = __popc(votes);
        __syncthreads();
        int at = base;
#pragma unroll
        for (int w = 0; w < PLAN_THREADS / 32; ++w) {
            if (w < warp) at += warp_sums[w];
            base += warp_sums[w];
        }
        if (mine) {
            const int r = row0 + at + __popc(votes & ((1u << lane) - 1u));
            p.place[i] = r;
            p.row[r] = i;
        }
        __syncthreads();
    }
    // rows behind the expert's last, and behind the last expert's
    for (int r = row0 + n + tid; r < row0 + (n + IMG_ROWS - 1) / IMG_ROWS * IMG_ROWS; r += PLAN_THREADS) p.row[r] = -1;
    for (int r = first_s[1] * IMG_ROWS + e * PLAN_THREADS + tid; r < p.rows; r += p.experts * PLAN_THREADS) p.row[r] = -1;
}

template <bool RB, bool YB>
__global__ void __launch_bounds__(THREADS) sum_kernel(const SumArgs a, int v4) {
    const int t = blockIdx.y;
    const int per = v4 ? 4 : 1;
    const int i = (blockIdx.x * THREADS + threadIdx.x) * per;
    if (i >= a.W) return;
    float s[4] = {0.f, 0.f, 0.f, 0.f};
    const size_t at = (size_t)t * a.W + i;
    for (int j = 0; j < a.top; ++j) {
        const int id = __ldg(a.ids + (size_t)t * a.top + j);
        if (id < 0 || id >= a.experts) continue;
        const float w = __ldg(a.weights + (size_t)t * a.top + j);
        const size_t p = ((size_t)t * a.top + j) * a.W + i;
        if (v4) {
            float v[4];
            if (RB) {
                const uint2 u = __ldg(reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(a.rows) + p));
                v[0] = bf16_lo(u.x), v[1] = bf16_hi(u.x), v[2] = bf16_lo(u.y), v[3] = bf16_hi(u.y);
            } else {
                const float4 u = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(a.rows) + p));
                v[0] = u.x, v[1] = u.y, v[2] = u.z, v[3] = u.w;
            }
#pragma unroll
            for (int c = 0; c < 4; ++c) s[c] = fmaf(w, v[c], s[c]);
        } else
            s[0] = fmaf(w, load1(a.rows, RB, p), s[0]);
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

cudaError_t launch_image_pack(const PackArgs& a, bool mx, cudaStream_t st) {
    const int kblocks = img_kblocks(mx, a.K);
    const long long units = (long long)a.rows * kblocks;
    unsigned g;
    if (const cudaError_t e = grid_of(units, WARPS * PACK_UNITS, &g)) return e;
#define PACK(MX, B, G) pack_kernel<MX, B, G><<<g, THREADS, 0, st>>>(a, kblocks, units)
    if (mx) {
        if (a.bf16) a.glu ? PACK(true, true, true) : PACK(true, true, false);
        else a.glu ? PACK(true, false, true) : PACK(true, false, false);
    } else {
        if (a.bf16) a.glu ? PACK(false, true, true) : PACK(false, true, false);
        else a.glu ? PACK(false, false, true) : PACK(false, false, false);
    }
#undef PACK
    return cudaGetLastError();
}

cudaError_t launch_image_unpack(const unsigned char* image, bool mx, int rows, int K, void* out, bool bf16, size_t ld, cudaStream_t st) {
    const int kblocks = img_kblocks(mx, K);
    const long long units = (long long)rows * kblocks;
    unsigned g;
    if (const cudaError_t e = grid_of(units, WARPS * PACK_UNITS, &g)) return e;
#define UNPACK(MX, B) unpack_kernel<MX, B><<<g, THREADS, 0, st>>>(image, K, kblocks, units, out, ld)
    if (mx) bf16 ? UNPACK(true, true) : UNPACK(true, false);
    else bf16 ? UNPACK(false, true) : UNPACK(false, false);
#undef UNPACK
    return cudaGetLastError();
}

cudaError_t launch_image_blocks(const uint8_t* blocks, int rows, int K, unsigned char* image, cudaStream_t st) {
    const int kblocks = img_kblocks(true, K);
    const long long units = (long long)rows * kblocks;
    unsigned g;
    if (const cudaError_t e = grid_of(units, WARPS, &g)) return e;
    blocks_kernel<<<g, THREADS, 0, st>>>(blocks, K, kblocks, units, image);
    return cudaGetLastError();
}

cudaError_t launch_plan(const int32_t* ids, const Plan& p, cudaStream_t st) {
    plan_kernel<<<p.experts, PLAN_THREADS, 0, st>>>(ids, p);
    return cudaGetLastError();
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
    if (a.rows_bf16) a.y_bf16 ? sum_kernel<true, true><<<g, THREADS, 0, st>>>(a, v4) : sum_kernel<true, false><<<g, THREADS, 0, st>>>(a, v4);
    else a.y_bf16 ? sum_kernel<false, true><<<g, THREADS, 0, st>>>(a, v4) : sum_kernel<false, false><<<g, THREADS, 0, st>>>(a, v4);
    return cudaGetLastError();
}

}  // namespace hm

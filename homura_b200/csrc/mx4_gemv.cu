// Few rows times 4-bit weights: y[m][n] = sum_k x[m][k] w[n][k], x f32 or bf16 as they are, w the image of image.h, f32 sums.
//
// Bound by the weights' 17/32 bytes each, if a weight costs few enough instructions: the codes go to f16 by conversion (exactly) and are multiplied
// on mma.sync m16n8k16, whose eight columns are the rows of x; a block of 32 values is two MMAs into accumulators of their own, which the block's
// scale then joins to the sum in f32.  x enters as f16: 2^e x with the row's largest value in [2^14, 2^15), so that a channel that stands out leaves the others their
// bits.  bf16 is one term: exact down to 2^-31 of the row's largest, then to 2^-39 of it (half a subnormal step).  f32 is two, the second 2^12 times what the first
// leaves: 2^-22 of a value, 2^-51 of the row's largest (a third would bring two more bits, which a row's sum in f32 does not keep).  So a launch of up to eight bf16 or four f32 rows has one MMA column block, eight f32 rows have two.
//
//   * a CTA = 128 features (a tile of the image) x its k-blocks; a producer warp copies tiles of 17 KB into a ring, eight warps multiply: four groups of 32
//     features, two halves of a k-block.  The k order of an MMA is free as long as both operands agree: lane t of a group of four takes values
//     8 t .. 8 t + 7 of a block, one word of codes.
//   * tiles that are fewer than the SMs share their k-blocks among the CTAs of a cluster, summed in rank order through distributed shared memory; otherwise
//     a CTA walks several tiles and converts x once.
// Measured (graph replays): one f32 row 896 -> 9728 5.4 us (4.6 MB: launch, x and two cluster barriers), seven bf16 rows 1536 -> 151936 29.4 us (128 MB, 0.66 of the
// measured copy bandwidth): 6.0 TB/s while tiles flow, at 60 % of the issue slots, behind 5 us of launch and x; 1187 tiles leave three CTAs a fifth one.  Eight f32 rows
// of the same size 46.2 us: twice the MMAs, one CTA per SM.
#include <algorithm>

#include "image.h"
#include "launch_attrs.h"
#include "mbarrier.cuh"

namespace hm {
namespace {

constexpr int MMA_WARPS = 8, THREADS = 32 + MMA_WARPS * 32;
constexpr int MAX_SLOTS = 8, MAX_SPLIT = 8;
constexpr int PART_LD = 9;  // floats of a feature's partial sums (eight rows), odd: free of bank conflicts

struct Shared {
    uint64_t full[MAX_SLOTS], empty[MAX_SLOTS];
    volatile int abort_flag;
    uint32_t top[8];        // largest finite value of a row, as bits
};

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1, const float (&c)[4]) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}
// A load that stays where it is written.
__device__ __forceinline__ uint4 load_now(const void* p) {
    uint4 v;
    asm volatile("ld.global.nc.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
    return v;
}
constexpr int X_TOP = 14;          // a row's largest value is brought into [2^X_TOP, 2^(X_TOP + 1))
constexpr int SUM_DOWN = 7;        // block sums join the f32 sum 2^-SUM_DOWN times: scales up to 2^100 then stay below its largest value
constexpr float LOW_UP = 4096.f;   // what the first term of an f32 leaves enters that many times

// 2^(byte j of w - 127 - SUM_DOWN); 255 counts as infinite here.
__device__ __forceinline__ float scale_of(uint32_t w, int j) {
    const uint32_t s = (j == 3 ? w >> 1 : w << (23 - 8 * j)) & 0x7F800000u;
    return __uint_as_float(max(s, 0x00400000u)) * (1.f / (1 << SUM_DOWN));
}
__device__ __forceinline__ uint32_t f16x2_rn(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

// 2^e brings a row's largest value to its place (rows below 2^-112: as far as a factor of 2^126 goes); the sums are 2^back times the row's.
__device__ __forceinline__ int row_exponent(uint32_t top) { return min(127 + X_TOP - (int)(top >> 23), 126); }
__device__ __forceinline__ int row_back(uint32_t top) { return SUM_DOWN - row_exponent(top); }
__device__ __forceinline__ float row_factor(uint32_t top) { return __uint_as_float((uint32_t)(127 + row_back(top)) << 23); }

// Elements of a column of x in shared memory: the k-blocks of a CTA and half a line, so that neighbouring columns lie in different banks.
__host__ __device__ inline int x_ld(int kb_per) { return kb_per * MX_K + 32; }
inline size_t smem_bytes(int slots, int kb_per, int cols) { return 1024 + (size_t)slots * MX_TILE + (size_t)cols * x_ld(kb_per) * 2 + 4 * IMG_ROWS * PART_LD * 4; }

// NB: blocks of eight columns; TERMS: f16 terms of x; XU: k-blocks of a row of x in a warp's registers.  Column of row m, term i: m + 8 i where the rows fill a block, else TERMS m + i.
template <int NB, int TERMS, int XU>
__global__ void __launch_bounds__(THREADS, 2) mx4_gemv_kernel(const MxGemvArgs a) {
    extern __shared__ __align__(1024) unsigned char dsm[];
    __shared__ Shared sh;
    unsigned char* ring = dsm + ((1024u - (s32(dsm) & 1023u)) & 1023u);
    const int ldx = x_ld(a.kb_per);
    uint16_t* xs = reinterpret_cast<uint16_t*>(ring + (size_t)a.slots * MX_TILE);
    const int cols = a.M * TERMS;
    float* parts = reinterpret_cast<float*>(xs + (size_t)cols * ldx);  // [tiles in turn: 2][2 halves][128 features][PART_LD]
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    pdl_launch_dependents();
    pdl_wait();
    int expert = 0, xrow0 = 0;
    if (a.ids) {
        expert = __ldg(a.ids + blockIdx.y);
        if (expert < 0 || expert >= a.experts) return;  // the whole cluster
        xrow0 = blockIdx.y / a.top;
    }
    const int rank = blockIdx.x % a.split, step = gridDim.x / a.split;
    const int kb0 = rank * a.kb_per, kb1 = min(a.kblocks, kb0 + a.kb_per), nkb = kb1 - kb0;
    if (tid == 0) {
        for (int s = 0; s < a.slots; ++s) { mb_init(&sh.full[s], 1); mb_init(&sh.empty[s], MMA_WARPS); }
        sh.abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    if (warp == MMA_WARPS) {
        asm volatile("bar.sync 2, 288;" ::: "memory");  // x is asked for first: behind the ring's tiles it would arrive after them
        if (lane == 0) {
            const unsigned char* w = a.w + expert * a.w_stride;
            bool ok = true;
            uint32_t issued = 0;
            int s = -1;
            uint32_t parity = 1;  // of the slot's use before
            for (int t = blockIdx.x / a.split; t < a.tiles && ok; t += step)
                for (int kb = kb0; kb < kb1; ++kb, ++issued) {
                    if (++s == a.slots) { s = 0; parity ^= 1u; }
                    if (issued >= (uint32_t)a.slots) ok = mb_wait(&sh.empty[s], parity, a.err_flag, &sh.abort_flag);
                    if (!ok) break;
                    mb_expect_tx(&sh.full[s], MX_TILE);
                    bulk_copy(ring + (size_t)s * MX_TILE, w + ((size_t)t * a.kblocks + kb) * MX_TILE, MX_TILE, &sh.full[s]);
                }
            mb_land_ring(sh.full, issued, (uint32_t)a.slots);  // always: a wait of the others may run out after this thread's last look at the flag
        }
    } else {
        // A warp takes a row of x: its largest finite value, then f16 terms.  Up to XU k-blocks (eight values of each per lane) are loaded once.
        constexpr bool B = TERMS == 1;
        constexpr int NW = B ? 1 : 2;
        const int k0 = kb0 * MX_K, m = warp;
        const size_t es = B ? 2 : 4;
        const char* row = static_cast<const char*>(a.x) + ((size_t)(xrow0 + m) * a.ldx + k0) * es;
        const bool aligned = ((uintptr_t)row & 15) == 0;
        uint4 w[XU][NW];
        auto fetch = [&](int b0) {
#pragma unroll
            for (int u = 0; u < XU; ++u) {
                const int k = (b0 + u) * MX_K + lane * 8;
                if (b0 + u >= nkb) break;
                if (aligned && k0 + k + 8 <= a.K) {
#pragma unroll
                    for (int e = 0; e < NW; ++e) w[u][e] = load_now(row + k * es + 16 * e);
                } else
                    load_ragged<8, B>(row, k, a.K - k0, w[u]);
            }
        };
        if (m < a.M) fetch(0);
        asm volatile("bar.arrive 2, 288;" ::: "memory");
        if (m < a.M) {
            float most = 0.f;
            for (int b0 = 0; b0 < nkb; b0 += XU) {
                if (b0) fetch(b0);
#pragma unroll
                for (int u = 0; u < XU; ++u) {
                    if (b0 + u >= nkb) break;
                    float v[8];
                    widen<8, B>(w[u], v);
#pragma unroll
                    for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf(v[e]));  // (leaves NaNs out)
                }
            }
            uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(most));
            if (top == 0x7F800000u) {  // without the infinities
                top = 0;
                for (int k = lane; k < min(a.K - k0, nkb * MX_K); k += 32) {
                    const uint32_t b = (B ? (uint32_t)__ldg(reinterpret_cast<const uint16_t*>(row) + k) << 16 : __ldg(reinterpret_cast<const uint32_t*>(row) + k)) & 0x7FFFFFFFu;
                    if (b < 0x7F800000u) top = max(top, b);
                }
                top = __reduce_max_sync(0xffffffffu, top);
            }
            if (lane == 0) sh.top[m] = top;
            const float up = __uint_as_float((uint32_t)(row_exponent(top) + 127) << 23);
            uint16_t* to = xs + (size_t)(NB == 2 ? m : TERMS * m) * ldx + lane * 8;
            for (int b0 = 0; b0 < nkb; b0 += XU) {
                if (nkb > XU) fetch(b0);
#pragma unroll
                for (int u = 0; u < XU; ++u) {
                    if (b0 + u >= nkb) break;
                    float v[8];
                    widen<8, B>(w[u], v);
                    uint32_t h[4], l[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float p = v[2 * e] * up, q = v[2 * e + 1] * up;
                        h[e] = f16x2_rn(p, q);
                        if (TERMS == 2) {  // what the first term leaves; nothing of an infinity
                            const float rp = p - f16_bits_to_f32((uint16_t)h[e]), rq = q - f16_bits_to_f32((uint16_t)(h[e] >> 16));
                            l[e] = f16x2_rn(fabsf(p) < __int_as_float(0x7F800000) ? rp * LOW_UP : 0.f, fabsf(q) < __int_as_float(0x7F800000) ? rq * LOW_UP : 0.f);
                        }
                    }
                    *reinterpret_cast<uint4*>(to + (b0 + u) * MX_K) = make_uint4(h[0], h[1], h[2], h[3]);
                    if (TERMS == 2) *reinterpret_cast<uint4*>(to + (b0 + u) * MX_K + (size_t)(NB == 2 ? a.M : 1) * ldx) = make_uint4(l[0], l[1], l[2], l[3]);
                }
            }
        }
        asm volatile("bar.sync 1, 256;" ::: "memory");
    }
    __syncwarp();
    const int fg = warp & 3, kh = (warp >> 2) & 1, g = lane >> 2, tl = lane & 3;
    int s = -1;
    uint32_t parity = 0;
    for (int t = blockIdx.x / a.split, turn = 0; t < a.tiles; t += step, turn ^= 1) {
        float* part = parts + (size_t)turn * 2 * IMG_ROWS * PART_LD;
        if (warp < MMA_WARPS) {
            float sum[2][NB][4];
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int e = 0; e < 4; ++e) sum[i][b][e] = 0.f;
            for (int kb = 0; kb < nkb; ++kb) {
                if (++s == a.slots) { s = 0; parity ^= 1u; }
                if (!__all_sync(0xffffffffu, mb_wait(&sh.full[s], parity, a.err_flag, &sh.abort_flag))) continue;
                const unsigned char* tile = ring + (size_t)s * MX_TILE;
                const uint32_t* sc = reinterpret_cast<const uint32_t*>(tile + kh * 512 + fg * 4);
                uint32_t scales[4];  // of features g, g + 8, g + 16, g + 24 of the group: a byte per block of this half
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    scales[i] = sc[(g + 8 * i) * 4];
                    if (__vcmpeq4(scales[i], 0xFFFFFFFFu))  // a block that is no number
#pragma unroll
                        for (int b = 0; b < NB; ++b) sum[i >> 1][b][2 * (i & 1)] = sum[i >> 1][b][2 * (i & 1) + 1] = __int_as_float(0x7FC00000);
                }
                const unsigned char* codes = tile + MX_SCALES + (fg * 32 + g) * 128 + tl * 4;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    uint4 xv[NB];
#pragma unroll
                    for (int b = 0; b < NB; ++b) {
                        const int col = NB == 2 ? b * a.M + min(g, a.M - 1) : min(g, cols - 1);  // columns that do not exist repeat the last
                        xv[b] = *reinterpret_cast<const uint4*>(xs + (size_t)col * ldx + kb * MX_K + (kh * 4 + j) * 32 + tl * 8);
                    }
#pragma unroll
                    for (int i = 0; i < 2; ++i) {  // features 16 i + g and 16 i + g + 8
                        uint32_t lo[4], hi[4];
                        const int piece = ((kh * 4 + j) ^ g) << 4;
                        mx_halves(*reinterpret_cast<const uint32_t*>(codes + i * 16 * 128 + piece), lo);
                        mx_halves(*reinterpret_cast<const uint32_t*>(codes + (i * 16 + 8) * 128 + piece), hi);
                        const float s0 = scale_of(scales[2 * i], j), s1 = scale_of(scales[2 * i + 1], j);
#pragma unroll
                        for (int b = 0; b < NB; ++b) {
                            const float zero[4] = {0.f, 0.f, 0.f, 0.f};
                            float c[4], d[4];
                            mma_f16(c, lo[0], hi[0], lo[1], hi[1], xv[b].x, xv[b].y, zero);
                            mma_f16(d, lo[2], hi[2], lo[3], hi[3], xv[b].z, xv[b].w, c);
                            sum[i][b][0] = fmaf(s0, d[0], sum[i][b][0]);
                            sum[i][b][1] = fmaf(s0, d[1], sum[i][b][1]);
                            sum[i][b][2] = fmaf(s1, d[2], sum[i][b][2]);
                            sum[i][b][3] = fmaf(s1, d[3], sum[i][b][3]);
                        }
                    }
                }
                __syncwarp();
                if (lane == 0) mb_arrive(&sh.empty[s]);
            }
            // terms of a row come together: in neighbouring columns of a lane, or in the same column of two blocks
            float* p = part + (size_t)kh * IMG_ROWS * PART_LD;
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float* q = p + (fg * 32 + i * 16 + h * 8 + g) * PART_LD;
                    if (NB == 2) {
                        q[2 * tl] = fmaf(sum[i][NB - 1][2 * h], 1.f / LOW_UP, sum[i][0][2 * h]);
                        q[2 * tl + 1] = fmaf(sum[i][NB - 1][2 * h + 1], 1.f / LOW_UP, sum[i][0][2 * h + 1]);
                    } else if (TERMS == 2) {
                        q[tl] = fmaf(sum[i][0][2 * h + 1], 1.f / LOW_UP, sum[i][0][2 * h]);
                    } else {
                        q[2 * tl] = sum[i][0][2 * h];
                        q[2 * tl + 1] = sum[i][0][2 * h + 1];
                    }
                }
            if (a.split == 1) asm volatile("bar.sync 1, 256;" ::: "memory");
        }
        if (a.split > 1) cluster_sync_all();  // one tile per cluster
        // thread: a feature and every second row (of those that fall to this CTA of a cluster)
        const int f = tid & 127, n = t * IMG_ROWS + f;
        if (warp < MMA_WARPS && n < a.N) {
            auto store = [&](int m, float v) {
                const size_t at = (a.ids ? blockIdx.y : m) * a.ldy + n;
                if (a.y_bf16) static_cast<uint16_t*>(a.y)[at] = (uint16_t)bf16x2_rne(v, 0.f);
                else static_cast<float*>(a.y)[at] = v;
            };
            const float* p = part + f * PART_LD;
            if (a.split == 1) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int m = 2 * i + (tid >> 7);
                    if (m < a.M) store(m, (p[m] + p[IMG_ROWS * PART_LD + m]) * row_factor(sh.top[m]));
                }
            } else {
                for (int m = rank + (tid >> 7) * a.split; m < a.M; m += 2 * a.split) {
                    // The CTAs scale their own part of a row: each brings its sum back before they are added, in 64 bits, where parts beyond the largest f32 of
                    // different signs still meet.
                    float q[MAX_SPLIT];
                    uint32_t top[MAX_SPLIT];
#pragma unroll
                    for (int r = 0; r < MAX_SPLIT; ++r)
                        if (r < a.split) {
                            q[r] = ld_dsmem_f32(dsmem_addr(p + m, r)) + ld_dsmem_f32(dsmem_addr(p + IMG_ROWS * PART_LD + m, r));
                            top[r] = __float_as_uint(ld_dsmem_f32(dsmem_addr(&sh.top[m], r)));
                        }
                    double v = 0.0;
#pragma unroll
                    for (int r = 0; r < MAX_SPLIT; ++r)
                        if (r < a.split) v += (double)q[r] * __hiloint2double((1023 + row_back(top[r])) << 20, 0);
                    store(m, (float)v);
                }
            }
        }
        if (a.split > 1) {
            cluster_sync_all();  // nobody ends while others read its sums
            break;
        }
    }
}

template <int NB, int TERMS>
cudaError_t launch(MxGemvArgs& a, int sm_count, cudaStream_t st) {
    constexpr size_t HALF = 112 * 1024, MOST = 225 * 1024;  // two CTAs of up to HALF share an SM
    const int cols = a.M * TERMS, rows = a.ids ? a.pairs : 1;
    a.split = 1;
    // Few tiles share their k-blocks among the CTAs of a cluster; so do rows too long for the shared memory of one.
    const long long ctas = (long long)a.tiles * rows;
    if (ctas * 2 <= 2 * sm_count) a.split = (int)std::min<long long>({2 * sm_count / ctas, (long long)MAX_SPLIT, (long long)a.kblocks});
    a.kb_per = (a.kblocks + a.split - 1) / a.split;
    while (a.split < MAX_SPLIT && smem_bytes(3, a.kb_per, cols) > MOST) {
        ++a.split;
        a.kb_per = (a.kblocks + a.split - 1) / a.split;
    }
    a.split = (a.kblocks + a.kb_per - 1) / a.kb_per;
    a.slots = MAX_SLOTS;
    if (a.split > 1) a.slots = std::min(a.slots, a.kb_per);
    const size_t limit = smem_bytes(3, a.kb_per, cols) <= HALF ? HALF : MOST;
    while (a.slots > 1 && smem_bytes(a.slots, a.kb_per, cols) > limit) --a.slots;
    const size_t smem = smem_bytes(a.slots, a.kb_per, cols);
    void (*const fn)(MxGemvArgs) = a.kb_per <= 2 ? mx4_gemv_kernel<NB, TERMS, 2> : mx4_gemv_kernel<NB, TERMS, 6>;
    cudaError_t e = ensure_dyn_smem(fn, smem);
    if (e != cudaSuccess) return e;
    const int per_sm = smem <= HALF ? 2 : 1;
    const dim3 grid(a.split > 1 || a.ids ? (unsigned)a.tiles * a.split : (unsigned)std::min(a.tiles, per_sm * sm_count), rows);
    return launch_after(fn, grid, THREADS, smem, a.split, st, a);
}

}  // namespace

cudaError_t launch_mx4_gemv(MxGemvArgs a, int sm_count, cudaStream_t st) {
    a.kblocks = img_kblocks(true, a.K);
    a.tiles = (a.N + IMG_ROWS - 1) / IMG_ROWS;
    if (a.bf16) return launch<1, 1>(a, sm_count, st);
    return a.M <= 4 ? launch<1, 2>(a, sm_count, st) : launch<2, 2>(a, sm_count, st);
}

}  // namespace hm

// Products of two operand images on the 5th-generation tensor cores: y[m][n] = sum_k x[m][k] w[n][k], 4-bit microscaled floats on both sides
// (tcgen05.mma kind::mxf4.block_scale, scales in tensor memory) or bf16 (kind::f16); f32 sums.  One group of rows, or groups of rows by
// expert, each with weights of its own (image.h, Plan).
//
//   * a unit = 128 features (the MMA's M: weights are its first operand) x up to 192 rows (its N, cut to the rows that exist), so that small groups
//     of rows cost what they are and an epilogue thread owns one feature: 32 neighbouring features of a row leave as one line without a transposition.
//   * one CTA per SM walks its units (persistent, static round robin): a warp copies k-blocks of 128 bytes per row into a ring of five slots, one issues
//     MMAs, eight read accumulators.  Two accumulators of 192 columns alternate; the scales of a slot have 24 columns of the tensor memory of their
//     own, so that nothing overwrites scales that an MMA still reads (5 * 24 + 384 = 504 of 512 columns).
//   * the tensor core truncates when it adds to an accumulator; accumulators cover CHUNK k-blocks (32 additions) and are summed in registers to nearest.
//   * units that are fewer than the SMs share their k-blocks among the CTAs of a cluster, whose partial tiles are summed in the order of their ranks
//     through distributed shared memory: no scratch outlives the launch.
#include "image.h"

#include <algorithm>

#include "launch_attrs.h"
#include "mbarrier.cuh"

namespace hm {
namespace {

constexpr int TN = 192;                      // rows of a unit at most
constexpr int CHUNK = 8;                     // k-blocks per accumulator
constexpr int SLOTS = 5;
constexpr int EPI_WARPS = 8, THREADS = 64 + EPI_WARPS * 32;
constexpr int A_SLOT = MX_TILE;              // scales (bf16: unused), 128 features
constexpr int B_SLOT = 2 * MX_SCALES + TN * 128;
constexpr int SLOT = A_SLOT + B_SLOT;
constexpr size_t SMEM = (size_t)SLOTS * SLOT + 1024;
constexpr int SF_COLS = 24, SF_BASE = 2 * TN;
constexpr int MAX_SPLIT = 16;
static_assert(SF_BASE + SLOTS * SF_COLS <= 512, "tensor memory");
static_assert(TN * IMG_ROWS * 4 <= SLOTS * SLOT, "partial tile");

__device__ __forceinline__ uint64_t desc_sw128(uint32_t smem_addr) {
    return (uint64_t)((smem_addr >> 4) & 0x3FFF) | (uint64_t)1 << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
// 32 rows of 16 bytes, eight rows of 128 bytes in a row, no swizzle
__device__ __forceinline__ uint64_t desc_scales(uint32_t smem_addr) { return (uint64_t)((smem_addr >> 4) & 0x3FFF) | (uint64_t)1 << 16 | (uint64_t)(128 >> 4) << 32 | (uint64_t)1 << 46; }
__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile("{ .reg .pred p; setp.ne.b32 p, %4, 0;\n"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p; }" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc) : "memory");
}
__device__ __forceinline__ void mma_mxf4(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sa, uint32_t sb, uint32_t acc) {
    asm volatile("{ .reg .pred p; setp.ne.b32 p, %6, 0;\n"
                 "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p; }" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(acc) : "memory");
}
__device__ __forceinline__ void copy_scales(uint32_t taddr, uint32_t smem_addr) {
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc_scales(smem_addr)) : "memory");
}
__device__ __forceinline__ void mma_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(s32(bar)) : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t (&r)[16], uint32_t addr) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(addr));
}
// Names the registers, so that no use of them moves in front of the wait.
__device__ __forceinline__ void tmem_wait(uint32_t (&r)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
                 :: "memory");
}

struct Shared {
    uint64_t full[SLOTS], empty[SLOTS], afull[2], aempty[2], done;
    uint32_t tmem;
    volatile int abort_flag;
    int units;
};

struct Unit {
    int expert, tile, row0, n;  // features tile * 128 ..; image rows row0 .. row0 + n
};
// Units of an expert: its rows fastest, so that units that run at the same time share weights.
__device__ __forceinline__ Unit unit_at(const ImageGemmArgs& a, const int* ufirst, int u) {
    Unit r;
    int rows = a.M, base = 0;
    r.expert = 0;
    if (a.first) {
        int lo = 0, hi = a.experts;  // the last expert whose first unit is at most u
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (ufirst[mid] <= u) lo = mid;
            else hi = mid;
        }
        r.expert = lo;
        u -= ufirst[lo];
        rows = __ldg(a.count + lo);
        base = __ldg(a.first + lo) * IMG_ROWS;
    }
    const int per = (rows + TN - 1) / TN, t = u % per;
    r.tile = u / per;
    r.row0 = base + t * TN;
    r.n = min(TN, rows - t * TN);
    return r;
}

__device__ __forceinline__ void store1(const ImageGemmArgs& a, int row, int f, float v) {
    if (a.bf16) static_cast<uint16_t*>(a.y)[(size_t)row * a.ldy + f] = (uint16_t)bf16x2_rne(v, 0.f);
    else static_cast<float*>(a.y)[(size_t)row * a.ldy + f] = v;
}
// A warp's 32 features (lane: one) of two rows (-1: none).  bf16: neighbouring lanes swap, so that each stores two features of one row.
__device__ __forceinline__ void store2(const ImageGemmArgs& a, int r0, int r1, int f, int lane, float v0, float v1) {
    if (!a.bf16 || !a.wide) {
        if (f < a.N && r0 >= 0) store1(a, r0, f, v0);
        if (f < a.N && r1 >= 0) store1(a, r1, f, v1);
        return;
    }
    const float got = __shfl_xor_sync(0xffffffffu, lane & 1 ? v0 : v1, 1);
    const int row = lane & 1 ? r1 : r0, g = f & ~1;
    if (row < 0 || g >= a.N) return;
    const uint32_t w = lane & 1 ? bf16x2_rne(got, v1) : bf16x2_rne(v0, got);
    uint16_t* y = static_cast<uint16_t*>(a.y) + (size_t)row * a.ldy + g;
    if (g + 1 < a.N) *reinterpret_cast<uint32_t*>(y) = w;
    else *y = (uint16_t)w;
}

template <bool MX>
__global__ void __launch_bounds__(THREADS, 1) image_gemm_kernel(const ImageGemmArgs a) {
    extern __shared__ __align__(1024) unsigned char dsm[];
    __shared__ Shared sh;
    __shared__ int ufirst[PLAN_EXPERTS];
    unsigned char* ring = dsm + ((1024u - (s32(dsm) & 1023u)) & 1023u);  // swizzle atoms need 1024-byte alignment
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        for (int s = 0; s < SLOTS; ++s) { mb_init(&sh.full[s], 1); mb_init(&sh.empty[s], 1); }
        for (int s = 0; s < 2; ++s) { mb_init(&sh.afull[s], 1); mb_init(&sh.aempty[s], EPI_WARPS); }
        mb_init(&sh.done, 1);
        sh.abort_flag = 0;
        if (!a.first) sh.units = (a.M + TN - 1) / TN * a.tiles;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(s32(&sh.tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (warp == 2 && a.first) {  // first unit of every expert
        int sum = 0;
        for (int i0 = 0; i0 < a.experts; i0 += 32) {
            const int i = i0 + lane;
            const int n = i < a.experts ? (__ldg(a.count + i) + TN - 1) / TN * a.tiles : 0;
            int inc = n;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int t = __shfl_up_sync(0xffffffffu, inc, o);
                if (lane >= o) inc += t;
            }
            if (i < a.experts) ufirst[i] = sum + inc - n;
            sum += __shfl_sync(0xffffffffu, inc, 31);
        }
        if (lane == 0) sh.units = sum;
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = sh.tmem;
    const int units = sh.units;
    const int rank = blockIdx.x % a.split, step = gridDim.x / a.split, u0 = blockIdx.x / a.split;
    const int kb0 = rank * a.kb_per, kb1 = min(a.kblocks, kb0 + a.kb_per);
    constexpr int TILE = MX ? MX_TILE : IMG_CODES;

    uint32_t issued = 0;
    if (warp == 0) {
        if (lane == 0) {
            bool ok = true;
            for (int u = u0; u < units && ok; u += step) {
                const Unit t = unit_at(a, ufirst, u);
                const unsigned char* w = a.w + t.expert * a.w_stride + (size_t)t.tile * a.kblocks * TILE;
                const unsigned char* x = a.x + (size_t)(t.row0 / IMG_ROWS) * a.kblocks * TILE;
                const size_t x_next = (size_t)a.kblocks * TILE;
                const int off = t.row0 % IMG_ROWS, n0 = min(t.n, IMG_ROWS - off), n1 = t.n - n0;  // rows in the first and in the second block
                const uint32_t b0 = (uint32_t)(n0 + 7) / 8 * 1024, b1 = (uint32_t)(n1 + 7) / 8 * 1024;
                const uint32_t bytes = (uint32_t)TILE + b0 + b1 + (MX ? (n1 > 0 ? 2u : 1u) * MX_SCALES : 0u);
                for (int kb = kb0; kb < kb1; ++kb, ++issued) {
                    const uint32_t s = issued % SLOTS;
                    if (issued >= SLOTS) ok = mb_wait(&sh.empty[s], ((issued / SLOTS) & 1u) ^ 1u, a.err_flag, &sh.abort_flag);
                    if (!ok) break;
                    unsigned char *sa = ring + (size_t)s * SLOT, *sb = sa + A_SLOT;
                    const unsigned char *wk = w + (size_t)kb * TILE, *xk = x + (size_t)kb * TILE;
                    mb_expect_tx(&sh.full[s], bytes);
                    bulk_copy(sa + (MX ? 0 : MX_SCALES), wk, TILE, &sh.full[s]);
                    if (MX) {
                        bulk_copy(sb, xk, MX_SCALES, &sh.full[s]);
                        if (n1 > 0) bulk_copy(sb + MX_SCALES, xk + x_next, MX_SCALES, &sh.full[s]);
                        xk += MX_SCALES;
                    }
                    bulk_copy(sb + 2 * MX_SCALES, xk + off * 128, b0, &sh.full[s]);
                    if (n1 > 0) bulk_copy(sb + 2 * MX_SCALES + n0 * 128, xk + x_next, b1, &sh.full[s]);
                }
            }
        }
    } else if (warp == 1) {
        if (lane == 0) {
            uint32_t i = 0, ci = 0;
            bool ok = true;
            for (int u = u0; u < units && ok; u += step) {
                const Unit t = unit_at(a, ufirst, u);
                const uint32_t n = (uint32_t)(t.n + 15) & ~15u, sf_off = (uint32_t)(t.row0 % IMG_ROWS) / 32;
                // D f32, both operands K-major, M 128, N n; bf16, or e2m1 with e8m0 scales
                const uint32_t idesc = MX ? 1u << 7 | 1u << 10 | (n >> 3) << 17 | 1u << 23 | (128u >> 4) << 24 : 1u << 4 | 1u << 7 | 1u << 10 | (n >> 3) << 17 | (128u >> 4) << 24;
                for (int kc = kb0; kc < kb1 && ok; kc += CHUNK, ++ci) {
                    const uint32_t buf = ci & 1u, d = tmem + buf * TN;
                    if (ci >= 2) ok = mb_wait(&sh.aempty[buf], ((ci >> 1) & 1u) ^ 1u, a.err_flag, &sh.abort_flag);
                    uint32_t more = 0;
                    for (int kb = kc; kb < min(kb1, kc + CHUNK) && ok; ++kb, ++i) {
                        const uint32_t s = i % SLOTS;
                        ok = mb_wait(&sh.full[s], (i / SLOTS) & 1u, a.err_flag, &sh.abort_flag);
                        if (!ok) break;
                        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                        const uint32_t sa = s32(ring + (size_t)s * SLOT), sb = sa + A_SLOT, wa = sa + MX_SCALES, xa = sb + 2 * MX_SCALES;
                        if (MX) {
                            const uint32_t fa = tmem + SF_BASE + s * SF_COLS, fb = fa + 8;
#pragma unroll
                            for (uint32_t h = 0; h < 2; ++h) {
                                copy_scales(fa + 4 * h, sa + 512 * h);
                                copy_scales(fb + 8 * h, sb + 512 * h);
                                copy_scales(fb + 8 * h + 4, sb + MX_SCALES + 512 * h);  // (not loaded where the unit ends in its first block: then nobody reads it)
                            }
#pragma unroll
                            for (uint32_t j = 0; j < 4; ++j) {
                                const uint32_t id = (j & 1) * 2;
                                mma_mxf4(d, desc_sw128(wa + j * 32), desc_sw128(xa + j * 32), idesc | id << 4 | id << 29, fa + 4 * (j >> 1), fb + 8 * (j >> 1) + sf_off, more);
                                more = 1;
                            }
                        } else {
#pragma unroll
                            for (uint32_t j = 0; j < 4; ++j) {
                                mma_f16(d, desc_sw128(wa + j * 32), desc_sw128(xa + j * 32), idesc, more);
                                more = 1;
                            }
                        }
                        mma_commit(&sh.empty[s]);
                    }
                    if (ok) mma_commit(&sh.afull[buf]);
                }
            }
        }
    } else {
        const int quarter = warp & 3, half = (warp - 2) >> 2;  // a warp reads its own quarter of the TMEM lanes; chunks of 16 rows alternate
        const uint32_t tbase = tmem + ((uint32_t)(quarter * 32) << 16);
        uint32_t ci = 0;
        float acc[TN / 2];
        for (int u = u0; u < units; u += step) {
            const Unit t = unit_at(a, ufirst, u);
            const int f = t.tile * IMG_ROWS + quarter * 32 + lane;
#pragma unroll
            for (int j = 0; j < TN / 2; ++j) acc[j] = 0.f;
            for (int kc = kb0; kc < kb1; kc += CHUNK, ++ci) {
                const uint32_t buf = ci & 1u;
                if (!__all_sync(0xffffffffu, mb_wait(&sh.afull[buf], (ci >> 1) & 1u, a.err_flag, &sh.abort_flag))) continue;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
                for (int c = 0; c < TN / 32; ++c) {
                    const int col = (2 * c + half) * 16;
                    if (col < t.n) {
                        uint32_t r[16];
                        tmem_ld16(r, tbase + buf * TN + col);
                        tmem_wait(r);
#pragma unroll
                        for (int j = 0; j < 16; ++j) acc[c * 16 + j] += __uint_as_float(r[j]);
                    }
                }
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) mb_arrive(&sh.aempty[buf]);
            }
            if (a.split > 1) {  // one unit per cluster: the ring is read, the partial tile [rows][128 features] takes its place
                float* part = reinterpret_cast<float*>(ring);
#pragma unroll
                for (int c = 0; c < TN / 32; ++c)
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        const int col = (2 * c + half) * 16 + j;
                        if (col < t.n) part[col * IMG_ROWS + quarter * 32 + lane] = acc[c * 16 + j];
                    }
                break;
            }
#pragma unroll
            for (int c = 0; c < TN / 32; ++c) {
                const int col = (2 * c + half) * 16;
                if (col < t.n) {
                    int row = -1;  // where row col + lane of the unit goes
                    if (lane < 16 && col + lane < t.n) row = a.row ? __ldg(a.row + t.row0 + col + lane) : t.row0 + col + lane;
#pragma unroll
                    for (int j = 0; j < 16; j += 2)
                        store2(a, __shfl_sync(0xffffffffu, row, j), __shfl_sync(0xffffffffu, row, j + 1), f, lane, acc[c * 16 + j], acc[c * 16 + j + 1]);
                }
            }
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (sh.abort_flag) {  // a wait ran out: the copies and MMAs in flight end before the CTA does and its accumulators are freed
        if (tid == 0) mb_land_ring(sh.full, issued, SLOTS);
        else if (tid == 32) {
            mma_commit(&sh.done);
            mb_land(&sh.done, 0);
        }
        __syncthreads();
    }
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    if (a.split > 1) {
        cluster_sync_all();
        const Unit t = unit_at(a, ufirst, u0);
        const float* part = reinterpret_cast<const float*>(ring);
        // a warp per row of 128 features; the ranks share the rows
        for (int col = rank * (THREADS / 32) + warp; col < t.n; col += a.split * (THREADS / 32)) {
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int r = 0; r < a.split; ++r) {
                const float4 p = ld_dsmem_f32x4(dsmem_addr(part + col * IMG_ROWS + lane * 4, r));
                v = make_float4(v.x + p.x, v.y + p.y, v.z + p.z, v.w + p.w);
            }
            const int row = a.row ? __ldg(a.row + t.row0 + col) : t.row0 + col, f = t.tile * IMG_ROWS + lane * 4;
            const float o[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (f + e < a.N) store1(a, row, f + e, o[e]);
        }
        cluster_sync_all();  // nobody ends while others read its tile
    }
}

}  // namespace

cudaError_t launch_image_gemm(ImageGemmArgs a, bool mx, int sm_count, cudaStream_t st) {
    a.kblocks = img_kblocks(mx, a.K);
    a.tiles = (a.N + IMG_ROWS - 1) / IMG_ROWS;
    a.wide = a.ldy % 2 == 0 && (uintptr_t)a.y % 4 == 0;
    const void* fn = mx ? reinterpret_cast<const void*>(image_gemm_kernel<true>) : reinterpret_cast<const void*>(image_gemm_kernel<false>);
    cudaError_t e = ensure_dyn_smem(fn, SMEM);
    if (e != cudaSuccess) return e;
    long long units;
    a.split = 1;
    if (a.first) {
        units = (long long)(a.pairs / TN + std::min(a.pairs, a.experts)) * a.tiles;  // at most
    } else {
        units = (long long)((a.M + TN - 1) / TN) * a.tiles;
        // Fewer units than half the SMs: their k-blocks are shared out, two at least for a CTA.
        if (units * 2 <= sm_count) a.split = (int)std::min<long long>(std::min(sm_count / units, (long long)MAX_SPLIT), (a.kblocks + 1) / 2);
    }
    if (units > 0x7FFFFFFF) return cudaErrorInvalidValue;
    if (a.split > 8 && (e = ensure_nonportable_clusters(fn)) != cudaSuccess) return e;
    a.kb_per = (a.kblocks + a.split - 1) / a.split;
    a.split = (a.kblocks + a.kb_per - 1) / a.kb_per;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(a.split > 1 ? (unsigned)units * a.split : (unsigned)std::min<long long>(units, sm_count));
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = SMEM;
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    if (a.split > 1) {
        at[0].id = cudaLaunchAttributeClusterDimension;
        at[0].val.clusterDim = {(unsigned)a.split, 1, 1};
        cfg.attrs = at;
        cfg.numAttrs = 1;
    }
    return mx ? cudaLaunchKernelEx(&cfg, image_gemm_kernel<true>, a) : cudaLaunchKernelEx(&cfg, image_gemm_kernel<false>, a);
}

}  // namespace hm

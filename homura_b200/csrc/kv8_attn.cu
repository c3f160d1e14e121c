// Softmax attention over the 8-bit paged cache:
//   out[row, head] = sum over the positions t <= row_pos whose page exists of softmax_t(scale q . k_t) v_t,   zeros where there is no such position.
// Page i of a row is shared[i] for i < n_shared and its sequence's page table entry behind them.
//
// kv8_stream_kernel   rows' contexts, eight (row, head) pairs of one key/value head at a time; bound by the bytes of the cache
// kv8_join_kernel     joins the parts of contexts that several CTAs share
//
// Arithmetic of the first.  A warp takes 32 tokens of a page for eight pairs on m16n8k16 MMAs of f16 with f32 sums:
//   scores [16 x 8 tokens] = Q [16 x dim] . K^T,   out [16 x 8 elements] = W [16 x 16 tokens] . V
// Codes are whole numbers below 128 and so exact in f16: a byte becomes the last bits of 1024 + byte (one permutation for two of them), from which 1152 is
// subtracted.  Rows 0 .. 7 of Q are the pairs' queries times a power of two and rounded, rows 8 .. 15 what that leaves (together 2^-22 of a value): the tile's
// two halves are added up after the product.  A token's key scale joins behind the product, its value scale goes into the weight, W = 2^(s - max) * scale, which
// enters the same way in two terms, times a power of two that follows the pair's largest W (granules of 2^-38 of it).  So the cache's values are used as they are,
// and results are f32 products but for 2^-22.  A step's 32 tokens have accumulators of their own, added up in f32 outside: tensor core sums are truncated.
//
// Work.  The pages of all rows, heads and tiles of eight pairs stand in one line, which the CTAs cut into equal lengths: contexts of any lengths keep all SMs
// busy to the end, and no length needs to be known on the host.  A CTA writes what it has as a whole and leaves the rest (its first and its last item) in `work`.
#include "kv8.h"

#include <cuda_fp16.h>

#include <algorithm>

#include "launch_attrs.h"
#include "mbarrier.cuh"
#include "rows.cuh"

namespace hm {
namespace {

constexpr int WARPS = 8, THREADS = WARPS * 32 + 32;
constexpr int PAIRS = 8;       // of an item
constexpr int TURN = WARPS / 2;    // pages that the warps take at once, two warps a page.  The stages are a multiple of it: a stage is always the same two warps', so
constexpr int MAX_STAGES = 12;     // that nobody waits for a stage's next page while the one in front of it is still on its way
constexpr size_t ROOM = 224 * 1024;  // shared memory of an SM for CTAs of this kernel, what they hold outside the dynamic part taken off
constexpr int LEAST_PAGES = TURN;  // of a CTA: fewer would only leave more to be joined
constexpr float LOG2E = 1.4426950408889634f;

// ---- the line of pages ------------------------------------------------------------------------------
struct Line {
    long long total, chunk;  // pages of all items; of a CTA
};

__device__ __forceinline__ int row_len(const Kv8AttnArgs& a, int m) {
    const int seq = __ldg(a.row_seq + m);
    return (unsigned)seq < (unsigned)a.pool.n_seq ? min(__ldg(a.row_pos + m), a.pool.max_pages * KV8_PAGE - 1) + 1 : 0;
}
__device__ __forceinline__ int row_pages(const Kv8AttnArgs& a, int m) { return max(0, (row_len(a, m) + KV8_PAGE - 1) / KV8_PAGE); }

// first[m]: pages of the rows in front of row m, first[M]: of all.  Every thread of the CTA takes part; ends with a barrier.
__device__ __forceinline__ Line make_line(const Kv8AttnArgs& a, int items, int ctas, int* first) {
    __shared__ int s_sum[THREADS / 32], s_most;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, per = (a.M + THREADS - 1) / THREADS, m0 = min(a.M, tid * per), m1 = min(a.M, m0 + per);
    if (tid == 0) s_most = 0;
    int sum = 0, most = 0;
    for (int m = m0; m < m1; ++m) {
        const int n = row_pages(a, m);
        first[m] = sum;
        sum += n;
        most = max(most, n);
    }
    int incl = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += up;
    }
    if (lane == 31) s_sum[warp] = incl;
    __syncthreads();
    most = __reduce_max_sync(0xffffffffu, most);
    if (lane == 0) atomicMax(&s_most, most);
    int before = incl - sum, all = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) {
        if (w < warp) before += s_sum[w];
        all += s_sum[w];
    }
    for (int m = m0; m < m1; ++m) first[m] += before;
    if (tid == 0) first[a.M] = all;
    __syncthreads();
    Line l;
    l.total = (long long)all * items;
    l.chunk = max((l.total + ctas - 1) / ctas, (long long)min(LEAST_PAGES, s_most));
    return l;
}

// A CTA's pages of one item.
struct Segment {
    int m, item, page, n, of;  // row, its item, first page, pages, pages of the whole item
};
__device__ __forceinline__ Segment segment_at(const Kv8AttnArgs& a, const int* first, int items, long long u, long long end) {
    int lo = 0, hi = a.M;  // the last row that begins at or in front of u; rows without pages are passed over
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if ((long long)first[mid] * items <= u) lo = mid;
        else hi = mid;
    }
    Segment s;
    s.m = lo;
    s.of = first[lo + 1] - first[lo];
    const long long off = u - (long long)first[lo] * items;
    s.item = (int)(off / s.of);
    s.page = (int)(off - (long long)s.item * s.of);
    s.n = (int)min((long long)(s.of - s.page), end - u);
    return s;
}

// ---- pieces of the arithmetic --------------------------------------------------------------------------
__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t h2_bits(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
// Two codes (bytes of w, chosen by `sel`: 0x4140 the first two, 0x4342 the others) as f16.
template <uint32_t SEL>
__device__ __forceinline__ uint32_t codes_f16(uint32_t w) {
    const uint32_t u = __byte_perm(w, 0x64646464u, SEL);
    return h2_bits(__hsub2(*reinterpret_cast<const __half2*>(&u), __half2half2(__ushort_as_half(0x6480))));
}
// x, y as f16, and what that leaves.
__device__ __forceinline__ void split_f16(float x, float y, uint32_t& hi, uint32_t& lo) {
    const __half2 h = __floats2half2_rn(x, y);
    const float2 f = __half22float2(h);
    hi = h2_bits(h);
    lo = h2_bits(__floats2half2_rn(x - f.x, y - f.y));
}
__device__ __forceinline__ float pow2_bits(int biased) { return __uint_as_float((uint32_t)biased << 23); }  // 2^(biased - 127), 1 <= biased <= 254
constexpr int UP = 14;         // queries and weights enter with their largest between 2^UP and 2^(UP + 1)
constexpr int LEAST_EXP = 14;  // smallest exponent field that a factor of 2^UP can be brought to

struct StreamShape {
    int dp, vp, ldo, block, stages;
    size_t q_at, merge_at, first_at, bytes;
};
__host__ __device__ inline StreamShape stream_shape(int dim, int vdim, int M, int stages) {
    StreamShape s;
    s.dp = kv8_pad(dim);
    s.vp = kv8_pad(vdim);
    s.ldo = s.vp + 4;
    s.block = (int)kv8_block_bytes(dim, vdim);
    s.stages = stages;
    s.q_at = (size_t)stages * s.block;
    s.merge_at = s.q_at + (size_t)s.dp / 16 * 32 * 16;
    s.first_at = s.merge_at + sizeof(float) * (WARPS / 2 * PAIRS * s.ldo);
    s.bytes = s.first_at + sizeof(int) * (M + 1);
    return s;
}

// What is left of an item in `work`: maximum and sum of every pair, then its elements (relative to the maximum, not divided).
__host__ __device__ inline size_t part_floats(int vp) { return PAIRS * (size_t)(vp + 4); }

__device__ __forceinline__ void consumers_sync() { asm volatile("bar.sync 1, 256;" ::: "memory"); }

template <bool BF16>
__device__ __forceinline__ void store4(const Kv8AttnArgs& a, int m, int head, int d, const float (&v)[4], bool wide) {
    const size_t at = (size_t)m * a.ldo + (size_t)head * a.pool.vdim + d;
    if (wide) {
        store_row<BF16, 4>(a.out, at, v);
        return;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float one[1] = {v[e]};
        if (d + e < a.pool.vdim) store_row<BF16, 1>(a.out, at + e, one);
    }
}

// VS: slabs of 32 value elements (at most).
template <bool BF16, int VS>
__global__ void __launch_bounds__(THREADS, VS <= 4 ? 2 : 1) kv8_stream_kernel(const Kv8AttnArgs a, int stages, int tiles, int wide) {
    extern __shared__ __align__(128) unsigned char dyn[];
    __shared__ uint64_t full[MAX_STAGES], empty[MAX_STAGES];
    __shared__ volatile int s_abort;
    __shared__ int s_there[MAX_STAGES];
    __shared__ float s_c[PAIRS];                                   // what scores are multiplied with
    __shared__ float s_m[WARPS / 2][PAIRS], s_l[WARPS / 2][PAIRS];
    const StreamShape sh = stream_shape(a.pool.dim, a.pool.vdim, a.M, stages);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, group = a.heads / a.pool.kv_heads, items = a.pool.kv_heads * tiles, ctas = gridDim.x;
    uint4* qf = reinterpret_cast<uint4*>(dyn + sh.q_at);
    float* merge = reinterpret_cast<float*>(dyn + sh.merge_at);
    int* first = reinterpret_cast<int*>(dyn + sh.first_at);
    if (tid == 0) {
        for (int s = 0; s < stages; ++s) {
            mb_init(&full[s], 1);
            mb_init(&empty[s], 2);
        }
        s_abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    const Line line = make_line(a, items, ctas, first);
    const long long u0 = min(line.total, blockIdx.x * line.chunk), u1 = min(line.total, u0 + line.chunk);
    pdl_launch_dependents();
    if (warp == WARPS) {
        // ---- copies ----
        uint32_t i = 0;
        bool go = true;
        for (long long u = u0; u < u1 && go;) {
            const Segment sg = segment_at(a, first, items, u, u1);
            const int kvh = sg.item / tiles;
            const int32_t* table = a.pool.page_table + (size_t)__ldg(a.row_seq + sg.m) * a.pool.max_pages;
            for (int p0 = 0; p0 < sg.n && go; p0 += 32) {
                const int p = sg.page + p0 + lane;
                const int id = p0 + lane < sg.n ? p < a.n_shared ? __ldg(a.shared + p) : __ldg(table + p) : 0;
                for (int j = 0; j < min(32, sg.n - p0); ++j, ++i) {
                    const int page = __shfl_sync(0xffffffffu, id, j), s = (int)(i % stages);
                    if (i >= (uint32_t)stages && !__all_sync(0xffffffffu, mb_wait(&empty[s], ((i / stages) & 1u) ^ 1u, a.err_flag, &s_abort))) {
                        go = false;
                        break;
                    }
                    if (lane == 0) {
                        const bool there = (unsigned)page < (unsigned)a.pool.n_pages;
                        s_there[s] = there;
                        if (there) {
                            mb_expect_tx(&full[s], (uint32_t)sh.block);
                            bulk_copy(dyn + (size_t)s * sh.block, a.pool.pages + ((size_t)page * a.pool.kv_heads + kvh) * sh.block, (uint32_t)sh.block, &full[s]);
                        } else {
                            mb_arrive(&full[s]);
                        }
                    }
                    __syncwarp();
                }
            }
            u += sg.n;
        }
        if (lane == 0) mb_land_ring(full, i, (uint32_t)stages);
        return;
    }

    // ---- rows without a context ----
    for (int m = blockIdx.x; m < a.M; m += ctas) {
        if (first[m + 1] != first[m] || (unsigned)__ldg(a.row_seq + m) >= (unsigned)a.pool.n_seq) continue;
        const float zero[1] = {0.f};
        for (int i = tid; i < a.heads * a.pool.vdim; i += WARPS * 32) store_row<BF16, 1>(a.out, (size_t)m * a.ldo + i, zero);
    }

    const int gid = lane >> 2, tig = lane & 3, slabs = sh.dp / 32, vslabs = sh.vp / 32;
    uint32_t i = 0;  // pages of this CTA so far
    for (long long u = u0; u < u1;) {
        const Segment sg = segment_at(a, first, items, u, u1);
        const int kvh = sg.item / tiles, tile = sg.item - kvh * tiles, pairs = min(PAIRS, group - tile * PAIRS), head0 = kvh * group + tile * PAIRS;
        const int len = row_len(a, sg.m);
        consumers_sync();  // the segment in front has read its queries
        {                  // warp w: the queries of pair w, eight elements a lane
            const int d0 = lane * 8;
            float x[8];
            uint32_t top = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                float one[1] = {0.f};
                if (warp < pairs && d0 + e < a.pool.dim) load_row<BF16, 1>(a.q, (size_t)sg.m * a.ldq + (size_t)(head0 + warp) * a.pool.dim + d0 + e, one);
                x[e] = one[0];
                top = max(top, __float_as_uint(one[0]) & 0x7FFFFFFFu);
            }
            top = __reduce_max_sync(0xffffffffu, top);
            const int ex = top >= 0x7F800000u ? 127 + UP : max((int)(top >> 23), LEAST_EXP);
            const float up = pow2_bits(254 + UP - ex);
            if (d0 < sh.dp) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint4 f;
                    split_f16(x[4 * h] * up, x[4 * h + 1] * up, f.x, f.y);
                    split_f16(x[4 * h + 2] * up, x[4 * h + 3] * up, f.z, f.w);
                    qf[(2 * (lane >> 2) + h) * 32 + warp * 4 + (lane & 3)] = f;
                }
            }
            if (lane == 0) s_c[warp] = a.scale * LOG2E * exp2f((float)(ex - 127 - UP));
        }
        consumers_sync();
        const float c = s_c[gid];
        float mx = -INFINITY, l = 0.f, o[VS][4][2];
        float ve = LEAST_EXP, largest = LEAST_EXP;  // exponent field of the unit of o, which follows the largest W so far (the exponent of that, as it was rounded down)
#pragma unroll
        for (int s = 0; s < VS; ++s)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[s][e][0] = o[s][e][1] = 0.f;
        const int half = warp & 1;
        for (int p = (int)(((uint32_t)(warp >> 1) - i) % TURN); p < sg.n; p += TURN) {
            const int st = (int)((i + p) % stages);
            if (!__all_sync(0xffffffffu, mb_wait(&full[st], ((i + p) / stages) & 1u, a.err_flag, &s_abort))) break;
            const int nt = len - ((sg.page + p) * KV8_PAGE + half * 32);  // tokens that are seen
            if (nt > 0 && s_there[st]) {
                const unsigned char* block = dyn + (size_t)st * sh.block;
                const float *ks = reinterpret_cast<const float*>(block) + half * 32, *vs = ks + KV8_PAGE;
                const unsigned char* kc = block + 8 * KV8_PAGE + (half * 32 + gid) * 32 + tig * 8;
                const unsigned char* vc = block + 8 * KV8_PAGE + KV8_PAGE * sh.dp + (half * 32 + tig) * 32 + gid * 4;
                float sc[4][4];
#pragma unroll
                for (int j = 0; j < 4; ++j) sc[j][0] = sc[j][1] = sc[j][2] = sc[j][3] = 0.f;
#pragma unroll 2
                for (int s = 0; s < slabs; ++s) {
                    const uint4 q0 = qf[2 * s * 32 + lane], q1 = qf[(2 * s + 1) * 32 + lane];
                    const uint32_t a0[4] = {q0.x, q0.y, q0.z, q0.w}, a1[4] = {q1.x, q1.y, q1.z, q1.w};
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const uint2 w = *reinterpret_cast<const uint2*>(kc + s * (KV8_PAGE * 32) + j * 256);
                        mma_f16(sc[j], a0, codes_f16<0x4140>(w.x), codes_f16<0x4342>(w.x));
                        mma_f16(sc[j], a1, codes_f16<0x4140>(w.y), codes_f16<0x4342>(w.y));
                    }
                }
                // column 2 tig + e of tile j is token 8 j + 4 e + tig
                float w[4][2], most = -INFINITY;
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int t = 8 * j + 4 * e + tig;
                        const float s = (sc[j][e] + sc[j][2 + e]) * (ks[t] * c);
                        w[j][e] = t < nt ? s : -INFINITY;
                        most = fmaxf(most, w[j][e]);
                    }
                most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
                most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
                const float now = fmaxf(mx, most), ref = now == -INFINITY ? 0.f : now, corr = exp2f(mx - ref);
                float top = 0.f;
                l *= corr;
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int t = 8 * j + 4 * e + tig;
                        const float pr = exp2f(w[j][e] - ref);
                        l += pr;
                        w[j][e] = t < nt ? pr * vs[t] : 0.f;
                        top = fmaxf(top, w[j][e]);
                    }
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                // the unit follows the maximum down and the weights up
                largest = fmaxf(fmaxf(largest + (mx - ref), (float)(__float_as_uint(top) >> 23)), (float)LEAST_EXP);
                const float ve_now = ceilf(largest);
                const float f = corr * exp2f(ve - ve_now), up = pow2_bits(254 + UP - (int)ve_now);
                mx = now;
                ve = ve_now;
                uint32_t wa[2][4];
#pragma unroll
                for (int j = 0; j < 4; ++j) split_f16(w[j][0] * up, w[j][1] * up, wa[j >> 1][(j & 1) * 2], wa[j >> 1][(j & 1) * 2 + 1]);
#pragma unroll
                for (int s = 0; s < VS; ++s) {
                    if (s >= vslabs) break;
                    float acc[4][4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[e][0] = acc[e][1] = acc[e][2] = acc[e][3] = 0.f;
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        uint32_t x[4];
#pragma unroll
                        for (int r = 0; r < 4; ++r) x[r] = *reinterpret_cast<const uint32_t*>(vc + s * (KV8_PAGE * 32) + (h * 16 + r * 4) * 32);
                        const uint32_t p01 = __byte_perm(x[0], x[1], 0x5140), p23 = __byte_perm(x[0], x[1], 0x7362), r01 = __byte_perm(x[2], x[3], 0x5140), r23 = __byte_perm(x[2], x[3], 0x7362);
                        mma_f16(acc[0], wa[h], codes_f16<0x4140>(p01), codes_f16<0x4140>(r01));
                        mma_f16(acc[1], wa[h], codes_f16<0x4342>(p01), codes_f16<0x4342>(r01));
                        mma_f16(acc[2], wa[h], codes_f16<0x4140>(p23), codes_f16<0x4140>(r23));
                        mma_f16(acc[3], wa[h], codes_f16<0x4342>(p23), codes_f16<0x4342>(r23));
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        o[s][e][0] = fmaf(o[s][e][0], f, acc[e][0] + acc[e][2]);
                        o[s][e][1] = fmaf(o[s][e][1], f, acc[e][1] + acc[e][3]);
                    }
                }
            }
            __syncwarp();
            if (lane == 0) mb_arrive(&empty[st]);
        }
        i += sg.n;
        u += sg.n;

        // ---- the warps' results added up: first those of warps 4 .. 7 to those of 0 .. 3, then these four ----
        l += __shfl_xor_sync(0xffffffffu, l, 1);
        l += __shfl_xor_sync(0xffffffffu, l, 2);
        const float down = exp2f(ve - (127 + UP));
#pragma unroll
        for (int s = 0; s < VS; ++s)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                o[s][e][0] *= down;
                o[s][e][1] *= down;
            }
        const int slot = warp & (WARPS / 2 - 1);
        float* mine = merge + ((size_t)slot * PAIRS + gid) * sh.ldo + tig * 8;  // elements 8 tig + 4 e + 0 .. 3 of a slab
        auto put = [&]() {
            if (tig == 0) {
                s_m[slot][gid] = mx;
                s_l[slot][gid] = l;
            }
#pragma unroll
            for (int s = 0; s < VS; ++s) {
                if (s >= vslabs) break;
#pragma unroll
                for (int e = 0; e < 2; ++e) *reinterpret_cast<float4*>(mine + s * 32 + 4 * e) = make_float4(o[s][0][e], o[s][1][e], o[s][2][e], o[s][3][e]);
            }
        };
        if (warp >= WARPS / 2) put();
        consumers_sync();
        if (warp < WARPS / 2) {
            const float om = s_m[slot][gid], now = fmaxf(mx, om), ref = now == -INFINITY ? 0.f : now, f0 = exp2f(mx - ref), f1 = exp2f(om - ref);
            l = fmaf(l, f0, s_l[slot][gid] * f1);
            mx = now;
#pragma unroll
            for (int s = 0; s < VS; ++s) {
                if (s >= vslabs) break;
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float4 x = *reinterpret_cast<const float4*>(mine + s * 32 + 4 * e);
                    o[s][0][e] = fmaf(o[s][0][e], f0, x.x * f1);
                    o[s][1][e] = fmaf(o[s][1][e], f0, x.y * f1);
                    o[s][2][e] = fmaf(o[s][2][e], f0, x.z * f1);
                    o[s][3][e] = fmaf(o[s][3][e], f0, x.w * f1);
                }
            }
            __syncwarp();
            put();
        }
        consumers_sync();
        const bool whole = sg.n == sg.of;
        float* part = static_cast<float*>(a.work) + (size_t)(2 * blockIdx.x + (sg.page == 0)) * part_floats(sh.vp);
        for (int k = tid; k < pairs * (sh.vp / 4); k += WARPS * 32) {
            const int pr = k / (sh.vp / 4), d = (k - pr * (sh.vp / 4)) * 4;
            float f[WARPS / 2], top = -INFINITY, sum = 0.f, v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < WARPS / 2; ++w) top = fmaxf(top, s_m[w][pr]);
            const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
            for (int w = 0; w < WARPS / 2; ++w) {
                f[w] = exp2f(s_m[w][pr] - ref);
                const float4 x = *reinterpret_cast<const float4*>(merge + ((size_t)w * PAIRS + pr) * sh.ldo + d);
                v[0] = fmaf(f[w], x.x, v[0]); v[1] = fmaf(f[w], x.y, v[1]); v[2] = fmaf(f[w], x.z, v[2]); v[3] = fmaf(f[w], x.w, v[3]);
                sum = fmaf(f[w], s_l[w][pr], sum);
            }
            if (whole) {
                const float inv = sum == 0.f ? 0.f : 1.0f / sum;
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] *= inv;
                if (d < a.pool.vdim) store4<BF16>(a, sg.m, head0 + pr, d, v, wide);
            } else {
                float* at = part + (size_t)pr * (sh.vp + 4);
                *reinterpret_cast<float4*>(at + 4 + d) = make_float4(v[0], v[1], v[2], v[3]);
                if (d == 0) {
                    at[0] = top;
                    at[1] = sum;
                }
            }
        }
    }
}

// One CTA per cut of the line: the item that a cut falls into, if the CTA in front of the cut holds its beginning.
template <bool BF16>
__global__ void __launch_bounds__(THREADS) kv8_join_kernel(const Kv8AttnArgs a, int tiles, int wide) {
    extern __shared__ int first[];
    const int tid = threadIdx.x, items = a.pool.kv_heads * tiles, group = a.heads / a.pool.kv_heads, ctas = gridDim.x + 1, cut = blockIdx.x + 1, vp = kv8_pad(a.pool.vdim);
    const Line line = make_line(a, items, ctas, first);
    pdl_wait();
    const long long u = cut * line.chunk;
    if (u >= line.total) return;
    const Segment sg = segment_at(a, first, items, u, line.total);
    if (sg.page == 0) return;
    const long long begin = u - sg.page, end = begin + sg.of;
    if (begin / line.chunk != cut - 1) return;
    const int last = (int)((end - 1) / line.chunk), kvh = sg.item / tiles, tile = sg.item - kvh * tiles, pairs = min(PAIRS, group - tile * PAIRS), head0 = kvh * group + tile * PAIRS;
    const float* work = static_cast<const float*>(a.work);
    for (int k = tid; k < pairs * (vp / 4); k += THREADS) {
        const int pr = k / (vp / 4), d = (k - pr * (vp / 4)) * 4;
        // the beginning is the second part of its CTA, what follows the first of theirs
        auto part = [&](int c) { return work + (size_t)(2 * c + (c == cut - 1)) * part_floats(vp) + (size_t)pr * (vp + 4); };
        float top = -INFINITY, sum = 0.f, v[4] = {0.f, 0.f, 0.f, 0.f};
        for (int c = cut - 1; c <= last; ++c) top = fmaxf(top, __ldcg(part(c)));
        const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll 4
        for (int c = cut - 1; c <= last; ++c) {
            const float* at = part(c);
            const float f = exp2f(__ldcg(at) - ref);
            const float4 x = __ldcg(reinterpret_cast<const float4*>(at + 4 + d));
            sum = fmaf(f, __ldcg(at + 1), sum);
            v[0] = fmaf(f, x.x, v[0]); v[1] = fmaf(f, x.y, v[1]); v[2] = fmaf(f, x.z, v[2]); v[3] = fmaf(f, x.w, v[3]);
        }
        const float inv = sum == 0.f ? 0.f : 1.0f / sum;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] *= inv;
        if (d < a.pool.vdim) store4<BF16>(a, sg.m, head0 + pr, d, v, wide);
    }
}

template <typename... KArgs, typename... Args>
cudaError_t launch_behind(void (*kern)(KArgs...), int grid, int threads, size_t smem, cudaStream_t st, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kern, KArgs(args)...);
}

template <bool BF16, int VS>
cudaError_t launch_stream(const Kv8AttnArgs& a, int sm_count, cudaStream_t st) {
    const int group = a.heads / a.pool.kv_heads, tiles = (group + PAIRS - 1) / PAIRS, size = BF16 ? 2 : 4;
    const int wide = a.pool.vdim % 4 == 0 && (((uintptr_t)a.out | a.ldo * size) & (4 * size - 1)) == 0;
    auto bytes = [&](int stages) { return stream_shape(a.pool.dim, a.pool.vdim, a.M, stages).bytes; };
    // two CTAs per SM where registers (VS) and shared memory let them
    const int per_sm = VS <= 4 && bytes(TURN) <= ROOM / 2 ? 2 : 1, ctas = per_sm * sm_count;
    int stages = MAX_STAGES;
    while (stages > TURN && bytes(stages) > ROOM / per_sm) stages -= TURN;
    const size_t smem = bytes(stages);
    cudaError_t e = ensure_dyn_smem(kv8_stream_kernel<BF16, VS>, smem);
    if (e == cudaSuccess) e = ensure_dyn_smem(kv8_join_kernel<BF16>, sizeof(int) * (a.M + 1));
    if (e != cudaSuccess) return e;
    kv8_stream_kernel<BF16, VS><<<(unsigned)ctas, THREADS, smem, st>>>(a, stages, tiles, wide);
    if ((e = cudaGetLastError()) != cudaSuccess) return e;
    return launch_behind(kv8_join_kernel<BF16>, ctas - 1, THREADS, sizeof(int) * (a.M + 1), st, a, tiles, wide);
}

template <bool BF16>
cudaError_t launch_typed(const Kv8AttnArgs& a, int sm_count, cudaStream_t st) {
    if (a.pool.vdim <= 64) return launch_stream<BF16, 2>(a, sm_count, st);
    if (a.pool.vdim <= 128) return launch_stream<BF16, 4>(a, sm_count, st);
    return launch_stream<BF16, 8>(a, sm_count, st);
}

}  // namespace

size_t kv8_attn_bytes(int, int vdim, int, int, int, int sm_count) { return sizeof(float) * 2 * 2 * (size_t)sm_count * part_floats(kv8_pad(vdim)); }

cudaError_t launch_kv8_attn(const Kv8AttnArgs& a, int sm_count, cudaStream_t st) { return a.bf16 ? launch_typed<true>(a, sm_count, st) : launch_typed<false>(a, sm_count, st); }

}  // namespace hm

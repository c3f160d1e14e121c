// Softmax attention over the 8-bit paged cache:
//   out[row, head] = sum over the positions t <= row_pos whose page exists of softmax_t(scale q . k_t) v_t,   zeros where there is no such position.
// Page i of a row is shared[i] for i < n_shared and its sequence's page table entry behind them.  Where there is enough of both rows and shared pages, these are taken on their own
// (kv8_prefix.cu), and what follows here begins behind them and joins both.
//
// kv8_stream_kernel   rows' contexts, eight (row, head) pairs of one key/value head at a time; bound by the bytes of the cache
// kv8_join_kernel     joins the parts of contexts that several CTAs share; launched where there can be such
//
// Arithmetic of the first.  A warp takes a piece, 32 tokens (half of a page), for eight pairs, on m16n8k32 MMAs of 8-bit whole numbers with 32-bit sums, whose B operands are the
// codes as they are cached:
//   scores [16 x 8 tokens] = Q [16 x dim] . K^T,   out [16 x 8 elements] = W [16 x 32 tokens] . V
// Queries and weights enter as digits of base 256: rows 0 .. 7 are the pairs' upper digits, rows 8 .. 15 the lower ones, so that a tile's two halves are added up
// after the product (the first times 256).  bf16 rows take two digits: a query is whole numbers up to 32639 for its largest element (2^-16 of that), a weight up to
// 65535 for the largest of its piece (2^-16 of that).  f32 rows take four, in two products: 2^-31 of the largest, or a value's own 24 bits.  Sums of digits times
// codes are exact; what f32 rounds is what one would round without digits.  A token's key scale joins behind the product, its value scale goes into the weight,
// W = 2^(s - max) * scale, so that the largest of a piece is found with it.
// Against f16 operands (codes become f16 by two instructions for two codes, queries and weights by two terms): 981 instructions for 32 tokens x 256 elements, of which
// a third made f16 of codes, 105 us for 64 sequences of 500 to 8000 tokens (366 MB).
//
// Work.  The pieces of all rows, heads and tiles of eight pairs stand in one line, which the CTAs cut into lengths of equal cost: contexts of any lengths keep all SMs busy to the
// end, and no length needs to be known on the host.  An item's beginning (queries, sums of the warps, barriers) counts as much as BEGIN pieces: with 0, 6, 12, 20 and 28 the 64
// sequences took 99, 91, 79, 75 and 77 us.  A CTA's warps take its pieces in turn, each with a ring of copies of its own; what they have of an item is added up in shared memory.  The
// CTA writes the items that it has as a whole and leaves the rest (its first and its last) in `work`, for kv8_join_kernel.
// Two kinds of items are no part of the line:
//   short ones where there are more than CTAs.  Adding up takes a CTA some 5 us, so that a team of 1 to 4 warps takes an item, as many warps as leave each item a team.  Where the table has
//   room for 40 pieces per warp of a team at most, 96 in all, these are all items, and there is nothing to join; with longer ones in between it is those of up to SOLO pieces, before the CTA
//   joins in with the line, as what a team has is not shared out.  Rows of 8 pairs over 2 heads of 128, all of one length, in teams / in the line, us: 100 rows of 500 tokens 14 / 25, 200 of 1100
//   28 / 44, 290 of 1500 46 / 60, 400 of 2500 (80 pieces, not in teams of 2: 93) 103, 800 of 500 46 / 89, 80 of 4000 (125 pieces, teams of 4) 53 / 47; with lengths from 1 to these the
//   teams gain as much.  The rest with SOLO: 64 rows of up to 500 own tokens behind a prefix 60 us in teams of 3, 67 by single warps; at the 64 sequences 16 pieces instead of 12 took 97 us.
//   all of them where there are no more than CTAs and the table has room for WHOLE pieces at most: a CTA takes an item, nothing is counted or joined.  One row of 14 heads over 2 of 64
//   elements: 64 tokens 6.6 us against 10.8, 1024 10.1 against 14.7, 2048 14.0 against 16.0, 3000 (94 pieces) 17.7 against 16.1;
//   16 rows of 3000 tokens 18.1 against 19.0.
// 64 sequences of 500 to 8000 tokens, 8 heads of 128: 74 us, 4.9 TB/s, three quarters of what a copy reaches; what is left is the start (7 us to the first scores) and the uneven end.  Three rows
// of 20000 to 32768 tokens: 22 us, of which the join takes 5.
// Slower where tried, at the 64 sequences with an even line (93 us with each of them): a range of pieces for every warp, which then has more partial items than are worth joining; whole
// pages for a warp, of which 12 do not fit twice; 16 warps with one piece each.
#include "kv8.h"

#include <algorithm>
#include <type_traits>

#include "kv8_rows.cuh"
#include "launch_attrs.h"
#include "mbarrier.cuh"

namespace hm {
namespace {

constexpr int PAIRS = KV8_PAIRS;   // of an item
constexpr int LEAST_PIECES = 12;   // of a CTA, one for each of its warps: fewer would only leave more to be joined
constexpr int BEGIN = 20;           // pieces that take a CTA as long as the beginning and end of an item
constexpr int WHOLE = 80;           // pieces that a CTA takes in less time than a join takes
constexpr int SOLO = 12;            // pieces that a team takes before its CTA joins in with the line
constexpr int TEAM_PIECES = 40, MOST_TEAM_PIECES = 96;  // pieces per warp, and of an item, up to which there is no line
constexpr int MAX_DEPTH = 4;
constexpr int MERGE_ROWS = 32;      // pairs' results of several warps that stand in shared memory when those of all are added up
constexpr size_t ROOM = 222 * 1024;  // shared memory of a CTA, beside the static
constexpr float LOG2E = 1.4426950408889634f;

// ---- the line of pieces -----------------------------------------------------------------------------
// An item is BEGIN units and one for every piece: what its queries, sums and barriers cost a CTA, so that those who have many short items have fewer pieces.
struct Line {
    long long total, chunk;  // units of all items; of a CTA
    bool solo;               // there are items of a few pieces
};

// Pieces of a row's items that stand in the line.
__device__ __forceinline__ int line_pieces(const Kv8AttnArgs& a, int m) {
    const int n = kv8_row_pieces(a, m);
    return n > a.solo ? n : 0;
}

// Units in the lower half, rows that have pieces in the line in the upper.
__device__ __forceinline__ int units_of(long long x) { return (int)(uint32_t)x; }
__device__ __forceinline__ int rows_of(long long x) { return (int)(x >> 32); }

// Every thread of the CTA adds up the units of some rows that follow one another, ceil(M / THREADS) of them; first[t]: units (of one item of each row) and rows in front of thread t's
// rows, first[THREADS]: of all.  Ends with a barrier.
template <int THREADS>
__device__ __forceinline__ Line make_line(const Kv8AttnArgs& a, int items, int ctas, long long* first) {
    __shared__ long long s_sum[THREADS / 32];
    __shared__ int s_most;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, per = (a.M + THREADS - 1) / THREADS, m0 = min(a.M, tid * per), m1 = min(a.M, m0 + per);
    if (tid == 0) s_most = 0;
    long long sum = 0;
    int most = 0;
    bool solo = false;
    for (int m = m0; m < m1; ++m) {
        const int n = kv8_row_pieces(a, m);
        if (n > a.solo) sum += (1ll << 32) + n + BEGIN;
        else solo |= n > 0;
        most = max(most, n);
    }
    long long incl = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long up = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += up;
    }
    if (lane == 31) s_sum[warp] = incl;
    __syncthreads();
    most = __reduce_max_sync(0xffffffffu, most);
    if (lane == 0) atomicMax(&s_most, most);
    long long before = incl - sum, all = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) {
        if (w < warp) before += s_sum[w];
        all += s_sum[w];
    }
    first[tid] = before;
    if (tid == 0) first[THREADS] = all;
    Line l;
    l.solo = __syncthreads_or(solo);
    l.total = (long long)units_of(all) * items;
    l.chunk = max((l.total + ctas - 1) / ctas, (long long)min(LEAST_PIECES, s_most) + BEGIN);
    return l;
}

// Pieces of one item that follow one another.
struct Segment {
    int m, item, at, n, of;  // row, its item, first piece (counted from own_from), pieces, pieces of the whole item
};
// The piece that unit u (of the line) stands for, or the item's first where it stands for the item's beginning (n is not set); `begin`: the item's first unit, `before`: pieces of
// the line in front of this one.
template <int THREADS>
__device__ __forceinline__ Segment unit_at(const Kv8AttnArgs& a, const long long* first, int items, long long u, long long& begin, long long& before) {
    const bool small = (unsigned long long)u >> 32 == 0;
    const int rank = small ? (int)((uint32_t)u / (uint32_t)items) : (int)(u / items);  // that many units of an item of every row are in front
    const int per = (a.M + THREADS - 1) / THREADS;
    int lo = 0, hi = (a.M + per - 1) / per;  // the last thread whose rows begin there or in front; those without pieces are passed over
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (units_of(first[mid]) <= rank) lo = mid;
        else hi = mid;
    }
    Segment s;
    int at = units_of(first[lo]), rows = rows_of(first[lo]);
    s.m = lo * per;
    for (s.of = line_pieces(a, s.m); s.of == 0 || rank >= at + s.of + BEGIN; s.of = line_pieces(a, ++s.m)) {
        at += s.of ? s.of + BEGIN : 0;
        rows += s.of > 0;
    }
    const long long off = u - (long long)at * items;  // below (of + BEGIN) * items
    const int units = s.of + BEGIN;
    s.item = small ? (int)((uint32_t)off / (uint32_t)units) : (int)(off / units);
    const int in = (int)(off - (long long)s.item * units);
    begin = u - in;
    s.at = max(0, in - BEGIN);
    s.n = 0;
    before = (long long)items * (at - rows * BEGIN) + (long long)s.item * s.of + s.at;
    return s;
}
// The segment behind s, `left` pieces from the end (not 0).
__device__ __forceinline__ void next_segment(const Kv8AttnArgs& a, int items, Segment& s, int left) {
    s.at = 0;
    if (++s.item == items) {
        s.item = 0;
        do s.of = line_pieces(a, ++s.m);
        while (s.of == 0);
    }
    s.n = min(s.of, left);
}

// ---- pieces of the arithmetic --------------------------------------------------------------------------
// c (+)= a . b; the first product of a sum begins with zeros.
template <bool UNSIGNED_A, bool FIRST>
__device__ __forceinline__ void mma_s8(int (&c)[4], const uint4& a, const uint2& b) {
    const int c0 = FIRST ? 0 : c[0], c1 = FIRST ? 0 : c[1], c2 = FIRST ? 0 : c[2], c3 = FIRST ? 0 : c[3];
    if constexpr (UNSIGNED_A)
        asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
            : "=r"(c[0]), "=r"(c[1]), "=r"(c[2]), "=r"(c[3])
            : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b.x), "r"(b.y), "r"(c0), "r"(c1), "r"(c2), "r"(c3));
    else
        asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
            : "=r"(c[0]), "=r"(c[1]), "=r"(c[2]), "=r"(c[3])
            : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b.x), "r"(b.y), "r"(c0), "r"(c1), "r"(c2), "r"(c3));
}
// 2^x; results below the normal range are zero.
__device__ __forceinline__ float exp2_ftz(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float pow2_bits(int biased) { return __uint_as_float((uint32_t)biased << 23); }  // 2^(biased - 127), 1 <= biased <= 254

// Digits of four values x[i], one word per digit, the lowest first (DIGITS 2: of 16 bits, else of 32).
template <int DIGITS>
__device__ __forceinline__ void digits_of(const uint32_t (&x)[4], uint32_t (&d)[DIGITS]) {
    const uint32_t a01 = __byte_perm(x[0], x[1], 0x5140), a23 = __byte_perm(x[2], x[3], 0x5140);  // digit 0 of both, digit 1 of both
    d[0] = __byte_perm(a01, a23, 0x5410);
    d[1] = __byte_perm(a01, a23, 0x7632);
    if constexpr (DIGITS == 4) {
        const uint32_t b01 = __byte_perm(x[0], x[1], 0x7362), b23 = __byte_perm(x[2], x[3], 0x7362);
        d[2] = __byte_perm(b01, b23, 0x5410);
        d[3] = __byte_perm(b01, b23, 0x7632);
    }
}
// What the upper and lower digits' sums of one or two products stand for.
template <int PASSES>
__device__ __forceinline__ float from_digits(const int (&c)[PASSES][4], int e) {
    const float low = (float)(c[PASSES - 1][e] * 256 + c[PASSES - 1][2 + e]);
    return PASSES == 1 ? low : fmaf((float)(c[0][e] * 256 + c[0][2 + e]), 65536.f, low);
}
constexpr float Q_MOST = 32639.f;   // two signed digits: 127 * 256 + 127
constexpr float W_PART = 65535.f / 65536.f;
// Queries are brought up by less than 2^128: those whose largest element is below 2^-112 (bf16) or 2^-98 have a step of 2^-127 for it.
constexpr float Q_LEAST = 1.925929944387236e-34f;  // 2^-112
constexpr int Q_LEAST_EX = 29;                     // exponent field of 2^-98
// Smallest exponent field that weights are brought up from: the last digit's step stays a normal number, 2^-126 or 2^-125
__device__ constexpr int w_least(bool bf16) { return bf16 ? 16 : 32; }

struct StreamShape {
    int dp, vp, ldo, kpart, vpart, queries;  // padded sizes, row of the warps' results, bytes of a piece's keys and values, words of 16 bytes of an item's queries
    size_t q_at, merge_at, bytes;
};
__host__ __device__ inline StreamShape stream_shape(int dim, int vdim, int passes, int warps, int depth) {
    StreamShape s;
    s.dp = kv8_pad(dim);
    s.vp = kv8_pad(vdim);
    s.ldo = s.vp + 8;
    s.kpart = kv8_part_bytes(dim);
    s.vpart = kv8_part_bytes(vdim);
    s.q_at = (size_t)warps * depth * (s.kpart + s.vpart);
    s.queries = s.dp / 32 * passes * 32;
    s.merge_at = s.q_at + 2 * sizeof(uint4) * s.queries;
    // a warp's own items have their queries in the same place
    const size_t merge = 2 * sizeof(uint4) * s.queries + sizeof(float) * MERGE_ROWS * s.ldo, own = sizeof(uint4) * s.queries * warps;
    s.bytes = s.q_at + (merge > own ? merge : own);
    return s;
}

// A query with the largest magnitude `top` (as bits): what its elements are multiplied with to be whole numbers (f32: a power of two that brings the largest to 2^29 .. 2^30; 0: it has an
// infinity or a NaN), and what its scores are multiplied with.
template <bool BF16>
__device__ __forceinline__ float query_factors(float scale, uint32_t top, float& up) {
    const bool finite = top < 0x7F800000u;
    const float most = fmaxf(__uint_as_float(top), Q_LEAST);
    const int ex = max((int)(top >> 23), Q_LEAST_EX);
    up = !finite ? 0.f : BF16 ? Q_MOST / most : pow2_bits(127 + 29 - (ex - 127));
    const float down = BF16 ? most / Q_MOST : exp2f((float)(ex - 127 - 29));
    return finite ? scale * LOG2E * down : __uint_as_float(0x7FC00000u);
}
// Eight elements of a query as signed digits, the upper two first, a product 32 words of 16 bytes behind the other.
template <bool BF16>
__device__ __forceinline__ void put_digits(const float (&x)[8], float up, uint4* to) {
    constexpr int PASSES = BF16 ? 1 : 2;
    uint32_t y[2][4], d[2][2 * PASSES];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const int whole = up != 0.f ? __float2int_rn(x[e] * up) : 0;
        y[e >> 2][e & 3] = BF16 ? (uint32_t)(whole + 0x80) ^ 0x80u : (uint32_t)(whole + 0x808080) ^ 0x808080u;
    }
    digits_of<2 * PASSES>(y[0], d[0]);
    digits_of<2 * PASSES>(y[1], d[1]);
#pragma unroll
    for (int h = 0; h < PASSES; ++h) {
        const int k = 2 * (PASSES - 1 - h);
        to[h * 32] = make_uint4(d[0][k + 1], d[0][k], d[1][k + 1], d[1][k]);
    }
}

// What is left of an item in `work`: maximum and sum of every pair, then its elements (relative to the maximum, not divided).
__host__ __device__ inline size_t part_floats(int vp) { return PAIRS * (size_t)(vp + 4); }

// Barrier of a team's warps, with an OR over their predicates.
__device__ __forceinline__ bool team_any(int team, int threads, bool v) {
    uint32_t r;
    asm volatile("{ .reg .pred p, q; setp.ne.u32 p, %1, 0; barrier.cta.red.or.aligned.pred q, %2, %3, p; selp.u32 %0, 1, 0, q; }" : "=r"(r) : "r"((uint32_t)v), "r"(1 + team), "r"(threads) : "memory");
    return r != 0;
}

// Parts in `work`: of CTA c its first item (0) and its last (1).
__device__ __forceinline__ float* cta_part(const Kv8AttnArgs& a, int vp, int cta, int which) { return static_cast<float*>(a.work) + (size_t)(2 * cta + which) * part_floats(vp); }

// References of the prefix's parts are those of products of weights and value scales, so that they may be more than 2^126 apart where the sums of weights that are relative to them are not: these are
// multiplied with the root of a factor twice.
// Joins four elements of a pair (relative to 2^top, with their sum; top is -inf where nothing was seen, so that the prefix's references alone count) with the parts of the prefix.
__device__ __forceinline__ void add_prefix(const Kv8AttnArgs& a, int vp, int kvh, int pair, int d, float& top, float& sum, float (&v)[4]) {
    const size_t pairs = (size_t)a.M * (a.heads / a.pool.kv_heads), step = (size_t)a.pool.kv_heads * pairs * (vp + 4);
    const float* at = a.prefix + ((size_t)kvh * pairs + pair) * (vp + 4);
    float most = top;
#pragma unroll 4
    for (int i = 0; i < a.prefix_n; ++i) most = fmaxf(most, __ldcg(at + i * step));
    const float ref = most == -INFINITY ? 0.f : most, root = exp2f(0.5f * (top - ref)), own = root * root;
    sum = sum * root * root;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] *= own;
#pragma unroll 4
    for (int i = 0; i < a.prefix_n; ++i) {
        const float2 ml = __ldcg(reinterpret_cast<const float2*>(at + i * step));
        if (ml.x == -INFINITY) continue;  // nothing seen
        const float r = exp2f(0.5f * (ml.x - ref)), f = r * r;
        const float4 x = __ldcg(reinterpret_cast<const float4*>(at + i * step + 4 + d));
        sum = fmaf(r * ml.y, r, sum);
        v[0] = fmaf(f, x.x, v[0]); v[1] = fmaf(f, x.y, v[1]); v[2] = fmaf(f, x.z, v[2]); v[3] = fmaf(f, x.w, v[3]);
    }
    top = most;
}

// The same for what a lane of a warp's own item has: elements 8 i + 2 tig + 0, 1 of a pair.
template <int VS>
__device__ __forceinline__ void add_prefix_to(const Kv8AttnArgs& a, int vp, int kvh, int pair, int tig, float& top, float& sum, float (&o)[VS * 4][2]) {
    const size_t pairs = (size_t)a.M * (a.heads / a.pool.kv_heads), step = (size_t)a.pool.kv_heads * pairs * (vp + 4);
    const float* at = a.prefix + ((size_t)kvh * pairs + pair) * (vp + 4);
    float most = top;
#pragma unroll 4
    for (int i = 0; i < a.prefix_n; ++i) most = fmaxf(most, __ldcg(at + i * step));
    const float ref = most == -INFINITY ? 0.f : most, root = exp2f(0.5f * (top - ref)), own = root * root;
    sum = sum * root * root;
#pragma unroll
    for (int s = 0; s < VS * 4; ++s) {
        o[s][0] *= own;
        o[s][1] *= own;
    }
#pragma unroll 1
    for (int i = 0; i < a.prefix_n; ++i) {
        const float2 ml = __ldcg(reinterpret_cast<const float2*>(at + i * step));
        const float r = ml.x == -INFINITY ? 0.f : exp2f(0.5f * (ml.x - ref)), f = r * r;
        if (ml.x != -INFINITY) sum = fmaf(r * ml.y, r, sum);
#pragma unroll
        for (int s = 0; s < VS * 4; ++s) {
            if (8 * s >= vp) break;
            const float2 x = __ldcg(reinterpret_cast<const float2*>(at + i * step + 4 + 8 * s + 2 * tig));
            o[s][0] = fmaf(f, x.x, o[s][0]);
            o[s][1] = fmaf(f, x.y, o[s][1]);
        }
    }
    top = most;
}

// VS: slabs of 32 value elements (at most).  A warp's ring holds `depth` pieces; the keys of a piece make room for those of a later one as soon as the scores are
// there, the values when the piece is done.
template <bool BF16, int VS, int WARPS>
__global__ void __launch_bounds__(WARPS * 32, 1) kv8_stream_kernel(const Kv8AttnArgs a, int depth, int tiles, int wide) {
    constexpr int PASSES = BF16 ? 1 : 2, THREADS = WARPS * 32;
    extern __shared__ __align__(128) unsigned char dyn[];
    __shared__ uint64_t bars[WARPS][2][MAX_DEPTH];
    __shared__ volatile int s_abort;
    __shared__ long long first[THREADS + 1];
    __shared__ uint64_t s_added;         // the sums of the segment in front have been read
    __shared__ float s_c[2][PAIRS];      // what scores are multiplied with
    __shared__ float s_m[MERGE_ROWS], s_l[MERGE_ROWS];
    const StreamShape sh = stream_shape(a.pool.dim, a.pool.vdim, PASSES, WARPS, depth);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, group = a.heads / a.pool.kv_heads, items = a.pool.kv_heads * tiles, ctas = gridDim.x;
    unsigned char* kbuf = dyn + (size_t)warp * depth * (sh.kpart + sh.vpart);
    unsigned char* vbuf = kbuf + (size_t)depth * sh.kpart;
    uint4* queries = reinterpret_cast<uint4*>(dyn + sh.q_at);  // of this segment and the one behind it
    float* merge = reinterpret_cast<float*>(dyn + sh.merge_at);
    uint64_t *kfull = bars[warp][0], *vfull = bars[warp][1];
    if (tid == 0) mb_init(&s_added, WARPS);
    if (lane == 0) {
        for (int s = 0; s < depth; ++s) {
            mb_init(&kfull[s], 1);
            mb_init(&vfull[s], 1);
        }
        s_abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    Line line{};
    if (a.whole) __syncthreads();
    else line = make_line<THREADS>(a, items, ctas, first);
    const long long u0 = min(line.total, blockIdx.x * line.chunk), u1 = min(line.total, u0 + line.chunk);
    Segment line_begin{};
    int count = 0;  // pieces of this CTA
    if (a.whole && (int)blockIdx.x < a.M * items) {
        line_begin.m = (int)blockIdx.x / items;
        line_begin.item = (int)blockIdx.x - line_begin.m * items;
        line_begin.of = line_begin.n = count = kv8_row_pieces(a, line_begin.m);
    } else if (u0 < u1) {
        long long begin, before, behind = (long long)items * (units_of(first[THREADS]) - rows_of(first[THREADS]) * BEGIN);
        if (u1 < line.total) unit_at<THREADS>(a, first, items, u1, begin, behind);
        line_begin = unit_at<THREADS>(a, first, items, u0, begin, before);
        count = (int)(behind - before);
        line_begin.n = min(line_begin.of - line_begin.at, count);
    }
    pdl_launch_dependents();

    // ---- rows without a context (where there is a prefix, kv8_join_kernel writes them) ----
    for (int m = blockIdx.x; m < a.M && a.prefix_n == 0; m += ctas) {
        if (kv8_row_pieces(a, m) > 0 || (unsigned)__ldg(a.row_seq + m) >= (unsigned)a.pool.n_seq) continue;
        const float zero[1] = {0.f};
        for (int i = tid; i < a.heads * a.pool.vdim; i += THREADS) store_row<BF16, 1>(a.out, (size_t)m * a.ldo + i, zero);
    }

    // ---- copies: `ahead` runs some pieces of this warp ahead of the arithmetic ----
    Segment sg{}, ahead{};
    int ahead_at = 0, ahead_begin = 0, ahead_page = -1;  // its piece, counted over the CTA (or the item that is this warp's own); the first of its segment; its page in the pool
    int end = 0, step = 1;                               // pieces of the CTA (of the item); this warp has every step-th
    const int32_t* ahead_table = nullptr;                // of its segment's sequence
    const unsigned char* ahead_head = nullptr;           // its head's block of page 0
    const uint32_t half = (uint32_t)(sh.kpart + sh.vpart), page_bytes = 2 * half * (uint32_t)a.pool.kv_heads;
    auto enter = [&]() {
        ahead_table = a.pool.page_table + (size_t)__ldg(a.row_seq + ahead.m) * a.pool.max_pages;
        ahead_head = a.pool.pages + (size_t)(ahead.item / tiles) * (2 * half);
    };
    auto settle = [&]() {
        if (ahead_at >= end) return;
        if (ahead_at >= ahead_begin + ahead.n) {
            do {
                ahead_begin += ahead.n;
                next_segment(a, items, ahead, end - ahead_begin);
            } while (ahead_at >= ahead_begin + ahead.n);
            enter();
        }
        const int p = (a.own_from + ahead.at + ahead_at - ahead_begin) >> 1;
        ahead_page = __ldg(p < a.n_shared ? a.shared + p : ahead_table + p);
    };
    // the piece that it stands at, null where there is none; on to the next
    auto take = [&]() -> const unsigned char* {
        const unsigned char* src = nullptr;
        if (ahead_at < end && (unsigned)ahead_page < (unsigned)a.pool.n_pages) src = ahead_head + (unsigned long long)(uint32_t)ahead_page * page_bytes + (((ahead.at + ahead_at - ahead_begin) & 1) ? half : 0u);
        ahead_at += step;
        settle();
        return src;
    };
    auto copy = [&](unsigned char* dst, const unsigned char* src, int bytes, uint64_t* bar) {
        if (lane == 0) {
            mb_expect_tx(bar, (uint32_t)bytes);
            bulk_copy(dst, src, (uint32_t)bytes, bar);
        }
    };
    uint32_t there = 0, phase = 0;  // bit s: slot s holds a piece; the parity of its next wait
    auto start = [&](const Segment& at, int from, int pieces, int stride, int slots) {
        ahead = at;
        ahead_at = from;
        ahead_begin = 0;
        end = pieces;
        step = stride;
        enter();
        settle();
        for (int s = 0; s < slots; ++s) {
            const unsigned char* src = take();
            there = (there & ~(1u << s)) | (src ? 1u << s : 0u);
            if (!src) continue;
            copy(kbuf + (size_t)s * sh.kpart, src, sh.kpart, &kfull[s]);
            copy(vbuf + (size_t)s * sh.vpart, src + sh.kpart, sh.vpart, &vfull[s]);
        }
    };

    // ---- queries: eight elements a lane ----
    static_assert(WARPS >= PAIRS, "a warp for every pair");
    auto fetch_query = [&](const Segment& of, int pr, float (&x)[8]) {
        const int kvh = of.item / tiles, tile = of.item - kvh * tiles, d0 = lane * 8;
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = 0.f;
        if (pr >= min(PAIRS, group - tile * PAIRS) || d0 >= a.pool.dim) return;
        const size_t at = (size_t)of.m * a.ldq + (size_t)(kvh * group + tile * PAIRS + pr) * a.pool.dim + d0;
        if (wide & 2) {
            float y[4], z[4];
            load_row<BF16, 4>(a.q, at, y);
            load_row<BF16, 4>(a.q, at + 4, z);
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = e < 4 ? y[e & 3] : z[e & 3];
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                float one[1] = {0.f};
                if (d0 + e < a.pool.dim) load_row<BF16, 1>(a.q, at + e, one);
                x[e] = one[0];
            }
        }
    };
    // as digits, in the order of the MMAs' operands; returns what the pair's scores are multiplied with
    auto put_query = [&](const float (&x)[8], int pr, uint4* to) -> float {
        uint32_t top = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(x[e]) & 0x7FFFFFFFu);
        float up;
        const float f = query_factors<BF16>(a.scale, __reduce_max_sync(0xffffffffu, top), up);
        if (lane * 8 < sh.dp) put_digits<BF16>(x, up, to + (lane >> 2) * PASSES * 32 + pr * 4 + (lane & 3));
        return f;
    };

    const int gid = lane >> 2, tig = lane & 3, slabs = sh.dp / 32, vslabs = sh.vp / 32;
    int i = 0, slot = 0, len = 0;  // this warp's next piece, counted over the CTA (or its own item), and its slot; tokens of the segment's row
    bool good = true;                         // no wait has run out
    bool alone = line.solo;                   // with items of this warp's team; then with the line
    const int teams = WARPS / a.team, team = warp / a.team, in_team = warp - team * a.team;
    int own = team * ctas + (int)blockIdx.x;  // those are every teams * ctas-th of all
    uint4* own_queries = queries + warp * sh.queries;  // where the line's queries and sums will stand
    float next_q[8];
    int begin = 0, turn = 0;
    bool joined = false, waited = false;  // at the line; for the prefix
    for (;;) {
        Segment behind{};
        int len_behind = 0;
        bool last = true;
        float c = 0.f;
        const uint4* qf;
        if (alone) {
            int m = 0, n = 0;
            for (; own < a.M * items; own += teams * ctas) {
                m = own / items;
                n = kv8_row_pieces(a, m);
                if (n > 0 && n <= a.solo) break;
            }
            if (own >= a.M * items || !good) {
                alone = false;
                continue;
            }
            sg = Segment{m, own - m * items, 0, n, n};
            own += teams * ctas;
            __syncwarp();
            start(sg, in_team, n, a.team, depth);
            len = kv8_row_len(a, m);
            begin = slot = 0;
            i = in_team;
            // lane (gid, tig): elements 8 tig .. 8 tig + 7 of every slab of pair gid
            const int kvh = sg.item / tiles, tile = sg.item - kvh * tiles;
            const bool is = gid < min(PAIRS, group - tile * PAIRS);
            const size_t q_at = (size_t)m * a.ldq + (size_t)(kvh * group + tile * PAIRS + (is ? gid : 0)) * a.pool.dim + 8 * tig;
            auto elements = [&](int s, float (&x)[8]) {
                const int left = is ? a.pool.dim - (32 * s + 8 * tig) : 0;
                if (wide & 2) {
                    float y[2][4] = {};
                    if (left > 0) {
                        load_row<BF16, 4>(a.q, q_at + 32 * s, y[0]);
                        load_row<BF16, 4>(a.q, q_at + 32 * s + 4, y[1]);
                    }
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[e] = y[e >> 2][e & 3];
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        float one[1] = {0.f};
                        if (e < left) load_row<BF16, 1>(a.q, q_at + 32 * s + e, one);
                        x[e] = one[0];
                    }
                }
            };
            uint32_t top = 0;
#pragma unroll 4
            for (int s = 0; s < slabs; ++s) {
                elements(s, next_q);
#pragma unroll
                for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(next_q[e]) & 0x7FFFFFFFu);
            }
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
            float up;
            c = query_factors<BF16>(a.scale, top, up);
#pragma unroll 2
            for (int s = 0; s < slabs; ++s) {
                elements(s, next_q);
                put_digits<BF16>(next_q, up, own_queries + s * PASSES * 32 + lane);
            }
            __syncwarp();
            qf = own_queries;
        } else {
            if (!joined) {
                joined = true;
                if (count == 0) break;
                sg = line_begin;
                if (warp < PAIRS) fetch_query(sg, warp, next_q);  // in front of the copies, behind which they would wait
                start(sg, warp, count, WARPS, good ? depth : 0);  // nothing into slots whose copies were given up
                len = kv8_row_len(a, sg.m);
                i = warp;
                begin = slot = 0;
                if (line.solo) __syncthreads();  // no warp has items of its own left
                if (warp < PAIRS) {
                    const float f = put_query(next_q, warp, queries);
                    if (lane == 0) s_c[0][warp] = f;
                }
                __syncthreads();
            }
            if (begin >= count) break;
            qf = queries + turn * sh.queries;
            c = s_c[turn][gid];
            last = begin + sg.n >= count;
            behind = sg;
            if (!last) {  // the next segment's queries are fetched now
                next_segment(a, items, behind, count - begin - sg.n);
                len_behind = kv8_row_len(a, behind.m);
                if (warp < PAIRS) fetch_query(behind, warp, next_q);
            }
        }
        const int kvh = sg.item / tiles, tile = sg.item - kvh * tiles, pairs = min(PAIRS, group - tile * PAIRS), head0 = kvh * group + tile * PAIRS;
        float mx = -INFINITY, l = 0.f, o[VS * 4][2];  // elements 8 i + 2 tig + 0, 1 of pair gid
#pragma unroll
        for (int s = 0; s < VS * 4; ++s) o[s][0] = o[s][1] = 0.f;
        for (; good && i < begin + sg.n; i += step) {
            const int nt = len - ((a.own_from + sg.at + i - begin) * KV8_HALF + 8 * tig);  // this lane's tokens are 8 tig .. 8 tig + 7: how many of them are seen
            const bool partial = nt + 8 * tig < KV8_HALF;
            const unsigned char* next = take();  // the piece that comes into this slot next
            unsigned char *keys = kbuf + (size_t)slot * sh.kpart, *values = vbuf + (size_t)slot * sh.vpart;
            if ((there >> slot) & 1u) {
                const uint32_t parity = (phase >> slot) & 1u;
                const unsigned char *kc = keys + KV8_HALF * 4 + gid * 32 + tig * 8, *vc = values + KV8_HALF * 4 + gid * 32 + tig * 8;
                if (!(good = __all_sync(0xffffffffu, mb_wait(&kfull[slot], parity, a.err_flag, &s_abort)))) break;
                int sc[4][PASSES][4];
                auto product = [&](int s, auto head) {
                    uint2 k[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) k[j] = *reinterpret_cast<const uint2*>(kc + s * (KV8_HALF * 32) + j * 256);
#pragma unroll
                    for (int h = 0; h < PASSES; ++h) {
                        const uint4 q = qf[(s * PASSES + h) * 32 + lane];
#pragma unroll
                        for (int j = 0; j < 4; ++j) mma_s8<false, decltype(head)::value>(sc[j][h], q, k[j]);
                    }
                };
                product(0, std::true_type{});
#pragma unroll VS <= 4 ? VS : 4
                for (int s = 1; s < slabs; ++s) product(s, std::false_type{});
                // column 2 tig + e of tile j is token 8 tig + 2 j + e
                float w[8], most = -INFINITY;
#pragma unroll
                for (int t = 0; t < 8; t += 4) {
                    const float4 x = *reinterpret_cast<const float4*>(keys + (8 * tig + t) * 4);
                    w[t] = from_digits<PASSES>(sc[t >> 1], 0) * (x.x * c);
                    w[t + 1] = from_digits<PASSES>(sc[t >> 1], 1) * (x.y * c);
                    w[t + 2] = from_digits<PASSES>(sc[(t >> 1) + 1], 0) * (x.z * c);
                    w[t + 3] = from_digits<PASSES>(sc[(t >> 1) + 1], 1) * (x.w * c);
                }
                __syncwarp();  // the keys have been read: the next ones may come
                if (next) copy(keys, next, sh.kpart, &kfull[slot]);
                if (partial)
#pragma unroll
                    for (int t = 0; t < 8; ++t) w[t] = t < nt ? w[t] : -INFINITY;
#pragma unroll
                for (int t = 0; t < 8; ++t) most = fmaxf(most, w[t]);
                most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
                most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
                const float now = fmaxf(mx, most), ref = now == -INFINITY ? 0.f : now, corr = exp2_ftz(mx - ref);
                mx = now;
                l *= corr;
                if (!(good = __all_sync(0xffffffffu, mb_wait(&vfull[slot], parity, a.err_flag, &s_abort)))) {
                    if (next) mb_land(&kfull[slot], parity ^ 1u);
                    break;
                }
                uint32_t top = 0;  // bits of the largest weight: of NaN where a scale is
                float sum = 0.f;
#pragma unroll
                for (int t = 0; t < 8; t += 4) {
                    const float4 y = *reinterpret_cast<const float4*>(values + (8 * tig + t) * 4);
                    float v[4] = {y.x, y.y, y.z, y.w};
                    if (partial)
#pragma unroll
                        for (int e = 0; e < 4; ++e) v[e] = t + e < nt ? v[e] : 0.f;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float pr = exp2_ftz(w[t + e] - ref);
                        sum += pr;
                        w[t + e] = pr * v[e];
                        top = max(top, __float_as_uint(w[t + e]));
                    }
                }
                l += sum;
                top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
                if (top >= 0x7F800000u) l = __uint_as_float(0x7FC00000u);
                const int ex = min(max((int)(top >> 23), w_least(BF16)), 254);
                // bf16: whole numbers up to 65535, f32: below 2^31, for the largest
                const float up = BF16 ? pow2_bits(127 + 15 - (ex - 127)) * W_PART : pow2_bits(127 + 30 - (ex - 127)), unit = exp2_ftz((float)(ex - 127 - (BF16 ? 15 : 30))) * (BF16 ? 1.f / W_PART : 1.f);
                uint4 wa[PASSES];
                {
                    uint32_t x[2][4], d[2][2 * PASSES];
#pragma unroll
                    for (int t = 0; t < 8; ++t) x[t >> 2][t & 3] = BF16 ? __float_as_uint(fmaf(w[t], up, 8388608.f)) : __float2uint_rn(w[t] * up);
                    digits_of<2 * PASSES>(x[0], d[0]);
                    digits_of<2 * PASSES>(x[1], d[1]);
#pragma unroll
                    for (int h = 0; h < PASSES; ++h) wa[h] = make_uint4(d[0][2 * (PASSES - 1 - h) + 1], d[0][2 * (PASSES - 1 - h)], d[1][2 * (PASSES - 1 - h) + 1], d[1][2 * (PASSES - 1 - h)]);
                }
                if (__any_sync(0xffffffffu, corr != 1.f)) {
#pragma unroll
                    for (int s = 0; s < VS * 4; ++s) {
                        o[s][0] *= corr;
                        o[s][1] *= corr;
                    }
                }
#pragma unroll
                for (int s = 0; s < VS; ++s) {
                    if (s >= vslabs) break;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint2 v = *reinterpret_cast<const uint2*>(vc + (s * 4 + e) * (8 * KV8_HALF));
                        int acc[PASSES][4];
#pragma unroll
                        for (int h = 0; h < PASSES; ++h) mma_s8<true, true>(acc[h], wa[h], v);
                        o[s * 4 + e][0] = fmaf(from_digits<PASSES>(acc, 0), unit, o[s * 4 + e][0]);
                        o[s * 4 + e][1] = fmaf(from_digits<PASSES>(acc, 1), unit, o[s * 4 + e][1]);
                    }
                }
                __syncwarp();
                phase ^= 1u << slot;
            } else if (next) {
                copy(keys, next, sh.kpart, &kfull[slot]);
            }
            if (next) copy(values, next + sh.kpart, sh.vpart, &vfull[slot]);
            there = (there & ~(1u << slot)) | (next ? 1u << slot : 0u);
            slot = slot + 1 == depth ? 0 : slot + 1;
        }

        l += __shfl_xor_sync(0xffffffffu, l, 1);
        l += __shfl_xor_sync(0xffffffffu, l, 2);
        if (alone) {
            if (a.team > 1) {  // the team's results to its first warp, by way of the others' first slot, which is free (32 * padded vdim bytes, and the scales' place)
                float* mine = reinterpret_cast<float*>(vbuf);
                if (in_team > 0) {
                    if (tig == 0) *reinterpret_cast<float2*>(mine + PAIRS * sh.vp + 2 * gid) = make_float2(mx, l);
#pragma unroll
                    for (int s = 0; s < VS * 4; ++s)
                        if (s < vslabs * 4) *reinterpret_cast<float2*>(mine + gid * sh.vp + 8 * (s ^ (gid & 3)) + 2 * tig) = make_float2(o[s][0], o[s][1]);
                }
                good = !team_any(team, a.team * 32, !good);
                if (in_team == 0) {
                    for (int w = 1; w < a.team; ++w) {
                        const float* from = reinterpret_cast<const float*>(vbuf + (size_t)w * depth * (sh.kpart + sh.vpart));
                        const float2 ml = *reinterpret_cast<const float2*>(from + PAIRS * sh.vp + 2 * gid);
                        const float now = fmaxf(mx, ml.x), ref = now == -INFINITY ? 0.f : now, f0 = exp2f(mx - ref), f1 = exp2f(ml.x - ref);
                        l = fmaf(l, f0, ml.y * f1);
                        mx = now;
#pragma unroll
                        for (int s = 0; s < VS * 4; ++s) {
                            if (s >= vslabs * 4) break;
                            const float2 x = *reinterpret_cast<const float2*>(from + gid * sh.vp + 8 * (s ^ (gid & 3)) + 2 * tig);
                            o[s][0] = fmaf(o[s][0], f0, x.x * f1);
                            o[s][1] = fmaf(o[s][1], f0, x.y * f1);
                        }
                    }
                }
                team_any(team, a.team * 32, false);  // they have been read
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // pieces are copied there again
                __syncwarp();
                if (in_team > 0) continue;
            }
            if (!waited) pdl_wait();  // the parts of the prefix are there
            waited = true;
            if (a.prefix_n) add_prefix_to<VS>(a, sh.vp, kvh, sg.m * group + tile * PAIRS + min(gid, pairs - 1), tig, mx, l, o);
            const float inv = l == 0.f ? 0.f : 1.0f / l;
#pragma unroll
            for (int s = 0; s < VS * 4; ++s)
                if (s < vslabs * 4 && gid < pairs) kv8_store2<BF16>(a, sg.m, head0 + gid, 8 * s + 2 * tig, o[s][0] * inv, o[s][1] * inv, wide & 1);
            continue;
        }
        // ---- the warps' results added up: `slots` warps at a time to those of the first `slots` warps, then these ----
        const int room = pairs <= 2 ? 2 : pairs <= 4 ? 4 : PAIRS, slots = min(WARPS, MERGE_ROWS / room);
        const int row = warp % slots * room + gid;
        float* mine = merge + (size_t)row * sh.ldo + tig * 2;
        auto put = [&]() {
            if (gid >= pairs) return;
            if (tig == 0) {
                s_m[row] = mx;
                s_l[row] = l;
            }
#pragma unroll
            for (int s = 0; s < VS * 4; ++s) {
                if (s >= vslabs * 4) break;
                *reinterpret_cast<float2*>(mine + s * 8) = make_float2(o[s][0], o[s][1]);
            }
        };
        if (begin > 0)  // the sums of the segment in front have been read by all
            good = __all_sync(0xffffffffu, mb_wait(&s_added, turn ^ 1, a.err_flag, &s_abort)) && good;
        for (int w0 = slots; w0 < WARPS; w0 += slots) {
            if (warp >= w0 && warp < w0 + slots) put();
            __syncthreads();
            if (warp < slots && warp + w0 < WARPS && gid < pairs) {
                const float om = s_m[row], now = fmaxf(mx, om), ref = now == -INFINITY ? 0.f : now, f0 = exp2f(mx - ref), f1 = exp2f(om - ref);
                l = fmaf(l, f0, s_l[row] * f1);
                mx = now;
#pragma unroll
                for (int s = 0; s < VS * 4; ++s) {
                    if (s >= vslabs * 4) break;
                    const float2 x = *reinterpret_cast<const float2*>(mine + s * 8);
                    o[s][0] = fmaf(o[s][0], f0, x.x * f1);
                    o[s][1] = fmaf(o[s][1], f0, x.y * f1);
                }
            }
            __syncthreads();
        }
        if (warp < slots) put();
        if (!last && warp < PAIRS) {
            const float f = put_query(next_q, warp, queries + (turn ^ 1) * sh.queries);
            if (lane == 0) s_c[turn ^ 1][warp] = f;
        }
        __syncthreads();
        const bool whole = sg.n == sg.of;
        float* part = cta_part(a, sh.vp, blockIdx.x, sg.at == 0);
        if (!waited) pdl_wait();  // the parts of the prefix are there
        waited = true;
        for (int k = tid; k < pairs * (sh.vp / 4); k += THREADS) {
            const int pr = k / (sh.vp / 4), d = (k - pr * (sh.vp / 4)) * 4;
            float top = -INFINITY, sum = 0.f, v[4] = {0.f, 0.f, 0.f, 0.f};
            for (int w = 0; w < slots; ++w) top = fmaxf(top, s_m[w * room + pr]);
            const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll 4
            for (int w = 0; w < slots; ++w) {
                const float f = exp2f(s_m[w * room + pr] - ref);
                const float4 x = *reinterpret_cast<const float4*>(merge + (size_t)(w * room + pr) * sh.ldo + d);
                v[0] = fmaf(f, x.x, v[0]); v[1] = fmaf(f, x.y, v[1]); v[2] = fmaf(f, x.z, v[2]); v[3] = fmaf(f, x.w, v[3]);
                sum = fmaf(f, s_l[w * room + pr], sum);
            }
            if (whole) {
                if (a.prefix_n) add_prefix(a, sh.vp, kvh, sg.m * group + tile * PAIRS + pr, d, top, sum, v);
                const float inv = sum == 0.f ? 0.f : 1.0f / sum;
                kv8_store2<BF16>(a, sg.m, head0 + pr, d, v[0] * inv, v[1] * inv, wide & 1);
                kv8_store2<BF16>(a, sg.m, head0 + pr, d + 2, v[2] * inv, v[3] * inv, wide & 1);
            } else {
                float* at = part + (size_t)pr * (sh.vp + 4);
                *reinterpret_cast<float4*>(at + 4 + d) = make_float4(v[0], v[1], v[2], v[3]);
                if (d == 0) {
                    at[0] = top;
                    at[1] = sum;
                }
            }
        }
        __syncwarp();
        if (lane == 0) mb_arrive(&s_added);
        begin += sg.n;
        turn ^= 1;
        sg = behind;
        len = len_behind;
    }
    if (!waited) pdl_wait();  // kv8_join_kernel waits for this launch alone
    // every copy has been waited for, unless a wait ran out: then what is still on its way has to land before this CTA's shared memory is another's
    if (!good)
        for (int s = 0; s < depth; ++s) {
            if (!((there >> s) & 1u)) continue;
            mb_land(&kfull[s], (phase >> s) & 1u);
            mb_land(&vfull[s], (phase >> s) & 1u);
        }
}

// One column of CTAs per cut of the line: the item that a cut falls into, if the CTA in front of the cut holds its beginning; a CTA has JOIN_PAIRS of its pairs.  A long context has a
// hundred parts and more: the warps share them, every lane with its elements of several parts in flight at once.  The CTAs behind those have rows that have nothing but the prefix.
constexpr int JOIN_THREADS = 256, JOIN_PAIRS = 2, JOIN_HEADS = 4;
template <bool BF16, int VS>
__global__ void __launch_bounds__(JOIN_THREADS) kv8_join_kernel(const Kv8AttnArgs a, int ctas, int tiles, int wide) {  // ctas: one more than cuts
    constexpr int THREADS = JOIN_THREADS, JW = THREADS / 32, NI = JOIN_PAIRS * VS * 8 / 32, AHEAD = 4;  // warps; groups of four elements a lane; parts in flight
    extern __shared__ __align__(128) unsigned char dyn[];                                               // factors [parts][JOIN_PAIRS], then the warps' sums
    __shared__ float s_top[JOIN_PAIRS], s_sum[JOIN_PAIRS];
    __shared__ long long first[THREADS + 1];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, items = a.pool.kv_heads * tiles, group = a.heads / a.pool.kv_heads, cut = blockIdx.x + 1, vp = kv8_pad(a.pool.vdim), quads = vp / 4;
    if (cut >= ctas) {
        pdl_wait();
        // a warp to JOIN_HEADS heads of all rows at a time, four elements a lane
        const int all = a.M * a.heads, step = ((int)gridDim.x - (ctas - 1)) * (int)gridDim.y * JW * JOIN_HEADS;
        const size_t all_pairs = (size_t)a.M * group, part = (size_t)a.pool.kv_heads * all_pairs * (vp + 4);
        for (int k = ((((cut - ctas) * (int)gridDim.y + (int)blockIdx.y) * JW) + warp) * JOIN_HEADS; k < all; k += step) {
            int m[JOIN_HEADS], head[JOIN_HEADS];
            const float* at[JOIN_HEADS];
            bool is[JOIN_HEADS];
#pragma unroll
            for (int j = 0; j < JOIN_HEADS; ++j) {
                const int r = min(k + j, all - 1);
                m[j] = r / a.heads;
                head[j] = r - m[j] * a.heads;
                const int kvh = head[j] / group;
                at[j] = a.prefix + ((size_t)kvh * all_pairs + (size_t)m[j] * group + (head[j] - kvh * group)) * (vp + 4);
                is[j] = k + j < all && kv8_row_pieces(a, m[j]) == 0 && (unsigned)__ldg(a.row_seq + m[j]) < (unsigned)a.pool.n_seq;
            }
            for (int d = 4 * lane; d < vp; d += 128) {
                float top[JOIN_HEADS], sum[JOIN_HEADS];
                float4 v[JOIN_HEADS];
#pragma unroll
                for (int j = 0; j < JOIN_HEADS; ++j) {
                    top[j] = -INFINITY;
                    sum[j] = 0.f;
                    v[j] = make_float4(0.f, 0.f, 0.f, 0.f);
                }
                for (int i = 0; i < a.prefix_n; ++i) {
                    float2 ml[JOIN_HEADS];
                    float4 x[JOIN_HEADS];
#pragma unroll
                    for (int j = 0; j < JOIN_HEADS; ++j) {
                        ml[j] = is[j] ? __ldcg(reinterpret_cast<const float2*>(at[j] + i * part)) : make_float2(-INFINITY, 0.f);
                        x[j] = is[j] ? __ldcg(reinterpret_cast<const float4*>(at[j] + i * part + 4 + d)) : make_float4(0.f, 0.f, 0.f, 0.f);
                    }
#pragma unroll
                    for (int j = 0; j < JOIN_HEADS; ++j) {
                        if (ml[j].x == -INFINITY) continue;  // nothing seen
                        const float now = fmaxf(top[j], ml[j].x), r0 = exp2f(0.5f * (top[j] - now)), r1 = exp2f(0.5f * (ml[j].x - now)), f0 = r0 * r0, f1 = r1 * r1;
                        top[j] = now;
                        sum[j] = fmaf(r1 * ml[j].y, r1, sum[j] * r0 * r0);
                        v[j].x = fmaf(f1, x[j].x, v[j].x * f0); v[j].y = fmaf(f1, x[j].y, v[j].y * f0); v[j].z = fmaf(f1, x[j].z, v[j].z * f0); v[j].w = fmaf(f1, x[j].w, v[j].w * f0);
                    }
                }
#pragma unroll
                for (int j = 0; j < JOIN_HEADS; ++j) {
                    if (!is[j]) continue;
                    const float inv = sum[j] == 0.f ? 0.f : 1.0f / sum[j];
                    kv8_store2<BF16>(a, m[j], head[j], d, v[j].x * inv, v[j].y * inv, wide & 1);
                    kv8_store2<BF16>(a, m[j], head[j], d + 2, v[j].z * inv, v[j].w * inv, wide & 1);
                }
            }
        }
        return;
    }
    const Line line = make_line<THREADS>(a, items, ctas, first);
    const long long u = cut * line.chunk;
    bool mine = u < line.total;
    long long begin = 0, before;
    Segment sg{};
    if (mine) {
        sg = unit_at<THREADS>(a, first, items, u, begin, before);
        mine = sg.at > 0 && (begin + BEGIN) / line.chunk == cut - 1;
    }
    const int kvh = sg.item / tiles, tile = sg.item - kvh * tiles, pr0 = (int)blockIdx.y * JOIN_PAIRS, pairs = min(JOIN_PAIRS, min(PAIRS, group - tile * PAIRS) - pr0), head0 = kvh * group + tile * PAIRS + pr0;
    const int parts = mine ? (int)((begin + BEGIN + sg.of - 1) / line.chunk) - (cut - 1) + 1 : 0;
    pdl_wait();
    if (!mine || pairs <= 0) return;
    // the beginning is the second part of its CTA, what follows the first of theirs
    auto part = [&](int i) -> const float* { return cta_part(a, vp, cut - 1 + i, i == 0) + (size_t)pr0 * (vp + 4); };
    float2* ml = reinterpret_cast<float2*>(dyn);  // reference and sum, then factor and sum
    float4* sums = reinterpret_cast<float4*>(dyn + (sizeof(float2) * JOIN_PAIRS * parts + 15) / 16 * 16);  // [JW][NI * 32]
    for (int k = tid; k < parts * JOIN_PAIRS; k += THREADS) ml[k] = k % JOIN_PAIRS < pairs ? __ldcg(reinterpret_cast<const float2*>(part(k / JOIN_PAIRS) + (size_t)(k % JOIN_PAIRS) * (vp + 4))) : make_float2(-INFINITY, 0.f);
    float4 acc[NI], x[AHEAD][NI];
    int off[NI];  // where a lane's groups stand in a part
#pragma unroll
    for (int n = 0; n < NI; ++n) {
        const int k = lane + 32 * n, pr = k / quads;
        acc[n] = make_float4(0.f, 0.f, 0.f, 0.f);
        off[n] = pr < pairs ? pr * (vp + 4) + 4 + (k - pr * quads) * 4 : -1;
    }
    auto fetch = [&](int i0) {
#pragma unroll
        for (int j = 0; j < AHEAD; ++j)
#pragma unroll
            for (int n = 0; n < NI; ++n) x[j][n] = i0 + j * JW < parts && off[n] >= 0 ? __ldcg(reinterpret_cast<const float4*>(part(i0 + j * JW) + off[n])) : make_float4(0.f, 0.f, 0.f, 0.f);
    };
    fetch(warp);  // on their way while the references are compared
    __syncthreads();
    if (warp < JOIN_PAIRS) {  // warp w: pair w
        float top = -INFINITY, sum = 0.f;
        for (int i = lane; i < parts; i += 32) top = fmaxf(top, ml[i * JOIN_PAIRS + warp].x);
        top = warp_max(top);
        const float ref = top == -INFINITY ? 0.f : top;
        for (int i = lane; i < parts; i += 32) {
            const float2 y = ml[i * JOIN_PAIRS + warp];
            const float f = exp2f(y.x - ref);
            ml[i * JOIN_PAIRS + warp].x = f;
            sum = fmaf(f, y.y, sum);
        }
        sum = warp_sum(sum);
        if (lane == 0) {
            s_top[warp] = top;
            s_sum[warp] = sum;
        }
    }
    __syncthreads();
    for (int i0 = warp; i0 < parts; i0 += AHEAD * JW) {
        if (i0 > warp) fetch(i0);
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
            if (i0 + j * JW >= parts) break;
#pragma unroll
            for (int n = 0; n < NI; ++n) {
                const float f = ml[(i0 + j * JW) * JOIN_PAIRS + min((lane + 32 * n) / quads, JOIN_PAIRS - 1)].x;
                acc[n].x = fmaf(f, x[j][n].x, acc[n].x); acc[n].y = fmaf(f, x[j][n].y, acc[n].y); acc[n].z = fmaf(f, x[j][n].z, acc[n].z); acc[n].w = fmaf(f, x[j][n].w, acc[n].w);
            }
        }
    }
#pragma unroll
    for (int n = 0; n < NI; ++n) sums[(warp * NI + n) * 32 + lane] = acc[n];
    __syncthreads();
    for (int k = tid; k < pairs * quads; k += THREADS) {
        const int pr = k / quads, d = (k - pr * quads) * 4;
        float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < JW; ++w) {
            const float4 y = sums[w * NI * 32 + k];
            v[0] += y.x; v[1] += y.y; v[2] += y.z; v[3] += y.w;
        }
        float top = s_top[pr], sum = s_sum[pr];
        if (a.prefix_n) add_prefix(a, vp, kvh, sg.m * group + tile * PAIRS + pr0 + pr, d, top, sum, v);
        const float inv = sum == 0.f ? 0.f : 1.0f / sum;
        kv8_store2<BF16>(a, sg.m, head0 + pr, d, v[0] * inv, v[1] * inv, wide & 1);
        kv8_store2<BF16>(a, sg.m, head0 + pr, d + 2, v[2] * inv, v[3] * inv, wide & 1);
    }
}

template <typename... KArgs, typename... Args>
cudaError_t launch_behind(void (*kern)(KArgs...), dim3 grid, int threads, size_t smem, cudaStream_t st, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
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

template <bool BF16, int VS, int WARPS>
cudaError_t launch_stream(const Kv8AttnArgs& a_in, int sm_count, cudaStream_t st) {
    Kv8AttnArgs a = a_in;
    const int group = a.heads / a.pool.kv_heads, tiles = (group + PAIRS - 1) / PAIRS, ctas = sm_count;
    const int wide = kv8_wide(a);
    auto bytes = [&](int depth) { return stream_shape(a.pool.dim, a.pool.vdim, BF16 ? 1 : 2, WARPS, depth).bytes; };
    int depth = MAX_DEPTH;
    while (depth > 1 && bytes(depth) > ROOM) --depth;
    // where there are more items than CTAs, a CTA would take them one by one
    const long all = (long)a.M * a.pool.kv_heads * tiles, most = std::max(0l, (long)a.pool.max_pages * (KV8_PAGE / KV8_HALF) - a.own_from);  // items; pieces of one
    a.team = 1;
    for (int t = 2; t <= 4; ++t)
        if (WARPS % t == 0 && all <= (long)ctas * (WARPS / t)) a.team = t;
    const long no_line = std::min(TEAM_PIECES * a.team, MOST_TEAM_PIECES);
    a.solo = all <= ctas ? 0 : most <= no_line ? (int)no_line : SOLO;
    a.whole = all <= ctas && most <= WHOLE;
    const bool own = most > 0 || a.prefix_n == 0, cut = own && !a.whole && most > a.solo, rest = a.prefix_n > 0 && !a.direct;
    const size_t smem = bytes(depth), join_smem = sizeof(float2) * JOIN_PAIRS * ctas + 16 + sizeof(float) * JOIN_THREADS * JOIN_PAIRS * VS;
    cudaError_t e = ensure_dyn_smem(kv8_stream_kernel<BF16, VS, WARPS>, smem);
    if (e == cudaSuccess) e = ensure_dyn_smem(kv8_join_kernel<BF16, VS>, join_smem);
    if (e != cudaSuccess) return e;
    if (own && a.prefix_n) {
        e = launch_behind(kv8_stream_kernel<BF16, VS, WARPS>, dim3((unsigned)ctas), WARPS * 32, smem, st, a, depth, tiles, wide);
    } else if (own) {
        kv8_stream_kernel<BF16, VS, WARPS><<<(unsigned)ctas, WARPS * 32, smem, st>>>(a, depth, tiles, wide);
        e = cudaGetLastError();
    }
    if (e != cudaSuccess || !(cut || rest)) return e;
    // a column of CTAs for every cut, then those of the rows that have nothing but the prefix
    const int columns = (std::min(group, PAIRS) + JOIN_PAIRS - 1) / JOIN_PAIRS, cuts = cut ? ctas - 1 : 0, at_once = JOIN_THREADS / 32 * JOIN_HEADS * columns;
    const long more = rest ? std::min(((long)a.M * a.heads + at_once - 1) / at_once, 4096l) : 0;
    return launch_behind(kv8_join_kernel<BF16, VS>, dim3((unsigned)(cuts + more), (unsigned)columns), JOIN_THREADS, join_smem, st, a, cuts + 1, tiles, wide);
}

// 12 warps (168 registers a thread) where their pieces fit, else eight.
template <bool BF16, int VS>
cudaError_t launch_warps(const Kv8AttnArgs& a, int sm_count, cudaStream_t st) {
    auto fits = [&](int warps) { return stream_shape(a.pool.dim, a.pool.vdim, BF16 ? 1 : 2, warps, 1).bytes <= ROOM; };
    if constexpr (VS <= 4)
        if (fits(12)) return launch_stream<BF16, VS, 12>(a, sm_count, st);
    return launch_stream<BF16, VS, 8>(a, sm_count, st);
}

template <bool BF16>
cudaError_t launch_typed(const Kv8AttnArgs& a, int sm_count, cudaStream_t st) {
    if (a.pool.vdim <= 64) return launch_warps<BF16, 2>(a, sm_count, st);
    if (a.pool.vdim <= 128) return launch_warps<BF16, 4>(a, sm_count, st);
    return launch_warps<BF16, 8>(a, sm_count, st);
}

}  // namespace

// `work`: parts of the line's cuts, then those of the prefix, then its sums.
static size_t line_floats(int vdim, int sm_count) { return 2 * (size_t)sm_count * part_floats(kv8_pad(vdim)); }
static size_t parts_floats(int kv_heads, int vdim, int M, int heads, int n_shared, int sm_count) { return (size_t)kv8_prefix_most_parts(kv_heads, M, heads, n_shared, sm_count) * M * heads * (kv8_pad(vdim) + 4); }

size_t kv8_attn_bytes(int kv_heads, int dim, int vdim, int M, int heads, int n_shared, int sm_count) {
    // rows of either type
    const Kv8Prefix p = kv8_prefix_plan(kv_heads, dim, vdim, 0, M, heads, n_shared, sm_count), q = kv8_prefix_plan(kv_heads, dim, vdim, 1, M, heads, n_shared, sm_count);
    return sizeof(float) * (line_floats(vdim, sm_count) + (p.parts ? parts_floats(kv_heads, vdim, M, heads, n_shared, sm_count) + std::max(p.sums, q.sums) : 0));
}

cudaError_t launch_kv8_attn(const Kv8AttnArgs& a_in, int sm_count, cudaStream_t st) {
    Kv8AttnArgs a = a_in;
    const Kv8Prefix p = kv8_prefix_plan(a.pool.kv_heads, a.pool.dim, a.pool.vdim, a.bf16, a.M, a.heads, a.n_shared, sm_count);
    a.own_from = 0;
    a.prefix_n = p.parts;
    a.direct = p.parts == 1;
    if (p.parts) {
        float* parts = static_cast<float*>(a.work) + line_floats(a.pool.vdim, sm_count);
        a.own_from = a.n_shared * (KV8_PAGE / KV8_HALF);
        const cudaError_t e = launch_kv8_prefix(a, p, parts, parts + parts_floats(a.pool.kv_heads, a.pool.vdim, a.M, a.heads, a.n_shared, sm_count), st);
        if (e != cudaSuccess) return e;
        a.prefix = parts;
    }
    return a.bf16 ? launch_typed<true>(a, sm_count, st) : launch_typed<false>(a, sm_count, st);
}

}  // namespace hm

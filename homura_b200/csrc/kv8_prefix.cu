// The shared pages of kv8_attn on the 5th-generation tensor cores: scores and sums of all rows over a prefix that is read once for 128 or 256 (row, head) pairs.
//
// Per block of 128 tokens (two pages), for 128 pairs of one key/value head, with f32 sums in tensor memory:
//   S [128 pairs x 128 tokens] = Q [128 x dim] . K^T         Q, K in shared memory
//   O [128 pairs x vdim]      += P [128 x 128 tokens] . V    P in tensor memory, where S was; V in shared memory, element by token
// Codes are whole numbers below 128, exact in f16.  A query row enters times a power of two (largest element 2^14 .. 2^15): a bf16 row is exact in one f16 term down to 2^-30 of
// its largest element, an f32 row takes two terms (2^-22 of a value).  A token's key scale joins the scores, its value scale the weights: P = 2^(s - ref) * scale enters as f16 in one
// term (2^-11 of itself) for bf16 rows, in two for f32 rows.  `ref` is a pair's reference in the units of P: it follows the largest s + log2(scale) of the tokens that the pair sees,
// with some room (2^8), so that O in tensor memory is hardly ever multiplied.  What other pairs see, and values whose own weights are next to nothing, have no part in it.  P is 2^15
// at most, and its smallest step, 2^-24, is 2^-31 of the largest product or less.  Scales count as 2^-100 at least and sums of weights, which are relative to the same
// reference, as 2^-20 of theirs, so that these stay finite.  Weights below 2^-126 of the reference are zero, which values above 2^100 bring near the largest.
//
// 24 warps: 0 .. 7 and 8 .. 15 turn scores into weights, two threads for every pair, a page each; 16 .. 18 make f16 of keys' codes, 19 .. 21 of values'; 22 copies pages; 23 issues the MMAs.  Two streams of
// blocks take turns on the tensor cores, so that one's MMAs run beside the other's exponentials: the two halves of 256 pairs over the same blocks (a block's codes are then converted once
// for both), or, for fewer pairs and f32 rows, whose two terms leave room for one tile of queries, the even and the odd blocks of 128 pairs.  Weights stand where their scores were; where
// two results of 64 elements leave room, a third place lets a stream's next scores come while its weights are still multiplied (256 rows of 32 heads behind 16384 tokens: 5 us less).
// The token axis is split where there are too few pairs for all SMs; splits form clusters that join what they have over their shared memory.  A row that has nothing but the prefix is then
// done, where that leaves one part; others, and further parts, go to `work`, relative to their references, to be joined with the rows' own pages.
//
// What bounds it: the instructions of the softmax.  256 rows of 32 heads over 4 of 64 elements: the schedulers issue in 7 of 10 cycles; exponentials fill 2050 cycles of a block of 256 pairs, the tensor
// cores 730; 117 us in all, 294 TFLOP/s.  A block took 4700 cycles and the whole 106 us while references followed scores alone: value scales in them cost one operation for two scores and the
// loads of their logarithms (8 us), counting from an origin a vote per block (1.5 us).  With 128 elements a block takes 7000, as the only place for keys is converted (4000)
// between two blocks' scores: 1021 rows of 12 heads, 91 us, the schedulers issue in 6 of 10.  Found slower, against 106 and 87 us: two places for keys and one for values (109 us for the
// 1021 rows); a pass that finds no maximum and is done again where a score exceeds its reference by too much, which a quarter of the blocks does with heavy-tailed scores; all six converting
// warps on keys, then on values (the 256 rows 117 us); a fourth warp for keys, which leaves 72 registers a thread (109 us there, 86 for the 1021 rows).
#include <algorithm>
#include <map>
#include <mutex>
#include <type_traits>
#include <utility>

#include "kv8.h"
#include "kv8_rows.cuh"
#include "launch_attrs.h"
#include "mbarrier.cuh"

namespace hm {
namespace {

constexpr int TILE = 128, BLOCK = 128;  // pairs of a tile, tokens of a block
constexpr int SOFT_WARPS = 16, CONV_WARPS = 3, THREADS = 768;  // those of keys, as many of values
constexpr int COPY_WARP = SOFT_WARPS + 2 * CONV_WARPS, MMA_WARP = COPY_WARP + 1;
constexpr int STREAM_WARPS = SOFT_WARPS / 2;
constexpr int MAX_RAW = 8;              // pages in flight or being converted
constexpr int RING = 5;                 // blocks whose scales are kept
constexpr int MOST_BUFS = 3;            // of scores
// Pieces of the streaming kernel (32 shared tokens, eight pairs) that take it as long as this kernel and its join.  us here / there at 16384, 24576 and 32768 pieces, rows of 16 heads over 2:
//   100 own tokens      64 rows              128 rows             256 rows             512 rows
//   bf16,  64 elements  33/31 34/36 37/42    30/26 35/39 38/45    33/22 30/29 36/35    30/28 32/36 32/45
//   bf16, 128 elements  41/36 42/44 45/51    40/33 45/47 49/54    42/29 40/37 45/45    39/36 42/47 42/58
//   f32,   64 elements  29/34 34/41 38/47    29/29 31/43 36/50    28/25 30/33 32/41    29/32 31/42 33/52
//   f32,  128 elements  38/41 43/52 49/61    38/39 42/55 47/64    36/35 39/47 43/58    37/44 40/58 43/72
//   none
//   bf16,  96 elements  30/34 31/41 34/48    26/29 29/39 33/50    26/24 25/32 29/40    22/28 25/39 25/49
//   f32,   64 elements  22/33 26/40 30/47    20/28 22/38 26/49    18/23 20/31 22/39    17/27 19/37 21/47
// One limit for all of them, where bf16 rows with tokens of their own gain but for 256 rows; f32 rows and rows without own tokens gain from fewer pieces on, at most sizes from 16384.
constexpr long LEAST_SHARED = 24576;
// Blocks of a stream whose products are one sum in tensor memory.  Its steps round towards zero, and values of one sign gather that: 1024 steps (64 blocks of f32 rows, whose two terms take 16
// steps each) 5.3e-5, 4096 of them 2.1e-4.  After 64 steps of f32 rows, 512 of bf16 rows, a thread adds what its pair has to f32 sums in `work`: 1.3e-6 at any length of f32 rows, which
// take 3 to 8 % longer for it (256 rows of 32 heads of 64 behind 16384 tokens 144 -> 150 us, 1021 rows of 32 heads of 128 there 810 -> 879).
__host__ __device__ constexpr int chunk_of(int terms) { return terms == 2 ? 4 : 64; }
constexpr int MOST_PARTS = 8;           // that are left to be joined with the rows' own pages
constexpr size_t ROOM = 226 * 1024;
constexpr uint32_t STATIC = 12800;      // of which what the kernel declares
constexpr float LOG2E = 1.4426950408889634f;
constexpr float SLACK = 8.f;            // how far a score may exceed its reference, as an exponent
constexpr float DROP = 7.f;             // a weight times its value scale enters as 2^DROP times what it is of the reference: 2^(SLACK + DROP) = 2^15
// Of value scales, in the reference.  A weight is below 2^(100 + SLACK + DROP) then, and a sum of 64 below 2^121; those of 2^23 blocks stay finite as 2^-SUM_DROP of theirs
constexpr float LEAST_LOG = -100.f;
constexpr int SUM_DROP = 20;
constexpr float FAR = 65536.f;          // references from here on are counted from a score, as f32 would leave too little of what is added to it

struct Shape {
    int dp, vp, katoms, kpart, half;  // padded sizes, pieces of 64 elements of keys, bytes of a half's keys, of a half
    int raw, kst, vst;                // pages of the ring, blocks of keys and of values as f16
    int bufs;                         // scores of so many tasks have a place in tensor memory: three where two results of 64 elements leave one more
    uint32_t q_tile, k_tile, v_tile, q_at, k_at, v_at, raw_at, bytes;
};
__host__ __device__ inline Shape shape_of(int dim, int vdim, int terms, int q_tiles) {
    Shape s;
    s.dp = kv8_pad(dim);
    s.vp = kv8_pad(vdim);
    s.katoms = (s.dp + 63) / 64;
    s.kpart = kv8_part_bytes(dim);
    s.half = (int)kv8_half_bytes(dim, vdim);
    s.bufs = s.vp <= 64 ? 3 : 2;
    s.q_tile = (uint32_t)terms * s.katoms * TILE * 128;
    s.k_tile = (uint32_t)s.katoms * BLOCK * 128;
    s.v_tile = 2u * s.vp * 128;
    // two blocks of values, then of keys, where they leave the ring three pages (a block and half of the next); then as many pages as fit
    const uint32_t page = 2u * s.half, room = (uint32_t)ROOM - STATIC - 1024 - q_tiles * s.q_tile;
    s.vst = s.k_tile + 2 * s.v_tile + 3 * page <= room ? 2 : 1;
    s.kst = 2 * s.k_tile + s.vst * s.v_tile + 3 * page <= room ? 2 : 1;
    s.raw = (int)((room - s.kst * s.k_tile - s.vst * s.v_tile) / page);
    if (s.raw > MAX_RAW) s.raw = MAX_RAW;
    s.q_at = 0;
    s.k_at = s.q_at + q_tiles * s.q_tile;
    s.v_at = s.k_at + s.kst * s.k_tile;
    s.raw_at = s.v_at + s.vst * s.v_tile;
    s.bytes = 1024 + s.raw_at + (uint32_t)s.raw * page;
    const uint32_t results = 1024 + 2u * TILE * (s.vp + 4) * 4u;  // the streams' results stand there at the end
    if (s.bytes < results) s.bytes = results;
    return s;
}

struct Shared {
    uint64_t raw_full[MAX_RAW], raw_empty[MAX_RAW], k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[MOST_BUFS], p_full[MOST_BUFS], pv_done[MOST_BUFS], sc_full[RING], q_full, done;
    uint32_t tmem;
    volatile int abort_flag;
    int longest;
    alignas(16) float ks[RING + 1][BLOCK];  // the last row: ones, for scores that have theirs
    alignas(16) float vs[RING][BLOCK];
    alignas(16) float lv[RING][BLOCK];  // log2 of the value scales
    int there[RING];   // bit i: page i of the block exists
    int raw_there[MAX_RAW];
    float half[2][2][2][TILE];  // [stream][turn][page of the block][pair]: what the two threads of a pair tell one another
};
static_assert(sizeof(Shared) <= STATIC, "");

__device__ __forceinline__ uint32_t desc_lo(uint32_t addr) { return ((addr >> 4) & 0x3FFF) | (1u << 16); }
constexpr uint32_t DESC_HI = (1024u >> 4) | (1u << 14) | (2u << 29);  // rows of 128 bytes in groups of eight, 128-byte swizzle
__device__ __forceinline__ uint32_t idesc_f16(int n) { return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(TILE >> 4) << 24); }  // f32 sums of f16, M 128, both K-major
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, bool accumulate) {
    asm volatile("{ .reg .pred p; .reg .b64 da, db; setp.ne.b32 p, %5, 0; mov.b64 da, {%1, %4}; mov.b64 db, {%2, %4};\n"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p; }" ::"r"(d), "r"(a_lo), "r"(b_lo), "r"(idesc), "n"(DESC_HI), "r"((uint32_t)accumulate) : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a_tmem, uint32_t b_lo, uint32_t idesc, bool accumulate) {
    asm volatile("{ .reg .pred p; .reg .b64 db; setp.ne.b32 p, %5, 0; mov.b64 db, {%2, %4};\n"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p; }" ::"r"(d), "r"(a_tmem), "r"(b_lo), "r"(idesc), "n"(DESC_HI), "r"((uint32_t)accumulate) : "memory");
}
__device__ __forceinline__ void mma_commit(uint64_t* bar) { asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(s32(bar)) : "memory"); }
__device__ __forceinline__ void tmem_ld32(uint32_t (&r)[32], uint32_t addr) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
                   "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
                 : "r"(addr));
}
// Names the registers, so that no use of them moves in front of the wait.
__device__ __forceinline__ void tmem_wait(uint32_t (&r)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                   "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
                 :: "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t (&r)[16], uint32_t addr) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(addr));
}
__device__ __forceinline__ void tmem_wait16(uint32_t (&r)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
                 :: "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t (&r)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
                 "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
                 : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ uint32_t elect_lane() {
    uint32_t p;
    asm volatile("{ .reg .pred P; .reg .b32 r; elect.sync r|P, 0xffffffff; selp.u32 %0, 1, 0, P; }" : "=r"(p));
    return p;
}
__device__ __forceinline__ float exp2_ftz(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Two f32 side by side: half the instructions of one by one.
__device__ __forceinline__ uint64_t pair_of(uint32_t lo, uint32_t hi) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(lo), "r"(hi));
    return r;
}
__device__ __forceinline__ uint64_t pair_of(float lo, float hi) { return pair_of(__float_as_uint(lo), __float_as_uint(hi)); }
__device__ __forceinline__ float2 of_pair(uint64_t v) {
    uint32_t lo, hi;
    asm("mov.b64 {%0, %1}, %2;" : "=r"(lo), "=r"(hi) : "l"(v));
    return make_float2(__uint_as_float(lo), __uint_as_float(hi));
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint32_t f16x2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ float f16_lo(uint32_t w) {
    float f;
    asm("{ .reg .b16 l, h; mov.b32 {l, h}, %1; cvt.f32.f16 %0, l; }" : "=f"(f) : "r"(w));
    return f;
}
__device__ __forceinline__ float f16_hi(uint32_t w) {
    float f;
    asm("{ .reg .b16 l, h; mov.b32 {l, h}, %1; cvt.f32.f16 %0, h; }" : "=f"(f) : "r"(w));
    return f;
}
// Four codes as f16: a byte with its sign bit turned becomes the last bits of 1024 + 128 + code, from which 1152 is subtracted.
__device__ __forceinline__ void codes_f16(uint32_t w, uint32_t& a, uint32_t& b) {
    w ^= 0x80808080u;
    const uint32_t x = __byte_perm(w, 0x64646464u, 0x4140), y = __byte_perm(w, 0x64646464u, 0x4342);
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(a) : "r"(x), "r"(0x64806480u));
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(b) : "r"(y), "r"(0x64806480u));
}

// Barrier of the two warps that share 32 pairs, with an OR over their predicates.
__device__ __forceinline__ bool both_any(int id, bool v) {
    uint32_t r;
    asm volatile("{ .reg .pred p, q; setp.ne.u32 p, %1, 0; barrier.cta.red.or.aligned.pred q, %2, 64, p; selp.u32 %0, 1, 0, q; }" : "=r"(r) : "r"((uint32_t)v), "r"(1 + id) : "memory");
    return r != 0;
}

// TERMS: f16 terms of queries and weights; PAIRED: the streams are two tiles of pairs over the same blocks.
template <bool BF16, int TERMS, bool PAIRED>
__global__ void __launch_bounds__(THREADS, 1) kv8_prefix_kernel(const Kv8AttnArgs a, int splits, int cluster, float* parts, float4* sums, int wide) {
    constexpr int CHUNK = chunk_of(TERMS);
    extern __shared__ __align__(128) unsigned char dsm[];
    __shared__ Shared sh;
    const Shape g = shape_of(a.pool.dim, a.pool.vdim, TERMS, PAIRED ? 2 : 1);
    unsigned char* base = dsm + ((1024u - (s32(dsm) & 1023u)) & 1023u);  // swizzled tiles need 1024-byte alignment
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, kvh = blockIdx.y, split = blockIdx.x % splits, tiles0 = blockIdx.x / splits * (PAIRED ? 2 : 1);
    const int group = a.heads / a.pool.kv_heads, pairs = a.M * group, ldo = g.vp + 4;
    pdl_launch_dependents();
    if (tid < BLOCK) sh.ks[RING][tid] = 1.f;
    if (tid == 0) {
        for (int s = 0; s < g.raw; ++s) {
            mb_init(&sh.raw_full[s], 1);
            mb_init(&sh.raw_empty[s], 2 * CONV_WARPS);
        }
        for (int s = 0; s < 2; ++s) {
            mb_init(&sh.k_full[s], CONV_WARPS);
            mb_init(&sh.k_empty[s], 1);
            mb_init(&sh.v_full[s], CONV_WARPS);
            mb_init(&sh.v_empty[s], 1);
        }
        for (int s = 0; s < MOST_BUFS; ++s) {
            mb_init(&sh.s_full[s], 1);
            mb_init(&sh.p_full[s], STREAM_WARPS);
            mb_init(&sh.pv_done[s], 1);
        }
        for (int s = 0; s < RING; ++s) mb_init(&sh.sc_full[s], CONV_WARPS);
        mb_init(&sh.q_full, SOFT_WARPS);
        mb_init(&sh.done, 1);
        sh.abort_flag = 0;
        sh.longest = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    // ---- the pair of a thread of the first warps, and how far it sees; its page of the blocks ----
    const int stream = (warp >> 3) & 1, side = (warp >> 2) & 1, tile = tiles0 + (PAIRED ? stream : 0), pair = tile * TILE + (tid & (TILE - 1));
    const bool mine = warp < SOFT_WARPS && pair < pairs;
    const int row = mine ? pair / group : 0;
    int len = 0;
    if (mine) {
        len = max(0, min(kv8_row_len(a, row), a.n_shared * KV8_PAGE));
    }
    {
        const int most = __reduce_max_sync(0xffffffffu, len);
        if (lane == 0 && warp < SOFT_WARPS) atomicMax(&sh.longest, most);
    }
    if (warp == MMA_WARP) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(s32(&sh.tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh.tmem, o_at0 = tmem + (uint32_t)g.bufs * BLOCK, o_step = g.bufs == 2 ? 128u : 64u;  // the streams' results, behind the scores
    const int longest = sh.longest, nb = (longest + BLOCK - 1) / BLOCK, per = (nb + splits - 1) / splits, b0 = min(nb, split * per), n = min(nb, b0 + per) - b0;  // this CTA's blocks
    const int tasks = PAIRED ? 2 * n : n;  // task j belongs to stream j & 1
    auto block_of = [&](int j) { return PAIRED ? j >> 1 : j; };  // counted from b0

    if (warp == COPY_WARP) {
        const int pages = min(a.n_shared - 2 * b0, 2 * n);
        bool ok = true;
        uint32_t i = 0;
        for (int p0 = 0; p0 < 2 * n && ok; p0 += 32) {
            const int id = p0 + lane < pages ? __ldg(a.shared + 2 * b0 + p0 + lane) : -1;
            for (int j = 0; j < min(32, 2 * n - p0); ++j, ++i) {
                const int page = __shfl_sync(0xffffffffu, id, j), s = (int)(i % g.raw);
                if (i >= (uint32_t)g.raw && !__all_sync(0xffffffffu, mb_wait(&sh.raw_empty[s], ((i / g.raw) & 1u) ^ 1u, a.err_flag, &sh.abort_flag))) {
                    ok = false;
                    break;
                }
                if (lane == 0) {
                    const bool there = (unsigned)page < (unsigned)a.pool.n_pages;
                    sh.raw_there[s] = there;
                    if (there) {
                        mb_expect_tx(&sh.raw_full[s], 2u * g.half);
                        bulk_copy(base + g.raw_at + (size_t)s * 2 * g.half, a.pool.pages + ((size_t)page * a.pool.kv_heads + kvh) * (size_t)(2 * g.half), 2u * g.half, &sh.raw_full[s]);
                    } else {
                        mb_arrive(&sh.raw_full[s]);  // what the slot holds is converted again, and not seen
                    }
                }
                __syncwarp();
            }
        }
        if (lane == 0) mb_land_ring(sh.raw_full, i, (uint32_t)g.raw);
    } else if (warp == MMA_WARP) {
        const uint32_t lead = elect_lane();
        const uint32_t id_s = idesc_f16(BLOCK), id_o = idesc_f16(g.vp);
        const uint32_t q_lo = desc_lo(s32(base + g.q_at)), k_lo = desc_lo(s32(base + g.k_at)), v_lo = desc_lo(s32(base + g.v_at));
        auto wait = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, mb_wait(bar, parity, a.err_flag, &sh.abort_flag)); };
        bool ok = tasks == 0 || wait(&sh.q_full, 0);
        int buf = 0;      // task j and the one `bufs` in front of it have the same place
        uint32_t turn = 0;  // j / bufs
        for (int j = 0; j < tasks + g.bufs && ok; ++j) {
            const uint32_t d_s = tmem + (uint32_t)buf * BLOCK;
            if (j >= g.bufs) {  // the product of that task; the first of a chunk begins with zeros
                const int t = j - g.bufs, b = block_of(t), s = t & 1;
                const uint32_t d_o = o_at0 + (uint32_t)s * o_step;
                const int vs = b & (g.vst - 1);  // one stage or two
                if ((!PAIRED || s == 0) && !(ok = wait(&sh.v_full[vs], (b >> (g.vst - 1)) & 1))) break;
                if (!(ok = wait(&sh.p_full[buf], (turn - 1) & 1))) break;
                tc_fence_after();
                const uint32_t v = v_lo + (uint32_t)vs * (g.v_tile / 16);
                if (lead) {
#pragma unroll
                    for (int h = 0; h < TERMS; ++h)
#pragma unroll
                        for (int k = 0; k < BLOCK / 16; ++k)
                            mma_ts(d_o, d_s + (k >> 1) * 32 + h * 16 + (k & 1) * 8, v + (uint32_t)(k >> 2) * (g.v_tile / 32) + (k & 3) * 2, id_o, ((t >> 1) & (CHUNK - 1)) != 0 || h > 0 || k > 0);
                    mma_commit(&sh.pv_done[buf]);
                    if (!PAIRED || s == 1) mma_commit(&sh.v_empty[vs]);
                }
                __syncwarp();
            }
            if (j < tasks) {
                const int b = block_of(j), s = j & 1;
                const int ks = b & (g.kst - 1);
                if ((!PAIRED || s == 0) && !(ok = wait(&sh.k_full[ks], (b >> (g.kst - 1)) & 1))) break;
                if (j >= g.bufs && !(ok = wait(&sh.pv_done[buf], (turn - 1) & 1))) break;  // the weights stand where the scores go
                tc_fence_after();
                if (lead) {
                    const uint32_t q = q_lo + (PAIRED ? (uint32_t)s * (g.q_tile / 16) : 0u), key = k_lo + (uint32_t)ks * (g.k_tile / 16);
                    bool more = false;
#pragma unroll
                    for (int h = 0; h < TERMS; ++h)
                        for (int k = 0; k < g.dp / 16; ++k) {
                            const uint32_t at = (uint32_t)(k >> 2) * (TILE * 128 / 16) + (k & 3) * 2;
                            mma_ss(d_s, q + (uint32_t)h * (g.q_tile / TERMS / 16) + at, key + at, id_s, more);
                            more = true;
                        }
                    mma_commit(&sh.s_full[buf]);
                    if (!PAIRED || s == 1) mma_commit(&sh.k_empty[ks]);
                }
                __syncwarp();
            }
            if (++buf == g.bufs) {
                buf = 0;
                ++turn;
            }
        }
        // what was issued has to end before the tensor memory is given back
        if (lead) mma_commit(&sh.done);
        __syncwarp();
        mb_land(&sh.done, 0);
    } else if (warp >= SOFT_WARPS) {
        // ---- codes to f16: keys (and the scales), values ----
        const bool values = warp >= SOFT_WARPS + CONV_WARPS;
        const int cw = (warp - SOFT_WARPS) % CONV_WARPS, units = values ? g.vp / 32 : g.dp / 32;
        auto wait = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, mb_wait(bar, parity, a.err_flag, &sh.abort_flag)); };
        // A lane's place in 32 rows of 32 bytes, and where it goes: a 16-byte piece of a row of 128 bytes has its number turned by the row's.  Lanes are dealt out so that eight of them read
        // and write eight different pieces of 16 bytes of the banks: values by rows and pieces, keys (whose row r is token t, kv8_key_row(t) = r) by the bits that make the last of t.
        const int h = (lane >> 1) & 3, y = lane >> 3;
        const int r0 = values ? (lane & 7) + 8 * (lane >> 4) : 8 * h + 2 * ((h & 1) ^ (y & 1)) + (lane & 1), c = values ? (h >> 1) ^ (y & 1) : (h >> 1) ^ (y >> 1);
        const int t0 = values ? r0 : ((r0 >> 1) & 3) * 8 + (r0 >> 3) * 2 + (r0 & 1), off = t0 * 128 + (((2 * c) ^ (t0 & 7)) << 4);
        const int part = (values ? g.kpart : 0) + KV8_HALF * 4 + r0 * 32 + c * 16, second = values ? 512 : 128;  // the lane's other place, whose token (element) is 16 behind
        const int more = (values ? g.vst : g.kst) - 1;  // stages but one
        int next = 0;                                   // slot of the next page, and the parity of its wait
        uint32_t parity = 0;
        bool ok = true;
        for (int b = 0; b < n; ++b) {
            const int st = b & more;
            int slot[2];
#pragma unroll
            for (int pg = 0; pg < 2; ++pg) {
                slot[pg] = next;
                ok = ok && wait(&sh.raw_full[next], parity);
                if (++next == g.raw) {
                    next = 0;
                    parity ^= 1u;
                }
            }
            if (ok && b > more) ok = wait(values ? &sh.v_empty[st] : &sh.k_empty[st], ((b >> more) - 1) & 1);
            if (!ok) break;
            if (!values) {
                // scales, and what there is of the block.  What stood in their ring is five blocks old.  The keys took the place of those of block b - 2 or b - 1, whose scores are done;
                // the products that stood in their place were done before: with three places for scores, those of block b - 5 at least
                const int ring = b % RING;
                for (int ph = cw; ph < 4; ph += CONV_WARPS) {
                    const unsigned char* from = base + g.raw_at + (size_t)slot[ph >> 1] * 2 * g.half + (size_t)(ph & 1) * g.half;
                    const float v = reinterpret_cast<const float*>(from + g.kpart)[lane];
                    sh.ks[ring][ph * 32 + lane] = reinterpret_cast<const float*>(from)[lane];
                    sh.vs[ring][ph * 32 + lane] = v;
                    sh.lv[ring][ph * 32 + lane] = fmaxf(__log2f(v), LEAST_LOG);  // of NaN: the least
                }
                if (cw == 0 && lane == 0) sh.there[ring] = (sh.raw_there[slot[0]] ? 1 : 0) | (sh.raw_there[slot[1]] ? 2 : 0);
                __syncwarp();
                if (lane == 0) mb_arrive(&sh.sc_full[ring]);
            }
            // a warp takes 32 elements of a half at a time: a lane 16 elements of two tokens, or 16 tokens of two elements
            const unsigned char* raw[2] = {base + g.raw_at + (size_t)slot[0] * 2 * g.half + part, base + g.raw_at + (size_t)slot[1] * 2 * g.half + part};
            unsigned char* tile = base + (values ? g.v_at + (uint32_t)st * g.v_tile : g.k_at + (uint32_t)st * g.k_tile);
            struct Unit {
                int ph, q;
                uint4 w0, w1;
            };
            auto settle = [&](Unit& u) {
                while (u.q >= units) {
                    u.q -= units;
                    ++u.ph;
                }
                if (u.ph >= 4) return;
                const unsigned char* from = raw[u.ph >> 1] + (u.ph & 1) * g.half + u.q * 1024;
                u.w0 = *reinterpret_cast<const uint4*>(from);
                u.w1 = *reinterpret_cast<const uint4*>(from + second);
            };
            auto convert = [&](const Unit& u) {
                unsigned char* to = tile + (values ? (uint32_t)(u.ph >> 1) * (g.v_tile / 2) + u.q * 4096 : (uint32_t)(u.q >> 1) * (BLOCK * 128) + u.ph * 4096);
                const int at = off ^ (((values ? u.ph : u.q) & 1) << 6);
                uint4 x, y;
                codes_f16(u.w0.x, x.x, x.y);
                codes_f16(u.w0.y, x.z, x.w);
                codes_f16(u.w0.z, y.x, y.y);
                codes_f16(u.w0.w, y.z, y.w);
                *reinterpret_cast<uint4*>(to + at) = x;
                *reinterpret_cast<uint4*>(to + (at ^ 16)) = y;
                codes_f16(u.w1.x, x.x, x.y);
                codes_f16(u.w1.y, x.z, x.w);
                codes_f16(u.w1.z, y.x, y.y);
                codes_f16(u.w1.w, y.z, y.w);
                *reinterpret_cast<uint4*>(to + at + 2048) = x;
                *reinterpret_cast<uint4*>(to + (at ^ 16) + 2048) = y;
            };
            Unit u{0, cw}, v;
            settle(u);
            while (u.ph < 4) {  // one is loaded while another is converted
                v.ph = u.ph;
                v.q = u.q + CONV_WARPS;
                settle(v);
                convert(u);
                if (v.ph >= 4) break;
                u.ph = v.ph;
                u.q = v.q + CONV_WARPS;
                settle(u);
                convert(v);
            }
            fence_async_smem();
            __syncwarp();
            if (lane == 0) {
                mb_arrive(values ? &sh.v_full[st] : &sh.k_full[st]);
                mb_arrive(&sh.raw_empty[slot[0]]);
                mb_arrive(&sh.raw_empty[slot[1]]);
            }
        }
    } else {
        // ---- scores to weights ----
        const uint32_t lanes = (uint32_t)(warp & 3) * 32 << 16, o_at = o_at0 + lanes + (uint32_t)stream * o_step;
        float c = 0.f;  // what scores are multiplied with
        if (n > 0) {
            // eight elements a lane, 8 or 16 lanes to a pair, so that a row is read by neighbours; the loads of several groups of pairs are on their way at once
            constexpr int MINE = (PAIRED ? 2 : 1) * TILE / SOFT_WARPS;
            constexpr int AHEAD = BF16 ? 4 : 2;
            const int lanes = 8 * g.katoms, at_once = 32 / lanes, sub = lane / lanes, d = 8 * (lane - sub * lanes);
            for (int r0 = warp * MINE + sub; r0 < (warp + 1) * MINE; r0 += AHEAD * at_once) {
                float x[AHEAD][8];
#pragma unroll
                for (int k = 0; k < AHEAD; ++k) {
                    const int r = r0 + k * at_once, p = tiles0 * TILE + r, m = p / group, left = r < (warp + 1) * MINE && p < pairs ? a.pool.dim - d : 0;
                    const size_t at = (size_t)m * a.ldq + (size_t)(kvh * group + p - m * group) * a.pool.dim + d;
                    if ((wide & 2) && left > 0) {
                        float y[2][4];
                        load_row<BF16, 4>(a.q, at, y[0]);
                        load_row<BF16, 4>(a.q, at + 4, y[1]);
#pragma unroll
                        for (int e = 0; e < 8; ++e) x[k][e] = y[e >> 2][e & 3];
                    } else {
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            float one[1] = {0.f};
                            if (e < left) load_row<BF16, 1>(a.q, at + e, one);
                            x[k][e] = one[0];
                        }
                    }
                }
#pragma unroll
                for (int k = 0; k < AHEAD; ++k) {
                    const int r = r0 + k * at_once;
                    if (r - sub >= (warp + 1) * MINE) break;  // eight pairs may be fewer than those at once
                    uint32_t top = 0;
#pragma unroll
                    for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(x[k][e]) & 0x7FFFFFFFu);
                    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
                    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
                    top = max(top, __shfl_xor_sync(0xffffffffu, top, 4));
                    if (lanes == 16) top = max(top, __shfl_xor_sync(0xffffffffu, top, 8));
                    const bool finite = top < 0x7F800000u;
                    const int ex = min(max((int)(top >> 23), 15), 254);
                    const float up = finite ? __uint_as_float((uint32_t)(254 + 14 - ex) << 23) * (a.scale < 0.f ? -1.f : 1.f) : 0.f;
                    if (d < (PAIRED ? 8 : 16)) sh.half[PAIRED ? r >> 7 : d >> 3][1][0][r & (TILE - 1)] = finite ? fabsf(a.scale) * LOG2E * exp2f((float)(ex - 127 - 14)) : __uint_as_float(0x7FC00000u);
                    uint32_t hi[4], lo[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float u = x[k][2 * e] * up, v = x[k][2 * e + 1] * up;
                        hi[e] = f16x2(u, v);
                        if (TERMS == 2) lo[e] = f16x2(u - f16_lo(hi[e]), v - f16_hi(hi[e]));
                    }
                    unsigned char* to = base + g.q_at + (uint32_t)(r >> 7) * g.q_tile + (d >> 6) * (TILE * 128) + (r & (TILE - 1)) * 128 + ((((d >> 3) & 7) ^ (r & 7)) << 4);
                    *reinterpret_cast<uint4*>(to) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                    if (TERMS == 2) *reinterpret_cast<uint4*>(to + g.q_tile / 2) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                }
            }
            fence_async_smem();
            __syncwarp();
            if (lane == 0) mb_arrive(&sh.q_full);
            asm volatile("barrier.cta.sync.aligned 9, %0;" ::"n"(SOFT_WARPS * 32) : "memory");
            c = sh.half[stream][1][0][tid & (TILE - 1)];  // both warps that have a pair read it in front of their first barrier, behind which the place is written again
        }
        bool ok = true;
        float ref = -INFINITY, unit = -INFINITY, l = 0.f;  // the pair's largest score + log2(value scale) at the last move; ref - DROP, which weights are relative to; 2^-SUM_DROP of the sum of the weights of this side
        float kept = -INFINITY;  // reference of the sums in memory
        float origin = 0.f;      // the score that all references are counted from
        float4* const sum_at = sums + ((size_t)(blockIdx.y * gridDim.x + blockIdx.x) * 2 + stream) * (g.vp / 4) * TILE + (tid & (TILE - 1));  // those of elements 4 i .. 4 i + 3 stand TILE i behind
        const int mine_n = PAIRED ? n : (n + 1 - stream) / 2, t0 = 64 * side;
        int buf = stream, before = 0;           // places of the scores of task 2 i + stream, and of the stream's task in front
        uint32_t turn = 0, turn_before = 0;     // parities of the waits for them
        for (int i = 0; i < mine_n; ++i) {
            const uint32_t s_at = tmem + lanes + (uint32_t)buf * BLOCK;
            const int b = PAIRED ? i : 2 * i + stream, ring = b % RING;
            ok = __all_sync(0xffffffffu, mb_wait(&sh.sc_full[ring], (b / RING) & 1, a.err_flag, &sh.abort_flag) && mb_wait(&sh.s_full[buf], turn, a.err_flag, &sh.abort_flag));
            tc_fence_after();
            const int seen = (sh.there[ring] >> side) & 1 ? len - (b0 + b) * BLOCK - t0 : 0;  // tokens of this side in front of the row's end
            bool special = __any_sync(0xffffffffu, seen < 64 || origin != 0.f);  // tokens to be left out, or an origin; scores are counted from theirs
            // tokens c0 .. c0 + 31 of this side that are seen, a bit for each
            auto visible = [&](int c0) -> uint32_t {
                const int k = seen - c0;
                return k <= 0 ? 0u : k >= 32 ? 0xffffffffu : (1u << k) - 1u;
            };
            const ulonglong2 *vs2 = reinterpret_cast<const ulonglong2*>(&sh.vs[ring][t0]), *lv2 = reinterpret_cast<const ulonglong2*>(&sh.lv[ring][t0]);  // two pairs of scales
            // Where a pair of the warp has an origin, scores are put in the place of their sums, counted from there; what they are multiplied with is one from then on.
            bool counted = false;
            auto count = [&](float by) {
                const float factor = counted ? 1.f : c;
                const float* keys = &sh.ks[counted ? RING : ring][t0];
#pragma unroll 1
                for (int c0 = 0; c0 < 64; c0 += 16) {
                    uint32_t x[16];
                    tmem_ld16(x, s_at + t0 + c0);
                    tmem_wait16(x);
#pragma unroll
                    for (int e = 0; e < 16; ++e) x[e] = __float_as_uint(__fsub_rn(__fmul_rn(__uint_as_float(x[e]), keys[c0 + e] * factor), by));  // rounded as scores in f32 are, so that the difference is exact
                    tmem_st16(s_at + t0 + c0, x);
                }
                tmem_st_wait();
                counted = true;
            };
            if (special && __any_sync(0xffffffffu, origin != 0.f)) count(origin);
            // ---- the largest score + log2(value scale) of both sides ----
            float top;
            auto find = [&](auto mask) {
                const ulonglong2* ks2 = reinterpret_cast<const ulonglong2*>(&sh.ks[decltype(mask)::value && counted ? RING : ring][t0]);
                const uint64_t c2 = decltype(mask)::value && counted ? pair_of(1.f, 1.f) : pair_of(c, c);  // joins a key's scale first: sums times either alone may leave f32
                top = -INFINITY;
#pragma unroll 1
                for (int c0 = 0; c0 < 64; c0 += 32) {
                    uint32_t x[32];
                    tmem_ld32(x, s_at + t0 + c0);
                    const uint32_t vis = decltype(mask)::value ? visible(c0) : 0u;
                    tmem_wait(x);
#pragma unroll
                    for (int e = 0; e < 32; e += 4) {
                        const ulonglong2 k = ks2[(c0 + e) >> 2], v = lv2[(c0 + e) >> 2];
#pragma unroll
                        for (int f = 0; f < 2; ++f) {
                            const float2 y = of_pair(fma2(pair_of(x[e + 2 * f], x[e + 2 * f + 1]), mul2(f ? k.y : k.x, c2), f ? v.y : v.x));
                            if (decltype(mask)::value) {
                                if ((vis >> (e + 2 * f)) & 1) top = fmaxf(top, y.x);
                                if ((vis >> (e + 2 * f + 1)) & 1) top = fmaxf(top, y.y);
                            } else {
                                top = fmaxf(fmaxf(top, y.x), y.y);
                            }
                        }
                    }
                }
            };
            auto tell = [&](int place) {  // two places in turn: the other side may be a step behind
                sh.half[stream][place & 1][side][tid & (TILE - 1)] = top;
                if (both_any(stream * 4 + (warp & 3), !ok)) return ok = false;
                top = fmaxf(top, sh.half[stream][place & 1][side ^ 1][tid & (TILE - 1)]);
                return true;
            };
            if (special) find(std::true_type{});
            else find(std::false_type{});
            if (!tell(i)) break;
            // A new reference that is far from the origin: counted from there, it is found again, twice: the second time the origin is exact, where the first sum with it was not
            auto far = [&]() { return top > ref + SLACK && fabsf(top) >= FAR && fabsf(top) < INFINITY; };
            if (__any_sync(0xffffffffu, far())) {
                special = true;
#pragma unroll 1
                for (int again = 1; ok && again <= 2; ++again) {
                    const float to = far() ? origin + top : origin, by = to - origin;
                    origin = to;
                    ref -= by;
                    unit -= by;
                    kept -= by;
                    count(counted ? by : origin);
                    find(std::true_type{});
                    tell(i + again);
                }
            }
            if (!ok) break;
            // ---- the reference, which moves only where it has to ----
            if (top > ref + SLACK) ref = top;
            const float now = ref - DROP;  // -inf while the pair has seen nothing
            const bool next_chunk = i > 0 && (i & (CHUNK - 1)) == 0;
            if (next_chunk || (i > 0 && __any_sync(0xffffffffu, now != unit))) {  // O is the product of the blocks so far, when the last of them is done
                ok = __all_sync(0xffffffffu, mb_wait(&sh.pv_done[before], turn_before, a.err_flag, &sh.abort_flag));
                tc_fence_after();
                const float root = unit == -INFINITY || now == unit ? 1.f : exp2_ftz(0.5f * (unit - now)), corr = root * root;
                l = l * root * root;  // stays in range where the factor does not: its weights may belong to small values
                if (next_chunk) {
                    const float down = kept == -INFINITY || now == kept ? 1.f : exp2_ftz(kept - now);
#pragma unroll 1
                    for (int c0 = 16 * side; c0 < g.vp; c0 += 32) {
                        uint32_t x[16];
                        tmem_ld16(x, o_at + c0);
#pragma unroll
                        for (int e = 0; e < 16; e += 4) {
                            float4* at = sum_at + (size_t)((c0 + e) / 4) * TILE;
                            const float4 y = i > CHUNK ? __ldcg(at) : make_float4(0.f, 0.f, 0.f, 0.f);
                            if (e == 0) tmem_wait16(x);
                            __stcg(at, make_float4(fmaf(y.x, down, __uint_as_float(x[e]) * corr), fmaf(y.y, down, __uint_as_float(x[e + 1]) * corr), fmaf(y.z, down, __uint_as_float(x[e + 2]) * corr),
                                                   fmaf(y.w, down, __uint_as_float(x[e + 3]) * corr)));
                        }
                    }
                    kept = now;
                } else {
#pragma unroll 1
                    for (int c0 = 16 * side; c0 < g.vp; c0 += 32) {
                        uint32_t x[16];
                        tmem_ld16(x, o_at + c0);
                        tmem_wait16(x);
#pragma unroll
                        for (int e = 0; e < 16; ++e) x[e] = __float_as_uint(__uint_as_float(x[e]) * corr);
                        tmem_st16(o_at + c0, x);
                    }
                }
            }
            unit = now;
            // ---- scores to weights ----
            const float shift = now == -INFINITY ? 0.f : now;
            const uint64_t shift2 = pair_of(-shift, -shift);
            uint64_t sum[2] = {0, 0};
            auto weigh = [&](auto mask) {
                const ulonglong2* ks2 = reinterpret_cast<const ulonglong2*>(&sh.ks[decltype(mask)::value && counted ? RING : ring][t0]);
                const uint64_t c2 = decltype(mask)::value && counted ? pair_of(1.f, 1.f) : pair_of(c, c);  // joins a key's scale first: sums times either alone may leave f32
#pragma unroll 1
                for (int c0 = 0; c0 < 64; c0 += 32) {
                    uint32_t x[32], p[TERMS][16];
                    tmem_ld32(x, s_at + t0 + c0);
                    const uint32_t vis = decltype(mask)::value ? visible(c0) : 0u;
                    tmem_wait(x);
#pragma unroll
                    for (int e = 0; e < 32; e += 4) {
                        const ulonglong2 k = ks2[(c0 + e) >> 2], v = vs2[(c0 + e) >> 2];
#pragma unroll
                        for (int f = 0; f < 2; ++f) {
                            float2 t = of_pair(fma2(pair_of(x[e + 2 * f], x[e + 2 * f + 1]), mul2(f ? k.y : k.x, c2), shift2));
                            if (decltype(mask)::value) {
                                if (!((vis >> (e + 2 * f)) & 1)) t.x = -INFINITY;
                                if (!((vis >> (e + 2 * f + 1)) & 1)) t.y = -INFINITY;
                            }
                            const uint64_t pp = pair_of(exp2_ftz(t.x), exp2_ftz(t.y));
                            sum[f] = add2(sum[f], pp);
                            float2 w = of_pair(mul2(pp, f ? v.y : v.x));
                            if (decltype(mask)::value) {  // scales of tokens that are not there may be anything
                                if (!((vis >> (e + 2 * f)) & 1)) w.x = 0.f;
                                if (!((vis >> (e + 2 * f + 1)) & 1)) w.y = 0.f;
                            }
                            uint32_t& hi = p[0][e / 2 + f];
                            hi = f16x2(w.x, w.y);
                            if (TERMS == 2) p[TERMS - 1][e / 2 + f] = f16x2(w.x - f16_lo(hi), w.y - f16_hi(hi));
                        }
                    }
#pragma unroll
                    for (int h = 0; h < TERMS; ++h) tmem_st16(s_at + t0 + c0 + 16 * h, p[h]);
                }
            };
            if (special) weigh(std::true_type{});
            else weigh(std::false_type{});
            const float2 sums = of_pair(add2(sum[0], sum[1]));
            l = fmaf(sums.x + sums.y, 1.f / (1 << SUM_DROP), l);
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mb_arrive(&sh.p_full[buf]);
            before = buf;
            turn_before = turn;
            if ((buf += 2) >= g.bufs) {
                buf -= g.bufs;
                turn ^= 1u;
            }
        }
        // all products are done: of this stream, and those that read what stands where the results go
        ok = __all_sync(0xffffffffu, mb_wait(&sh.done, 0, a.err_flag, &sh.abort_flag)) && ok;
        tc_fence_after();
        // ---- what this stream has: into shared memory, where queries, keys and values stood ----
        sh.half[stream][mine_n & 1][side][tid & (TILE - 1)] = l;
        both_any(stream * 4 + (warp & 3), false);
        l += sh.half[stream][mine_n & 1][side ^ 1][tid & (TILE - 1)];
        const float down = kept == -INFINITY || kept == unit ? 1.f : exp2_ftz(kept - unit);
        float* to = reinterpret_cast<float*>(base) + (size_t)(stream * TILE + (tid & (TILE - 1))) * ldo;
        if (side == 0) *reinterpret_cast<float2*>(to) = make_float2(unit == -INFINITY && l != 0.f ? 0.f : origin + unit + SUM_DROP, l);  // a sum that is NaN is not passed over
#pragma unroll 1
        for (int c0 = 16 * side; c0 < g.vp; c0 += 32) {
            uint32_t x[16];
            tmem_ld16(x, o_at + c0);
            tmem_wait16(x);
            const bool some = ok && mine_n > 0;
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
                float4 y = some ? make_float4(__uint_as_float(x[e]), __uint_as_float(x[e + 1]), __uint_as_float(x[e + 2]), __uint_as_float(x[e + 3])) : make_float4(0.f, 0.f, 0.f, 0.f);
                if (some && mine_n > CHUNK) {
                    const float4 z = __ldcg(sum_at + (size_t)((c0 + e) / 4) * TILE);
                    y = make_float4(fmaf(z.x, down, y.x), fmaf(z.y, down, y.y), fmaf(z.z, down, y.z), fmaf(z.w, down, y.w));
                }
                constexpr float F = 1.f / (1 << SUM_DROP);
                *reinterpret_cast<float4*>(to + 4 + c0 + e) = make_float4(y.x * F, y.y * F, y.z * F, y.w * F);
            }
        }
    }
    __syncwarp();
    tc_fence_before();
    if (cluster > 1) cluster_sync_all();
    else __syncthreads();
    if (warp == MMA_WARP) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    // ---- the splits of a cluster (and the two streams of a tile) joined: a warp to a pair, the CTAs take turns ----
    const int rank = cluster > 1 ? (int)cluster_ctarank() : 0, rows = PAIRED ? 2 * TILE : TILE, sources = PAIRED ? cluster : 2 * cluster;
    constexpr int AT_ONCE = 4;  // sources whose loads are on their way together
    const int step = cluster * (THREADS / 32), last = min(rows, pairs - tiles0 * TILE) - 1, d = min(4 * lane, g.vp - 4);
    for (int r = rank * (THREADS / 32) + warp; r <= last; r += step) {
        float top = -INFINITY, l = 0.f;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int s0 = 0; s0 < sources; s0 += AT_ONCE) {
            float m[AT_ONCE], lm[AT_ONCE];
            float4 x[AT_ONCE];
#pragma unroll
            for (int k = 0; k < AT_ONCE; ++k) {  // source s: CTA s, or CTA s / 2 and stream s % 2
                const int s = s0 + k;
                m[k] = -INFINITY;
                if (s >= sources) continue;
                const uint32_t at = dsmem_addr(reinterpret_cast<const float*>(base) + (size_t)(PAIRED ? r : r + (s & 1) * TILE) * ldo, (uint32_t)(PAIRED ? s : s >> 1));
                m[k] = ld_dsmem_f32(at);
                lm[k] = ld_dsmem_f32(at + 4);
                x[k] = ld_dsmem_f32x4(at + 16 + 4 * d);
            }
#pragma unroll
            for (int k = 0; k < AT_ONCE; ++k) {
                if (m[k] == -INFINITY) continue;  // nothing seen
                const float now = fmaxf(top, m[k]), r0 = exp2_ftz(0.5f * (top - now)), r1 = exp2_ftz(0.5f * (m[k] - now)), f0 = r0 * r0, f1 = r1 * r1;
                top = now;
                l = fmaf(r1 * lm[k], r1, l * r0 * r0);
                v.x = fmaf(f1, x[k].x, v.x * f0); v.y = fmaf(f1, x[k].y, v.y * f0); v.z = fmaf(f1, x[k].z, v.z * f0); v.w = fmaf(f1, x[k].w, v.w * f0);
            }
        }
        const int p = tiles0 * TILE + r, m = p / group;
        if (a.direct && kv8_row_pieces(a, m) == 0) {  // the row has nothing else
            if ((unsigned)__ldg(a.row_seq + m) >= (unsigned)a.pool.n_seq || 4 * lane >= g.vp) continue;
            const int head = kvh * group + p - m * group;
            const float inv = l == 0.f ? 0.f : 1.0f / l;
            kv8_store2<BF16>(a, m, head, 4 * lane, v.x * inv, v.y * inv, wide & 1);
            kv8_store2<BF16>(a, m, head, 4 * lane + 2, v.z * inv, v.w * inv, wide & 1);
            continue;
        }
        float* to = parts + (((size_t)(split / cluster) * a.pool.kv_heads + kvh) * pairs + p) * (g.vp + 4);
        if (lane == 0) *reinterpret_cast<float2*>(to) = make_float2(top, l);
        if (4 * lane < g.vp) *reinterpret_cast<float4*>(to + 4 + 4 * lane) = v;
    }
    if (cluster > 1) cluster_sync_all();  // nobody leaves while a peer reads its shared memory
}

template <bool BF16, int TERMS, bool PAIRED>
cudaError_t launch(const Kv8AttnArgs& a, const Kv8Prefix& p, float* parts, float* sums, cudaStream_t st) {
    const Shape g = shape_of(a.pool.dim, a.pool.vdim, TERMS, PAIRED ? 2 : 1);
    const int wide = kv8_wide(a);
    const cudaError_t e = ensure_dyn_smem(kv8_prefix_kernel<BF16, TERMS, PAIRED>, g.bytes);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(p.groups * p.splits), (unsigned)a.pool.kv_heads);
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = g.bytes;
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)p.cluster;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = p.cluster > 1 ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kv8_prefix_kernel<BF16, TERMS, PAIRED>, a, p.splits, p.cluster, parts, reinterpret_cast<float4*>(sums), wide);
}

// Clusters of CTAs that have an SM each which the current device holds at the same time; asked once per size.
int clusters_at_once(int cluster, int sm_count) {
    static std::mutex mu;
    static std::map<std::pair<int, int>, int> known;
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return sm_count / cluster;
    std::lock_guard<std::mutex> lk(mu);
    const auto key = std::make_pair(dev, cluster);
    const auto it = known.find(key);
    if (it != known.end()) return it->second;
    int n = 0;
    const size_t smem = shape_of(128, 128, 1, 2).bytes;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)cluster);
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)cluster;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    if (ensure_dyn_smem(kv8_prefix_kernel<true, 1, true>, smem) != cudaSuccess || cudaOccupancyMaxActiveClusters(&n, kv8_prefix_kernel<true, 1, true>, &cfg) != cudaSuccess) {
        cudaGetLastError();
        n = sm_count / cluster;
    }
    return known[key] = n;
}

}  // namespace

Kv8Prefix kv8_prefix_plan(int kv_heads, int dim, int vdim, int bf16, int M, int heads, int n_shared, int sm_count) {
    Kv8Prefix p{};
    const long pairs = (long)M * (heads / kv_heads);
    // wider heads do not fit tensor memory (two streams of scores and results) or shared memory.  Up to 16 pairs are two items of the streaming kernel at most, which reads 2.5 TB/s of a prefix
    // twice while its codes are converted here at 2 TB/s
    if (n_shared < 1 || dim > 128 || vdim > 128 || pairs <= 2 * KV8_PAIRS) return p;
    const long group = heads / kv_heads, pieces = (long)M * kv_heads * ((group + KV8_PAIRS - 1) / KV8_PAIRS) * n_shared * (KV8_PAGE / KV8_HALF);
    if (pieces < LEAST_SHARED) return p;
    const long tiles = (pairs + TILE - 1) / TILE;
    p.paired = bf16 && tiles > 1;
    const long groups = p.paired ? (tiles + 1) / 2 : tiles, items = groups * kv_heads, blocks = (n_shared + 1) / 2;
    // A CTA per SM: splits and clusters with the least time, in blocks; four for a CTA's beginning and end, one for every part that is left to be joined.
    const long most = std::min<long>({blocks, 64, std::max<long>(1, (2l * sm_count + items - 1) / items)});
    double best = 0.0;
    for (int cluster = 8; cluster > 0; --cluster)
        for (int s = cluster; s <= most && s <= cluster * MOST_PARTS; s += cluster) {
            const long at_once = std::max(1, cluster > 1 ? clusters_at_once(cluster, sm_count) : sm_count);
            const double cost = (double)((items * s / cluster + at_once - 1) / at_once) * ((double)((blocks + s - 1) / s) * (p.paired ? 2.0 : 1.0) + 4.0) + s / cluster;
            if (p.splits == 0 || cost < best) {
                best = cost;
                p.splits = s;
                p.cluster = cluster;
            }
        }
    p.groups = (int)groups;
    p.parts = p.splits / p.cluster;
    const long of_cta = (blocks + p.splits - 1) / p.splits;
    if ((p.paired ? of_cta : (of_cta + 1) / 2) > chunk_of(bf16 ? 1 : 2)) p.sums = 2 * (size_t)TILE * kv8_pad(vdim) * items * p.splits;
    return p;
}

int kv8_prefix_most_parts(int kv_heads, int M, int heads, int n_shared, int sm_count) {
    const long tiles = ((long)M * (heads / kv_heads) + TILE - 1) / TILE, items = (tiles + 1) / 2 * kv_heads;
    return (int)std::min<long>({(n_shared + 1) / 2, MOST_PARTS, std::max<long>(1, (2l * sm_count + items - 1) / items)});
}

cudaError_t launch_kv8_prefix(const Kv8AttnArgs& a, const Kv8Prefix& p, float* parts, float* sums, cudaStream_t st) {
    if (!a.bf16) return launch<false, 2, false>(a, p, parts, sums, st);
    return p.paired ? launch<true, 1, true>(a, p, parts, sums, st) : launch<true, 1, false>(a, p, parts, sums, st);
}

}  // namespace hm

// Products of two operand images on the 5th-generation tensor cores: y[m][n] = sum_k x[m][k] w[n][k], 4-bit microscaled floats on both sides
// (tcgen05.mma kind::mxf4.block_scale, scales in tensor memory) or bf16 (kind::f16); f32 sums.  One group of rows, or groups of rows by
// expert, each with weights of its own (image.h, Plan).
//
//   * a unit = 128 features (the MMA's M: weights are its first operand) x up to 192 rows (its N, cut to the rows that exist), so that small groups
//     of rows cost what they are: with 16 rows per expert the weights are streamed once and nothing else counts.
//   * one CTA per SM walks its units (persistent, static round robin): a warp copies k-blocks of 128 bytes per row into a ring of four slots, one issues
//     MMAs, eight read accumulators.  Two accumulators of 192 columns alternate; the scales of a slot have 24 columns of the tensor memory of their
//     own, so that nothing overwrites scales that an MMA still reads (4 * 24 + 384 = 480 of 512 columns).
//   * the tensor core truncates when it adds to an accumulator; accumulators cover CHUNK k-blocks (32 additions) and are summed in registers to nearest.
//   * units that are fewer than half the SMs share their k-blocks among the CTAs of a cluster, whose partial tiles are summed in the order of their
//     ranks through distributed shared memory: no scratch outlives the launch.
// Measured (graph replays): 1999 x 17920 x 1536 4-bit to bf16 32 us = 3.4 PFLOP/s, 2.1 times the measured bf16 rate; the GPU is at its power limit then (990 W,
// 1.73 GHz).  A k-block takes 402 clocks of MMAs, 584 with its six scale copies, and 96 KB of shared-memory traffic with the staged results: copies in, operands
// out and results fill two thirds of that pipe.  64 rows x 8960 -> 1536 in clusters of seven 6.9 us; 32 experts x 16 rows, 60 MB of weights, 11.8 us from the L2, 15.7 from
// memory.
// Taken back: pairs of CTAs (cta_group::2, half the rows loaded per CTA; 34.5 us: five slots do not cover the way from CTA to CTA, six leave too little
// shared memory for the results, 40 us), scales written to the
// tensor memory by four more warps instead of copied (38 us), waits by one lane of a warp (34 us), groups cut into units of equal sizes (within 5 % either way).
#include "image.h"

#include <algorithm>

#include "launch_attrs.h"
#include "mbarrier.cuh"

namespace hm {
namespace {

constexpr int TN = 192;                      // rows of a unit at most
constexpr int CHUNK = 8;                     // k-blocks per accumulator
constexpr int SLOTS = 4;
constexpr int EPI_WARPS = 8, THREADS = 64 + EPI_WARPS * 32;
constexpr int A_SLOT = MX_TILE;              // scales (bf16: unused), 128 features
constexpr int B_SLOT = 2 * MX_SCALES + TN * 128;
constexpr int SLOT = A_SLOT + B_SLOT;
constexpr int STAGE_LD = IMG_ROWS * 2 + 16;      // bytes of a staged row of 128 bf16: eight of them begin in different banks
constexpr int STAGE_HALF = 32 * STAGE_LD;        // ... and 16 rows of 128 f32
constexpr size_t SMEM = (size_t)SLOTS * SLOT + 4 * STAGE_HALF + 1024;
constexpr int SF_COLS = 24, SF_BASE = 2 * TN;
constexpr int MAX_SPLIT = 8;
static_assert(SF_BASE + SLOTS * SF_COLS <= 512 && TN % 64 == 0, "tensor memory");
static_assert(TN * IMG_ROWS * 4 <= SLOTS * SLOT, "partial tile");

// The warps that copy and multiply stay converged: every lane runs their loops and one, elected in place, issues.  Addresses and
// descriptors then live in uniform registers; issued from a branch of lane 0 a k-block cost 1300 clocks whatever its MMAs took.
//
// Shared-memory descriptors, upper word: rows of 128 bytes in groups of eight, 128-byte swizzle; and 32 rows of 16 bytes, eight rows of 128 bytes in a row.
constexpr uint32_t DESC_TILE = (1024 >> 4) | 1u << 14 | 2u << 29, DESC_SCALES = (128 >> 4) | 1u << 14;
__device__ __forceinline__ uint32_t desc_lo(uint32_t smem_addr) { return ((smem_addr >> 4) & 0x3FFF) | 1u << 16; }
// A k-block: four MMAs of 32 bytes per row, whose end arrives at `done`.  more: adds to the accumulator (0: the first MMA replaces it).
__device__ __forceinline__ void step_bf16(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t more, uint64_t* done) {
    asm volatile("{ .reg .pred p, e;\n .reg .b64 x0, x1, x2, x3, y0, y1, y2, y3;\n .reg .b32 t;\n"
                 "setp.ne.b32 p, %4, 0;\n"
                 "mov.b64 x0, {%1, %5};\n mov.b64 y0, {%2, %5};\n"
                 "add.u32 t, %1, 2;\n mov.b64 x1, {t, %5};\n add.u32 t, %2, 2;\n mov.b64 y1, {t, %5};\n"
                 "add.u32 t, %1, 4;\n mov.b64 x2, {t, %5};\n add.u32 t, %2, 4;\n mov.b64 y2, {t, %5};\n"
                 "add.u32 t, %1, 6;\n mov.b64 x3, {t, %5};\n add.u32 t, %2, 6;\n mov.b64 y3, {t, %5};\n"
                 "elect.sync _|e, 0xffffffff;\n"
                 "@e tcgen05.mma.cta_group::1.kind::f16 [%0], x0, y0, %3, p;\n"
                 "@e tcgen05.mma.cta_group::1.kind::f16 [%0], x1, y1, %3, 1;\n"
                 "@e tcgen05.mma.cta_group::1.kind::f16 [%0], x2, y2, %3, 1;\n"
                 "@e tcgen05.mma.cta_group::1.kind::f16 [%0], x3, y3, %3, 1;\n"
                 "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%6]; }" ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(more), "n"(DESC_TILE), "r"(s32(done)) : "memory");
}
// The same on 4-bit codes.  The scales of a block of 128 rows are two times 512 bytes, one for either half of the 256 values, which go to four columns each for
// all four warps' lanes: features sa -> fa, fa + 4; rows sb -> fb, fb + 8, and of a second block (two) fb + 4, fb + 12.  An MMA of 64 values takes two of a
// column's four bytes (hi: the idesc of the upper two); the unit's rows begin at column fb + off.
__device__ __forceinline__ void step_mx(uint32_t d, uint32_t sa, uint32_t a, uint32_t sb, uint32_t b, uint32_t idesc, uint32_t fa, uint32_t off, uint32_t two, uint32_t more, uint64_t* done) {
    asm volatile("{ .reg .pred p, q, e;\n .reg .b64 x0, x1, x2, x3, y0, y1, y2, y3, s0, s1, s2, s3, s4, s5;\n .reg .b32 t, hi, f4, f8, f12, f16, f20, b0, b1;\n"
                 "setp.ne.b32 p, %9, 0;\n setp.ne.b32 q, %8, 0;\n"
                 "mov.b64 s0, {%1, %12};\n add.u32 t, %1, 32;\n mov.b64 s1, {t, %12};\n"
                 "mov.b64 s2, {%3, %12};\n add.u32 t, %3, 32;\n mov.b64 s3, {t, %12};\n"
                 "add.u32 t, %3, 64;\n mov.b64 s4, {t, %12};\n add.u32 t, %3, 96;\n mov.b64 s5, {t, %12};\n"
                 "add.u32 f4, %6, 4;\n add.u32 f8, %6, 8;\n add.u32 f12, %6, 12;\n add.u32 f16, %6, 16;\n add.u32 f20, %6, 20;\n"
                 "add.u32 b0, f8, %7;\n add.u32 b1, f16, %7;\n or.b32 hi, %5, %13;\n"
                 "mov.b64 x0, {%2, %11};\n mov.b64 y0, {%4, %11};\n"
                 "add.u32 t, %2, 2;\n mov.b64 x1, {t, %11};\n add.u32 t, %4, 2;\n mov.b64 y1, {t, %11};\n"
                 "add.u32 t, %2, 4;\n mov.b64 x2, {t, %11};\n add.u32 t, %4, 4;\n mov.b64 y2, {t, %11};\n"
                 "add.u32 t, %2, 6;\n mov.b64 x3, {t, %11};\n add.u32 t, %4, 6;\n mov.b64 y3, {t, %11};\n"
                 "elect.sync _|e, 0xffffffff;\n and.pred q, q, e;\n"
                 "@e tcgen05.cp.cta_group::1.32x128b.warpx4 [%6], s0;\n"
                 "@e tcgen05.cp.cta_group::1.32x128b.warpx4 [f4], s1;\n"
                 "@e tcgen05.cp.cta_group::1.32x128b.warpx4 [f8], s2;\n"
                 "@e tcgen05.cp.cta_group::1.32x128b.warpx4 [f16], s3;\n"
                 "@q tcgen05.cp.cta_group::1.32x128b.warpx4 [f12], s4;\n"
                 "@q tcgen05.cp.cta_group::1.32x128b.warpx4 [f20], s5;\n"
                 "@e tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], x0, y0, %5, [%6], [b0], p;\n"
                 "@e tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], x1, y1, hi, [%6], [b0], 1;\n"
                 "@e tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], x2, y2, %5, [f4], [b1], 1;\n"
                 "@e tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], x3, y3, hi, [f4], [b1], 1;\n"
                 "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%10]; }" ::"r"(d), "r"(sa), "r"(a), "r"(sb), "r"(b), "r"(idesc), "r"(fa), "r"(off), "r"(two), "r"(more), "r"(s32(done)), "n"(DESC_TILE),
                 "n"(DESC_SCALES), "n"(2u << 4 | 2u << 29)
                 : "memory");
}
__device__ __forceinline__ void mma_commit(uint64_t* bar) {
    asm volatile("{ .reg .pred e;\n elect.sync _|e, 0xffffffff;\n @e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0]; }" ::"r"(s32(bar)) : "memory");
}
// Copies of a k-block into a slot: features (`TILE` bytes), the rows' scales and codes of one or two (two) blocks of the rows' image.
struct Copies {
    uint64_t w, x0, x1;      // in the images: features; rows, or with scales these; the second block's
    uint32_t b0, b1, bytes;  // bytes of the rows' parts, and of all copies
    uint32_t two;
};
__device__ __forceinline__ void copy_bf16(const Copies& c, uint32_t bar, uint32_t wa, uint32_t xa) {
    asm volatile("{ .reg .pred e, q;\n .reg .b64 st;\n .reg .b32 t;\n"
                 "setp.ne.b32 q, %9, 0;\n add.u32 t, %5, %6;\n"
                 "elect.sync _|e, 0xffffffff;\n and.pred q, q, e;\n"
                 "@e mbarrier.arrive.expect_tx.shared::cta.b64 st, [%0], %8;\n"
                 "@e cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%4], [%1], %10, [%0];\n"
                 "@e cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%5], [%2], %6, [%0];\n"
                 "@q cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [t], [%3], %7, [%0]; }" ::"r"(bar), "l"(c.w), "l"(c.x0), "l"(c.x1), "r"(wa), "r"(xa), "r"(c.b0), "r"(c.b1), "r"(c.bytes), "r"(c.two), "n"(IMG_CODES)
                 : "memory");
}
// xs: the slot's place for the rows' scales, two times MX_SCALES in front of their codes; off: bytes in front of the first row's codes.
__device__ __forceinline__ void copy_mx(const Copies& c, uint32_t bar, uint32_t wa, uint32_t xs, uint64_t off) {
    asm volatile("{ .reg .pred e, q;\n .reg .b64 st, y0, y1;\n .reg .b32 s1, d0, d1;\n"
                 "setp.ne.b32 q, %8, 0;\n add.u32 s1, %5, %10;\n add.u32 d0, s1, %10;\n add.u32 d1, d0, %6;\n"
                 "add.u64 y0, %2, %11;\n add.u64 y1, %3, %10;\n"
                 "elect.sync _|e, 0xffffffff;\n and.pred q, q, e;\n"
                 "@e mbarrier.arrive.expect_tx.shared::cta.b64 st, [%0], %9;\n"
                 "@e cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%4], [%1], %12, [%0];\n"
                 "@e cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%5], [%2], %10, [%0];\n"
                 "@e cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [d0], [y0], %6, [%0];\n"
                 "@q cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [s1], [%3], %10, [%0];\n"
                 "@q cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [d1], [y1], %7, [%0]; }" ::"r"(bar), "l"(c.w), "l"(c.x0), "l"(c.x1), "r"(wa), "r"(xs), "r"(c.b0), "r"(c.b1), "r"(c.two), "r"(c.bytes), "n"(MX_SCALES),
                 "l"(off), "n"(MX_TILE)
                 : "memory");
}
// 32 features (the warp's lanes of the tensor memory) x 32 rows: a lane has one feature of all rows, or, BF16, the fragments that stmatrix takes: of eight
// rows and eight features lane 4 f + r has feature f, rows 2 r and 2 r + 1.
template <bool BF16>
__device__ __forceinline__ int value_row(int lane, int j) { return BF16 ? (j >> 2 & 3) * 8 + (lane & 3) * 2 + (j & 1) : j; }
template <bool BF16>
__device__ __forceinline__ int value_feature(int lane, int j) { return BF16 ? (j >> 4) * 16 + (j >> 1 & 1) * 8 + (lane >> 2) : lane; }
template <bool BF16>
__device__ __forceinline__ void tmem_read(float (&r)[32], uint32_t addr) {
    if (BF16) {
#pragma unroll
        for (int h = 0; h < 32; h += 16)
            asm volatile("tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                         : "=f"(r[h]), "=f"(r[h + 1]), "=f"(r[h + 2]), "=f"(r[h + 3]), "=f"(r[h + 4]), "=f"(r[h + 5]), "=f"(r[h + 6]), "=f"(r[h + 7]), "=f"(r[h + 8]), "=f"(r[h + 9]), "=f"(r[h + 10]), "=f"(r[h + 11]),
                           "=f"(r[h + 12]), "=f"(r[h + 13]), "=f"(r[h + 14]), "=f"(r[h + 15])
                         : "r"(addr + ((uint32_t)h << 16)));
    } else {
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                     : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]), "=f"(r[8]), "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15]),
                       "=f"(r[16]), "=f"(r[17]), "=f"(r[18]), "=f"(r[19]), "=f"(r[20]), "=f"(r[21]), "=f"(r[22]), "=f"(r[23]), "=f"(r[24]), "=f"(r[25]), "=f"(r[26]), "=f"(r[27]), "=f"(r[28]), "=f"(r[29]), "=f"(r[30]), "=f"(r[31])
                     : "r"(addr));
    }
}
// Names the registers, so that no use of them moves in front of the wait.
__device__ __forceinline__ void tmem_wait(float (&r)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+f"(r[0]), "+f"(r[1]), "+f"(r[2]), "+f"(r[3]), "+f"(r[4]), "+f"(r[5]), "+f"(r[6]), "+f"(r[7]), "+f"(r[8]), "+f"(r[9]), "+f"(r[10]), "+f"(r[11]), "+f"(r[12]), "+f"(r[13]), "+f"(r[14]), "+f"(r[15]),
                   "+f"(r[16]), "+f"(r[17]), "+f"(r[18]), "+f"(r[19]), "+f"(r[20]), "+f"(r[21]), "+f"(r[22]), "+f"(r[23]), "+f"(r[24]), "+f"(r[25]), "+f"(r[26]), "+f"(r[27]), "+f"(r[28]), "+f"(r[29]), "+f"(r[30]), "+f"(r[31])
                 :: "memory");
}

struct Shared {
    uint64_t full[SLOTS], empty[SLOTS], afull[2], aempty[2], done;
    uint32_t tmem;
    volatile int abort_flag;
    int units;
    int rows[2][TN];  // places of a unit's rows in y, -1: none; units alternate
};

// Units begin at rows 0 or 64 of a block: their scales then begin at an even column of the tensor memory (32 rows to a column), as an MMA wants them; an odd one
// is a misaligned address.
struct Unit {
    int expert, tile, row0, n;  // features tile * 128 ..; image rows row0 .. row0 + n
};
// Groups of rows, in shared memory: an expert's first unit, rows, and first image row.
struct Groups {
    int unit[PLAN_EXPERTS], rows[PLAN_EXPERTS], base[PLAN_EXPERTS];
};
// A warp reads the plan; returns the number of units.  Groups that do not fit (a plan of other pairs) have no rows.
__device__ __forceinline__ int read_groups(const ImageGemmArgs& a, Groups& g, int lane) {
    int sum = 0;
    for (int i0 = 0; i0 < a.experts; i0 += 32) {
        const int i = i0 + lane;
        int rows = 0, base = 0;
        if (i < a.experts) {
            const int n = __ldg(a.count + i), b = __ldg(a.first + i);
            base = b * IMG_ROWS;
            rows = n > 0 && n <= a.pairs && b >= 0 && b <= (a.rows - n) / IMG_ROWS ? n : 0;
        }
        const int units = (rows + TN - 1) / TN * a.tiles;
        int inc = units;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int t = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += t;
        }
        if (i < a.experts) {
            g.unit[i] = sum + inc - units;
            g.rows[i] = rows;
            g.base[i] = base;
        }
        sum += __shfl_sync(0xffffffffu, inc, 31);
    }
    return sum;
}
// Units of an expert: its rows fastest, so that units that run at the same time share weights.
__device__ __forceinline__ Unit unit_at(const ImageGemmArgs& a, const Groups& g, int u) {
    Unit r;
    int rows = a.M, base = 0;
    r.expert = 0;
    if (a.first) {
        int lo = 0, hi = a.experts;  // the last expert whose first unit is at most u
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (g.unit[mid] <= u) lo = mid;
            else hi = mid;
        }
        r.expert = __shfl_sync(0xffffffffu, lo, 0);  // the same in all lanes: uniform for the compiler too
        rows = __shfl_sync(0xffffffffu, g.rows[lo], 0);
        base = __shfl_sync(0xffffffffu, g.base[lo], 0);
        u -= __shfl_sync(0xffffffffu, g.unit[lo], 0);
    }
    const int per = (rows + TN - 1) / TN, t = u % per;
    r.tile = u / per;
    r.row0 = base + t * TN;
    r.n = min(TN, rows - t * TN);
    return r;
}

// An epilogue warp has 32 features (lane: one) of 32 rows; the four warps of a half bring the rows of 128 features together in shared memory (two buffers in turn,
// one barrier each) and store them as whole lines, 16 bytes per lane.  Stored from the registers, 4 bytes per lane and a place in y for each, the same tile took
// three times as long; as bulk copies of one row each, twice.
struct Stage {
    unsigned char* buf;  // [2][STAGE_HALF]
    uint32_t used;       // buffers so far
    int bar;             // named barrier of the half's warps
};
template <typename T, int ROWS, int LD>
__device__ __forceinline__ void stage_out(const ImageGemmArgs& a, Stage& st, const unsigned char* buf, const int* rows, int n0, int et) {
    constexpr int PER = 16 / sizeof(T), PIECES = IMG_ROWS / PER;  // values of a piece, pieces of a row
    asm volatile("bar.sync %0, 128;" ::"r"(st.bar) : "memory");
    const int nf = min(IMG_ROWS, a.N - n0);
#pragma unroll
    for (int i = 0; i < ROWS * PIECES / 128; ++i) {
        const int piece = i * 128 + et, row = rows[piece / PIECES], c = piece % PIECES * PER;
        if (row < 0 || c >= nf) continue;
        const uint4 v = *reinterpret_cast<const uint4*>(buf + piece / PIECES * LD + piece % PIECES * 16);
        T* y = static_cast<T*>(a.y) + (size_t)row * a.ldy + n0 + c;
        if (a.wide && c + PER <= nf) *reinterpret_cast<uint4*>(y) = v;
        else {
            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int e = 0; e < PER; ++e)
                if (c + e < nf) y[e] = sizeof(T) == 2 ? (T)(w[e / 2] >> (16 * (e & 1))) : (T)w[e % 4];
        }
    }
}
template <bool BF16>
__device__ __forceinline__ void emit(const ImageGemmArgs& a, Stage& st, const int* rows, int n0, int et, const float (&v)[32]) {
    if (BF16) {
        unsigned char* buf = st.buf + (st.used++ & 1u) * STAGE_HALF;
        const int lane = et & 31;
        // eight rows by 32 features at a time: thread 8 g + i names row i of the features' group g
        const uint32_t at = s32(buf) + (lane & 7) * STAGE_LD + (et & 96) * 2 + (lane >> 3) * 16;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(at + j * 8 * STAGE_LD), "r"(bf16x2_rne(v[4 * j], v[4 * j + 1])), "r"(bf16x2_rne(v[4 * j + 2], v[4 * j + 3])),
                         "r"(bf16x2_rne(v[16 + 4 * j], v[16 + 4 * j + 1])), "r"(bf16x2_rne(v[16 + 4 * j + 2], v[16 + 4 * j + 3]))
                         : "memory");
        stage_out<uint16_t, 32, STAGE_LD>(a, st, buf, rows, n0, et);
    } else {
#pragma unroll
        for (int h = 0; h < 32; h += 16) {
            unsigned char* buf = st.buf + (st.used++ & 1u) * STAGE_HALF;
            float* d = reinterpret_cast<float*>(buf) + et;
#pragma unroll
            for (int j = 0; j < 16; ++j) d[j * IMG_ROWS] = v[h + j];
            stage_out<uint32_t, 16, IMG_ROWS * 4>(a, st, buf, rows + h, n0, et);
        }
    }
}

__device__ __forceinline__ void store1(const ImageGemmArgs& a, int row, int f, float v) {
    if (a.bf16) static_cast<uint16_t*>(a.y)[(size_t)row * a.ldy + f] = (uint16_t)bf16x2_rne(v, 0.f);
    else static_cast<float*>(a.y)[(size_t)row * a.ldy + f] = v;
}

template <bool MX, bool BF16>
__global__ void __launch_bounds__(THREADS, 1) image_gemm_kernel(const ImageGemmArgs a) {
    extern __shared__ __align__(1024) unsigned char dsm[];
    __shared__ Shared sh;
    __shared__ Groups groups;
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
    pdl_wait();
    if (warp == 2 && a.first) {
        const int n = read_groups(a, groups, lane);
        if (lane == 0) sh.units = n;
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = __shfl_sync(0xffffffffu, sh.tmem, 0), ring_at = __shfl_sync(0xffffffffu, s32(ring), 0);
    const int units = __shfl_sync(0xffffffffu, sh.units, 0);
    const int rank = blockIdx.x % a.split, step = gridDim.x / a.split, u0 = blockIdx.x / a.split;
    const int kb0 = rank * a.kb_per, kb1 = min(a.kblocks, kb0 + a.kb_per);
    constexpr int TILE = MX ? MX_TILE : IMG_CODES;

    uint32_t issued = 0;
    if (warp == 0) {
        bool ok = true;
        Unit t = u0 < units ? unit_at(a, groups, u0) : Unit{};
        for (int u = u0; u < units && ok; u += step) {
            Unit next = t;
            const int off = t.row0 % IMG_ROWS, n0 = min(t.n, IMG_ROWS - off), n1 = t.n - n0;  // rows in the first and in the second block
            Copies c;
            c.b0 = (uint32_t)(n0 + 7) / 8 * 1024;
            c.b1 = (uint32_t)(n1 + 7) / 8 * 1024;
            c.two = n1 > 0;
            c.bytes = (uint32_t)TILE + c.b0 + c.b1 + (MX ? (1 + c.two) * MX_SCALES : 0u);
            c.w = (uint64_t)__cvta_generic_to_global(a.w + t.expert * a.w_stride + ((size_t)t.tile * a.kblocks + kb0) * TILE);
            c.x0 = (uint64_t)__cvta_generic_to_global(a.x + ((size_t)(t.row0 / IMG_ROWS) * a.kblocks + kb0) * TILE);
            c.x1 = c.x0 + (size_t)a.kblocks * TILE;
            if (!MX) c.x0 += off * 128;
            for (int kb = kb0; kb < kb1; ++kb, ++issued, c.w += TILE, c.x0 += TILE, c.x1 += TILE) {
                const uint32_t s = issued % SLOTS, sa = ring_at + s * SLOT, sb = sa + A_SLOT;
                if (issued >= SLOTS) ok = mb_wait(&sh.empty[s], ((issued / SLOTS) & 1u) ^ 1u, a.err_flag, &sh.abort_flag);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                if (MX) copy_mx(c, s32(&sh.full[s]), sa, sb, MX_SCALES + off * 128);
                else copy_bf16(c, s32(&sh.full[s]), sa + MX_SCALES, sb + 2 * MX_SCALES);
                if (kb == kb0 && u + step < units) next = unit_at(a, groups, u + step);  // looked up while copies and MMAs run
            }
            t = next;
        }
    } else if (warp == 1) {
        // No wait's result decides anything here: where one has run out, the others return at once and the MMAs read what is there, whose
        // results nobody uses.
        uint32_t i = 0, ci = 0;
        Unit t = u0 < units ? unit_at(a, groups, u0) : Unit{};
        for (int u = u0; u < units; u += step) {
            Unit next = t;
            const uint32_t off = (uint32_t)t.row0 % IMG_ROWS, n = ((uint32_t)t.n + 15) & ~15u, two = t.n + off > IMG_ROWS;
            // D f32, both operands K-major, M 128, N n; bf16, or e2m1 with e8m0 scales
            const uint32_t idesc = MX ? 1u << 7 | 1u << 10 | (n >> 3) << 17 | 1u << 23 | (128u >> 4) << 24 : 1u << 4 | 1u << 7 | 1u << 10 | (n >> 3) << 17 | (128u >> 4) << 24;
            for (int kc = kb0; kc < kb1; kc += CHUNK, ++ci) {
                const uint32_t buf = ci & 1u, d = tmem + buf * TN;
                if (ci >= 2) mb_wait(&sh.aempty[buf], ((ci >> 1) & 1u) ^ 1u, a.err_flag, &sh.abort_flag);
                const int ke = min(kb1, kc + CHUNK);
                for (int kb = kc; kb < ke; ++kb, ++i) {
                    const uint32_t s = i % SLOTS;
                    mb_wait(&sh.full[s], (i / SLOTS) & 1u, a.err_flag, &sh.abort_flag);
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const uint32_t sa = desc_lo(ring_at + s * SLOT), wa = sa + (MX_SCALES >> 4), sb = sa + (A_SLOT >> 4), xa = sb + (2 * MX_SCALES >> 4);
                    if (MX) step_mx(d, sa, wa, sb, xa, idesc, tmem + SF_BASE + s * SF_COLS, off / 32, two, kb > kc, &sh.empty[s]);
                    else step_bf16(d, wa, xa, idesc, kb > kc, &sh.empty[s]);
                    if (kb == kb0 && u + step < units) next = unit_at(a, groups, u + step);
                }
                mma_commit(&sh.afull[buf]);
            }
            t = next;
        }
    } else {
        const int quarter = warp & 3, half = (warp - 2) >> 2;  // a warp reads its own quarter of the TMEM lanes; chunks of 32 rows alternate
        const uint32_t tbase = tmem + ((uint32_t)(quarter * 32) << 16) + half * 32;
        const int et = tid - 64, qt = quarter * 32 + lane;
        uint32_t ci = 0, ui = 0;
        Stage st{ring + (size_t)SLOTS * SLOT + half * 2 * STAGE_HALF, 0, 2 + half};
        const bool whole = kb1 - kb0 <= CHUNK && a.split == 1;  // one accumulator per unit
        Unit t, next = u0 < units ? unit_at(a, groups, u0) : Unit{};
        for (int u = u0; u < units; u += step, ++ui) {
            t = next;
            if (u + step < units) next = unit_at(a, groups, u + step);
            const int n0 = t.tile * IMG_ROWS, *rows = sh.rows[ui & 1] + half * 32;
            // (nobody reads the entries of the unit before the last: its readers have met at the barrier of the last one)
            if (et < TN) {
                const int row = et < t.n ? (a.row ? __ldg(a.row + t.row0 + et) : t.row0 + et) : -1;
                sh.rows[ui & 1][et] = a.row && row >= a.pairs ? -1 : row;
            }
            asm volatile("bar.sync 1, 256;" ::: "memory");
            if (whole) {  // small code: the loops of the other warps stay in the instruction cache
                const uint32_t buf = ci & 1u;
                const bool ok = __all_sync(0xffffffffu, mb_wait(&sh.afull[buf], (ci >> 1) & 1u, a.err_flag, &sh.abort_flag));
                ++ci;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                float v[32];
                if (half * 32 < t.n) tmem_read<BF16>(v, tbase + buf * TN);
#pragma unroll 1
                for (int col = 0; col + half * 32 < t.n; col += 64) {
                    float now[32];
                    tmem_wait(v);
#pragma unroll
                    for (int j = 0; j < 32; ++j) now[j] = v[j];
                    if (col + 64 + half * 32 < t.n) tmem_read<BF16>(v, tbase + buf * TN + col + 64);  // the next rows, while these leave
                    else {
                        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                        if (ok && lane == 0) mb_arrive(&sh.aempty[buf]);
                    }
                    emit<BF16>(a, st, rows + col, n0, qt, now);
                }
                if (half * 32 >= t.n && ok && lane == 0) mb_arrive(&sh.aempty[buf]);
                continue;
            }
            float acc[TN / 64][32];
#pragma unroll
            for (int c = 0; c < TN / 64; ++c)
#pragma unroll
                for (int j = 0; j < 32; ++j) acc[c][j] = 0.f;
            for (int kc = kb0; kc < kb1; kc += CHUNK, ++ci) {
                const uint32_t buf = ci & 1u;
                if (!__all_sync(0xffffffffu, mb_wait(&sh.afull[buf], (ci >> 1) & 1u, a.err_flag, &sh.abort_flag))) continue;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
                for (int c = 0; c < TN / 64; ++c) {
                    if (c * 64 + half * 32 < t.n) {
                        float v[32];
                        tmem_read<BF16>(v, tbase + buf * TN + c * 64);
                        tmem_wait(v);
#pragma unroll
                        for (int j = 0; j < 32; ++j) acc[c][j] += v[j];
                    }
                }
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) mb_arrive(&sh.aempty[buf]);
            }
            if (a.split > 1) {  // one unit per cluster: the ring is read, the partial tile [rows][128 features] takes its place
                float* part = reinterpret_cast<float*>(ring);
#pragma unroll
                for (int c = 0; c < TN / 64; ++c)
#pragma unroll
                    for (int j = 0; j < 32; ++j) {
                        const int col = c * 64 + half * 32 + value_row<BF16>(lane, j);
                        if (col < t.n) part[col * IMG_ROWS + quarter * 32 + value_feature<BF16>(lane, j)] = acc[c][j];
                    }
                break;
            }
#pragma unroll
            for (int c = 0; c < TN / 64; ++c)
                if (c * 64 + half * 32 < t.n) emit<BF16>(a, st, rows + c * 64, n0, qt, acc[c]);
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (sh.abort_flag) {  // a wait ran out: the copies and MMAs in flight end before the CTA does and its accumulators are freed
        if (warp == 0) mb_land_ring(sh.full, issued, SLOTS);
        else if (warp == 1) {
            mma_commit(&sh.done);
            mb_land(&sh.done, 0);
        }
        __syncthreads();
    }
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    if (a.split > 1) {
        cluster_sync_all();
        const Unit t = unit_at(a, groups, u0);
        const float* part = reinterpret_cast<const float*>(ring);
        // a warp per row of 128 features; the ranks share the rows
        for (int col = rank * (THREADS / 32) + warp; col < t.n; col += a.split * (THREADS / 32)) {
            const float* at = part + col * IMG_ROWS + lane * 4;
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
            float4 p[MAX_SPLIT];  // all are asked for before the first is added
#pragma unroll
            for (int r = 0; r < MAX_SPLIT; ++r)
                if (r < a.split) p[r] = ld_dsmem_f32x4(dsmem_addr(at, r));
#pragma unroll
            for (int r = 0; r < MAX_SPLIT; ++r)
                if (r < a.split) v = make_float4(v.x + p[r].x, v.y + p[r].y, v.z + p[r].z, v.w + p[r].w);
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
    a.wide = a.ldy * (a.bf16 ? 2 : 4) % 16 == 0 && (uintptr_t)a.y % 16 == 0;
    void (*const kernels[2][2])(ImageGemmArgs) = {{image_gemm_kernel<false, false>, image_gemm_kernel<false, true>}, {image_gemm_kernel<true, false>, image_gemm_kernel<true, true>}};
    void (*const fn)(ImageGemmArgs) = kernels[mx][a.bf16 != 0];
    cudaError_t e = ensure_dyn_smem(fn, SMEM);
    if (e != cudaSuccess) return e;
    long long units;
    a.split = 1;
    if (a.first) {
        units = (long long)(a.pairs / TN + std::min(a.pairs, a.experts)) * a.tiles;  // at most
    } else {
        units = (long long)((a.M + TN - 1) / TN) * a.tiles;
        // Fewer units than half the SMs: their k-blocks are shared out, two at least for a CTA, as far as all clusters run at once (a cluster stays within the 16 or
        // 18 SMs of a GPC: twelve clusters of twelve took two rounds, 17 us where seven each take one).
        if (units * 2 <= sm_count) {
            for (a.split = (int)std::min<long long>(MAX_SPLIT, (a.kblocks + 1) / 2); a.split > 1 && units > 8LL * (16 / a.split); --a.split) {
            }
        }
    }
    if (units > 0x7FFFFFFF) return cudaErrorInvalidValue;
    a.kb_per = (a.kblocks + a.split - 1) / a.split;
    a.split = (a.kblocks + a.kb_per - 1) / a.kb_per;
    return launch_after(fn, dim3(a.split > 1 ? (unsigned)units * a.split : (unsigned)std::min<long long>(units, sm_count)), THREADS, SMEM, a.split, st, a);
}

}  // namespace hm

// Operand images of the tensor cores: rows of bf16 or of 4-bit microscaled floats, products of two images, products grouped by expert
// (image.cu, image_gemm.cu, mx4_gemv.cu).
#pragma once
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "common.cuh"

namespace hm {

// An image is tiles [blocks of 128 rows][k-blocks], a tile the shared-memory picture of 128 rows of 128 bytes: 64 bf16, or 256 codes of 4 bits (the
// value with the even index in the low half of its byte); 16-byte pieces XOR-ed by row & 7, the 128-byte swizzle of the MMA's operands.  In
// front of a tile of codes stand its 1024 scale bytes, as the tensor memory takes them: for either half of the 256 values, [32 rows][4 groups of 32 rows][4
// blocks of 32 values].  bf16 images are those of hm_pack_bf16_tc.  What a row has beyond K is zero; rows beyond the last are not written.
constexpr int IMG_ROWS = 128;
constexpr int IMG_CODES = IMG_ROWS * 128;  // bytes of a tile without its scales
constexpr int MX_SCALES = 1024;
constexpr int MX_TILE = MX_SCALES + IMG_CODES;
constexpr int MX_K = 256, BF_K = 64;       // values of a k-block
__host__ __device__ inline int img_kblocks(bool mx, int K) { return mx ? (K + MX_K - 1) / MX_K : (K + BF_K - 1) / BF_K; }
__host__ __device__ inline size_t img_tile(bool mx) { return mx ? MX_TILE : IMG_CODES; }
inline size_t img_bytes(bool mx, int rows, int K) { return ((size_t)rows + IMG_ROWS - 1) / IMG_ROWS * img_kblocks(mx, K) * img_tile(mx); }
// Byte of the scale of row r (of the block), block b (of 32 values of the k-block) in front of its tile.
__host__ __device__ inline int mx_scale_at(int r, int b) { return (b >> 2) * 512 + (r & 31) * 16 + (r >> 5) * 4 + (b & 3); }

// ---- plan of rows grouped by expert: int32 words ------------------------------------------------
//   first [experts + 1]   first block of 128 image rows of an expert; the last is the number of blocks
//   count [experts]       rows of an expert
//   place [pairs]         image row of a pair; -1: none
//   row [blocks * 128]    pair of an image row; -1: none
// An expert's rows keep the order of the pairs and start at a block of their own, so that its tiles are whole tiles of the image.
constexpr int PLAN_EXPERTS = 1024;
__host__ __device__ inline int plan_blocks(int pairs, int experts) { return pairs / IMG_ROWS + (pairs < experts ? pairs : experts); }
struct Plan {
    int32_t *first, *count, *place, *row;
    int pairs, experts, rows;  // rows: of the image, at most
};
inline size_t plan_ints(int pairs, int experts) { return 2 * (size_t)experts + 1 + pairs + (size_t)plan_blocks(pairs, experts) * IMG_ROWS; }
inline Plan plan_at(int32_t* p, int pairs, int experts) {
    return Plan{p, p + experts + 1, p + 2 * experts + 1, p + 2 * experts + 1 + pairs, pairs, experts, plan_blocks(pairs, experts) * IMG_ROWS};
}
cudaError_t launch_plan(const int32_t* ids, const Plan& p, cudaStream_t st);

struct PackArgs {
    const void* x;        // rows of K values, or of 2 K with glu: silu(first K) * last K
    int bf16, glu;
    size_t ldx;           // elements from row to row
    int rows, K;          // rows: of x
    const int32_t* place; // optional, [rows * top]: row r of x goes to the image rows place[r * top ..], -1: none
    int top, image_rows;
    unsigned char* image;
};
cudaError_t launch_image_pack(const PackArgs& a, bool mx, cudaStream_t st);
cudaError_t launch_image_unpack(const unsigned char* image, bool mx, int rows, int K, void* out, bool bf16, size_t ld, cudaStream_t st);
// GGUF blocks of 17 bytes [rows][K / 32] -> image.
cudaError_t launch_image_blocks(const uint8_t* blocks, int rows, int K, unsigned char* image, cudaStream_t st);

struct SumArgs {
    const void *rows, *resid;  // [tokens * top][W]; [tokens][W] f32 or null
    int rows_bf16, y_bf16;
    const int32_t* ids;        // [tokens * top]
    const float* weights;
    int tokens, top, experts, W;
    void* y;
};
cudaError_t launch_expert_sum(const SumArgs& a, cudaStream_t st);

struct ImageGemmArgs {
    const unsigned char *x, *w;
    size_t w_stride;      // bytes from an expert's image to the next
    int M, N, K;          // M: rows without a plan
    void* y;
    size_t ldy;           // elements
    int bf16;             // y is bf16
    const int32_t* first; // plan (null: one group of M rows): rows go to y[row[image row]]
    const int32_t *count, *row;
    int experts, pairs, rows;  // rows: of the image, at most
    int* err_flag;
    // filled in by launch_image_gemm
    int kblocks, tiles, split, kb_per, wide;
};
cudaError_t launch_image_gemm(ImageGemmArgs a, bool mx, int sm_count, cudaStream_t st);

struct MxGemvArgs {
    const void* x;
    int bf16;
    size_t ldx;
    int M;                // rows, 1 .. 8; with ids: 1, and `pairs` of them
    const unsigned char* w;
    size_t w_stride;
    int N, K;
    void* y;
    size_t ldy;
    int y_bf16;
    const int32_t* ids;   // optional, [pairs]: pair p is row p / top of x times the image of expert ids[p]; left as it is where there is none
    int pairs, top, experts;
    int* err_flag;
    // filled in by launch_mx4_gemv
    int kblocks, tiles, split, kb_per, slots;
};
constexpr int MX_GEMV_K = 32768;  // widest row
cudaError_t launch_mx4_gemv(MxGemvArgs a, int sm_count, cudaStream_t st);

// Launch that may begin while the kernel in front of it ends (each of these kernels waits for that before it touches memory).  Short kernels let the next one
// begin at once; the plan and the products do not: what stood by for their end took 1 to 3 us of a chain plan, pack, product.
template <typename... P, typename... A>
inline cudaError_t launch_after(void (*k)(P...), dim3 grid, int threads, size_t smem, int cluster, cudaStream_t st, A... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim = {(unsigned)cluster, 1, 1};
    cfg.attrs = at;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, k, args...);
}

// ---- codes and scales ---------------------------------------------------------------------------
#ifdef __CUDACC__
// Eight values of [-8, 8] (or beyond: they saturate) to the nearest codes, ties to even; v[0] in the lowest four bits.
__device__ __forceinline__ uint32_t mx_codes(const float (&v)[8]) {
    uint32_t r;
    asm("{ .reg .b8 a, b, c, d;\n"
        "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n"
        "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n"
        "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n"
        "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n"
        "mov.b32 %0, {a, b, c, d}; }"
        : "=r"(r)
        : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
    return r;
}
// What a lane loads at once: up to 16 bytes.
template <int BYTES> struct Words { using type = uint4; };
template <> struct Words<8> { using type = uint2; };
template <> struct Words<4> { using type = uint32_t; };
// V values from element k of a row of n on; those beyond are zero.
template <int V, bool BF16, typename Word>
__device__ __forceinline__ void load_ragged(const char* x, int k, int n, Word* w) {
    uint32_t* o = reinterpret_cast<uint32_t*>(w);
#pragma unroll
    for (int e = 0; e < V; ++e) {
        if (BF16) {
            const uint32_t b = k + e < n ? __ldg(reinterpret_cast<const uint16_t*>(x) + k + e) : 0u;
            o[e / 2] = e & 1 ? o[e / 2] | b << 16 : b;
        } else
            o[e] = k + e < n ? __ldg(reinterpret_cast<const uint32_t*>(x) + k + e) : 0u;
    }
}
template <int V, bool BF16, typename Word>
__device__ __forceinline__ void widen(const Word* w, float (&v)[V]) {
    const uint32_t* o = reinterpret_cast<const uint32_t*>(w);
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = BF16 ? (e & 1 ? bf16_hi(o[e / 2]) : bf16_lo(o[e / 2])) : __uint_as_float(o[e]);
}
// Eight codes as four words of two f16.
__device__ __forceinline__ void mx_halves(uint32_t codes, uint32_t (&h)[4]) {
    asm("{ .reg .b8 a, b, c, d;\n"
        "mov.b32 {a, b, c, d}, %4;\n"
        "cvt.rn.f16x2.e2m1x2 %0, a;\n"
        "cvt.rn.f16x2.e2m1x2 %1, b;\n"
        "cvt.rn.f16x2.e2m1x2 %2, c;\n"
        "cvt.rn.f16x2.e2m1x2 %3, d; }"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
        : "r"(codes));
}
// 2^(s - 127), 255: NaN.
__device__ __forceinline__ float mx_scale(uint32_t s) { return __uint_as_float(s == 0 ? 0x00400000u : s == 255u ? 0x7FC00000u : s << 23); }
#endif

}  // namespace hm

// Rotary positions: the first `rot` elements of every head as rot / 2 pairs (a, b), each turned by turns[i] * position of a full turn:
//   a' = mult (a cos - b sin),  b' = mult (a sin + b cos)
// Pairs are neighbours (2 i, 2 i + 1) or stand half of `rot` apart; the elements behind `rot` are copied.
//
// Angles: turns * position in 64 bits, less its nearest quarter, leaves at most an eighth of a turn, which f32 holds to 2^-28; so a far position is as
// exact as a near one.  A block has `rows` rows: it computes their sines and cosines once, in shared memory, and all heads take them from there; the elements that a thread
// begins with are on their way meanwhile.  What bounds it is bytes, for few rows the chain of a position's load, its sine, a barrier and the rows'
// elements.  8191 rows of 14 heads (and 2 beside them) of 128 in bf16: 13.0 us (4.5 TB/s) against 15.4 with one row to a block and elements loaded behind the sines.  Blocks of 128 threads:
// 12.3 us there, but 3.5 instead of 2.8 us for 64 rows of 36 heads.
#include "rope.h"

#include "rows.cuh"

namespace hm {
namespace {

constexpr int RT = 256;

// V elements per access (1 where sizes or addresses are not multiples of 16 bytes).
template <bool BF16, int V, bool NEXT>
__global__ void __launch_bounds__(RT) rope_kernel(const RopeArgs a, int rows) {
    extern __shared__ float2 cs[];  // [rows][rot / 2] cosine and sine
    const int half = a.rot / 2, m0 = blockIdx.x * rows, tid = threadIdx.x, here = min(rows, a.M - m0);
    const int rest = a.y == a.x ? 0 : a.dim - a.rot;
    // pieces of a head: V elements of both halves, or V / 2 pairs; then V elements that are copied
    const int turned = NEXT ? (V == 1 ? half : a.rot / V) : half / V, pieces = turned + rest / V, of_row = a.heads * pieces, all = here * of_row;
    constexpr bool TWO = !NEXT || V == 1;  // a piece is two runs of V elements
    const int step = NEXT ? 1 : half;
    struct Piece {
        int r, p;
        size_t x, y;
        float u[V], w[V];
    };
    auto load = [&](int i, Piece& s) {
        s.r = i / of_row;
        const int j = i - s.r * of_row, h = j / pieces;
        s.p = j - h * pieces;
        const int at = s.p >= turned ? a.rot + (s.p - turned) * V : NEXT && V == 1 ? 2 * s.p : s.p * V;
        s.x = (size_t)(m0 + s.r) * a.ldx + (size_t)h * a.dim + at;
        s.y = (size_t)(m0 + s.r) * a.ldy + (size_t)h * a.dim + at;
        load_row<BF16, V>(a.x, s.x, s.u);
        if (TWO && s.p < turned) load_row<BF16, V>(a.x, s.x + step, s.w);
    };
    Piece s;
    int i = tid;
    if (i < all) load(i, s);
    for (int k = tid; k < here * half; k += RT) {
        const int r = k / half, j = k - r * half;
        const double t = a.turns[j] * (double)__ldg(a.pos + m0 + r), q = rint(4.0 * t);
        float sn, c;
        sincospif(2.0f * (float)(t - 0.25 * q), &sn, &c);
        const int quarter = (int)((long long)q & 3);
        const float cc = quarter & 1 ? -sn : c, ss = quarter & 1 ? c : sn;  // turned by one quarter, or by none; then by a half
        cs[k] = make_float2((quarter & 2 ? -cc : cc) * a.magnitude, (quarter & 2 ? -ss : ss) * a.magnitude);
    }
    __syncthreads();
    while (i < all) {
        const float2* t = cs + s.r * half;
        if (s.p >= turned) {
            store_row<BF16, V>(a.y, s.y, s.u);
        } else if constexpr (TWO) {
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float2 z = t[s.p * V + e];
                const float x = s.u[e], y = s.w[e];
                s.u[e] = fmaf(x, z.x, -(y * z.y));
                s.w[e] = fmaf(x, z.y, y * z.x);
            }
            store_row<BF16, V>(a.y, s.y, s.u);
            store_row<BF16, V>(a.y, s.y + step, s.w);
        } else {
#pragma unroll
            for (int e = 0; e < V; e += 2) {
                const float2 z = t[(s.p * V + e) / 2];
                const float x = s.u[e], y = s.u[e + 1];
                s.u[e] = fmaf(x, z.x, -(y * z.y));
                s.u[e + 1] = fmaf(x, z.y, y * z.x);
            }
            store_row<BF16, V>(a.y, s.y, s.u);
        }
        i += RT;
        if (i < all) load(i, s);
    }
}

template <bool BF16, int V>
cudaError_t launch_v(const RopeArgs& a, int sm_count, cudaStream_t st) {
    // rows until every thread has something to do, 16 at most, but no fewer blocks than four for every SM
    const int pieces = a.heads * (a.neighbours ? (V == 1 ? a.rot / 2 : a.rot / V) : a.rot / 2 / V);
    int rows = 1;
    while (rows < 16 && rows * pieces < RT && ((long)a.M + 2 * rows - 1) / (2 * rows) >= 4 * sm_count) rows *= 2;
    const unsigned grid = (unsigned)(((long)a.M + rows - 1) / rows);
    const size_t smem = sizeof(float2) * (size_t)(a.rot / 2) * rows;
    if (a.neighbours) rope_kernel<BF16, V, true><<<grid, RT, smem, st>>>(a, rows);
    else rope_kernel<BF16, V, false><<<grid, RT, smem, st>>>(a, rows);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_rope(const RopeArgs& a, int sm_count, cudaStream_t st) {
    const int size = a.bf16 ? 2 : 4, v = 16 / size;
    const bool wide = (((uintptr_t)a.x | (uintptr_t)a.y | (a.ldx * size) | (a.ldy * size) | ((size_t)a.dim * size)) & 15) == 0 && a.rot % (a.neighbours ? v : 2 * v) == 0;
    if (a.bf16) return wide ? launch_v<true, 8>(a, sm_count, st) : launch_v<true, 1>(a, sm_count, st);
    return wide ? launch_v<false, 4>(a, sm_count, st) : launch_v<false, 1>(a, sm_count, st);
}

}  // namespace hm

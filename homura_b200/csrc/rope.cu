// Rotary positions: the first `rot` elements of every head as rot / 2 pairs (a, b), each turned by turns[i] * position of a full turn:
//   a' = mult (a cos - b sin),  b' = mult (a sin + b cos)
// Pairs are neighbours (2 i, 2 i + 1) or stand half of `rot` apart; the elements behind `rot` are copied.
//
// Angles: turns * position in 64 bits, less its nearest quarter, leaves at most an eighth of a turn, which f32 holds to 2^-28; so a far position is as
// exact as a near one.  A block computes the sines and cosines of its rows once, in shared memory, and all heads take them from there.
#include "rope.h"

#include "rows.cuh"

namespace hm {
namespace {

constexpr int RT = 256;

// One row per blockIdx.x; V elements per access (1 where sizes or addresses are not multiples of 16 bytes).
template <bool BF16, int V, bool NEXT>
__global__ void __launch_bounds__(RT) rope_kernel(const RopeArgs a) {
    extern __shared__ float2 cs[];  // [rot / 2] cosine and sine
    const int half = a.rot / 2, m = blockIdx.x, tid = threadIdx.x;
    const int pos = a.pos[m];
    for (int i = tid; i < half; i += RT) {
        const double t = a.turns[i] * (double)pos, q = rint(4.0 * t);
        float s, c;
        sincospif(2.0f * (float)(t - 0.25 * q), &s, &c);
        const int quarter = (int)((long long)q & 3);
        const float cc = quarter & 1 ? -s : c, ss = quarter & 1 ? c : s;  // turned by one quarter, or by none; then by a half
        cs[i] = make_float2((quarter & 2 ? -cc : cc) * a.magnitude, (quarter & 2 ? -ss : ss) * a.magnitude);
    }
    __syncthreads();
    const int rest = a.y == a.x ? 0 : a.dim - a.rot;
    // pieces of a head: V elements of both halves, or V / 2 pairs; then V elements that are copied
    const int turned = NEXT ? (V == 1 ? half : a.rot / V) : half / V, pieces = turned + rest / V;
    for (int i = tid; i < a.heads * pieces; i += RT) {
        const int h = i / pieces, p = i - h * pieces;
        const size_t xb = (size_t)m * a.ldx + (size_t)h * a.dim, yb = (size_t)m * a.ldy + (size_t)h * a.dim;
        if (p >= turned) {
            float v[V];
            const int at = a.rot + (p - turned) * V;
            load_row<BF16, V>(a.x, xb + at, v);
            store_row<BF16, V>(a.y, yb + at, v);
        } else if constexpr (!NEXT || V == 1) {
            const int at = NEXT ? 2 * p : p * V, step = NEXT ? 1 : half;
            float u[V], w[V];
            load_row<BF16, V>(a.x, xb + at, u);
            load_row<BF16, V>(a.x, xb + at + step, w);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float2 t = cs[p * V + e];
                const float x = u[e], z = w[e];
                u[e] = fmaf(x, t.x, -(z * t.y));
                w[e] = fmaf(x, t.y, z * t.x);
            }
            store_row<BF16, V>(a.y, yb + at, u);
            store_row<BF16, V>(a.y, yb + at + step, w);
        } else {
            float u[V];
            load_row<BF16, V>(a.x, xb + p * V, u);
#pragma unroll
            for (int e = 0; e < V; e += 2) {
                const float2 t = cs[(p * V + e) / 2];
                const float x = u[e], z = u[e + 1];
                u[e] = fmaf(x, t.x, -(z * t.y));
                u[e + 1] = fmaf(x, t.y, z * t.x);
            }
            store_row<BF16, V>(a.y, yb + p * V, u);
        }
    }
}

template <bool BF16, int V>
cudaError_t launch_v(const RopeArgs& a, cudaStream_t st) {
    const size_t smem = sizeof(float2) * (a.rot / 2);
    if (a.neighbours) rope_kernel<BF16, V, true><<<(unsigned)a.M, RT, smem, st>>>(a);
    else rope_kernel<BF16, V, false><<<(unsigned)a.M, RT, smem, st>>>(a);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_rope(const RopeArgs& a, cudaStream_t st) {
    const int size = a.bf16 ? 2 : 4, v = 16 / size;
    const bool wide = (((uintptr_t)a.x | (uintptr_t)a.y | (a.ldx * size) | (a.ldy * size) | ((size_t)a.dim * size)) & 15) == 0 && a.rot % (a.neighbours ? v : 2 * v) == 0;
    if (a.bf16) return wide ? launch_v<true, 8>(a, st) : launch_v<true, 1>(a, st);
    return wide ? launch_v<false, 4>(a, st) : launch_v<false, 1>(a, st);
}

}  // namespace hm

// Softmax attention over the 8-bit paged cache:
//   out[row, head] = sum over the positions t <= row_pos whose page exists of softmax_t(scale q . k_t) v_t,   zeros where there is no such position.
// Page i of a row is shared[i] for i < n_shared and its sequence's page table entry behind them.
//
// One CTA per row and head, a page at a time with the running maximum and sum; everything in f32.
#include "kv8.h"
#include "rows.cuh"

namespace hm {
namespace {

constexpr int AT = 128;

template <bool BF16>
__global__ void __launch_bounds__(AT) kv8_attn_kernel(const Kv8AttnArgs a) {
    __shared__ float q_s[KV8_MAX_DIM], p_s[KV8_PAGE], part[AT];
    __shared__ float s_corr, s_max, s_sum;
    const int h = blockIdx.x, m = blockIdx.y, tid = threadIdx.x, dim = a.pool.dim, vdim = a.pool.vdim;
    const int seq = a.row_seq[m];
    if ((unsigned)seq >= (unsigned)a.pool.n_seq) return;
    const int len = min(a.row_pos[m], a.pool.max_pages * KV8_PAGE - 1) + 1, kvh = h / (a.heads / a.pool.kv_heads);
    for (int d = tid; d < dim; d += AT) {
        float x[1];
        load_row<BF16, 1>(a.q, (size_t)m * a.ldq + (size_t)h * dim + d, x);
        q_s[d] = x[0] * (a.scale * 1.4426950408889634f);
    }
    if (tid == 0) {
        s_max = -INFINITY;
        s_sum = 0.f;
    }
    float o[KV8_MAX_DIM / AT] = {};
    __syncthreads();
    for (int pi = 0; pi * KV8_PAGE < len; ++pi) {
        const int page = pi < a.n_shared ? a.shared[pi] : a.pool.page_table[(size_t)seq * a.pool.max_pages + pi];
        if ((unsigned)page >= (unsigned)a.pool.n_pages) continue;
        const unsigned char* block = a.pool.pages + ((size_t)page * a.pool.kv_heads + kvh) * kv8_block_bytes(dim, vdim);
        const float* scales = reinterpret_cast<const float*>(block);
        const unsigned char *kc = block + 8 * KV8_PAGE, *vc = kc + KV8_PAGE * kv8_pad(dim);
        const int nt = min(KV8_PAGE, len - pi * KV8_PAGE), t = tid >> 1;
        float s = 0.f;
        for (int d = tid & 1; d < dim; d += 2) s = fmaf(q_s[d], (float)((int)kc[(d >> 5) * (KV8_PAGE * 32) + kv8_key_row(t) * 32 + (d & 31)] - 128), s);
        part[tid] = s;
        __syncthreads();
        if (tid < 32) {
            float e[2];
            for (int i = 0; i < 2; ++i) {
                const int u = tid + 32 * i;
                e[i] = u < nt ? (part[2 * u] + part[2 * u + 1]) * scales[u] : -INFINITY;
            }
            const float old = s_max, mx = fmaxf(old, warp_max(fmaxf(e[0], e[1]))), ref = mx == -INFINITY ? 0.f : mx;
            e[0] = exp2f(e[0] - ref);
            e[1] = exp2f(e[1] - ref);
            const float l = warp_sum(e[0] + e[1]);
            for (int i = 0; i < 2; ++i) p_s[tid + 32 * i] = tid + 32 * i < nt ? e[i] * scales[KV8_PAGE + tid + 32 * i] : 0.f;
            __syncwarp();
            if (tid == 0) {
                s_corr = exp2f(old - ref);
                s_sum = fmaf(s_sum, s_corr, l);
                s_max = mx;
            }
        }
        __syncthreads();
        for (int i = 0; i < KV8_MAX_DIM / AT; ++i) {
            const int d = tid + i * AT;
            if (d >= vdim) break;
            float v = 0.f;
            for (int u = 0; u < nt; ++u) v = fmaf(p_s[u], (float)((int)vc[(d >> 5) * (KV8_PAGE * 32) + u * 32 + (d & 31)] - 128), v);
            o[i] = fmaf(o[i], s_corr, v);
        }
        __syncthreads();
    }
    for (int i = 0; i < KV8_MAX_DIM / AT; ++i) {
        const int d = tid + i * AT;
        if (d >= vdim) break;
        const float y[1] = {s_sum == 0.f ? 0.f : o[i] / s_sum};
        store_row<BF16, 1>(a.out, (size_t)m * a.ldo + (size_t)h * vdim + d, y);
    }
}

}  // namespace

size_t kv8_attn_bytes(int, int, int, int, int, int) { return 16; }

cudaError_t launch_kv8_attn(const Kv8AttnArgs& a, int, cudaStream_t st) {
    const dim3 grid((unsigned)a.heads, (unsigned)a.M);
    if (a.bf16) kv8_attn_kernel<true><<<grid, AT, 0, st>>>(a);
    else kv8_attn_kernel<false><<<grid, AT, 0, st>>>(a);
    return cudaGetLastError();
}

}  // namespace hm

// Rows of f32 or bf16 elements in device memory, taken V consecutive elements at a time: one access of V elements (16 bytes, or 8 of four bf16), or one element.
#pragma once
#include "common.cuh"

namespace hm {

template <bool BF16, int V>
__device__ __forceinline__ void load_row(const void* base, size_t at, float (&v)[V]) {
    if constexpr (V == 1) {
        v[0] = BF16 ? bf16_bits_to_f32(static_cast<const uint16_t*>(base)[at]) : static_cast<const float*>(base)[at];
    } else if constexpr (BF16) {
        uint32_t w[V / 2];
        if constexpr (V == 8) {
            const uint4 u = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(base) + at);
            w[0] = u.x; w[1] = u.y; w[2] = u.z; w[3] = u.w;
        } else {
            const uint2 u = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(base) + at);
            w[0] = u.x; w[1] = u.y;
        }
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {
            v[2 * i] = bf16_lo(w[i]);
            v[2 * i + 1] = bf16_hi(w[i]);
        }
    } else {
        const float4 u = *reinterpret_cast<const float4*>(static_cast<const float*>(base) + at);
        v[0] = u.x; v[1] = u.y; v[2] = u.z; v[3] = u.w;
    }
}

template <bool BF16, int V>
__device__ __forceinline__ void store_row(void* base, size_t at, const float (&v)[V]) {
    if constexpr (V == 1) {
        if (BF16) static_cast<uint16_t*>(base)[at] = (uint16_t)bf16x2_rne(v[0], 0.f);
        else static_cast<float*>(base)[at] = v[0];
    } else if constexpr (BF16) {
        uint32_t w[V / 2];
#pragma unroll
        for (int i = 0; i < V / 2; ++i) w[i] = bf16x2_rne(v[2 * i], v[2 * i + 1]);
        if constexpr (V == 8) *reinterpret_cast<uint4*>(static_cast<uint16_t*>(base) + at) = make_uint4(w[0], w[1], w[2], w[3]);
        else *reinterpret_cast<uint2*>(static_cast<uint16_t*>(base) + at) = make_uint2(w[0], w[1]);
    } else {
        *reinterpret_cast<float4*>(static_cast<float*>(base) + at) = make_float4(v[0], v[1], v[2], v[3]);
    }
}

}  // namespace hm

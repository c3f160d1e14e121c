// Rotary positions of rows of heads (rope.cu).
#pragma once
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace hm {

constexpr int ROPE_MAX_DIM = 1024;  // elements of a head

struct RopeArgs {
    const void* x;         // [M] rows of heads * dim elements, ldx apart
    void* y;               // the same, ldy apart; may be x
    size_t ldx, ldy;
    int bf16;
    int M, heads, dim, rot;
    int neighbours;        // pairs are (2 i, 2 i + 1); else (i, i + rot / 2)
    const int32_t* pos;    // [M]
    const double* turns;   // [rot / 2] turns per position
    float magnitude;       // the rotated elements are multiplied with this
};
cudaError_t launch_rope(const RopeArgs& a, int sm_count, cudaStream_t st);

}  // namespace hm

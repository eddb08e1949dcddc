// What the decode kernels of the 4-bit cache share: the call's operands, the division of its tiles
// among persistent CTAs, and the scratch through which they hand over to the finishing kernel.
#pragma once

#include "kv4.cuh"

namespace asu {
namespace kv4 {

constexpr int kTile = 64;  // entries a tile

struct Operands {
    const __nv_bfloat16* q;
    int64_t q_token, q_head;  // elements
    const uint8_t* pool;
    uint64_t pool_token, pool_pitch;  // bytes
    int32_t pool_rows;
    const int32_t* slots;
    int64_t slots_token;
    int32_t tokens, heads, topk;
    float scale_log2;  // scale * log2(e): the kernels' exponentials are powers of two
    bool q_aligned;    // every q row starts on 16 bytes
    __nv_bfloat16* out;
    float* lse;
    __nv_bfloat16* weights;
    int32_t* status;
};

// Row (token of one part of the call) r has `tiles` consecutive units; CTA i takes the units
// [start(i), start(i + 1)), which differ by one at most.  A row that lies in several CTAs' ranges is
// joined afterwards.  The division depends on the call's sizes alone, so results repeat.
struct Division {
    int32_t rows, tiles, ctas;
    __host__ __device__ __forceinline__ int64_t units() const { return static_cast<int64_t>(rows) * tiles; }
    __host__ __device__ __forceinline__ int64_t start(int i) const { return units() * i / ctas; }
    __host__ __device__ __forceinline__ int cta_of(int64_t u) const {
        return static_cast<int>(((u + 1) * ctas - 1) / units());
    }
    // Scratch slot of CTA i's piece of a row that starts at unit `row_start`: a CTA's range holds at
    // most two pieces of rows, one at its start and one at its end.
    __host__ __device__ __forceinline__ int piece(int i, int64_t row_start) const {
        return 2 * i + (start(i) >= row_start ? 0 : 1);
    }
};

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return reinterpret_cast<const uint32_t&>(v);
}

// kv4_decode_wide.cu: any number of heads up to 128, at the cost of 128.
int64_t wide_workspace(int64_t tokens, int64_t topk, bool weights);
int launch_wide(cudaStream_t stream, const Operands& op, void* workspace);

}  // namespace kv4
}  // namespace asu

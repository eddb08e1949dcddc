// What the decode kernels of the 4-bit cache share: the call's operands, the division of its tiles
// among persistent CTAs, and the scratch through which they hand over to the finishing kernel.
#pragma once

#include "kv4.cuh"

namespace asu {
namespace kv4 {

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
// [start(i), start(i + 1)), `each` of them and one more in the first `more` CTAs.  A row that lies in
// several CTAs' ranges is joined afterwards.  The division depends on the call's sizes alone, so results
// repeat.  All in 32 bits: 64-bit divisions were a third of the kernels' code.
struct Division {
    int32_t rows, tiles, ctas, each, more;
    Division() = default;
    Division(int64_t rows_, int64_t tiles_, int64_t most) {
        rows = static_cast<int32_t>(rows_);
        tiles = static_cast<int32_t>(tiles_);
        const int64_t units = rows_ * tiles_;  // below 2^26: tokens, entries and parts are bounded
        ctas = static_cast<int32_t>(units < most ? units : most);
        each = static_cast<int32_t>(units / ctas);
        more = static_cast<int32_t>(units % ctas);
    }
    __host__ __device__ __forceinline__ int32_t start(int32_t i) const { return i * each + (i < more ? i : more); }
    __host__ __device__ __forceinline__ int32_t cta_of(int32_t u) const {
        const int32_t first = more * (each + 1);
        return u < first ? u / (each + 1) : more + (u - first) / each;
    }
    // Scratch slot of CTA i's piece of a row that starts at unit `row_start`: a CTA's range holds at
    // most two pieces of rows, one at its start and one at its end.
    __host__ __device__ __forceinline__ int32_t piece(int32_t i, int32_t row_start) const {
        return 2 * i + (start(i) >= row_start ? 0 : 1);
    }
};

// Walks the units of a CTA's range.
struct Walk {
    int32_t u, row, tile;
    __device__ __forceinline__ Walk(const Division& d, int32_t start) {
        u = start;
        row = start / d.tiles;
        tile = start - row * d.tiles;
    }
    __device__ __forceinline__ void next(const Division& d) {
        ++u;
        if (++tile == d.tiles) {
            tile = 0;
            ++row;
        }
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

// kv4_decode.cu
int64_t decode_workspace(int64_t tokens, int64_t heads, int64_t topk, bool weights);
int launch_decode(cudaStream_t stream, const Operands& op, void* workspace);

}  // namespace kv4
}  // namespace asu

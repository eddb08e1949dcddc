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

// Row (token) r has `tiles` consecutive units; CTA i takes the units [start(i), start(i + 1)).  Either all CTAs take
// the same number of units, `each` and one more in the first `more` of them, wherever rows begin and end; or every row
// is cut in `parts` of `each` units (the last may be shorter) and a CTA takes one.  Both end when the CTA with the most
// units does; the second spares CTAs a change of rows in the middle of their range (q, the output), which costs as
// much as `change` units, and leaves fewer pieces to join.  It depends on the call's sizes alone, so results
// repeat.  All in 32 bits: 64-bit divisions were a third of the kernels' code.
struct Division {
    int32_t rows, tiles, ctas, each, more, parts;  // parts 0: the first kind
    Division() = default;
    Division(int64_t rows_, int64_t tiles_, int64_t most, int64_t change) {
        rows = static_cast<int32_t>(rows_);
        tiles = static_cast<int32_t>(tiles_);
        const int64_t units = rows_ * tiles_;  // below 2^26: tokens, entries and parts are bounded
        ctas = static_cast<int32_t>(units < most ? units : most);
        each = static_cast<int32_t>(units / ctas);
        more = static_cast<int32_t>(units % ctas);
        parts = 0;
        if (rows_ <= most) {
            int64_t cut = most / rows_ < tiles_ ? most / rows_ : tiles_;
            const int64_t per = (tiles_ + cut - 1) / cut;
            if (per <= each + (more > 0) + change) {
                cut = (tiles_ + per - 1) / per;
                parts = static_cast<int32_t>(cut);
                each = static_cast<int32_t>(per);
                ctas = static_cast<int32_t>(rows_ * cut);
                more = 0;
            }
        }
    }
    __host__ __device__ __forceinline__ int32_t start(int32_t i) const {
        if (parts > 0) return i / parts * tiles + i % parts * each;
        return i * each + (i < more ? i : more);
    }
    __host__ __device__ __forceinline__ int32_t cta_of(int32_t u) const {
        if (parts > 0) return u / tiles * parts + u % tiles / each;
        const int32_t first = more * (each + 1);
        return u < first ? u / (each + 1) : more + (u - first) / each;
    }
    // Does any row lie in several CTAs' ranges, so that there are pieces?  (Ranges of unequal sizes cannot all start with
    // a row: the units are a multiple of `tiles`.)
    bool shares() const { return parts > 0 ? parts > 1 : tiles > 1 && (more > 0 || each % tiles != 0); }
    // Scratch slot of CTA i's piece of a row that starts at unit `row_start`: a CTA's range holds at
    // most two pieces of rows, one at its start and one at its end.
    __host__ __device__ __forceinline__ int32_t piece(int32_t i, int32_t row_start) const {
        if (parts > 0) return 2 * i;
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

__device__ __forceinline__ void shared_store16(uint32_t at, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}

// 32 latents as four 16-byte chunks of a swizzled row; chunk i goes to `at` with i in address bits 4 and 5.
__device__ __forceinline__ void dequantise(const uint4& code, uint32_t scales, uint32_t at) {
    const uint32_t w[4] = {code.x, code.y, code.z, code.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        __nv_bfloat162 s, c;
        scale_pair(scales, i / 2, s, c);
        uint32_t v[4];
        unpack_word(w[i], s, c, v);
        shared_store16(at ^ (i << 4), v[0], v[1], v[2], v[3]);
    }
}

// 8 values that start on any element.
__device__ __forceinline__ uint4 load_unaligned(const __nv_bfloat16* p) {
    uint32_t w[4];
    const unsigned short* s = reinterpret_cast<const unsigned short*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i)
        w[i] = static_cast<uint32_t>(__ldg(s + 2 * i)) | (static_cast<uint32_t>(__ldg(s + 2 * i + 1)) << 16);
    return make_uint4(w[0], w[1], w[2], w[3]);
}

__device__ __forceinline__ bool is_there(const Operands& op, int64_t token, int e) {
    const int32_t s = __ldg(op.slots + token * op.slots_token + e);
    return s >= 0 && s < op.pool_rows;
}

// Entry e's weight from the sum over the heads.  A head whose scores are not numbers makes the sum NaN, for entries that
// are not there too (their 0 times its factor): those stay at 0.
__device__ __forceinline__ float weight_of(const Operands& op, int64_t token, int e, float sum) {
    return sum == sum || is_there(op, token, e) ? sum : 0.0f;
}

inline int64_t align256(int64_t x) { return (x + 255) / 256 * 256; }

// kv4_decode.cu: up to kTallHeads heads
constexpr int kTallHeads = 64;
int64_t tall_workspace(int64_t tokens, int64_t heads, int64_t topk, bool weights);
int64_t tall_weights(int64_t heads, int64_t topk);  // bytes of it for a token's weights
int launch_tall(cudaStream_t stream, const Operands& op, void* workspace);
// kv4_decode_wide.cu: more
int64_t wide_workspace(int64_t tokens, int64_t topk, bool weights);
int64_t wide_weights(int64_t topk);
int launch_wide(cudaStream_t stream, const Operands& op, void* workspace);

}  // namespace kv4
}  // namespace asu

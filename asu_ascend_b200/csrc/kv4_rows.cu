// Write and read side of the 4-bit MLA cache: bf16 / fp16 rows -> 416-byte rows, and back to bf16.
//
// Mathematics, per group of 16 values with a = max |x|:
//   s = a / 7 rounded to a number with three bits behind the point (ties to even), clamped to the
//       scale byte's range [2^-18, 15360]
//   n = clamp(rint(x / s), -7, 7) + 8
// s is at most 1/16 below a / 7, so x / s stays below 7.5 and no value of an unclamped group is off
// by more than s / 2.  Both roundings have exact ties among 16-bit inputs (x / s = k + 1/2), so the
// quotients must be the correctly rounded ones: a / 7 is an IEEE division, and x * (1 / s) is
// corrected by one residual step (Markstein 1990), which gives every quotient that is representable
// exactly -- the ties are.
//
// One warp per row, one lane per group: the lane loads its 32 bytes, needs no exchange with other
// lanes for the maximum, and stores 8 bytes of nibbles and one scale byte; 8 lanes move the
// rope part.  Bound by HBM: 1152 bytes in and 416 out per row (the other way round when reading).
#include <cuda_fp16.h>

#include "kv4.cuh"

namespace asu {
namespace {

using namespace kv4;

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;

template <typename T>
__device__ __forceinline__ float to_float(T v);
template <>
__device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_float<__half>(__half v) { return __half2float(v); }

// 8 consecutive 16-bit values; kVec: 16-byte aligned.
template <bool kVec>
__device__ __forceinline__ uint4 load8(const uint16_t* p) {
    if constexpr (kVec) {
        return __ldg(reinterpret_cast<const uint4*>(p));
    } else {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
            w[i] = static_cast<uint32_t>(__ldg(p + 2 * i)) | (static_cast<uint32_t>(__ldg(p + 2 * i + 1)) << 16);
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
}

template <typename T, bool kVec>
__global__ void __launch_bounds__(kThreads)
kv4_pack_kernel(const uint16_t* __restrict__ src, int64_t src_pitch, int64_t n, const int32_t* __restrict__ slots,
                uint8_t* __restrict__ pool, int64_t pool_rows, uint64_t pool_pitch, int32_t* status) {
    pdl_wait();
    pdl_trigger();
    const int lane = threadIdx.x & 31;
    int32_t bits = 0;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5); i < n;
         i += static_cast<int64_t>(gridDim.x) * kWarps) {
        const int64_t slot = slots != nullptr ? static_cast<int64_t>(__ldg(slots + i)) : i;
        if (slot == kNotFound) continue;
        if (slot < 0 || slot >= pool_rows) {
            bits |= ASU_ST_BAD_QUERY;
            continue;
        }
        const uint16_t* row = src + i * src_pitch;
        uint8_t* dst = pool + static_cast<uint64_t>(slot) * pool_pitch;
        uint4 raw[2];
        raw[0] = load8<kVec>(row + lane * kGroup);
        raw[1] = load8<kVec>(row + lane * kGroup + 8);
        uint4 rope = make_uint4(0, 0, 0, 0);
        if (lane < kRope / 8) rope = load8<kVec>(row + kLatent + lane * 8);

        float x[kGroup];
        const T* v = reinterpret_cast<const T*>(raw);
        float a = 0.0f;
        bool finite = true;
#pragma unroll
        for (int k = 0; k < kGroup; ++k) {
            x[k] = to_float(v[k]);
            a = fmaxf(a, fabsf(x[k]));
            finite &= fabsf(x[k]) < INFINITY;
        }
        if (!finite) {  // NaN is stored as 0, an infinity as the largest value of the largest scale
            bits |= ASU_ST_BAD_SOURCE;
#pragma unroll
            for (int k = 0; k < kGroup; ++k) x[k] = x[k] == x[k] ? fminf(fmaxf(x[k], -3e38f), 3e38f) : 0.0f;
        }
        uint32_t sb = __float_as_uint(__fdiv_rn(a, 7.0f));
        sb = (sb + 0x7ffffu + ((sb >> 20) & 1u)) >> 20;
        const int byte = min(max(static_cast<int>(sb) - ((127 - kScaleBias) << 3), 0), 255);
        const float s = __uint_as_float(scale_bits(byte) << 16);
        const float inv = __frcp_rn(s);
        uint32_t word[2] = {0, 0};
#pragma unroll
        for (int k = 0; k < kGroup; ++k) {
            float y = x[k] * inv;
            y = fmaf(fmaf(-y, s, x[k]), inv, y);
            y = fminf(fmaxf(y, -7.0f), 7.0f);
            // 1.5 * 2^23 + 8 is even: the sum rounds to the nearest integer, ties to even
            const uint32_t code = __float_as_uint(y + 12582920.0f) & 15u;
            word[k / 8] |= code << (4 * ((k % 8) / 2 + 4 * (k % 2)));
        }
        *reinterpret_cast<uint2*>(dst + lane * 8) = make_uint2(word[0], word[1]);
        dst[kScaleOffset + lane] = static_cast<uint8_t>(byte);
        if (lane < kRope / 8) {
            if constexpr (!std::is_same<T, __nv_bfloat16>::value) {
                const T* h = reinterpret_cast<const T*>(&rope);
                uint32_t w[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const __nv_bfloat162 p = __floats2bfloat162_rn(to_float(h[2 * k]), to_float(h[2 * k + 1]));
                    w[k] = reinterpret_cast<const uint32_t&>(p);
                }
                rope = make_uint4(w[0], w[1], w[2], w[3]);
            }
            *reinterpret_cast<uint4*>(dst + kRopeOffset + lane * 16) = rope;
        }
    }
    if (bits) flag_status(status, 0, bits);
}

__global__ void __launch_bounds__(kThreads)
kv4_unpack_kernel(const uint8_t* __restrict__ pool, int64_t pool_rows, uint64_t pool_pitch,
                  const int32_t* __restrict__ slots, int64_t n, uint16_t* __restrict__ dst, int64_t dst_pitch,
                  int32_t* status) {
    pdl_wait();
    pdl_trigger();
    const int lane = threadIdx.x & 31;
    int32_t bits = 0;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5); i < n;
         i += static_cast<int64_t>(gridDim.x) * kWarps) {
        const int64_t slot = slots != nullptr ? static_cast<int64_t>(__ldg(slots + i)) : i;
        uint4 o[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
        uint4 rope = make_uint4(0, 0, 0, 0);
        if (slot >= 0 && slot < pool_rows) {
            const uint8_t* row = pool + static_cast<uint64_t>(slot) * pool_pitch;
            const uint2 w = __ldg(reinterpret_cast<const uint2*>(row + lane * 8));
            const uint32_t byte = __ldg(row + kScaleOffset + lane);
            if (lane < kRope / 8) rope = __ldg(reinterpret_cast<const uint4*>(row + kRopeOffset + lane * 16));
            __nv_bfloat162 s, c;
            scale_pair(byte, s, c);
            unpack_word(w.x, s, c, reinterpret_cast<uint32_t*>(&o[0]));
            unpack_word(w.y, s, c, reinterpret_cast<uint32_t*>(&o[1]));
        } else if (slot != kNotFound) {
            bits |= ASU_ST_BAD_QUERY;
        }
        uint16_t* to = dst + i * dst_pitch;
        reinterpret_cast<uint4*>(to + lane * kGroup)[0] = o[0];
        reinterpret_cast<uint4*>(to + lane * kGroup)[1] = o[1];
        if (lane < kRope / 8) *reinterpret_cast<uint4*>(to + kLatent + lane * 8) = rope;
    }
    if (bits) flag_status(status, 0, bits);
}

dim3 grid_for(int64_t n) {
    const int64_t blocks = (n + kWarps - 1) / kWarps;
    return dim3(static_cast<unsigned>(blocks < (1 << 20) ? blocks : (1 << 20)));
}

bool pool_ok(const void* pool, int64_t rows, uint64_t pitch) {
    return reinterpret_cast<uintptr_t>(pool) % 16 == 0 && pitch % 16 == 0 && pitch >= kRowBytes && rows > 0;
}

}  // namespace
}  // namespace asu

using namespace asu;

extern "C" int asu_kv4_pack(void* stream, const void* src, int32_t src_dtype, int64_t src_pitch, int64_t n,
                            const int32_t* slots, void* pool, int64_t pool_rows, uint64_t pool_pitch,
                            int32_t* status) {
    if (n == 0) return ASU_OK;
    if (n < 0 || src == nullptr || pool == nullptr || pool_rows <= 0 || (slots == nullptr && n > pool_rows) ||
        src_pitch < 0 || (src_dtype != ASU_DTYPE_BF16 && src_dtype != ASU_DTYPE_FP16) ||
        pool_pitch < static_cast<uint64_t>(kRowBytes))
        return ASU_ERR_ARG;
    if (!pool_ok(pool, pool_rows, pool_pitch) || reinterpret_cast<uintptr_t>(src) % 2 != 0) return ASU_ERR_ALIGN;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool vec = reinterpret_cast<uintptr_t>(src) % 16 == 0 && src_pitch % 8 == 0;
    const uint16_t* p = static_cast<const uint16_t*>(src);
    uint8_t* d = static_cast<uint8_t*>(pool);
    auto run = [&](auto kernel) {
        return launch_pdl(kernel, grid_for(n), dim3(kThreads), 0, s, p, src_pitch, n, slots, d, pool_rows, pool_pitch,
                          status);
    };
    if (src_dtype == ASU_DTYPE_BF16)
        return vec ? run(kv4_pack_kernel<__nv_bfloat16, true>) : run(kv4_pack_kernel<__nv_bfloat16, false>);
    return vec ? run(kv4_pack_kernel<__half, true>) : run(kv4_pack_kernel<__half, false>);
}

extern "C" int asu_kv4_unpack(void* stream, const void* pool, int64_t pool_rows, uint64_t pool_pitch,
                              const int32_t* slots, int64_t n, void* dst, int64_t dst_pitch, int32_t* status) {
    if (n == 0) return ASU_OK;
    if (n < 0 || dst == nullptr || pool == nullptr || pool_rows <= 0 || (slots == nullptr && n > pool_rows) ||
        dst_pitch < kDim || pool_pitch < static_cast<uint64_t>(kRowBytes))
        return ASU_ERR_ARG;
    if (!pool_ok(pool, pool_rows, pool_pitch) || reinterpret_cast<uintptr_t>(dst) % 16 != 0 || dst_pitch % 8 != 0)
        return ASU_ERR_ALIGN;
    return launch_pdl(kv4_unpack_kernel, grid_for(n), dim3(kThreads), 0, static_cast<cudaStream_t>(stream),
                      static_cast<const uint8_t*>(pool), pool_rows, pool_pitch, slots, n,
                      static_cast<uint16_t*>(dst), dst_pitch, status);
}

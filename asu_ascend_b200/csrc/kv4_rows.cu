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
// A warp takes two rows at a time.  Writing, a lane has a group: it loads its 32 bytes, needs no exchange with
// other lanes for the maximum, and stores 8 bytes of nibbles and one scale byte; 8 lanes move the rope part.
// Reading, a lane has two words 32 apart, so that every store of the warp is of consecutive bytes.
// 65536 rows (1152 bytes here, 416 there), bf16 or fp16: 27 us to write, 3.8 TB/s (one row at a time 30 us, four 35), and
// neither instructions nor memory are at their limit, as a warp loads, computes and stores in turn; 20 us to read, 5.0 TB/s.
#include <cuda_fp16.h>

#include "kv4.cuh"

namespace asu {
namespace {

using namespace kv4;

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kRows = 2;  // a warp's rows at a time, their loads together

template <typename T>
__device__ __forceinline__ float to_float(T v);
template <>
__device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_float<__half>(__half v) { return __half2float(v); }

// The largest magnitude of 16 values; NaN if there is one.
template <typename T>
__device__ __forceinline__ float largest(const uint4 (&raw)[2]) {
    const uint32_t w[8] = {raw[0].x, raw[0].y, raw[0].z, raw[0].w, raw[1].x, raw[1].y, raw[1].z, raw[1].w};
    using Pair = std::conditional_t<std::is_same<T, __half>::value, __half2, __nv_bfloat162>;
    Pair m = __habs2(reinterpret_cast<const Pair&>(w[0]));
#pragma unroll
    for (int k = 1; k < 8; ++k) m = __hmax2_nan(m, __habs2(reinterpret_cast<const Pair&>(w[k])));
    return to_float(__hmax_nan(m.x, m.y));
}

// 8 consecutive 16-bit values of a row that is aligned to kAlign bytes.
template <int kAlign>
__device__ __forceinline__ uint4 load8(const uint16_t* p) {
    if constexpr (kAlign >= 16) {
        return __ldg(reinterpret_cast<const uint4*>(p));
    } else {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
            w[i] = static_cast<uint32_t>(__ldg(p + 2 * i)) | (static_cast<uint32_t>(__ldg(p + 2 * i + 1)) << 16);
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
}

// 16 of them: a whole sector in one load where the alignment allows it.
template <int kAlign>
__device__ __forceinline__ void load16(const uint16_t* p, uint4 (&v)[2]) {
    if constexpr (kAlign == 32) {
        asm("ld.global.nc.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
            : "=r"(v[0].x), "=r"(v[0].y), "=r"(v[0].z), "=r"(v[0].w), "=r"(v[1].x), "=r"(v[1].y), "=r"(v[1].z),
              "=r"(v[1].w)
            : "l"(p));
    } else {
        v[0] = load8<kAlign>(p);
        v[1] = load8<kAlign>(p + 8);
    }
}

template <typename T, int kAlign>
__global__ void __launch_bounds__(kThreads)
kv4_pack_kernel(const uint16_t* __restrict__ src, int64_t src_pitch, int64_t n, const int32_t* __restrict__ slots,
                uint8_t* __restrict__ pool, int64_t pool_rows, uint64_t pool_pitch, int32_t* status) {
    pdl_wait();
    pdl_trigger();
    const int lane = threadIdx.x & 31;
    int32_t bits = 0;
    for (int64_t i0 = (static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5)) * kRows; i0 < n;
         i0 += static_cast<int64_t>(gridDim.x) * kWarps * kRows) {
        int64_t slot[kRows];
        uint4 raw[kRows][2], rope[kRows];
#pragma unroll
        for (int m = 0; m < kRows; ++m) {
            const int64_t i = i0 + m < n ? i0 + m : i0;
            slot[m] = i0 + m >= n ? kNotFound : slots != nullptr ? static_cast<int64_t>(__ldg(slots + i)) : i;
            const uint16_t* row = src + i * src_pitch;
            load16<kAlign>(row + lane * kGroup, raw[m]);
            rope[m] = lane < kRope / 8 ? load8<kAlign>(row + kLatent + lane * 8) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int m = 0; m < kRows; ++m) {
            if (slot[m] == kNotFound) continue;
            if (slot[m] < 0 || slot[m] >= pool_rows) {
                bits |= ASU_ST_BAD_QUERY;
                continue;
            }
            uint8_t* dst = pool + static_cast<uint64_t>(slot[m]) * pool_pitch;
            const float a = largest<T>(raw[m]);
            float x[kGroup];
            const T* v = reinterpret_cast<const T*>(raw[m]);
#pragma unroll
            for (int k = 0; k < kGroup; ++k) x[k] = to_float(v[k]);
            float top = a;
            if (!(a < INFINITY)) {  // NaN is stored as 0, an infinity as the largest value of the largest scale
                bits |= ASU_ST_BAD_SOURCE;
                top = 0.0f;
#pragma unroll
                for (int k = 0; k < kGroup; ++k) {
                    x[k] = x[k] == x[k] ? x[k] : 0.0f;
                    top = fmaxf(top, fabsf(x[k]));
                }
            }
            uint32_t sb = __float_as_uint(__fdiv_rn(top, 7.0f));
            sb = (sb + 0x7ffffu + ((sb >> 20) & 1u)) >> 20;
            const int byte = min(max(static_cast<int>(sb) - ((127 - kScaleBias) << 3), 0), 255);
            const float s = __uint_as_float(scale_bits(byte) << 16);
            const float inv = __frcp_rn(s);
            if (byte == 255) {  // only there can a quotient round to more than 7
#pragma unroll
                for (int k = 0; k < kGroup; ++k) x[k] = fminf(fmaxf(x[k], -7.0f * s), 7.0f * s);
            }
            // 1.5 * 2^23 + 8 is even: the sum with it rounds to the nearest integer, ties to even, and its bits are
            // kMagic + code.  The word adds them up as they are, each at its place, and the magic ones cancel.
            constexpr uint32_t kMagic = 0x4b400000u;
            uint32_t word[2] = {0u - kMagic * 0x11111111u, 0u - kMagic * 0x11111111u};
            const uint64_t inv2 = pair(inv, inv), minus_s2 = pair(-s, -s), magic2 = pair(12582920.0f, 12582920.0f);
#pragma unroll
            for (int k = 0; k < kGroup; k += 2) {
                const uint64_t x2 = pair(x[k], x[k + 1]);
                uint64_t y2 = mul2(x2, inv2);
                y2 = fma2(fma2(y2, minus_s2, x2), inv2, y2);
                float y[2];
                unpair(add2(y2, magic2), y[0], y[1]);
#pragma unroll
                for (int i = 0; i < 2; ++i) word[k / 8] += __float_as_uint(y[i]) << (4 * ((k % 8) / 2 + 4 * i));
            }
            *reinterpret_cast<uint2*>(dst + lane * 8) = make_uint2(word[0], word[1]);
            dst[kScaleOffset + lane] = static_cast<uint8_t>(byte);
            if (lane < kRope / 8) {
                if constexpr (!std::is_same<T, __nv_bfloat16>::value) {
                    const T* h = reinterpret_cast<const T*>(&rope[m]);
                    uint32_t w[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const __nv_bfloat162 p = __floats2bfloat162_rn(to_float(h[2 * k]), to_float(h[2 * k + 1]));
                        w[k] = reinterpret_cast<const uint32_t&>(p);
                    }
                    rope[m] = make_uint4(w[0], w[1], w[2], w[3]);
                }
                *reinterpret_cast<uint4*>(dst + kRopeOffset + lane * 16) = rope[m];
            }
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
    for (int64_t i0 = (static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5)) * kRows; i0 < n;
         i0 += static_cast<int64_t>(gridDim.x) * kWarps * kRows) {
        uint32_t w[kRows][2], byte[kRows][2];
        uint4 rope[kRows];
        uint32_t there = 0;
#pragma unroll
        for (int m = 0; m < kRows; ++m) {
            const int64_t i = i0 + m;
            const int64_t slot = i >= n ? kNotFound : slots != nullptr ? static_cast<int64_t>(__ldg(slots + i)) : i;
            if (slot >= 0 && slot < pool_rows) {
                const uint8_t* row = pool + static_cast<uint64_t>(slot) * pool_pitch;
#pragma unroll
                for (int h = 0; h < 2; ++h) {  // a lane's words 32 apart, so that its stores are next to its neighbours'
                    w[m][h] = __ldg(reinterpret_cast<const uint32_t*>(row) + h * 32 + lane);
                    byte[m][h] = __ldg(row + kScaleOffset + h * 16 + lane / 2);
                }
                if (lane < kRope / 8) rope[m] = __ldg(reinterpret_cast<const uint4*>(row + kRopeOffset + lane * 16));
                there |= 1u << m;
            } else if (slot != kNotFound) {
                bits |= ASU_ST_BAD_QUERY;
            }
        }
#pragma unroll
        for (int m = 0; m < kRows; ++m) {
            if (i0 + m >= n) break;
            uint4 o[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
            if ((there >> m) & 1u) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    __nv_bfloat162 s, c;
                    scale_pair(byte[m][h], s, c);
                    unpack_word(w[m][h], s, c, reinterpret_cast<uint32_t*>(&o[h]));
                }
            } else {
                rope[m] = make_uint4(0, 0, 0, 0);
            }
            uint16_t* to = dst + (i0 + m) * dst_pitch;
            reinterpret_cast<uint4*>(to)[lane] = o[0];
            reinterpret_cast<uint4*>(to)[32 + lane] = o[1];
            if (lane < kRope / 8) *reinterpret_cast<uint4*>(to + kLatent + lane * 8) = rope[m];
        }
    }
    if (bits) flag_status(status, 0, bits);
}

dim3 grid_for(int64_t n) {
    const int64_t blocks = (n + kWarps * kRows - 1) / (kWarps * kRows);
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
    const uint16_t* p = static_cast<const uint16_t*>(src);
    uint8_t* d = static_cast<uint8_t*>(pool);
    auto run = [&](auto kernel) {
        return launch_pdl(kernel, grid_for(n), dim3(kThreads), 0, s, p, src_pitch, n, slots, d, pool_rows, pool_pitch,
                          status);
    };
    // 32-byte loads for rows that allow them, 16-byte ones, or single values
    const uint64_t start = reinterpret_cast<uintptr_t>(src) | static_cast<uint64_t>(src_pitch) * 2;
    if (src_dtype == ASU_DTYPE_BF16)
        return start % 32 == 0   ? run(kv4_pack_kernel<__nv_bfloat16, 32>)
               : start % 16 == 0 ? run(kv4_pack_kernel<__nv_bfloat16, 16>)
                                 : run(kv4_pack_kernel<__nv_bfloat16, 2>);
    return start % 32 == 0   ? run(kv4_pack_kernel<__half, 32>)
           : start % 16 == 0 ? run(kv4_pack_kernel<__half, 16>)
                             : run(kv4_pack_kernel<__half, 2>);
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

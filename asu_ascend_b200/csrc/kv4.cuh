// The 4-bit MLA row: 512 latent values and 64 position-encoded ones in 416 bytes (13 sectors).
//
//   [0, 256)    512 nibbles n in 1..15: value (n - 8) * s.  Eight values share a 32-bit word; value
//               2j is nibble j, value 2j + 1 nibble j + 4, so that (word >> 4j) & 0x000f000f is the
//               pair (2j, 2j + 1) in the two halves of a register, ready for packed arithmetic
//   [256, 288)  32 scale bytes, one per 16 values: b stands for s = (1 + (b & 7) / 8) * 2^((b >> 3) - 18)
//   [288, 416)  64 bf16
//
// A value has 3 significant bits from the nibble and 4 from the scale: exact in bf16, so the tensor
// cores multiply exactly the numbers that the row stands for.
#pragma once

#include <cuda_bf16.h>

#include "asu_common.cuh"

namespace asu {
namespace kv4 {

constexpr int kLatent = ASU_KV4_LATENT;
constexpr int kRope = ASU_KV4_ROPE;
constexpr int kDim = kLatent + kRope;
constexpr int kGroup = ASU_KV4_GROUP;
constexpr int kRowBytes = ASU_KV4_ROW_BYTES;
constexpr int kScaleOffset = kLatent / 2;
constexpr int kRopeOffset = kScaleOffset + kLatent / kGroup;
constexpr int kScaleBias = 18;
static_assert(kRopeOffset + 2 * kRope == kRowBytes, "row layout");

// bf16 bits of a scale byte: exponent and the three mantissa bits move in one shift.
__host__ __device__ __forceinline__ uint32_t scale_bits(uint32_t b) { return (b << 4) + ((127 - kScaleBias) << 7); }

// Four pairs of bf16 (the word's 8 values in order) from a word of nibbles and its scale as a
// bf16 pair.  0x4300 | n is 128 + n; (128 + n) * s - 136 * s is (n - 8) * s, and every term is
// exact: 136 s = 17 * (8 + m) * 2^e needs 8 bits at most (17 * 15 = 255).  3 instructions a pair.
__device__ __forceinline__ void unpack_word(uint32_t w, __nv_bfloat162 s, __nv_bfloat162 c, uint32_t out[4]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const uint32_t bits = ((w >> (4 * j)) & 0x000f000fu) | 0x43004300u;
        const __nv_bfloat162 v = __hfma2(reinterpret_cast<const __nv_bfloat162&>(bits), s, c);
        out[j] = reinterpret_cast<const uint32_t&>(v);
    }
}

// The scale pair (s, s) of a byte, and c = -136 s.
__device__ __forceinline__ void scale_pair(uint32_t byte, __nv_bfloat162& s, __nv_bfloat162& c) {
    const uint32_t b = scale_bits(byte);
    const uint32_t both = b | (b << 16);
    s = reinterpret_cast<const __nv_bfloat162&>(both);
    c = __hmul2(s, __float2bfloat162_rn(-136.0f));
}

// The same for byte `i` of a register of scale bytes.
__device__ __forceinline__ void scale_pair(uint32_t bytes, int i, __nv_bfloat162& s, __nv_bfloat162& c) {
    const uint32_t both = __byte_perm(bytes, 0, 0x4040 | (i << 8) | i) * 16u + ((127 - kScaleBias) << 7) * 0x10001u;
    s = reinterpret_cast<const __nv_bfloat162&>(both);
    c = __hmul2(s, __float2bfloat162_rn(-136.0f));
}

// Pairs of floats in one register pair: one instruction for two.
__device__ __forceinline__ uint64_t pair(float lo, float hi) {
    uint64_t v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(lo), "f"(hi));
    return v;
}
__device__ __forceinline__ void unpair(uint64_t v, float& lo, float& hi) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}

}  // namespace kv4
}  // namespace asu

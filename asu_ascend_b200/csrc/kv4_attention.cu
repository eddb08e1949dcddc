// Sparse MLA attention of decode tokens over the 4-bit cache.
//
//   s_hj = scale * q_h . k_j over the entries j whose slot is not -1     (576 wide)
//   out_h = sum_j p_hj v_j,  p_h = softmax(s_h),  v_j = the first 512 of k_j
//   lse_h = log sum_j exp s_hj,   weights_j = sum_h p_hj
// A token without any entry: out 0, lse -inf, weights 0.
//
// One CTA per (token, head); every warp takes each fourth entry, holds 16 latents and 2 rope values a
// lane, and keeps its own running maximum and sum; the four are joined at the end.
#include "kv4_decode.cuh"

namespace asu {
namespace {

using namespace kv4;

constexpr int kThreads = 128;
constexpr int kWarps = kThreads / 32;

__global__ void __launch_bounds__(kThreads)
kv4_decode_kernel(const __nv_bfloat16* __restrict__ q, int64_t q_token, int64_t q_head, const uint8_t* __restrict__ pool,
                  int64_t pool_token, int64_t pool_rows, uint64_t pool_pitch, const int32_t* __restrict__ slots,
                  int64_t slots_token, int heads, int topk, float scale, __nv_bfloat16* __restrict__ out,
                  float* __restrict__ lse, float* __restrict__ logits, int32_t* status) {
    pdl_wait();
    pdl_trigger();
    __shared__ float s_m[kWarps], s_l[kWarps];
    __shared__ float s_o[kWarps][kLatent];
    const int h = blockIdx.x, t = blockIdx.y;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const __nv_bfloat16* qr = q + t * q_token + h * q_head;
    float qv[18];
#pragma unroll
    for (int i = 0; i < 16; ++i) qv[i] = __bfloat162float(qr[lane * 16 + i]);
    qv[16] = __bfloat162float(qr[kLatent + lane * 2]);
    qv[17] = __bfloat162float(qr[kLatent + lane * 2 + 1]);
    float acc[16] = {};
    float m = -INFINITY, l = 0.0f;
    int32_t bits = 0;
    for (int j = warp; j < topk; j += kWarps) {
        const int32_t slot = slots[t * slots_token + j];
        float s = -INFINITY;
        if (slot >= 0 && slot < pool_rows) {
            const uint8_t* row = pool + t * pool_token + static_cast<uint64_t>(slot) * pool_pitch;
            const uint2 w = *reinterpret_cast<const uint2*>(row + lane * 8);
            __nv_bfloat162 sc, c;
            scale_pair(row[kScaleOffset + lane], sc, c);
            uint32_t p[8];
            unpack_word(w.x, sc, c, p);
            unpack_word(w.y, sc, c, p + 4);
            float v[16];
            float dot = 0.0f;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                v[i] = __uint_as_float(i % 2 ? p[i / 2] & 0xffff0000u : p[i / 2] << 16);
                dot = fmaf(qv[i], v[i], dot);
            }
            const uint32_t r = *reinterpret_cast<const uint32_t*>(row + kRopeOffset + lane * 4);
            dot = fmaf(qv[16], __uint_as_float(r << 16), dot);
            dot = fmaf(qv[17], __uint_as_float(r & 0xffff0000u), dot);
#pragma unroll
            for (int d = 16; d > 0; d >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, d);
            s = dot * scale;
            const float mn = fmaxf(m, s);
            const float old = __expf(m - mn), e = __expf(s - mn);
            m = mn;
            l = l * old + e;
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[i] = acc[i] * old + e * v[i];
        } else if (slot != kNotFound) {
            bits |= ASU_ST_BAD_QUERY;
        }
        if (logits != nullptr && lane == 0) logits[(static_cast<int64_t>(t) * heads + h) * topk + j] = s;
    }
    if (lane == 0) {
        s_m[warp] = m;
        s_l[warp] = l;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) s_o[warp][lane * 16 + i] = acc[i];
    __syncthreads();
    float mm = -INFINITY, ll = 0.0f;
    for (int w = 0; w < kWarps; ++w) mm = fmaxf(mm, s_m[w]);
    const float base = mm == -INFINITY ? 0.0f : mm;
    for (int w = 0; w < kWarps; ++w) ll += s_l[w] * __expf(s_m[w] - base);
    const float inv = ll > 0.0f ? 1.0f / ll : 0.0f;
    for (int i = threadIdx.x; i < kLatent; i += kThreads) {
        float o = 0.0f;
        for (int w = 0; w < kWarps; ++w) o += s_o[w][i] * __expf(s_m[w] - base);
        out[(static_cast<int64_t>(t) * heads + h) * kLatent + i] = __float2bfloat16(o * inv);
    }
    if (threadIdx.x == 0) lse[static_cast<int64_t>(t) * heads + h] = ll > 0.0f ? mm + logf(ll) : -INFINITY;
    if (bits && lane == 0) flag_status(status, 0, bits);
}

__global__ void __launch_bounds__(256)
kv4_weights_kernel(const float* __restrict__ logits, const float* __restrict__ lse, int heads, int topk,
                   __nv_bfloat16* __restrict__ weights) {
    pdl_wait();
    pdl_trigger();
    const int t = blockIdx.y;
    const int j = blockIdx.x * blockDim.x + threadIdx.x;
    if (j >= topk) return;
    float w = 0.0f;
    for (int h = 0; h < heads; ++h) {
        const float s = logits[(static_cast<int64_t>(t) * heads + h) * topk + j];
        if (s != -INFINITY) w += __expf(s - lse[static_cast<int64_t>(t) * heads + h]);
    }
    weights[static_cast<int64_t>(t) * topk + j] = __float2bfloat16(w);
}

int64_t workspace_bytes(int64_t tokens, int64_t heads, int64_t topk, bool weights) {
    if (heads > 32) return wide_workspace(tokens, topk, weights);
    return weights ? tokens * heads * topk * 4 : 0;
}

}  // namespace
}  // namespace asu

using namespace asu;

extern "C" int64_t asu_kv4_attention_workspace_bytes(int64_t tokens, int64_t heads, int64_t topk, int32_t weights) {
    if (tokens < 0 || heads < 0 || topk < 0 || tokens > ASU_KV4_MAX_TOKENS || heads > ASU_KV4_MAX_HEADS ||
        topk > ASU_KV4_MAX_TOPK)
        return -1;
    return workspace_bytes(tokens, heads, topk, weights != 0);
}

extern "C" int asu_kv4_attention(void* stream, const void* q, int64_t q_token_stride, int64_t q_head_stride,
                                 const void* pool, int64_t pool_rows, uint64_t pool_pitch, uint64_t pool_token_stride,
                                 const int32_t* slots, int64_t slots_token_stride, int64_t tokens, int64_t heads,
                                 int64_t topk, float scale, void* out, float* lse, void* weights, void* workspace,
                                 int64_t workspace_size, int32_t* status) {
    if (tokens < 0 || heads < 0 || topk < 0 || tokens > ASU_KV4_MAX_TOKENS || heads > ASU_KV4_MAX_HEADS ||
        topk > ASU_KV4_MAX_TOPK || pool_rows < 0 || pool_rows > 0x7fffffff || q_token_stride < 0 || q_head_stride < 0 ||
        slots_token_stride < 0 || pool_pitch < static_cast<uint64_t>(kRowBytes) || !(scale > 0.0f) ||
        !(scale < INFINITY))
        return ASU_ERR_ARG;
    if (tokens == 0 || heads == 0) return ASU_OK;
    if (!q || !out || !lse || (topk && (!slots || !pool))) return ASU_ERR_ARG;
    const int64_t need = workspace_bytes(tokens, heads, topk, weights != nullptr);
    if (need > 0 && (workspace == nullptr || workspace_size < need)) return ASU_ERR_ARG;
    if (reinterpret_cast<uintptr_t>(q) % 2 || reinterpret_cast<uintptr_t>(pool) % 16 || pool_pitch % 16 ||
        pool_token_stride % 16 || reinterpret_cast<uintptr_t>(out) % 16 || reinterpret_cast<uintptr_t>(lse) % 4 ||
        reinterpret_cast<uintptr_t>(workspace) % 16)
        return ASU_ERR_ALIGN;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (heads > 32) {
        Operands op;
        op.q = static_cast<const __nv_bfloat16*>(q);
        op.q_token = q_token_stride;
        op.q_head = q_head_stride;
        op.pool = static_cast<const uint8_t*>(pool);
        op.pool_token = pool_token_stride;
        op.pool_pitch = pool_pitch;
        op.pool_rows = static_cast<int32_t>(pool_rows);
        op.slots = slots;
        op.slots_token = slots_token_stride;
        op.tokens = static_cast<int32_t>(tokens);
        op.heads = static_cast<int32_t>(heads);
        op.topk = static_cast<int32_t>(topk);
        op.scale_log2 = scale * 1.4426950408889634f;
        op.q_aligned = reinterpret_cast<uintptr_t>(q) % 16 == 0 && q_token_stride % 8 == 0 && q_head_stride % 8 == 0;
        op.out = static_cast<__nv_bfloat16*>(out);
        op.lse = lse;
        op.weights = static_cast<__nv_bfloat16*>(weights);
        op.status = status;
        return launch_wide(s, op, workspace);
    }
    float* logits = weights != nullptr ? static_cast<float*>(workspace) : nullptr;
    int rc = launch_pdl(kv4_decode_kernel, dim3(static_cast<unsigned>(heads), static_cast<unsigned>(tokens)),
                        dim3(kThreads), 0, s, static_cast<const __nv_bfloat16*>(q), q_token_stride, q_head_stride,
                        static_cast<const uint8_t*>(pool), static_cast<int64_t>(pool_token_stride), pool_rows,
                        pool_pitch, slots, slots_token_stride, static_cast<int>(heads), static_cast<int>(topk), scale,
                        static_cast<__nv_bfloat16*>(out), lse, logits, status);
    if (rc != ASU_OK || weights == nullptr || topk == 0) return rc;
    return launch_pdl(kv4_weights_kernel,
                      dim3(static_cast<unsigned>((topk + 255) / 256), static_cast<unsigned>(tokens)), dim3(256), 0, s,
                      static_cast<const float*>(logits), static_cast<const float*>(lse), static_cast<int>(heads),
                      static_cast<int>(topk), static_cast<__nv_bfloat16*>(weights));
}

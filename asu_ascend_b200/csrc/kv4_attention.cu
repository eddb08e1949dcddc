// C entry point of sparse MLA attention over the 4-bit cache.
//
//   s_hj = scale * q_h . k_j over the entries j whose slot is not -1     (576 wide)
//   out_h = sum_j p_hj v_j,  p_h = softmax(s_h),  v_j = the first 512 of k_j
//   lse_h = log sum_j exp s_hj,   weights_j = sum_h p_hj
// A token without any entry: out 0, lse -inf, weights 0.
#include "kv4_decode.cuh"

#include <algorithm>

using namespace asu;
using namespace asu::kv4;

// Up to kTallHeads heads the kernel whose products have the heads as columns, above it the one whose products
// have them as 128 rows.  One and the other in us, 2048 entries, each token's rows in a pool of its own, inputs in
// rotation (none in L2):
//   heads             16        32         64        80       128
//   128 tokens  55 / 120  63 / 122  101 / 128   - / 131   - / 139
//   32 tokens   23 /  37  25 /  38   33 /  38   - /  39   - /  41
// The first, taking 64 heads at a time, needed 167 and 54 us for 80 heads.  For one token they are within 2 us of each
// other.
static int64_t decode_workspace(int64_t tokens, int64_t heads, int64_t topk, bool weights) {
    return heads <= kTallHeads ? tall_workspace(tokens, heads, topk, weights) : wide_workspace(tokens, topk, weights);
}

// Weights need the softmax weights of every head until a token's sum is known: two bytes a (padded) head and entry.
// Calls of more tokens than kWeightsBytes of them hold are done in parts of the same size, one after the other
// in the stream and in the same workspace.  128 heads x 2048 entries: 496 tokens, some 600 us of work a part.
constexpr int64_t kWeightsBytes = 256ll << 20;
static int64_t tokens_at_once(int64_t tokens, int64_t heads, int64_t topk, bool weights) {
    if (!weights) return tokens;
    const int64_t most = kWeightsBytes / (heads <= kTallHeads ? tall_weights(heads, topk) : wide_weights(topk));
    const int64_t parts = (tokens + most - 1) / most;
    return (tokens + parts - 1) / parts;
}

// Of the largest part, whether that is the last one or one before.
static int64_t call_workspace(int64_t tokens, int64_t heads, int64_t topk, bool weights) {
    const int64_t some = tokens_at_once(tokens, heads, topk, weights), rest = tokens % some;
    const int64_t bytes = decode_workspace(some, heads, topk, weights);
    return rest > 0 ? std::max(bytes, decode_workspace(rest, heads, topk, weights)) : bytes;
}

extern "C" int64_t asu_kv4_attention_workspace_bytes(int64_t tokens, int64_t heads, int64_t topk, int32_t weights) {
    if (tokens < 0 || heads < 0 || topk < 0 || tokens > ASU_KV4_MAX_TOKENS || heads > ASU_KV4_MAX_HEADS ||
        topk > ASU_KV4_MAX_TOPK)
        return -1;
    return tokens && heads ? call_workspace(tokens, heads, topk, weights != 0 && topk > 0) : 0;
}

extern "C" int asu_kv4_attention(void* stream, const void* q, int64_t q_token_stride, int64_t q_head_stride,
                                 const void* pool, int64_t pool_rows, uint64_t pool_pitch, uint64_t pool_token_stride,
                                 const int32_t* slots, int64_t slots_token_stride, int64_t tokens, int64_t heads,
                                 int64_t topk, float scale, void* out, float* lse, void* weights, void* workspace,
                                 int64_t workspace_size, int32_t* status) {
    if (tokens < 0 || heads < 0 || topk < 0 || tokens > ASU_KV4_MAX_TOKENS || heads > ASU_KV4_MAX_HEADS ||
        topk > ASU_KV4_MAX_TOPK || pool_rows < 0 || pool_rows > 0x7fffffff || q_token_stride < 0 || q_head_stride < 0 ||
        slots_token_stride < 0 || pool_pitch < static_cast<uint64_t>(kRowBytes))
        return ASU_ERR_ARG;
    const float scale_log2 = scale * 1.4426950408889634f;
    if (!(scale_log2 > 0.0f) || !(scale_log2 < INFINITY)) return ASU_ERR_ARG;
    if (tokens == 0 || heads == 0) return ASU_OK;
    if (!q || !out || !lse || (topk && (!slots || !pool))) return ASU_ERR_ARG;
    if (topk == 0) weights = nullptr;
    const int64_t need = call_workspace(tokens, heads, topk, weights != nullptr);
    if (need > 0 && (workspace == nullptr || workspace_size < need)) return ASU_ERR_ARG;
    if (reinterpret_cast<uintptr_t>(q) % 2 || reinterpret_cast<uintptr_t>(pool) % 16 || pool_pitch % 16 ||
        pool_token_stride % 16 || reinterpret_cast<uintptr_t>(out) % 32 || reinterpret_cast<uintptr_t>(lse) % 4 ||
        reinterpret_cast<uintptr_t>(workspace) % 32 || reinterpret_cast<uintptr_t>(slots) % 4 ||
        reinterpret_cast<uintptr_t>(weights) % 2)
        return ASU_ERR_ALIGN;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
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
    op.heads = static_cast<int32_t>(heads);
    op.topk = static_cast<int32_t>(topk);
    op.scale_log2 = scale_log2;
    op.q_aligned = reinterpret_cast<uintptr_t>(q) % 16 == 0 && q_token_stride % 8 == 0 && q_head_stride % 8 == 0;
    op.out = static_cast<__nv_bfloat16*>(out);
    op.lse = lse;
    op.weights = static_cast<__nv_bfloat16*>(weights);
    op.status = status;
    const int64_t some = tokens_at_once(tokens, heads, topk, weights != nullptr);
    for (int64_t t = 0; t < tokens; t += some) {
        op.tokens = static_cast<int32_t>(std::min(some, tokens - t));
        const int rc = op.heads <= kTallHeads ? launch_tall(s, op, workspace) : launch_wide(s, op, workspace);
        if (rc != ASU_OK) return rc;
        op.q += some * op.q_token;
        op.pool += static_cast<uint64_t>(some) * op.pool_token;
        op.slots += some * op.slots_token;
        op.out += some * op.heads * kLatent;
        op.lse += some * op.heads;
        if (weights != nullptr) op.weights += some * op.topk;
    }
    return ASU_OK;
}

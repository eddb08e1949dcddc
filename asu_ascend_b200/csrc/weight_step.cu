// Slot pools that evict by accumulated attention weight, one pool per request row: the last step's
// weights, the eviction and the resolve of this step's keys in one launch.
//
//   U_s = decay * score_s + sum of last_weight over the entries with last_slot == s (in entry order)
//   candidates: resident slots that no key of this step is in and whose key is below keep_from
//   E = min(max(0, min(free_target, S) - free_count), candidates) with the lowest (U, slot) leave:
//       their keys are unmapped, their slots pushed on the free stack in rising order
//   resolve: a resident key is a hit; the first occurrence of a missing key pops the stack (top
//       first, in query order), later ones are hits; an empty stack leaves slot -1
//
// One CTA of 1024 threads per row.  Thread t owns the slots [t * IPT_S, (t + 1) * IPT_S) and keeps
// their scores and keys in registers, so that ranks in slot order come from a block scan and the row
// is read and written once.  A request's step is a serial chain of block barriers over a few dozen
// KB: latency-bound, not bandwidth-bound.
//  * Scores are sums of non-negative floats, whose bit patterns order like integers.  The E-th
//    lowest is found bit by bit from the top: 31 block-wide counts of "below the trial value".
//    No sort and no histogram; the result does not depend on scheduling.
//  * Ties at the threshold go to the lower slots: one packed scan ranks the slots below it
//    and the ties together.
//  * The products and sums of U are rounded one by one (no fma), so that a plain
//    decay-then-add gives the same bits and the same victims.
#include "asu_common.cuh"

#include <cuda_bf16.h>

namespace asu {
namespace {

constexpr int kThreads = 1024;
constexpr int32_t kEmptyKey = -1;

enum : uint8_t { kInvalid = 0, kHit = 1, kMiss = 2, kBad = 3 };

__device__ __forceinline__ uint32_t hash_slot(int32_t key, int log2h) {
    return (static_cast<uint32_t>(key) * 0x9E3779B1u) >> (32 - log2h);
}

// Sum of one small count per thread over the block; `buf` holds 32 ints.  One barrier: alternate two
// buffers between back-to-back calls.
__device__ __forceinline__ int block_sum_1b(int v, int* buf) {
    const int lane = threadIdx.x & 31;
    v = __reduce_add_sync(0xffffffffu, v);
    if (lane == 0) buf[threadIdx.x >> 5] = v;
    __syncthreads();
    return __reduce_add_sync(0xffffffffu, buf[lane]);
}

__device__ __forceinline__ float weight_at(const void* w, int dtype, uint64_t i) {
    if (dtype == ASU_DTYPE_FP32) return __ldcg(static_cast<const float*>(w) + i);
    const uint16_t b = __ldcg(static_cast<const unsigned short*>(w) + i);
    return __uint_as_float(static_cast<uint32_t>(b) << 16);
}

template <int IPT_Q, int IPT_S>
__global__ void __launch_bounds__(kThreads)
weight_step_kernel(int32_t* __restrict__ t2s, int32_t* __restrict__ s2t, float* __restrict__ score,
                   int32_t* __restrict__ stack, int32_t* __restrict__ count, const int32_t* last_slot,
                   const void* __restrict__ last_weight, int weight_dtype, uint32_t last_count, float decay,
                   const int32_t* __restrict__ keep_from, const int32_t* __restrict__ query, int32_t* slot_out,
                   uint8_t* __restrict__ hit_mask, uint8_t* __restrict__ install_mask, int32_t* __restrict__ evicted,
                   uint32_t ev_stride, int32_t* __restrict__ ev_count, int64_t* __restrict__ stats, int32_t* status,
                   uint32_t K, uint32_t S, uint32_t Q, uint32_t target, int log2h) {
    pdl_wait();
    pdl_trigger();
    extern __shared__ int32_t smem[];
    const uint32_t H = 1u << log2h;
    float* s_sum = reinterpret_cast<float*>(smem);          // [S] decayed score + weights
    int32_t* s_claim = smem + S;                            // [S] first entry naming the slot; later the victims
    int32_t* s_hkey = s_claim + S;                          // [H] hash: key
    int32_t* s_hpos = s_hkey + H;                           // [H] hash: first position of the key
    int32_t* s_hval = s_hpos + H;                           // [H] hash: installed slot
    uint8_t* s_asked = reinterpret_cast<uint8_t*>(s_hval + H);  // [S] a key of this step is in the slot
    __shared__ int buf_a[32], buf_b[32];
    __shared__ int n_hits, n_valid, n_double;
    const int tid = threadIdx.x;
    const uint32_t r = blockIdx.x;
    int32_t* trow = t2s + static_cast<uint64_t>(r) * K;
    int32_t* srow = s2t + static_cast<uint64_t>(r) * S;
    float* crow = score + static_cast<uint64_t>(r) * S;
    int32_t* krow = stack + static_cast<uint64_t>(r) * S;
    int32_t bits = 0;

    // ---- loads; shared-memory set-up ----
    const int32_t free0 = ld_cg(count + r);
    const int32_t bound = keep_from != nullptr ? __ldg(keep_from + r) : INT32_MAX;
    int32_t key[IPT_Q], g[IPT_Q];
#pragma unroll
    for (int j = 0; j < IPT_Q; ++j) {
        const uint32_t pos = tid + j * kThreads;
        key[j] = -1;
        g[j] = kNotFound;
        if (pos < Q) {
            key[j] = __ldg(query + static_cast<uint64_t>(r) * Q + pos);
            if (static_cast<uint32_t>(key[j]) < K) g[j] = ld_cg(trow + key[j]);
        }
    }
    int32_t owner[IPT_S];
#pragma unroll
    for (int j = 0; j < IPT_S; ++j) {
        const uint32_t s = tid * IPT_S + j;
        owner[j] = kNotFound;
        if (s < S) {
            owner[j] = ld_cg(srow + s);
            s_sum[s] = __fmul_rn(__ldcg(crow + s), decay);
            s_claim[s] = INT32_MAX;
            s_asked[s] = 0;
        }
    }
    for (uint32_t i = tid; i < H; i += kThreads) {
        s_hkey[i] = kEmptyKey;
        s_hpos[i] = INT32_MAX;
    }
    if (tid == 0) n_hits = n_valid = n_double = 0;
    if (free0 < 0 || free0 > static_cast<int32_t>(S)) {  // uniform across the block
        if (tid == 0) {
            flag_status(status, r, ASU_ST_BAD_STATE);
            ev_count[r] = 0;
        }
        for (uint32_t i = tid; i < Q; i += kThreads) {
            slot_out[static_cast<uint64_t>(r) * Q + i] = kNotFound;
            hit_mask[static_cast<uint64_t>(r) * Q + i] = 0;
            install_mask[static_cast<uint64_t>(r) * Q + i] = 0;
        }
        return;
    }
    __syncthreads();

    // ---- the last step's entries claim their slots; this step's keys are classified ----
    const uint64_t last_row = static_cast<uint64_t>(r) * last_count;
    for (uint32_t p = tid; p < last_count; p += kThreads) {
        const int32_t s = __ldcg(last_slot + last_row + p);
        if (static_cast<uint32_t>(s) < S) atomicMin(&s_claim[s], static_cast<int32_t>(p));
        else if (s != kNotFound) bits |= ASU_ST_BAD_QUERY;
    }
    uint8_t st[IPT_Q];
    int32_t hidx[IPT_Q];
    int valid_local = 0;
#pragma unroll
    for (int j = 0; j < IPT_Q; ++j) {
        const int32_t pos = tid + j * kThreads;
        st[j] = kInvalid;
        hidx[j] = -1;
        if (static_cast<uint32_t>(pos) >= Q) continue;
        if (static_cast<uint32_t>(key[j]) >= K) {
            bits |= ASU_ST_BAD_QUERY;
            continue;
        }
        ++valid_local;
        if (static_cast<uint32_t>(g[j]) < S) {
            st[j] = kHit;
            s_asked[g[j]] = 1;
        } else if (g[j] == kNotFound) {
            st[j] = kMiss;
            uint32_t h = hash_slot(key[j], log2h);
            while (true) {  // terminates: at most Q <= H distinct keys
                const int32_t old = atomicCAS(&s_hkey[h], kEmptyKey, key[j]);
                if (old == kEmptyKey || old == key[j]) break;
                h = (h + 1) & (H - 1);
            }
            hidx[j] = static_cast<int32_t>(h);
            atomicMin(&s_hpos[h], pos);
        } else {
            st[j] = kBad;
            bits |= ASU_ST_BAD_STATE;
        }
    }
    __syncthreads();

    // ---- weights onto the sums: only the first entry of a slot writes it ----
    for (uint32_t p = tid; p < last_count; p += kThreads) {
        const int32_t s = __ldcg(last_slot + last_row + p);
        if (static_cast<uint32_t>(s) >= S) continue;
        const float w = weight_at(last_weight, weight_dtype, last_row + p);
        if (!(w >= 0.0f) || w == INFINITY) bits |= ASU_ST_BAD_WEIGHT;
        if (s_claim[s] == static_cast<int32_t>(p)) {
            if (w >= 0.0f && w < INFINITY) s_sum[s] = __fadd_rn(s_sum[s], w);
        } else {
            n_double = 1;
        }
    }
    __syncthreads();
    if (n_double) {  // uniform; a slot named more than once: its first entry adds the others in order
        for (uint32_t p = tid; p < last_count; p += kThreads) {
            const int32_t s = __ldcg(last_slot + last_row + p);
            if (static_cast<uint32_t>(s) >= S || s_claim[s] != static_cast<int32_t>(p)) continue;
            float u = s_sum[s];
            for (uint32_t i = p + 1; i < last_count; ++i) {
                if (__ldcg(last_slot + last_row + i) != s) continue;
                const float w = weight_at(last_weight, weight_dtype, last_row + i);
                if (w >= 0.0f && w < INFINITY) u = __fadd_rn(u, w);
            }
            s_sum[s] = u;
        }
        __syncthreads();
    }

    // ---- who leaves ----
    uint32_t u[IPT_S];
    bool may[IPT_S];
    int cand_local = 0;
#pragma unroll
    for (int j = 0; j < IPT_S; ++j) {
        const uint32_t s = tid * IPT_S + j;
        may[j] = false;
        u[j] = 0;
        if (s < S && owner[j] >= 0) {
            const float v = s_sum[s];
            u[j] = __float_as_uint(v);
            may[j] = !s_asked[s] && owner[j] < bound;
        }
        cand_local += may[j];
    }
    const int32_t tgt = static_cast<int32_t>(target < S ? target : S);
    int32_t E = tgt > free0 ? tgt - free0 : 0;
    uint32_t cut = 0;  // the E-th lowest U among the candidates
    int below = 0;     // candidates under it
    if (E > 0) {       // uniform
        const int n = block_sum_1b(cand_local, buf_a);
        if (E > n) E = n;
        for (int b = 30; b >= 0; --b) {
            const uint32_t trial = cut | (1u << b);
            int c = 0;
#pragma unroll
            for (int j = 0; j < IPT_S; ++j) c += may[j] && u[j] < trial;
            c = block_sum_1b(c, (b & 1) ? buf_a : buf_b);
            if (c < E) {
                cut = trial;
                below = c;
            }
        }
        __syncthreads();
    }
    bool gone[IPT_S];
    if (E > 0) {
        int packed = 0;
#pragma unroll
        for (int j = 0; j < IPT_S; ++j)
            packed += may[j] ? (u[j] < cut ? 1 : (u[j] == cut ? 1 << 16 : 0)) : 0;
        int total = 0;
        packed = block_exclusive_scan_1b(packed, buf_a, &total);
        int rank = packed & 0xffff, ties = packed >> 16;
        const int quota = E - below;
        rank += min(ties, quota);
#pragma unroll
        for (int j = 0; j < IPT_S; ++j) {
            const int32_t s = tid * IPT_S + j;
            const bool tie = may[j] && u[j] == cut;
            gone[j] = may[j] && (u[j] < cut || (tie && ties < quota));
            ties += tie;
            if (!gone[j]) continue;
            s_claim[rank] = s;
            st_cg(krow + free0 + rank, s);
            evicted[static_cast<uint64_t>(r) * ev_stride + rank] = owner[j];
            if (static_cast<uint32_t>(owner[j]) < K) st_cg(trow + owner[j], kNotFound);
            else bits |= ASU_ST_BAD_STATE;
            st_cg(srow + s, kNotFound);
            ++rank;
        }
    } else {
#pragma unroll
        for (int j = 0; j < IPT_S; ++j) gone[j] = false;
    }
#pragma unroll
    for (int j = 0; j < IPT_S; ++j) {
        const uint32_t s = tid * IPT_S + j;
        if (s < S) __stcg(crow + s, gone[j] || owner[j] < 0 ? 0.0f : __uint_as_float(u[j]));
    }
    for (int i = E + tid; i < tgt; i += kThreads) evicted[static_cast<uint64_t>(r) * ev_stride + i] = kNotFound;
    if (tid == 0) ev_count[r] = E;
    const int32_t free1 = free0 + E;
    __syncthreads();  // victims listed and unmapped

    // ---- first occurrences of missing keys pop the stack in query order ----
    int32_t slot[IPT_Q];
    bool first[IPT_Q], inst[IPT_Q];
    int taken = 0;
#pragma unroll
    for (int j = 0; j < IPT_Q; ++j) {
        const int32_t pos = tid + j * kThreads;
        first[j] = st[j] == kMiss && s_hpos[hidx[j]] == pos;
        int total = 0;
        const int before = block_exclusive_scan_1b(first[j], (j & 1) ? buf_a : buf_b, &total);
        slot[j] = st[j] == kHit ? g[j] : kNotFound;
        inst[j] = false;
        if (first[j]) {
            const int32_t k = taken + before;
            int32_t s = kNotFound;
            if (k < free1) {
                s = k < E ? s_claim[E - 1 - k] : ld_cg(krow + (free0 - 1 - (k - E)));
                if (static_cast<uint32_t>(s) >= S) {
                    bits |= ASU_ST_BAD_STATE;
                    s = kNotFound;
                }
            }
            if (s >= 0) {
                st_cg(trow + key[j], s);
                st_cg(srow + s, key[j]);
                inst[j] = true;
            } else {
                bits |= ASU_ST_SHORTAGE;
            }
            s_hval[hidx[j]] = s;
            slot[j] = s;
        }
        taken += total;
    }
    const int32_t n_inst = taken < free1 ? taken : free1;
    __syncthreads();  // installed slots visible
    int hits_local = 0;
#pragma unroll
    for (int j = 0; j < IPT_Q; ++j) {
        const uint32_t pos = tid + j * kThreads;
        bool hit = st[j] == kHit;
        if (st[j] == kMiss && !first[j]) {
            slot[j] = s_hval[hidx[j]];
            hit = slot[j] >= 0;
        }
        hits_local += hit;
        if (pos < Q) {
            const uint64_t o = static_cast<uint64_t>(r) * Q + pos;
            slot_out[o] = slot[j];
            hit_mask[o] = hit;
            install_mask[o] = inst[j];
        }
    }
    hits_local = __reduce_add_sync(0xffffffffu, hits_local);
    valid_local = __reduce_add_sync(0xffffffffu, valid_local);
    if ((tid & 31) == 0) {
        if (hits_local) atomicAdd(&n_hits, hits_local);
        if (valid_local) atomicAdd(&n_valid, valid_local);
    }
    if (bits) flag_status(status, r, bits);
    __syncthreads();
    if (tid == 0) {
        st_cg(count + r, free1 - n_inst);
        if (stats != nullptr) {
            unsigned long long* row =
                reinterpret_cast<unsigned long long*>(stats + static_cast<uint64_t>(r) * ASU_LRU_STAT_COLS);
            atomicAdd(row + ASU_LRU_STAT_HITS, static_cast<unsigned long long>(n_hits));
            atomicAdd(row + ASU_LRU_STAT_MISSES, static_cast<unsigned long long>(n_valid - n_hits));
            atomicAdd(row + ASU_LRU_STAT_INSTALLS, static_cast<unsigned long long>(n_inst));
            atomicAdd(row + ASU_LRU_STAT_SHORTAGES, static_cast<unsigned long long>(n_valid - n_hits - n_inst));
            atomicAdd(row + ASU_LRU_STAT_EVICTIONS, static_cast<unsigned long long>(E));
        }
    }
}

int log2_ceil(uint32_t x) {
    int l = 0;
    while ((1u << l) < x) ++l;
    return l;
}

template <int IPT_Q, int IPT_S>
int launch(cudaStream_t s, int32_t* t2s, int32_t* s2t, float* score, int32_t* stack, int32_t* count,
           const int32_t* last_slot, const void* last_weight, int dtype, uint32_t last_count, float decay,
           const int32_t* keep_from, const int32_t* query, int32_t* slot_out, uint8_t* hit, uint8_t* inst,
           int32_t* evicted, uint32_t ev_stride, int32_t* ev_count, int64_t* stats, int32_t* status, uint32_t R,
           uint32_t K, uint32_t S, uint32_t Q, uint32_t target) {
    const auto kernel = weight_step_kernel<IPT_Q, IPT_S>;
    int max_dynamic = 0;
    const int rc = asu_max_dynamic_smem(reinterpret_cast<const void*>(kernel), &max_dynamic);
    if (rc != ASU_OK) return rc;
    // hash load factor 1/2, or up to 1 where S and Q are both large (it still ends: Q <= H)
    int log2h = log2_ceil(2 * (Q < 16 ? 16 : Q));
    size_t smem = 9ull * S + 12ull * (1ull << log2h);
    if (smem > static_cast<size_t>(max_dynamic)) {
        --log2h;
        smem = 9ull * S + 12ull * (1ull << log2h);
    }
    if (smem > static_cast<size_t>(max_dynamic)) return ASU_ERR_ARG;
    return launch_pdl(kernel, dim3(R), dim3(kThreads), smem, s, t2s, s2t, score, stack, count, last_slot, last_weight,
                      dtype, last_count, decay, keep_from, query, slot_out, hit, inst, evicted, ev_stride, ev_count,
                      stats, status, K, S, Q, target, log2h);
}

}  // namespace
}  // namespace asu

using namespace asu;

extern "C" int asu_weight_step(void* stream, int32_t* token_to_slot, int32_t* slot_to_token, float* score,
                               int32_t* free_stack, int32_t* free_count, const int32_t* last_slot,
                               const void* last_weight, int32_t weight_dtype, uint32_t last_count, float decay,
                               const int32_t* keep_from, const int32_t* query, int32_t* slot_out, uint8_t* hit_mask,
                               uint8_t* install_mask, int32_t* evicted, uint32_t evicted_stride,
                               int32_t* evicted_count, int64_t* stats, int32_t* status, uint32_t req_num,
                               uint32_t key_space, uint32_t slot_count, uint32_t query_count, uint32_t free_target) {
    if (req_num == 0) return ASU_OK;
    if (!token_to_slot || !slot_to_token || !score || !free_stack || !free_count || !evicted_count ||
        (query_count && (!query || !slot_out || !hit_mask || !install_mask)))
        return ASU_ERR_ARG;
    if (req_num > 0x7fffffffu || key_space == 0 || key_space > 0x7fffffffu || slot_count == 0 ||
        slot_count > 16384u || query_count > 4096u || last_count > 4096u || !(decay >= 0.0f) || !(decay <= 1.0f))
        return ASU_ERR_ARG;
    if (last_count && (!last_slot || !last_weight ||
                       (weight_dtype != ASU_DTYPE_BF16 && weight_dtype != ASU_DTYPE_FP32)))
        return ASU_ERR_ARG;
    if (last_count && query_count) {  // slot_out may be last_slot itself, row for row, and nothing in between
        const uintptr_t a = reinterpret_cast<uintptr_t>(last_slot), b = reinterpret_cast<uintptr_t>(slot_out);
        const uint64_t an = 4ull * req_num * last_count, bn = 4ull * req_num * query_count;
        if (a < b + bn && b < a + an && (a != b || last_count != query_count)) return ASU_ERR_ARG;
    }
    const uint32_t tgt = free_target < slot_count ? free_target : slot_count;
    if (tgt > 0 && (evicted == nullptr || evicted_stride < tgt)) return ASU_ERR_ARG;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
#define ASU_WEIGHT_CASE(NQ, NS)                                                                                       \
    if (query_count <= kThreads * NQ && slot_count <= kThreads * NS)                                                  \
        return launch<NQ, NS>(s, token_to_slot, slot_to_token, score, free_stack, free_count, last_slot, last_weight, \
                              weight_dtype, last_count, decay, keep_from, query, slot_out, hit_mask, install_mask,    \
                              evicted, evicted_stride, evicted_count, stats, status, req_num, key_space, slot_count,  \
                              query_count, free_target);
    ASU_WEIGHT_CASE(2, 2)
    ASU_WEIGHT_CASE(2, 8)
    ASU_WEIGHT_CASE(2, 16)
    ASU_WEIGHT_CASE(4, 16)
#undef ASU_WEIGHT_CASE
    return ASU_ERR_ARG;
}

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
// One CTA of 1024 threads per row.  A request's step is a serial chain of dependent loads and block barriers
// over a few dozen KB: a call takes 14 to 15 us for 1 x 10240 slots and 20 for 128 x 8192 (from a cold L2), of which
// the loads are 5 to 8, the threshold 3 to 4, and every instruction of all threads costs 8 cycles.
//  * A warp owns a run of slots and takes 32 of them at a time: loads are of whole lines, shared memory has
//    no bank conflicts, and ranks in slot order need the ballots and one exchange of a count per warp.
//    (With a run of slots for each thread, strided, and a sum over the block for every bit of the
//    threshold, the step took 51 and 36 us.)
//  * Scores are sums of non-negative floats, whose bit patterns order like integers.  The E-th lowest is
//    found by three counts of digits, of 11, 11 and 9 bits, and fewer when a digit's slots leave all.
//    Counts are integers: the result does not depend on scheduling.
//  * Ties at the threshold go to the lower slots.
//  * Victims are listed in shared memory first and written out of the list: their five stores then run once
//    for 1024 victims, not once for 32 slots of a warp (20 -> 14 us for 1 x 10240).
//  * A slot that the last step names several times gets its weights in their order: each round of
//    additions takes the first entry that is left of every slot.
//  * The products and sums of U are rounded one by one (no fma), so that a plain
//    decay-then-add gives the same bits and the same victims.
#include "asu_common.cuh"

#include <cuda_bf16.h>

namespace asu {
namespace {

constexpr int kThreads = 1024;
constexpr int32_t kEmptyKey = -1;
constexpr int kBins = 2048;  // of the first two digits; 512 of the last
constexpr int kHistogram = 2 * kBins + 512;

enum : uint8_t { kInvalid = 0, kHit = 1, kMiss = 2, kBad = 3 };

__device__ __forceinline__ uint32_t hash_slot(int32_t key, int log2h) {
    return (static_cast<uint32_t>(key) * 0x9E3779B1u) >> (32 - log2h);
}

__device__ __forceinline__ float weight_at(const void* w, int dtype, uint64_t i) {
    if (dtype == ASU_DTYPE_FP32) return __ldcg(static_cast<const float*>(w) + i);
    const uint16_t b = __ldcg(static_cast<const unsigned short*>(w) + i);
    return __uint_as_float(static_cast<uint32_t>(b) << 16);
}

// Sum of the warps' values before this warp, and of all.
__device__ __forceinline__ int before_warp(const int* per_warp, int* total) {
    const int lane = threadIdx.x & 31, v = per_warp[lane];
    *total = __reduce_add_sync(0xffffffffu, v);
    return __reduce_add_sync(0xffffffffu, lane < static_cast<int>(threadIdx.x >> 5) ? v : 0);
}

// IPT_Q: keys, and entries of the last step, a thread at most; IPT_S: slots.
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
    extern __shared__ __align__(16) int32_t smem[];
    const uint32_t H = 1u << log2h;
    const uint32_t slots16 = (S + 15) & ~15u;                       // the arrays start on 16 bytes
    int32_t* s_count = smem;                                        // [kHistogram] candidates by digit
    uint8_t* s_asked = reinterpret_cast<uint8_t*>(smem + kHistogram);  // [S] a key of this step is in the slot
    int32_t* s_hkey = smem + kHistogram + slots16 / 4;              // [H] hash: key
    int32_t* s_hpos = s_hkey + H;                                   // [H] hash: first position of the key
    int32_t* s_claim = s_hpos + H;    // [S] first entry left that names the slot; later the victims
    int32_t* s_hval = s_claim + slots16;                            // [H] hash: installed slot
    float* s_sum = reinterpret_cast<float*>(s_hval + H);            // [S] decayed score + weights
    __shared__ int buf_a[32], buf_b[32], buf_q[32];
    __shared__ int n_hits, n_valid;
    __shared__ int s_digit[3];  // of the threshold; candidates below it; in it
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t below_lane = (1u << lane) - 1;
    const uint32_t r = blockIdx.x;
    int32_t* trow = t2s + static_cast<uint64_t>(r) * K;
    int32_t* srow = s2t + static_cast<uint64_t>(r) * S;
    float* crow = score + static_cast<uint64_t>(r) * S;
    int32_t* krow = stack + static_cast<uint64_t>(r) * S;
    int32_t bits = 0;
    // the warp's keys, entries and slots: item j of the lane
    const int per_q = (Q + kThreads - 1) / kThreads, per_s = (S + kThreads - 1) / kThreads;
    auto pos_of = [&](int j) { return static_cast<uint32_t>((warp * per_q + j) * 32 + lane); };
    auto slot_of = [&](int j) { return static_cast<uint32_t>((warp * per_s + j) * 32 + lane); };

    // ---- loads; shared-memory set-up ----
    const int32_t free0 = ld_cg(count + r);
    const int32_t bound = keep_from != nullptr ? __ldg(keep_from + r) : INT32_MAX;
    int32_t key[IPT_Q], g[IPT_Q];
#pragma unroll
    for (int j = 0; j < IPT_Q; ++j) {
        key[j] = -1;
        if (j < per_q && pos_of(j) < Q) key[j] = __ldg(query + static_cast<uint64_t>(r) * Q + pos_of(j));
    }
    const uint64_t last_row = static_cast<uint64_t>(r) * last_count;
    int32_t named[IPT_Q];  // the entries' slots
    float w[IPT_Q];        // and weights
#pragma unroll
    for (int j = 0; j < IPT_Q; ++j) {
        const uint32_t p = tid + j * kThreads;
        named[j] = p < last_count ? __ldcg(last_slot + last_row + p) : kNotFound;
        w[j] = p < last_count ? weight_at(last_weight, weight_dtype, last_row + p) : 0.0f;
    }
    int32_t owner[IPT_S];
    float faded[IPT_S];
#pragma unroll
    for (int j = 0; j < IPT_S; ++j) {
        const bool mine = j < per_s && slot_of(j) < S;
        owner[j] = mine ? ld_cg(srow + slot_of(j)) : kNotFound;
        faded[j] = mine ? __ldcg(crow + slot_of(j)) : 0.0f;
    }
    auto fill = [&](int32_t* from, const int32_t* to, int v) {
        for (int4* p = reinterpret_cast<int4*>(from) + tid; p < reinterpret_cast<const int4*>(to); p += kThreads)
            *p = make_int4(v, v, v, v);
    };
    fill(s_count, s_hkey, 0);  // and s_asked
    fill(s_hkey, s_hpos, kEmptyKey);
    fill(s_hpos, s_hval, INT32_MAX);  // and s_claim
    if (tid == 0) n_hits = n_valid = 0;
    const int32_t tgt = static_cast<int32_t>(target < S ? target : S);
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
        for (int i = tid; i < tgt; i += kThreads) evicted[static_cast<uint64_t>(r) * ev_stride + i] = kNotFound;
        return;
    }
#pragma unroll
    for (int j = 0; j < IPT_Q; ++j)
        g[j] = static_cast<uint32_t>(key[j]) < K ? ld_cg(trow + key[j]) : kNotFound;
#pragma unroll
    for (int j = 0; j < IPT_S; ++j) {
        if (j >= per_s || slot_of(j) >= S) continue;
        const float v = __fmul_rn(faded[j], decay);
        if (!(v >= 0.0f) && owner[j] >= 0) bits |= ASU_ST_BAD_STATE;
        s_sum[slot_of(j)] = v > 0.0f ? v : 0.0f;  // never -0: the bits are ordered as unsigned ones
    }
    __syncthreads();

    // ---- the last step's entries claim their slots; this step's keys are classified ----
#pragma unroll
    for (int j = 0; j < IPT_Q; ++j) {
        if (static_cast<uint32_t>(named[j]) >= S) {
            if (named[j] != kNotFound) bits |= ASU_ST_BAD_QUERY;
            named[j] = kNotFound;
            continue;
        }
        if (!(w[j] >= 0.0f) || w[j] == INFINITY) {
            bits |= ASU_ST_BAD_WEIGHT;
            named[j] = kNotFound;
            continue;
        }
        atomicMin(&s_claim[named[j]], tid + j * kThreads);
    }
    uint8_t st[IPT_Q];
    int32_t hidx[IPT_Q];
    int valid_local = 0;
#pragma unroll
    for (int j = 0; j < IPT_Q; ++j) {
        st[j] = kInvalid;
        hidx[j] = -1;
        if (j >= per_q || pos_of(j) >= Q) continue;
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
            atomicMin(&s_hpos[h], static_cast<int32_t>(pos_of(j)));
        } else {
            st[j] = kBad;
            bits |= ASU_ST_BAD_STATE;
        }
    }
    __syncthreads();

    // ---- weights onto the sums: a slot's entries one after the other, in as many rounds as a slot has ----
    while (true) {
        int left = 0;
#pragma unroll
        for (int j = 0; j < IPT_Q; ++j) {
            const int32_t s = named[j];
            if (s == kNotFound) continue;
            if (s_claim[s] == tid + j * kThreads) {
                s_sum[s] = __fadd_rn(s_sum[s], w[j]);
                s_claim[s] = INT32_MAX;  // no entry's own: who reads it meanwhile stays for the next round
                named[j] = kNotFound;
            } else {
                left = 1;
            }
        }
        if (!__syncthreads_or(left)) break;
#pragma unroll
        for (int j = 0; j < IPT_Q; ++j)
            if (named[j] != kNotFound) atomicMin(&s_claim[named[j]], tid + j * kThreads);
        __syncthreads();
    }

    // ---- who leaves ----
    uint32_t u[IPT_S];  // score bits; all ones where the slot is no candidate
#pragma unroll
    for (int j = 0; j < IPT_S; ++j) {
        u[j] = 0xffffffffu;
        if (j >= per_s || slot_of(j) >= S) continue;
        const float v = s_sum[slot_of(j)];
        __stcg(crow + slot_of(j), owner[j] < 0 ? 0.0f : v);
        if (owner[j] >= 0 && owner[j] < bound && !s_asked[slot_of(j)]) u[j] = __float_as_uint(v);
    }
    int32_t E = tgt > free0 ? tgt - free0 : 0;
    uint32_t cut = 0, whole = 0;  // the E-th lowest U among the candidates; all under `whole` leave
    int quota = 0;                // and so many of those at cut
    if (E > 0) {                  // uniform
        int below = 0;
#pragma unroll 1
        for (int pass = 0; pass < 3; ++pass) {
            const int shift = pass == 0 ? 20 : pass == 1 ? 9 : 0;
            const int width = pass == 2 ? 9 : 11;
            int32_t* bins = s_count + pass * kBins;
#pragma unroll
            for (int j = 0; j < IPT_S; ++j) {
                if (j >= per_s) break;
                if ((u[j] ^ cut) >> (shift + width) == 0)
                    atomicAdd(&bins[(u[j] >> shift) & ((1u << width) - 1)], 1);
            }
            __syncthreads();
            const int2 c = pass < 2 || tid < 256 ? reinterpret_cast<const int2*>(bins)[tid] : make_int2(0, 0);
            const int sum = __reduce_add_sync(0xffffffffu, c.x + c.y);
            if (lane == 0) buf_a[warp] = sum;
            __syncthreads();
            int total;
            int before = below + before_warp(buf_a, &total);
            if (pass == 0 && E > total) E = total;
            if (E == 0) break;
            if (before < E && E <= before + sum) {  // one warp
                int x = c.x + c.y;
#pragma unroll
                for (int d = 1; d < 32; d <<= 1) {
                    const int y = __shfl_up_sync(0xffffffffu, x, d);
                    if (lane >= d) x += y;
                }
                before += x - c.x - c.y;
                if (before < E && E <= before + c.x + c.y) {  // one thread
                    const bool second = E > before + c.x;
                    s_digit[0] = 2 * tid + second;
                    s_digit[1] = before + (second ? c.x : 0);
                    s_digit[2] = second ? c.y : c.x;
                }
            }
            __syncthreads();
            cut |= static_cast<uint32_t>(s_digit[0]) << shift;
            below = s_digit[1];
            whole = cut;
            quota = E - below;
            if (quota == s_digit[2]) {  // they leave all
                whole = cut + (1u << shift);
                quota = 0;
                break;
            }
        }
    }
    if (E > 0) {
        int mine = 0;  // of the warp: those under `whole`, and those at cut from bit 16 on
#pragma unroll
        for (int j = 0; j < IPT_S; ++j) {
            if (j >= per_s) break;
            mine += __popc(__ballot_sync(0xffffffffu, u[j] < whole));
            if (quota > 0) mine += __popc(__ballot_sync(0xffffffffu, u[j] == cut)) << 16;
        }
        if (lane == 0) buf_b[warp] = mine;
        __syncthreads();
        int total;
        int before = before_warp(buf_b, &total), ties = before >> 16;
        before = (before & 0xffff) + min(ties, quota);
        int32_t* s_key = reinterpret_cast<int32_t*>(s_sum);  // the sums are done with
#pragma unroll
        for (int j = 0; j < IPT_S; ++j) {
            if (j >= per_s) break;
            bool leaves = u[j] < whole;
            uint32_t all = __ballot_sync(0xffffffffu, leaves);
            if (quota > 0) {
                const bool tie = u[j] == cut;
                const uint32_t all_ties = __ballot_sync(0xffffffffu, tie);
                leaves |= tie && ties + __popc(all_ties & below_lane) < quota;
                ties += __popc(all_ties);
                all = __ballot_sync(0xffffffffu, leaves);
            }
            if (leaves) {
                const int rank = before + __popc(all & below_lane);
                s_claim[rank] = static_cast<int32_t>(slot_of(j));
                s_key[rank] = owner[j];
            }
            before += __popc(all);
        }
        __syncthreads();
        for (int i = tid; i < E; i += kThreads) {
            const int32_t s = s_claim[i], k = s_key[i];
            st_cg(krow + free0 + i, s);
            evicted[static_cast<uint64_t>(r) * ev_stride + i] = k;
            if (static_cast<uint32_t>(k) < K) st_cg(trow + k, kNotFound);
            else bits |= ASU_ST_BAD_STATE;
            st_cg(srow + s, kNotFound);
            __stcg(crow + s, 0.0f);
        }
    }
    for (int i = E + tid; i < tgt; i += kThreads) evicted[static_cast<uint64_t>(r) * ev_stride + i] = kNotFound;
    if (tid == 0) ev_count[r] = E;
    const int32_t free1 = free0 + E;

    // ---- first occurrences of missing keys pop the stack in query order ----
    uint32_t first = 0, inst = 0;
    int firsts = 0;
#pragma unroll
    for (int j = 0; j < IPT_Q; ++j) {
        const bool f = st[j] == kMiss && s_hpos[hidx[j]] == static_cast<int32_t>(pos_of(j));
        first |= static_cast<uint32_t>(f) << j;
        firsts += __popc(__ballot_sync(0xffffffffu, f));
    }
    if (lane == 0) buf_q[warp] = firsts;
    __syncthreads();  // victims listed and unmapped
    int taken;
    int before = before_warp(buf_q, &taken);
    int32_t slot[IPT_Q];
#pragma unroll
    for (int j = 0; j < IPT_Q; ++j) {
        const bool f = (first >> j) & 1u;
        const uint32_t all = __ballot_sync(0xffffffffu, f);
        slot[j] = st[j] == kHit ? g[j] : kNotFound;
        if (f) {
            const int32_t k = before + __popc(all & below_lane);
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
                inst |= 1u << j;
            } else {
                bits |= ASU_ST_SHORTAGE;
            }
            s_hval[hidx[j]] = s;
            slot[j] = s;
        }
        before += __popc(all);
    }
    const int32_t n_inst = taken < free1 ? taken : free1;
    __syncthreads();  // installed slots visible
    int hits_local = 0;
#pragma unroll
    for (int j = 0; j < IPT_Q; ++j) {
        bool hit = st[j] == kHit;
        if (st[j] == kMiss && !((first >> j) & 1u)) {
            slot[j] = s_hval[hidx[j]];
            hit = slot[j] >= 0;
        }
        hits_local += hit;
        if (j < per_q && pos_of(j) < Q) {
            const uint64_t o = static_cast<uint64_t>(r) * Q + pos_of(j);
            slot_out[o] = slot[j];
            hit_mask[o] = hit;
            install_mask[o] = (inst >> j) & 1u;
        }
    }
    hits_local = __reduce_add_sync(0xffffffffu, hits_local);
    valid_local = __reduce_add_sync(0xffffffffu, valid_local);
    if (lane == 0) {
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
    const size_t slots16 = (static_cast<size_t>(S) + 15) & ~size_t{15};
    size_t smem = 4ull * kHistogram + 9 * slots16 + 12ull * (1ull << log2h);
    if (smem > static_cast<size_t>(max_dynamic)) {
        --log2h;
        smem = 4ull * kHistogram + 9 * slots16 + 12ull * (1ull << log2h);
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
    if (query_count <= kThreads * NQ && last_count <= kThreads * NQ && slot_count <= kThreads * NS)                   \
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

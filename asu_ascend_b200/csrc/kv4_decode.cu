// Sparse decode attention over the 4-bit cache for up to 64 heads, on the tcgen05 tensor cores.
//
// A row of 416 bytes meets 1088 multiply-adds for each head.  The products take the 128 entries of a tile
// (scores) or 128 latents (output) as their 128 rows and the heads as their columns, so that few heads
// cost little more than the reading of the dequantised rows from shared memory:
//   scores  S^T [128 entries x kN heads] = K Q^T          36 products of K = 16
//   output  O^T [4 x 128 latents x kN]  += V^T P^T        32 products
// Heads are padded to kN = 16, 32 or 64 (a product with both operands in shared memory takes 40 cycles for
// 32 columns or fewer, 48 for 64).
//
// Shared memory, 217 KB with 64 heads: q, 9 blocks of [kN heads x 64 values]; the tile's dequantised rows, 8
// blocks of [128 entries x 64 latents] and one of the rope part, all 128-byte rows in the 128-byte
// swizzle.  A latent block serves both products: entries x latents with the latents contiguous is K-major
// for the scores and M-major for the output.  The weights P [128 entries x kN] take the rope block's
// place once the scores are made.  There is no room for a second tile; its parts are released one after the
// other instead: latents 0..255 after the first half of the output products, the rest after the second,
// and the scores' products start on a part while the next is being filled.
//
// Tensor memory: O^T 4 kN columns, S^T kN.  A softmax thread's lane is an entry, so it holds all the heads of
// its entry and the maximum over the entries would be an exchange between 128 threads.  It is not needed in
// every tile: any reference close to it will do, as bf16 and fp32 carry 2^-126 .. 2^127.  The
// reference is the maximum of a piece's first tile and moves only when a score exceeds it by 2^40,
// which the threads vote on.  Sums of the weights stay with the threads until the piece is done.
//
// 13 warps: 4 softmax, 8 that load rows into registers and dequantise (the next tile's loads are issued as
// soon as a tile is stored, and fly during its products), one that issues the products.
//
// Tokens cut into 2 to 8 equal parts are joined by the cluster of their CTAs, if all clusters run at once, others by a
// second kernel, 5 to 8 us after the first.  The second kernel and the cluster, in us: 61 x 64 x 1024 over one pool 32.1 /
// 29.5, with weights 39.2 / 36.8; the weights of an uncut token, 1 x 16 x 100, 12.9 / 11.4; 32 x 32 x 2048 over one pool 22.1
// / 21.8, but over a pool a token 23.4 / 25.2.
//
// 128 tokens x 16 heads x 2048 entries take 55 us, 61 x 64 x 1024 29 us (inputs in rotation, none in L2).
// A tile is a chain of 3.3 us: the output products of its first half 0.35, two halves to dequantise 0.7 to 0.85
// each (shared memory: 128 KB stored, and the products' rows read at the same time), the scores' second half 0.45,
// the softmax 0.45, four hand-overs of 0.15; the loads of rows are hidden.  Tried and slower, 16 heads: tiles of 64
// entries twice (both buffers are held while one is filled: 78 us); rows through asynchronous copies and 16 warps
// that dequantise and make the softmax (62 us); four quarters instead of two halves (58 us: loads of 32 bytes a
// row instead of 128); every tile dequantised twice, into tensor memory for the scores (99 us: instructions and
// loads); products of single warps with rows dequantised in registers (79 us).
#include <atomic>

#include "kv4_decode.cuh"
#include "tcgen05.cuh"

namespace asu {
namespace kv4 {
namespace {

constexpr int kThreads = 13 * 32;
constexpr int kTile = 128;
constexpr int kBlock = kTile * 128;  // bytes of a [128 entries x 64] block
constexpr float kMaxGrowth = 40.0f;  // base 2
// Minus the reference while there is none: any finite score exceeds it, and a score of -inf still gives a weight of 0
// (with +inf here it would give NaN).
constexpr float kNoReference = 3.4028235e38f;
constexpr int kMaxParts = 8;         // CTAs of a cluster

// Every barrier is waited for in every phase by each of its waiters, and its next phase depends on them: a
// phase is never two ahead of one that waits for it.
enum Bar {
    kFullLow,   // latents 0..255 of the tile are dequantised (8 warps)
    kFullHigh,  // 256..511 and rope (8 warps)
    kFreeLow,   // the output products of latents 0..255 are done
    kOutput,    // all of them: the rest of the rows and the weights are free
    kScores,    // the tile's scores are made
    kWeights,   // its weights are in shared memory and the scores read (128 threads)
    kQuery,     // the token's q is in place (128 threads)
    kDrain,
    kBars
};

template <int kN>
struct Layout {
    static constexpr int kQBlock = kN * 128;  // bytes of a [kN heads x 64] block
    static constexpr int kQ = 0;
    static constexpr int kRows = (9 * kQBlock + 1023) / 1024 * 1024;
    static constexpr int kRope = kRows + 8 * kBlock;  // later the weights
    static constexpr int kBarsAt = kRope + kBlock;
    static constexpr int kBytes = kBarsAt + 8 * kBars + 1024;  // the base is rounded up to 1024
    static constexpr uint32_t kColS = 4 * kN;
};

struct Scratch {
    float* ml;         // [2 * ctas][2][kN] reference (base 2) and sum of a piece
    float* o;          // [2 * ctas][kN][512] its output
    float* ref;        // [tokens][tiles][kN] the reference of a tile's weights
    __nv_bfloat16* p;  // [tokens][tiles][128][kN] a tile's weights
};

// What a slot that is not there reads: a row of zeros.
__device__ __align__(16) const uint32_t g_zero_row[kRowBytes / 4] = {
#define ASU_ZERO4 0x88888888u, 0x88888888u, 0x88888888u, 0x88888888u
#define ASU_ZERO16 ASU_ZERO4, ASU_ZERO4, ASU_ZERO4, ASU_ZERO4
    ASU_ZERO16, ASU_ZERO16, ASU_ZERO16, ASU_ZERO16
#undef ASU_ZERO16
#undef ASU_ZERO4
};

// Loads that stay where they are written: the compiler would move plain ones down to their use and expose
// their latency.
__device__ __forceinline__ uint4 load16(const uint8_t* p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "l"(p));
    return v;
}
__device__ __forceinline__ uint32_t load2(const uint8_t* p) {
    unsigned short v;
    asm volatile("ld.global.nc.u16 %0, [%1];" : "=h"(v) : "l"(p));
    return v;
}

// Floats in the order of signed integers, and back.
__device__ __forceinline__ int ordered(float x) {
    const int i = __float_as_int(x);
    return i ^ ((i >> 31) & 0x7fffffff);
}
__device__ __forceinline__ float unordered(int i) { return __int_as_float(i ^ ((i >> 31) & 0x7fffffff)); }

// A token's CTAs are a cluster: when all have written their pieces, each joins a share of the heads and sums the
// weights of its own tiles.  That spares the second launch and its way to every SM.  `smem` is free: [9][kN] factors
// of the pieces and lse, and [3][kN] of a tile's weights.
template <int kN>
__device__ __forceinline__ void join_in_cluster(const Operands& op, const Division& div, const Scratch& scratch,
                                                float* smem) {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    const int parts = div.parts, token = blockIdx.x / parts, rank = blockIdx.x % parts;
    const int first_cta = token * parts;
    float(*s_factor)[kN] = reinterpret_cast<float(*)[kN]>(smem);
    float* s_lse = s_factor[kMaxParts];  // base 2
    if (parts == 1) {  // the outputs are written, and only weights are asked for
        if (threadIdx.x < kN)
            s_lse[threadIdx.x] = static_cast<int>(threadIdx.x) < op.heads
                                     ? op.lse[static_cast<int64_t>(token) * op.heads + threadIdx.x] * 1.4426950408889634f
                                     : -INFINITY;
    } else if (threadIdx.x < kN) {
        const int h = threadIdx.x;
        float m[kMaxParts], l[kMaxParts], top = -INFINITY, sum = 0.0f;
#pragma unroll
        for (int p = 0; p < kMaxParts; ++p) {
            const float* ml = scratch.ml + 4 * (first_cta + (p < parts ? p : 0)) * kN + h;
            m[p] = p < parts ? __ldcg(ml) : -INFINITY;
            l[p] = __ldcg(ml + kN);
            top = fmaxf(top, m[p]);
        }
#pragma unroll
        for (int p = 0; p < kMaxParts; ++p) {
            m[p] = m[p] == -INFINITY ? 0.0f : exp2_fast(m[p] - top);
            sum = fmaf(l[p], m[p], sum);
        }
        const float inv = sum != 0.0f ? 1.0f / sum : 0.0f;  // a NaN goes on
#pragma unroll
        for (int p = 0; p < kMaxParts; ++p) s_factor[p][h] = m[p] * inv;
        s_lse[h] = sum != 0.0f && h < op.heads ? top + log2f(sum) : -INFINITY;
        if (rank == 0 && h < op.heads)
            op.lse[static_cast<int64_t>(token) * op.heads + h] =
                sum != 0.0f ? (top + log2f(sum)) * 0.6931471805599453f : -INFINITY;
    }
    __syncthreads();
    const int t = threadIdx.x & 127, group = threadIdx.x >> 7;  // three groups, and a warp that looks on
    if (group >= 3) return;
    constexpr int kHeads = 4;  // at a time: their loads fly together
    const int share = (op.heads + parts - 1) / parts;
    const int last = min(op.heads, (rank + 1) * share);
    for (int h0 = rank * share + group * kHeads; parts > 1 && h0 < last; h0 += 3 * kHeads) {
        float4 acc[kHeads] = {};
#pragma unroll 2
        for (int p = 0; p < parts; ++p) {
            float4 v[kHeads];
#pragma unroll
            for (int k = 0; k < kHeads; ++k) {
                const int64_t row = static_cast<int64_t>(2 * (first_cta + p)) * kN + min(h0 + k, last - 1);
                v[k] = __ldcg(reinterpret_cast<const float4*>(scratch.o + row * kLatent) + t);
            }
#pragma unroll
            for (int k = 0; k < kHeads; ++k) {
                const float f = s_factor[p][min(h0 + k, last - 1)];
                acc[k].x = fmaf(v[k].x, f, acc[k].x), acc[k].y = fmaf(v[k].y, f, acc[k].y);
                acc[k].z = fmaf(v[k].z, f, acc[k].z), acc[k].w = fmaf(v[k].w, f, acc[k].w);
            }
        }
#pragma unroll
        for (int k = 0; k < kHeads; ++k)
            if (h0 + k < last)
                reinterpret_cast<uint2*>(op.out + (static_cast<int64_t>(token) * op.heads + h0 + k) * kLatent)[t] =
                    make_uint2(pack_bf16(acc[k].x, acc[k].y), pack_bf16(acc[k].z, acc[k].w));
    }
    if (op.weights == nullptr) return;
    float* s_tile = s_factor[kMaxParts + 1 + group];
    for (int u = div.start(blockIdx.x) + group; u < div.start(blockIdx.x + 1); u += 3) {
        const uint4* p = reinterpret_cast<const uint4*>(scratch.p + (static_cast<int64_t>(u) * kTile + t) * kN);
        uint4 v[kN / 8];
#pragma unroll
        for (int i = 0; i < kN / 8; ++i) v[i] = __ldcg(p + i);
        if (t < kN) {
            const float ref = __ldcg(scratch.ref + static_cast<int64_t>(u) * kN + t);
            s_tile[t] = s_lse[t] == -INFINITY ? 0.0f : exp2_fast(ref - s_lse[t]);
        }
        asm volatile("bar.sync %0, 128;" ::"r"(2 + group) : "memory");
        const int e = (u - token * div.tiles) * kTile + t;
        float w = 0.0f;
#pragma unroll
        for (int i = 0; i < kN / 8; ++i) {
            const uint32_t x[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                w = fmaf(__uint_as_float(x[k] << 16), s_tile[i * 8 + 2 * k], w);
                w = fmaf(__uint_as_float(x[k] & 0xffff0000u), s_tile[i * 8 + 2 * k + 1], w);
            }
        }
        if (e < op.topk)
            op.weights[static_cast<int64_t>(token) * op.topk + e] = __float2bfloat16(weight_of(op, token, e, w));
        asm volatile("bar.sync %0, 128;" ::"r"(2 + group) : "memory");
    }
}

// kJoin: a token's CTAs are a cluster and join their pieces themselves.
template <int kN, bool kJoin>
__global__ void __launch_bounds__(kThreads, 1)
kv4_decode_kernel(const Operands op, const Division div, const Scratch scratch) {
    using L = Layout<kN>;
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint32_t s_tmem;
    __shared__ int s_dead;
    __shared__ float s_minus_ref[kN];  // minus the reference, base 2
    __shared__ float s_fade[kN];       // what a new reference multiplies sums and output by; later 1 / sum
    __shared__ __align__(8) int s_top[4][kN];       // each softmax warp's maximum, or sum
    const uint32_t base = (tc::smem_u32(smem_raw) + 1023u) & ~1023u;
    auto bar = [&](int which) { return base + L::kBarsAt + 8u * which; };
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    volatile int* dead = &s_dead;
    // A wait that runs out sets the flag, and then no other one waits: every loop goes through to its end, on
    // whatever the buffers hold, so that each barrier is met by all; the status says that it happened.
    auto warp_wait = [&](int which, uint32_t phase) {
        tc::mbar_wait(bar(which), phase & 1, dead);
        __syncwarp();
    };

    if (tid == 0) {
        s_dead = 0;
        tc::mbar_init(bar(kFullLow), 8);
        tc::mbar_init(bar(kFullHigh), 8);
        tc::mbar_init(bar(kFreeLow), 1);
        tc::mbar_init(bar(kOutput), 1);
        tc::mbar_init(bar(kScores), 1);
        tc::mbar_init(bar(kWeights), 128);
        tc::mbar_init(bar(kQuery), 128);
        tc::mbar_init(bar(kDrain), 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 12) tc::tmem_alloc<512>(tc::smem_u32(&s_tmem));
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    // All columns, although few heads need fewer: they start at 0, whatever else runs on the SM, and the
    // addresses below are constants.
    if (tid == 0 && s_tmem != 0) *dead = 1;
    pdl_wait();

    const int32_t u0 = div.start(blockIdx.x), u1 = div.start(blockIdx.x + 1);
    const int tiles = div.tiles;

    if (warp >= 4 && warp < 12) {
        // ---- rows: global memory -> registers -> dequantised blocks ----
        // lane = 8 q + 2 rr + lp: row rr of four, latents 32 * (2 q + lp) .. of either half.  Eight
        // consecutive lanes store to four rows x two chunks, which the swizzle spreads over all banks.
        const int quarter = lane >> 3, lp = lane & 1;
        const int row0 = (warp - 4) * 4 + ((lane >> 1) & 3);  // and row0 + 32, 64, 96
        const int chunk = 2 * quarter + lp, rope_chunk = lp * 4 + quarter;
        int32_t bits = 0;
        uint4 low[4], high[4], rope[4];
        uint32_t low_scales[4], high_scales[4];
        int32_t slot[4];
        Walk ahead(div, u0);
        auto load_slots = [&] {
            const int32_t* row = op.slots + ahead.row * op.slots_token;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int e = ahead.tile * kTile + i * 32 + row0;
                slot[i] = ahead.u < u1 && e < op.topk ? __ldg(row + e) : kNotFound;
            }
        };
        auto load_rows = [&] {
            const uint8_t* pool = op.pool + static_cast<uint64_t>(ahead.row) * op.pool_token;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const bool there = slot[i] >= 0 && slot[i] < op.pool_rows;
                if (!there && slot[i] != kNotFound) bits |= ASU_ST_BAD_QUERY;
                const uint8_t* p = there ? pool + static_cast<uint64_t>(slot[i]) * op.pool_pitch
                                         : reinterpret_cast<const uint8_t*>(g_zero_row);
                low[i] = load16(p + chunk * 16);
                high[i] = load16(p + 128 + chunk * 16);
                rope[i] = load16(p + kRopeOffset + rope_chunk * 16);
                low_scales[i] = load2(p + kScaleOffset + chunk * 2);
                high_scales[i] = load2(p + kScaleOffset + 16 + chunk * 2);
            }
        };
        load_slots();
        load_rows();
        ahead.next(div);
        load_slots();
        const uint32_t at = base + L::kRows + quarter * kBlock + row0 * 128 + (((lp * 4) ^ (row0 & 7)) << 4);
        const uint32_t rope_at = base + L::kRope + row0 * 128 + ((rope_chunk ^ (row0 & 7)) << 4);
        const uint32_t count = u1 - u0;
        for (uint32_t n = 0; n < count; ++n) {
            if (n >= 1) warp_wait(kFreeLow, n - 1);
#pragma unroll
            for (int i = 0; i < 4; ++i) dequantise(low[i], low_scales[i], at + i * 32 * 128);
            tc::fence_async_shared();
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(bar(kFullLow));
            if (n >= 1) warp_wait(kOutput, n - 1);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                dequantise(high[i], high_scales[i], at + 4 * kBlock + i * 32 * 128);
                shared_store16(rope_at + i * 32 * 128, rope[i].x, rope[i].y, rope[i].z, rope[i].w);
            }
            tc::fence_async_shared();
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(bar(kFullHigh));
            load_rows();
            ahead.next(div);
            load_slots();
        }
        if (bits) flag_status(op.status, 0, bits);
    } else if (warp == 12) {
        // ---- the products, all by one lane.  (The branch has to be that of elect.sync itself: with a plain
        // lane number, or its result kept, the issue of a product takes 80 cycles instead of 30.) ----
        if (tc::elect_one()) {
            constexpr uint32_t kDescS = tc::instruction(128, kN, false, false);
            constexpr uint32_t kDescO = tc::instruction(128, kN, true, true);
            const uint32_t desc_q = tc::operand(base + L::kQ, 0);
            const uint32_t desc_k = tc::operand(base + L::kRows, 0);
            const uint32_t desc_v = tc::operand(base + L::kRows, kBlock);
            const uint32_t desc_p = tc::operand(base + L::kRope, 0);
            auto wait = [&](int which, uint32_t phase) { tc::mbar_wait(bar(which), phase & 1, dead); };
            uint32_t n = 0, segment = 0;
            for (Walk at(div, u0); at.u < u1; at.next(div), ++n) {
                const bool first = at.u == u0 || at.tile == 0;
                if (first) wait(kQuery, segment++);
#pragma unroll 1
                for (int part = 0; part < 2; ++part) {
                    wait(part ? kFullHigh : kFullLow, n);
                    tc::fence_after();
#pragma unroll
                    for (int i = 0; i < 5; ++i) {
                        if (i == 4 && part == 0) continue;
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            tc::mma_ss(L::kColS, desc_k + (4 * part + i) * (kBlock / 16) + 2 * k,
                                       desc_q + (4 * part + i) * (L::kQBlock / 16) + 2 * k, kDescS, part || i || k);
                    }
                }
                tc::commit(bar(kScores));
                wait(kWeights, n);
                tc::fence_after();
#pragma unroll 1
                for (int t = 0; t < 4; ++t) {
#pragma unroll
                    for (int k = 0; k < kTile / 16; ++k)
                        tc::mma_ss(t * kN, desc_v + t * (2 * kBlock / 16) + k * (2048 / 16), desc_p + k * (2048 / 16),
                                   kDescO, !first || k);
                    if (t == 1) tc::commit(bar(kFreeLow));
                }
                tc::commit(bar(kOutput));
            }
        }
        __syncwarp();
    } else {
        // ---- softmax: a thread an entry of the tile; for the output, a thread a latent of 128 ----
        const uint32_t lanes = static_cast<uint32_t>(warp * 32) << 16;
        auto softmax_sync = [] { asm volatile("bar.sync 1, 128;" ::: "memory"); };  // these four warps
        auto load_q = [&](int token) {
            const __nv_bfloat16* q = op.q + token * op.q_token + (tid & 7) * 8;
            const uint32_t to0 = base + L::kQ + (((tid ^ (tid >> 3)) & 7) << 4);
#pragma unroll 1
            for (int h = tid >> 3; h < kN; h += 16) {
                const bool there = h < op.heads;
                const __nv_bfloat16* from = q + (there ? h : 0) * op.q_head;
                if (op.q_aligned || !there) {
#pragma unroll
                    for (int k = 0; k < 9; ++k)
                        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to0 + k * L::kQBlock + h * 128),
                                     "l"(from + k * 64), "r"(there ? 16 : 0)
                                     : "memory");
                } else {
#pragma unroll 1
                    for (int k = 0; k < 9; ++k) {
                        const uint4 v = load_unaligned(from + k * 64);
                        shared_store16(to0 + k * L::kQBlock + h * 128, v.x, v.y, v.z, v.w);
                    }
                }
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
            tc::fence_async_shared();
            tc::mbar_arrive(bar(kQuery));
        };
        constexpr int kC = kN < 32 ? kN : 32;  // columns at a time
        float l[kN];                           // this thread's entries' weights by head
        Walk at(div, u0);
        load_q(at.row);
        auto slot_here = [&](const Walk& w) -> bool {
            const int e = w.tile * kTile + tid;
            if (w.u >= u1 || e >= op.topk) return false;
            const int32_t s = __ldg(op.slots + w.row * op.slots_token + e);
            return s >= 0 && s < op.pool_rows;
        };
        bool there = slot_here(at);
        for (uint32_t n = 0; at.u < u1; ++n) {
            const int token = at.row, tile = at.tile;
            const bool first = at.u == u0 || tile == 0;
            const bool last = at.u + 1 == u1 || tile + 1 == tiles;
            if (first) {
#pragma unroll
                for (int h = 0; h < kN; ++h) l[h] = 0.0f;
            }
            warp_wait(kScores, n);
            if (n >= 1) warp_wait(kOutput, n - 1);  // long done: these scores came after it
            tc::fence_after();
            // does a score exceed its reference by too much?
            bool over = false;
            if (!first) {
#pragma unroll 1
                for (int c0 = 0; c0 < kN; c0 += kC) {
                    uint32_t s[kC];
                    tc::tmem_load(lanes + L::kColS + c0, s);
                    tc::tmem_wait_load(s);
                    float top = -INFINITY;
#pragma unroll
                    for (int h = 0; h < kC; ++h)
                        top = fmaxf(top, fmaf(__uint_as_float(s[h]), op.scale_log2, s_minus_ref[c0 + h]));
                    over |= top > kMaxGrowth;
                }
                over &= there;
            }
            if (tc::any_of<128>(over || first)) {
                // new references: the maxima over the tile's entries, of this tile alone in a piece's first
#pragma unroll 1
                for (int c0 = 0; c0 < kN; c0 += kC) {
                    uint32_t s[kC];
                    tc::tmem_load(lanes + L::kColS + c0, s);
                    tc::tmem_wait_load(s);
#pragma unroll
                    for (int h = 0; h < kC; ++h) {
                        const float x = there ? __uint_as_float(s[h]) * op.scale_log2 : -INFINITY;
                        const int top = __reduce_max_sync(0xffffffffu, ordered(x));
                        if (lane == h) s_top[warp][c0 + h] = top;
                    }
                }
                softmax_sync();
                if (tid < kN) {
                    const float top = unordered(max(max(s_top[0][tid], s_top[1][tid]), max(s_top[2][tid], s_top[3][tid])));
                    // a piece whose entries so far are all missing has none
                    const float old = first ? kNoReference : s_minus_ref[tid];
                    const float now = fminf(old, -top);
                    s_fade[tid] = old == now ? 1.0f : old == kNoReference ? 0.0f : exp2_fast(now - old);
                    s_minus_ref[tid] = now;
                }
                softmax_sync();
                if (!first) {
#pragma unroll
                    for (int h = 0; h < kN; ++h) l[h] *= s_fade[h];
#pragma unroll 1
                    for (int c0 = 0; c0 < 4 * kN; c0 += kC) {
                        uint32_t o[kC];
                        tc::tmem_load(lanes + c0, o);
                        tc::tmem_wait_load(o);
#pragma unroll
                        for (int h = 0; h < kC; ++h) o[h] = __float_as_uint(__uint_as_float(o[h]) * s_fade[(c0 + h) % kN]);
                        tc::tmem_store(lanes + c0, o);
                    }
                    tc::tmem_wait_store();
                }
            }
            const int64_t unit = static_cast<int64_t>(token) * tiles + tile;
            if (op.weights != nullptr && tid < kN) scratch.ref[unit * kN + tid] = -s_minus_ref[tid];
#pragma unroll
            for (int c0 = 0; c0 < kN; c0 += kC) {
                uint32_t s[kC];
                tc::tmem_load(lanes + L::kColS + c0, s);
                tc::tmem_wait_load(s);
                // The weights are rounded to bf16, as the tensor cores take them beside bf16 rows: half a step, 2^-8 of
                // each at most, which the sums average out (0.0020 off the exact output in the mean instead of the
                // 0.0017 that the output's own rounding leaves).  Their sum l takes them before the rounding.
                uint32_t p[kC / 2];
#pragma unroll
                for (int h = 0; h < kC; h += 2) {
                    float a = exp2_fast(fmaf(__uint_as_float(s[h]), op.scale_log2, s_minus_ref[c0 + h]));
                    float b = exp2_fast(fmaf(__uint_as_float(s[h + 1]), op.scale_log2, s_minus_ref[c0 + h + 1]));
                    a = there ? a : 0.0f;
                    b = there ? b : 0.0f;
                    l[c0 + h] += a;
                    l[c0 + h + 1] += b;
                    p[h / 2] = pack_bf16(a, b);
                }
                const uint32_t to = base + L::kRope + tid * 128;
#pragma unroll
                for (int i = 0; i < kC / 8; ++i)
                    shared_store16(to + (((c0 / 8 + i) ^ (tid & 7)) << 4), p[4 * i], p[4 * i + 1], p[4 * i + 2],
                                   p[4 * i + 3]);
                if (op.weights != nullptr) {
                    uint4* out = reinterpret_cast<uint4*>(scratch.p + (unit * kTile + tid) * kN + c0);
#pragma unroll
                    for (int i = 0; i < kC / 8; ++i)
                        out[i] = make_uint4(p[4 * i], p[4 * i + 1], p[4 * i + 2], p[4 * i + 3]);
                }
            }
            tc::fence_async_shared();
            tc::fence_before();
            tc::mbar_arrive(bar(kWeights));
            at.next(div);
            there = slot_here(at);
            if (last) {
                // this token's scores are all made: the next one's q comes beside the output products
                if (at.u < u1) load_q(at.row);
                // Sums over the entries: within the warps, then the four.  In each step a lane passes half of its
                // heads on and adds the partner's to the other half.
#pragma unroll
                for (int d = 16, count = kN / 2; d > 0; d >>= 1, count >>= 1) {
                    const bool upper = (lane & d) != 0;
                    if (count == 0) l[0] += __shfl_xor_sync(0xffffffffu, l[0], d);
#pragma unroll
                    for (int h = 0; h < count; ++h) {
                        const float other = __shfl_xor_sync(0xffffffffu, upper ? l[h] : l[h + count], d);
                        l[h] = (upper ? l[h + count] : l[h]) + other;
                    }
                }
                if constexpr (kN == 16) s_top[warp][lane / 2] = __float_as_int(l[0]);
                if constexpr (kN == 32) s_top[warp][lane] = __float_as_int(l[0]);
                if constexpr (kN == 64)
                    *reinterpret_cast<int2*>(&s_top[warp][2 * lane]) =
                        make_int2(__float_as_int(l[0]), __float_as_int(l[1]));
                softmax_sync();
                const int row_start = token * tiles;
                const bool whole = row_start >= u0 && row_start + tiles <= u1;
                const int piece = div.piece(blockIdx.x, row_start);
                if (tid < kN) {
                    const float sum = (__int_as_float(s_top[0][tid]) + __int_as_float(s_top[1][tid])) +
                                      (__int_as_float(s_top[2][tid]) + __int_as_float(s_top[3][tid]));
                    if (whole) {
                        s_fade[tid] = sum != 0.0f ? 1.0f / sum : 0.0f;  // a NaN goes on
                        if (tid < op.heads)
                            op.lse[static_cast<int64_t>(token) * op.heads + tid] =
                                sum != 0.0f ? (log2f(sum) - s_minus_ref[tid]) * 0.6931471805599453f : -INFINITY;
                    } else {
                        scratch.ml[piece * 2 * kN + tid] = sum != 0.0f ? -s_minus_ref[tid] : -INFINITY;
                        scratch.ml[(piece * 2 + 1) * kN + tid] = sum;
                    }
                }
                softmax_sync();
                warp_wait(kOutput, n);
                tc::fence_after();
#pragma unroll 1
                for (int c0 = 0; c0 < 4 * kN; c0 += kC) {
                    uint32_t o[kC];
                    tc::tmem_load(lanes + c0, o);
                    tc::tmem_wait_load(o);
                    const int latent = c0 / kN * 128 + tid, h0 = c0 % kN;
                    if (whole) {
                        __nv_bfloat16* to = op.out + (static_cast<int64_t>(token) * op.heads + h0) * kLatent + latent;
#pragma unroll
                        for (int h = 0; h < kC; ++h)
                            if (h0 + h < op.heads)
                                to[h * kLatent] = __float2bfloat16(__uint_as_float(o[h]) * s_fade[h0 + h]);
                    } else {
                        float* to = scratch.o + (static_cast<int64_t>(piece) * kN + h0) * kLatent + latent;
#pragma unroll
                        for (int h = 0; h < kC; ++h) to[h * kLatent] = __uint_as_float(o[h]);
                    }
                }
                tc::fence_before();
            }
        }
    }
    pdl_trigger();
    if constexpr (kJoin) {
        __syncwarp();
        join_in_cluster<kN>(op, div, scratch, reinterpret_cast<float*>(smem_raw));
    }
    __syncthreads();
    if (s_dead && tid == 0) flag_status(op.status, 0, ASU_ST_TIMEOUT);
    if (warp == 12) {
        // Nothing of this block may be in flight when its tensor memory goes and its barriers with it,
        // whatever way the loops were left.
        if (tc::elect_one()) {
            tc::commit(bar(kDrain));
            for (int i = 0; i < tc::kSpinLimit && !tc::mbar_try(bar(kDrain), 0); ++i) {
            }
        }
        __syncwarp();
        tc::fence_after();
        tc::tmem_free<512>(s_tmem);
    }
}

// Joins the pieces of tokens that several CTAs share, and sums the weights over the heads.
//   blocks y < joins: two heads of a token, 4 latents a thread
//   other blocks:     two tiles, an entry a thread: weights_j = sum_h p_hj 2^(ref_h - lse_h)
// Loads that do not depend on one another are issued together: the blocks are short and wait for little else.
template <int kN>
__global__ void __launch_bounds__(256)
kv4_finish_kernel(const Operands op, const Division div, const Scratch scratch) {
    pdl_wait();
    pdl_trigger();
    __shared__ float s_factor[2][kN];
    const int token = blockIdx.x, joins = (op.heads + 1) / 2;
    const int tid = threadIdx.x & 127, part = threadIdx.x >> 7;
    const int first = token * div.tiles;
    const int i0 = div.cta_of(first), i1 = div.cta_of(first + div.tiles - 1);
    constexpr int kBatch = 4;  // pieces at a time
    // running reference (base 2) and sum of a head; factors of what is there and of the next pieces
    float m = -INFINITY, l = 0.0f, old, f[kBatch];
    float pm[kBatch], pl[kBatch];
    auto load_ml = [&](int i, int head) {
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
            const bool here = i + k <= i1;
            const float* ml = scratch.ml + div.piece(here ? i + k : i, first) * 2 * kN + head;
            pm[k] = here ? __ldcg(ml) : -INFINITY;
            pl[k] = __ldcg(ml + kN);
        }
    };
    auto join = [&] {
        float top = m;
#pragma unroll
        for (int k = 0; k < kBatch; ++k) top = fmaxf(top, pm[k]);
        old = m == -INFINITY ? 0.0f : exp2_fast(m - top);
        l *= old;
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
            f[k] = pm[k] == -INFINITY ? 0.0f : exp2_fast(pm[k] - top);
            l = fmaf(pl[k], f[k], l);
        }
        m = top;
    };
    if (static_cast<int>(blockIdx.y) < joins) {
        const int head = 2 * blockIdx.y + part;
        if (i0 == i1 || head >= op.heads) return;  // written by its one CTA
        float4 acc = make_float4(0, 0, 0, 0);
        for (int i = i0; i <= i1; i += kBatch) {
            load_ml(i, head);
            float4 v[kBatch];
#pragma unroll
            for (int k = 0; k < kBatch; ++k) {
                const int64_t row = static_cast<int64_t>(div.piece(i + k, first)) * kN + head;
                v[k] = i + k <= i1 ? __ldcg(reinterpret_cast<const float4*>(scratch.o + row * kLatent) + tid)
                                   : make_float4(0, 0, 0, 0);
            }
            join();
            acc.x *= old, acc.y *= old, acc.z *= old, acc.w *= old;
#pragma unroll
            for (int k = 0; k < kBatch; ++k) {
                acc.x = fmaf(v[k].x, f[k], acc.x), acc.y = fmaf(v[k].y, f[k], acc.y);
                acc.z = fmaf(v[k].z, f[k], acc.z), acc.w = fmaf(v[k].w, f[k], acc.w);
            }
        }
        const float inv = l != 0.0f ? 1.0f / l : 0.0f;
        reinterpret_cast<uint2*>(op.out + (static_cast<int64_t>(token) * op.heads + head) * kLatent)[tid] =
            make_uint2(pack_bf16(acc.x * inv, acc.y * inv), pack_bf16(acc.z * inv, acc.w * inv));
        if (tid == 0)
            op.lse[static_cast<int64_t>(token) * op.heads + head] =
                l != 0.0f ? (m + log2f(l)) * 0.6931471805599453f : -INFINITY;
        return;
    }
    const int tile = 2 * (blockIdx.y - joins) + part;
    const bool here = tile < div.tiles;
    const int64_t unit = static_cast<int64_t>(token) * div.tiles + (here ? tile : 0);
    const uint4* p = reinterpret_cast<const uint4*>(scratch.p + (unit * kTile + tid) * kN);
    uint4 v[kN / 8];
#pragma unroll
    for (int i = 0; i < kN / 8; ++i) v[i] = __ldcg(p + i);
    if (tid < kN) {
        const float ref = __ldcg(scratch.ref + unit * kN + tid);
        float lse = -INFINITY;  // base 2; the joining blocks may not have written it yet
        if (tid < op.heads) {
            if (i0 == i1) {
                lse = op.lse[static_cast<int64_t>(token) * op.heads + tid] * 1.4426950408889634f;
            } else {
                for (int i = i0; i <= i1; i += kBatch) {
                    load_ml(i, tid);
                    join();
                }
                if (l != 0.0f) lse = m + log2f(l);
            }
        }
        s_factor[part][tid] = lse == -INFINITY ? 0.0f : exp2_fast(ref - lse);
    }
    __syncthreads();
    const int e = tile * kTile + tid;
    if (!here || e >= op.topk) return;
    float w = 0.0f;
#pragma unroll
    for (int i = 0; i < kN / 8; ++i) {
        const uint32_t x[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            w = fmaf(__uint_as_float(x[k] << 16), s_factor[part][i * 8 + 2 * k], w);
            w = fmaf(__uint_as_float(x[k] & 0xffff0000u), s_factor[part][i * 8 + 2 * k + 1], w);
        }
    }
    op.weights[static_cast<int64_t>(token) * op.topk + e] = __float2bfloat16(weight_of(op, token, e, w));
}

int columns_of(int64_t heads) { return heads <= 16 ? 16 : heads <= 32 ? 32 : 64; }

int64_t tiles_of(int64_t topk) { return topk > 0 ? (topk + kTile - 1) / kTile : 1; }  // no entry: one empty tile

Division division(int64_t tokens, int64_t topk, int sms) { return Division(tokens, tiles_of(topk), sms, 1); }

void layout(const Division& d, int n, bool weights, int64_t (&at)[5]) {
    const int64_t units = static_cast<int64_t>(d.rows) * d.tiles;
    const int64_t pieces = d.shares() ? 2ll * d.ctas : 0;
    at[0] = 0;
    at[1] = at[0] + align256(pieces * 2 * n * 4);
    at[2] = at[1] + align256(pieces * n * kLatent * 4);
    at[3] = at[2] + (weights ? align256(units * n * 4) : 0);
    at[4] = at[3] + (weights ? units * kTile * n * 2 : 0);
}

// How many clusters of that many CTAs the device can run at once; asked once per device.
template <int kN>
int most_clusters(int parts, int bytes) {
    static std::atomic<int> known[64][kMaxParts + 1];  // 1 + the answer
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
    int n = known[dev][parts].load(std::memory_order_relaxed) - 1;
    if (n >= 0) return n;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = static_cast<unsigned>(parts);
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(parts));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = bytes;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&n, kv4_decode_kernel<kN, true>, &cfg) != cudaSuccess) {
        cudaGetLastError();
        n = 0;
    }
    known[dev][parts].store(n + 1, std::memory_order_relaxed);
    return n;
}

template <int kN>
int launch(cudaStream_t s, const Operands& op, void* workspace) {
    const Division d = division(op.tokens, op.topk, asu_sm_count());
    int64_t at[5];
    layout(d, kN, op.weights != nullptr, at);
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    const Scratch scratch = {reinterpret_cast<float*>(ws + at[0]), reinterpret_cast<float*>(ws + at[1]),
                             reinterpret_cast<float*>(ws + at[2]), reinterpret_cast<__nv_bfloat16*>(ws + at[3])};
    int max_dynamic = 0;
    int rc = asu_max_dynamic_smem(reinterpret_cast<const void*>(kv4_decode_kernel<kN, false>), &max_dynamic);
    if (rc != ASU_OK) return rc;
    if (max_dynamic < Layout<kN>::kBytes) return ASU_ERR_ARG;
    if (d.parts > (op.weights != nullptr ? 0 : 1) && d.parts <= kMaxParts) {
        rc = asu_max_dynamic_smem(reinterpret_cast<const void*>(kv4_decode_kernel<kN, true>), &max_dynamic);
        if (rc != ASU_OK) return rc;
        // All of the SM's shared memory: blocks of a cluster wait for one another while they hold tensor memory, which
        // another kernel's cluster on the same SMs must not wait for while it holds some.
        if (max_dynamic >= Layout<kN>::kBytes && most_clusters<kN>(d.parts, max_dynamic) >= op.tokens)
            return launch_pdl_clusters(kv4_decode_kernel<kN, true>, dim3(d.ctas), dim3(kThreads), max_dynamic, s,
                                       static_cast<unsigned>(d.parts), op, d, scratch);
    }
    rc = launch_pdl(kv4_decode_kernel<kN, false>, dim3(d.ctas), dim3(kThreads), Layout<kN>::kBytes, s, op, d, scratch);
    if (rc != ASU_OK || (!d.shares() && op.weights == nullptr)) return rc;
    return launch_pdl(kv4_finish_kernel<kN>,
                      dim3(static_cast<unsigned>(op.tokens),
                           static_cast<unsigned>((op.heads + 1) / 2 + (op.weights != nullptr ? (d.tiles + 1) / 2 : 0))),
                      dim3(256), 0, s, op, d, scratch);
}

}  // namespace

int64_t tall_workspace(int64_t tokens, int64_t heads, int64_t topk, bool weights) {
    int64_t at[5];
    layout(division(tokens, topk, asu_sm_count()), columns_of(heads), weights, at);
    return at[4];
}

int64_t tall_weights(int64_t heads, int64_t topk) { return tiles_of(topk) * columns_of(heads) * (4 + 2 * kTile); }

int launch_tall(cudaStream_t s, const Operands& op, void* workspace) {
    switch (columns_of(op.heads)) {
        case 16: return launch<16>(s, op, workspace);
        case 32: return launch<32>(s, op, workspace);
        default: return launch<64>(s, op, workspace);
    }
}

}  // namespace kv4
}  // namespace asu

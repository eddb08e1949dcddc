// Sparse decode attention over the 4-bit cache, on the tcgen05 tensor cores.
//
// A row of 416 bytes meets 1088 multiply-adds for each head.  The products take the 128 entries of a tile
// (scores) or 128 latents (output) as their 128 rows and the heads as their columns, so that few heads
// cost little more than the reading of the dequantised rows from shared memory:
//   scores  S^T [128 entries x kN heads] = K Q^T          36 products of K = 16
//   output  O^T [4 x 128 latents x kN]  += V^T P^T        32 products
// Heads are taken kN = 16 or 32 at a time; more are several rows of work.
//
// Shared memory, 225 KB with 32 heads: q, 9 blocks of [kN heads x 64 values]; the tile's dequantised rows, 8
// blocks of [128 entries x 64 latents] and one of the rope part, all 128-byte rows in the 128-byte
// swizzle; the weights P [128 entries x kN]; and the 4-bit part of the next tile's rows.  A latent block
// serves both products: entries x latents with the latents contiguous is K-major for the scores and M-major
// for the output.  There is no room for a second dequantised tile; its parts are released one after the
// other instead: the rope block after the scores, latents 0..255 after the first half of the output
// products, the rest after the second, and the scores' products start on a part while the next is filled.
//
// Tensor memory: O^T 4 kN columns, S^T kN.  A thread's lane is an entry, so the maximum over the entries would
// be an exchange between 128 threads.  It is not needed in every tile: any reference close to it will do, as
// bf16 and fp32 carry 2^-126 .. 2^127.  The reference is the maximum of a piece's first tile and moves
// only when a score exceeds it by 2^40, which the threads vote on.  Sums of the weights stay with the
// threads until the piece is done.
//
// 19 warps.  Dequantising a tile, its scores, their softmax and the output products wait for one another
// all around, so the same 16 warps do both kinds of work, each kind in a quarter of the time that four
// warps of its own took: they dequantise the tile, and when the scores are there, four warps a quarter of
// the entries make a quarter of the heads each.  Two warps copy rows, asynchronously (a tile's 53 KB on
// their way to registers instead do not fit into what the shared memory leaves of the L1 cache: their issue
// alone took 2 us).  One issues the products.
#include "kv4_decode.cuh"
#include "tcgen05.cuh"

namespace asu {
namespace kv4 {
namespace {

constexpr int kWorkers = 16 * 32;
constexpr int kThreads = kWorkers + 3 * 32;
constexpr int kTile = 128;
constexpr int kBlock = kTile * 128;        // bytes of a [128 entries x 64] block
constexpr int kRawHalf = kTile * (128 + 16);  // bytes of a tile's 256 latents in 4 bits: nibbles, then scales
constexpr float kMaxGrowth = 40.0f;  // base 2

// Every barrier is waited for in every phase by each of its waiters, and its next phase depends on them: a
// phase is never two ahead of one that waits for it.
enum Bar {
    kLowHere,   // the 4-bit latents 0..255 of the tile are in shared memory (64 threads' copies)
    kLowRead,   // and have been read (16 warps)
    kHighHere,  // the same of 256..511
    kHighRead,
    kFullLow,   // latents 0..255 of the tile are dequantised (16 warps)
    kFullHigh,  // 256..511 (16 warps) and the rope part (2)
    kFreeLow,   // the output products of latents 0..255 are done
    kOutput,    // all of them: the rest of the rows and the weights are free
    kScores,    // the tile's scores are made
    kWeights,   // its weights are in shared memory and the scores read (16 warps)
    kQuery,     // the row of work's q is in place (16 warps)
    kDrain,
    kBars
};

template <int kN>
struct Layout {
    static constexpr int kQBlock = kN * 128;  // bytes of a [kN heads x 64] block
    static constexpr int kWeightRow = kN == 32 ? 64 : 128;  // bytes; with 16 heads there is room for padding
    static constexpr int kQ = 0;
    static constexpr int kRows = 9 * kQBlock;
    static constexpr int kRope = kRows + 8 * kBlock;
    static constexpr int kP = kRope + kBlock;
    static constexpr int kRaw = kP + kTile * kWeightRow;
    static constexpr int kBarsAt = kRaw + 2 * kRawHalf;
    static constexpr int kBytes = kBarsAt + 8 * kBars + 1024;  // the base is rounded up to 1024
    static constexpr uint32_t kColS = 4 * kN;
    static_assert(kRows % 1024 == 0 && kP % 1024 == 0, "swizzled blocks start on 1024 bytes");
};

struct Scratch {
    float* ml;         // [2 * ctas][2][kN] reference (base 2) and sum of a piece
    float* o;          // [2 * ctas][kN][512] its output
    float* ref;        // [rows of work][tiles][kN] the reference of a tile's weights
    __nv_bfloat16* p;  // [rows of work][tiles][128][kN] a tile's weights
};

__device__ __forceinline__ void shared_store16(uint32_t at, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}

__device__ __forceinline__ uint4 shared_load16(uint32_t at) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at));
    return v;
}
__device__ __forceinline__ uint32_t shared_load2(uint32_t at) {
    unsigned short v;
    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(at));
    return v;
}
__device__ __forceinline__ void copy16(uint32_t to, const void* from, bool there) {  // zeros where not there
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(there ? 16 : 0) : "memory");
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

// Floats in the order of signed integers, and back.
__device__ __forceinline__ int ordered(float x) {
    const int i = __float_as_int(x);
    return i ^ ((i >> 31) & 0x7fffffff);
}
__device__ __forceinline__ float unordered(int i) { return __int_as_float(i ^ ((i >> 31) & 0x7fffffff)); }

template <int kC>
__device__ __forceinline__ void load_shared(float (&v)[kC], const float* from) {
#pragma unroll
    for (int i = 0; i < kC; i += 4) {
        const float4 x = *reinterpret_cast<const float4*>(from + i);
        v[i] = x.x, v[i + 1] = x.y, v[i + 2] = x.z, v[i + 3] = x.w;
    }
}

// The weights of an entry and 2 kW heads, the part-th such group, into the entry's row of chunks of 8 heads:
// 128-byte rows, chunk ^ row % 8, or 64-byte rows, chunk ^ row / 2 % 4 ...
template <int kW>
__device__ __forceinline__ void store_weights(uint32_t base, int entry, int part, const uint32_t (&p)[kW]) {
    if constexpr (kW == 2) {
        const uint32_t to = base + entry * 128 + (((part >> 1) ^ (entry & 7)) << 4) + (part & 1) * 8;
        asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(to), "r"(p[0]), "r"(p[1]) : "memory");
    } else {
        shared_store16(base + entry * 64 + ((part ^ ((entry >> 1) & 3)) << 4), p[0], p[1], p[2], p[3]);
    }
}
// ... and to global memory.
template <int kW>
__device__ __forceinline__ void store_weights(__nv_bfloat16* to, const uint32_t (&p)[kW]) {
    if constexpr (kW == 2) *reinterpret_cast<uint2*>(to) = make_uint2(p[0], p[1]);
    else *reinterpret_cast<uint4*>(to) = make_uint4(p[0], p[1], p[2], p[3]);
}

__device__ __forceinline__ void workers_sync() { asm volatile("bar.sync 1, %0;" ::"n"(kWorkers) : "memory"); }

template <int kN>
__global__ void __launch_bounds__(kThreads, 1)
kv4_decode_kernel(const Operands op, const Division div, const Scratch scratch) {
    using L = Layout<kN>;
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint32_t s_tmem;
    __shared__ int s_dead;
    __shared__ __align__(16) float s_minus_ref[kN];  // minus the reference, base 2; +inf while there is none
    __shared__ __align__(16) float s_fade[kN];       // what a new reference multiplies sums and output by; later 1 / sum
    __shared__ int s_top[4][kN];                     // by quarters of the entries: maximum, or sum
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
    auto warp_arrive = [&](int which) {
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(bar(which));
    };

    if (tid == 0) {
        s_dead = 0;
        tc::mbar_init(bar(kFullLow), 16);
        tc::mbar_init(bar(kFullHigh), 16 + 2);
        tc::mbar_init(bar(kLowHere), 64);
        tc::mbar_init(bar(kLowRead), 16);
        tc::mbar_init(bar(kHighHere), 64);
        tc::mbar_init(bar(kHighRead), 16);
        tc::mbar_init(bar(kFreeLow), 1);
        tc::mbar_init(bar(kOutput), 1);
        tc::mbar_init(bar(kScores), 1);
        tc::mbar_init(bar(kWeights), 16);
        tc::mbar_init(bar(kQuery), 16);
        tc::mbar_init(bar(kDrain), 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 16) tc::tmem_alloc<512>(tc::smem_u32(&s_tmem));
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    // All columns, although few heads need fewer: they start at 0, whatever else runs on the SM, and the
    // addresses below are constants.
    if (tid == 0 && s_tmem != 0) *dead = 1;
    pdl_wait();

    const int32_t u0 = div.start(blockIdx.x), u1 = div.start(blockIdx.x + 1);
    const int tiles = div.tiles;

    if (warp == 16) {
        // ---- the products, all by one lane.  (The branch has to be that of elect.sync itself: with a plain
        // lane number, or its result kept, the issue of a product takes 80 cycles instead of 30.) ----
        if (tc::elect_one()) {
            constexpr uint32_t kDescS = tc::instruction(128, kN, false, false);
            constexpr uint32_t kDescO = tc::instruction(128, kN, true, true);
            const uint32_t desc_q = tc::operand(base + L::kQ, 0);
            const uint32_t desc_k = tc::operand(base + L::kRows, 0);
            const uint32_t desc_v = tc::operand(base + L::kRows, kBlock);
            const uint32_t desc_p = tc::operand(base + L::kP, 0);
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
                            tc::mma_ss<tc::operand_high(128), tc::operand_high(128)>(
                                L::kColS, desc_k + (4 * part + i) * (kBlock / 16) + 2 * k,
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
                        tc::mma_ss<tc::operand_high(128), tc::operand_high(L::kWeightRow)>(
                            t * kN, desc_v + t * (2 * kBlock / 16) + k * (2048 / 16), desc_p + k * L::kWeightRow, kDescO,
                            !first || k);
                    if (t == 1) tc::commit(bar(kFreeLow));
                }
                tc::commit(bar(kOutput));
            }
        }
        __syncwarp();
    } else if (warp > 16) {
        // ---- rows: asynchronous copies, a tile ahead; a warp 64 rows of it.  An entry that is not there copies
        // nothing and leaves zeros: finite values, whose weights are 0. ----
        const int row0 = (warp - 17) * 64;
        int32_t bits = 0;
        Walk at(div, u0);
        int token = at.row % op.tokens;
        int32_t slot[2];
        auto load_slots = [&] {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int e = at.tile * kTile + row0 + i * 32 + lane;
                slot[i] = at.u < u1 && e < op.topk ? __ldg(op.slots + token * op.slots_token + e) : kNotFound;
            }
        };
        load_slots();
        // 9 lanes a row and half: 8 chunks of nibbles, swizzled, and the scales
        const int lane_row = lane / 9, piece = lane - lane_row * 9;
        const uint32_t rope = base + L::kRope + (row0 + (lane >> 3)) * 128;
        const uint32_t count = u1 - u0;
        for (uint32_t n = 0; n < count; ++n) {
            const uint64_t pool = reinterpret_cast<uint64_t>(op.pool) + static_cast<uint64_t>(token) * op.pool_token;
            uint64_t from[2];
            uint32_t valid[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const bool there = slot[i] >= 0 && slot[i] < op.pool_rows;
                if (!there && slot[i] != kNotFound) bits |= ASU_ST_BAD_QUERY;
                valid[i] = __ballot_sync(0xffffffffu, there);
                from[i] = pool + static_cast<uint64_t>(there ? slot[i] : 0) * op.pool_pitch;
            }
            const int row = at.row;
            at.next(div);
            if (at.row != row && ++token == op.tokens) token = 0;
            load_slots();
#pragma unroll 1
            for (int half = 0; half < 2; ++half) {
                if (n >= 1) warp_wait(half ? kHighRead : kLowRead, n - 1);
                const uint32_t raw = base + L::kRaw + half * kRawHalf;
                const int offset = piece < 8 ? half * 128 + piece * 16 : kScaleOffset + half * 16;
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int r = 0; r < 33; r += 3) {
                        const int mine = r + lane_row;
                        const uint64_t src = __shfl_sync(0xffffffffu, from[i], mine & 31) + offset;
                        const int to_row = row0 + i * 32 + mine;
                        const uint32_t to = raw + (piece < 8 ? to_row * 128 + ((piece ^ (to_row & 7)) << 4)
                                                             : kTile * 128 + to_row * 16);
                        if (lane < 27 && mine < 32)
                            copy16(to, reinterpret_cast<const void*>(src), (valid[i] >> (mine & 31)) & 1u);
                    }
                asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar(half ? kHighHere : kLowHere))
                             : "memory");
            }
            if (n >= 1) warp_wait(kScores, n - 1);
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int r = 0; r < 32; r += 4) {  // 8 lanes a row, into the swizzled block
                    const int mine = r + (lane >> 3);
                    const uint64_t src = __shfl_sync(0xffffffffu, from[i], mine) + kRopeOffset + (lane & 7) * 16;
                    copy16(rope + (i * 32 + r) * 128 + (((lane ^ mine) & 7) << 4), reinterpret_cast<const void*>(src),
                           (valid[i] >> mine) & 1u);
                }
            asm volatile("cp.async.wait_all;" ::: "memory");
            tc::fence_async_shared();
            warp_arrive(kFullHigh);
        }
        if (bits) flag_status(op.status, 0, bits);
    } else {
        // ---- rows: lane = 8 q + 2 rr + lp has row rr of four, latents 32 * (2 q + lp) .. of either half.  Eight
        // consecutive lanes read and store four rows x two chunks: all banks, on both sides (a row is 72 words, 8
        // more than a multiple of 32, and the blocks are swizzled). ----
        const int quarter = lane >> 3, lp = lane & 1;
        const int row0 = warp * 4 + ((lane >> 1) & 3);  // and row0 + 64
        const int chunk = 2 * quarter + lp;
        const uint32_t raw = base + L::kRaw + row0 * 128 + ((chunk ^ (row0 & 7)) << 4);
        const uint32_t raw_scales = base + L::kRaw + kTile * 128 + row0 * 16 + chunk * 2;
        const uint32_t rows_at = base + L::kRows + quarter * kBlock + row0 * 128 + (((lp * 4) ^ (row0 & 7)) << 4);
        auto dequantise_half = [&](int half) {
            uint4 code[2];
            uint32_t scales[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                code[i] = shared_load16(raw + half * kRawHalf + i * 64 * 128);
                scales[i] = shared_load2(raw_scales + half * kRawHalf + i * 64 * 16);
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) dequantise(code[i], scales[i], rows_at + half * 4 * kBlock + i * 64 * 128);
            tc::fence_async_shared();
        };
        // ---- softmax: this thread's entry of the tile, and its warp's heads ----
        constexpr int kC = kN / 4;
        const int part = warp >> 2;   // heads part * kC ..; of the output, latents part * 128 ..
        const int entry = (warp & 3) * 32 + lane;
        const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
        float l[kC];  // the entries' weights by head
        // the row of work's q, zero for heads beyond the last: 8 lanes a block of a head
        auto copy_q = [&](int row) {
            const int token = row % op.tokens, head0 = row / op.tokens * kN;
            const int h = tid >> 3;
            if (h < kN) {
                const bool there = head0 + h < op.heads;
                const __nv_bfloat16* from = op.q + token * op.q_token + (there ? head0 + h : 0) * op.q_head + (tid & 7) * 8;
                const uint32_t to = base + L::kQ + h * 128 + (((tid ^ h) & 7) << 4);
                if (op.q_aligned || !there) {
#pragma unroll
                    for (int k = 0; k < 9; ++k) copy16(to + k * L::kQBlock, from + k * 64, there);
                } else {
#pragma unroll 1
                    for (int k = 0; k < 9; ++k) {
                        const uint4 v = load_unaligned(from + k * 64);
                        shared_store16(to + k * L::kQBlock, v.x, v.y, v.z, v.w);
                    }
                }
            }
        };

        Walk at(div, u0);
        int token = at.row % op.tokens;
        copy_q(at.row);
        auto slot_here = [&]() -> int32_t {
            const int e = at.tile * kTile + entry;
            return at.u < u1 && e < op.topk ? __ldg(op.slots + token * op.slots_token + e) : kNotFound;
        };
        int32_t slot = slot_here();
        for (uint32_t n = 0; at.u < u1; ++n) {
            const int row = at.row, tile = at.tile;
            const bool first = at.u == u0 || tile == 0;
            const bool last = at.u + 1 == u1 || tile + 1 == tiles;
            const bool there = slot >= 0 && slot < op.pool_rows;
#pragma unroll 1
            for (int half = 0; half < 2; ++half) {
                warp_wait(half ? kHighHere : kLowHere, n);
                if (n >= 1) warp_wait(half ? kOutput : kFreeLow, n - 1);
                dequantise_half(half);
                __syncwarp();
                if (lane == 0) {
                    tc::mbar_arrive(bar(half ? kFullHigh : kFullLow));
                    tc::mbar_arrive(bar(half ? kHighRead : kLowRead));
                }
            }
            if (first) {  // q is on its way since the piece before
                asm volatile("cp.async.wait_all;" ::: "memory");
                tc::fence_async_shared();
                warp_arrive(kQuery);
#pragma unroll
                for (int h = 0; h < kC; ++h) l[h] = 0.0f;
            }
            warp_wait(kScores, n);
            tc::fence_after();
            uint32_t s[kC];
            tc::tmem_load(lanes + L::kColS + part * kC, s);
            tc::tmem_wait_load(s);
            // does a score exceed its reference by too much?
            float minus_ref[kC];
            bool over = false;
            if (!first) {
                load_shared(minus_ref, s_minus_ref + part * kC);
#pragma unroll
                for (int h = 0; h < kC; ++h)
                    over |= fmaf(__uint_as_float(s[h]), op.scale_log2, minus_ref[h]) > kMaxGrowth;
                over &= there;
            }
            if (tc::any_of<kWorkers>(over || first)) {
                // new references: the maxima over the tile's entries, of this tile alone in a piece's first
#pragma unroll
                for (int h = 0; h < kC; ++h) {
                    const float x = there ? __uint_as_float(s[h]) * op.scale_log2 : -INFINITY;
                    const int top = __reduce_max_sync(0xffffffffu, ordered(x));
                    if (lane == h) s_top[warp & 3][part * kC + h] = top;
                }
                workers_sync();
                if (tid < kN) {
                    const float top = unordered(max(max(s_top[0][tid], s_top[1][tid]), max(s_top[2][tid], s_top[3][tid])));
                    // while all entries of a piece were missing there is no reference: +inf here, so that
                    // the next score of any size exceeds it
                    const float old = first ? INFINITY : s_minus_ref[tid];
                    const float now = fminf(old, -top);
                    s_fade[tid] = old == now ? 1.0f : old == INFINITY ? 0.0f : exp2_fast(now - old);
                    s_minus_ref[tid] = now;
                }
                workers_sync();
                load_shared(minus_ref, s_minus_ref + part * kC);
                if (!first) {
#pragma unroll
                    for (int h = 0; h < kC; ++h) l[h] *= s_fade[part * kC + h];
#pragma unroll 1
                    for (int c0 = 0; c0 < kN; c0 += 16) {
                        uint32_t o[16];
                        tc::tmem_load(lanes + part * kN + c0, o);
                        tc::tmem_wait_load(o);
#pragma unroll
                        for (int h = 0; h < 16; ++h) o[h] = __float_as_uint(__uint_as_float(o[h]) * s_fade[c0 + h]);
                        tc::tmem_store(lanes + part * kN + c0, o);
                    }
                    tc::tmem_wait_store();
                }
            }
            const int64_t unit = static_cast<int64_t>(row) * tiles + tile;
            uint32_t p[kC / 2];
#pragma unroll
            for (int h = 0; h < kC; h += 2) {
                float a = exp2_fast(fmaf(__uint_as_float(s[h]), op.scale_log2, minus_ref[h]));
                float b = exp2_fast(fmaf(__uint_as_float(s[h + 1]), op.scale_log2, minus_ref[h + 1]));
                a = there ? a : 0.0f;
                b = there ? b : 0.0f;
                l[h] += a;
                l[h + 1] += b;
                p[h / 2] = pack_bf16(a, b);
            }
            store_weights(base + L::kP, entry, part, p);
            tc::fence_async_shared();
            tc::fence_before();
            warp_arrive(kWeights);
            if (op.weights != nullptr) {
                store_weights(scratch.p + (unit * kTile + entry) * kN + part * kC, p);
                if (entry < kC) scratch.ref[unit * kN + part * kC + entry] = -s_minus_ref[part * kC + entry];
            }
            at.next(div);
            const int was = token;
            if (at.row != row && ++token == op.tokens) token = 0;
            slot = slot_here();
            if (last) {
                // this row's scores are all made: the next one's q comes beside the output products
                if (at.u < u1) copy_q(at.row);
                // sums over the entries: within the warps, then the four quarters
#pragma unroll
                for (int h = 0; h < kC; ++h) {
                    float x = l[h];
#pragma unroll
                    for (int d = 16; d > 0; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
                    if (lane == h) s_top[warp & 3][part * kC + h] = __float_as_int(x);
                }
                workers_sync();
                const int head0 = row / op.tokens * kN;
                const int row_start = row * tiles;
                const bool whole = row_start >= u0 && row_start + tiles <= u1;
                const int piece = div.piece(blockIdx.x, row_start);
                if (tid < kN) {
                    const float sum = (__int_as_float(s_top[0][tid]) + __int_as_float(s_top[1][tid])) +
                                      (__int_as_float(s_top[2][tid]) + __int_as_float(s_top[3][tid]));
                    if (whole) {
                        s_fade[tid] = sum > 0.0f ? 1.0f / sum : 0.0f;
                        if (head0 + tid < op.heads)
                            op.lse[static_cast<int64_t>(was) * op.heads + head0 + tid] =
                                sum > 0.0f ? (log2f(sum) - s_minus_ref[tid]) * 0.6931471805599453f : -INFINITY;
                    } else {
                        scratch.ml[piece * 2 * kN + tid] = sum > 0.0f ? -s_minus_ref[tid] : -INFINITY;
                        scratch.ml[(piece * 2 + 1) * kN + tid] = sum;
                    }
                }
                workers_sync();
                warp_wait(kOutput, n);
                tc::fence_after();
                const int latent = part * 128 + entry;
                __nv_bfloat16* out = op.out + (static_cast<int64_t>(was) * op.heads + head0) * kLatent + latent;
                float* partial = scratch.o + static_cast<int64_t>(piece) * kN * kLatent + latent;
#pragma unroll 1
                for (int c0 = 0; c0 < kN; c0 += 16) {
                    uint32_t o[16];
                    tc::tmem_load(lanes + part * kN + c0, o);
                    tc::tmem_wait_load(o);
#pragma unroll
                    for (int h = 0; h < 16; ++h) {
                        if (!whole) partial[(c0 + h) * kLatent] = __uint_as_float(o[h]);
                        else if (head0 + c0 + h < op.heads)
                            out[(c0 + h) * kLatent] = __float2bfloat16(__uint_as_float(o[h]) * s_fade[c0 + h]);
                    }
                }
                tc::fence_before();
            }
        }
    }
    pdl_trigger();
    __syncthreads();
    if (s_dead && tid == 0) flag_status(op.status, 0, ASU_ST_TIMEOUT);
    if (warp == 16) {
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

// Joins the pieces of rows that several CTAs share, and sums the weights over the heads.
//   blocks y < heads: one head of a token, 4 latents a thread
//   other blocks:     one tile, an entry a thread: weights_j = sum_h p_hj 2^(ref_h - lse_h)
template <int kN>
__global__ void __launch_bounds__(128)
kv4_finish_kernel(const Operands op, const Division div, const Scratch scratch) {
    pdl_wait();
    pdl_trigger();
    __shared__ float s_factor[ASU_KV4_MAX_HEADS];
    const int token = blockIdx.x, tid = threadIdx.x;
    // reference and sum (base 2) of a head over its pieces; the CTAs of its row
    auto total = [&](int head, int& i0, int& i1, float& m, float& l) {
        const int first = (head / kN * op.tokens + token) * div.tiles;
        i0 = div.cta_of(first);
        i1 = div.cta_of(first + div.tiles - 1);
        if (i0 == i1) return;
        m = -INFINITY, l = 0.0f;
#pragma unroll 4
        for (int i = i0; i <= i1; ++i) m = fmaxf(m, scratch.ml[div.piece(i, first) * 2 * kN + head % kN]);
#pragma unroll 4
        for (int i = i0; i <= i1; ++i) {
            const float* ml = scratch.ml + div.piece(i, first) * 2 * kN + head % kN;
            l += ml[kN] * (ml[0] == -INFINITY ? 0.0f : exp2_fast(ml[0] - m));
        }
    };
    if (static_cast<int>(blockIdx.y) < op.heads) {
        const int head = blockIdx.y;
        int i0, i1;
        float m, l;
        total(head, i0, i1, m, l);
        if (i0 == i1) return;  // written by its one CTA
        const int first = (head / kN * op.tokens + token) * div.tiles;
        float4 acc = make_float4(0, 0, 0, 0);
#pragma unroll 4
        for (int i = i0; i <= i1; ++i) {
            const int piece = div.piece(i, first);
            const float pm = scratch.ml[piece * 2 * kN + head % kN];
            const float f = pm == -INFINITY ? 0.0f : exp2_fast(pm - m);
            const float4 v =
                reinterpret_cast<const float4*>(scratch.o + (static_cast<int64_t>(piece) * kN + head % kN) * kLatent)[tid];
            acc.x += v.x * f, acc.y += v.y * f, acc.z += v.z * f, acc.w += v.w * f;
        }
        const float inv = l > 0.0f ? 1.0f / l : 0.0f;
        reinterpret_cast<uint2*>(op.out + (static_cast<int64_t>(token) * op.heads + head) * kLatent)[tid] =
            make_uint2(pack_bf16(acc.x * inv, acc.y * inv), pack_bf16(acc.z * inv, acc.w * inv));
        if (tid == 0)
            op.lse[static_cast<int64_t>(token) * op.heads + head] =
                l > 0.0f ? (m + log2f(l)) * 0.6931471805599453f : -INFINITY;
        return;
    }
    const int tile = blockIdx.y - op.heads;
    const int parts = (op.heads + kN - 1) / kN;
    for (int head = tid; head < parts * kN; head += 128) {  // the joining blocks may not have written lse yet
        float f = 0.0f;
        if (head < op.heads) {
            int i0, i1;
            float m, l;
            total(head, i0, i1, m, l);
            const float lse = i0 == i1 ? op.lse[static_cast<int64_t>(token) * op.heads + head] * 1.4426950408889634f
                                       : (l > 0.0f ? m + log2f(l) : -INFINITY);
            const int64_t unit = static_cast<int64_t>(head / kN * op.tokens + token) * div.tiles + tile;
            if (lse != -INFINITY) f = exp2_fast(scratch.ref[unit * kN + head % kN] - lse);
        }
        s_factor[head] = f;
    }
    __syncthreads();
    const int e = tile * kTile + tid;
    if (e >= op.topk) return;
    float w = 0.0f;
    for (int part = 0; part < parts; ++part) {
        const int64_t unit = static_cast<int64_t>(part * op.tokens + token) * div.tiles + tile;
        const uint4* p = reinterpret_cast<const uint4*>(scratch.p + (unit * kTile + tid) * kN);
#pragma unroll
        for (int i = 0; i < kN / 8; ++i) {
            const uint4 v = __ldg(p + i);
            const uint32_t x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                w = fmaf(__uint_as_float(x[k] << 16), s_factor[part * kN + i * 8 + 2 * k], w);
                w = fmaf(__uint_as_float(x[k] & 0xffff0000u), s_factor[part * kN + i * 8 + 2 * k + 1], w);
            }
        }
    }
    op.weights[static_cast<int64_t>(token) * op.topk + e] = __float2bfloat16(w);
}

int64_t align256(int64_t x) { return (x + 255) / 256 * 256; }

int columns_of(int64_t heads) { return heads <= 16 ? 16 : 32; }

Division division(int64_t tokens, int64_t heads, int64_t topk, int sms) {
    const int n = columns_of(heads);
    return Division((heads + n - 1) / n * tokens, topk > 0 ? (topk + kTile - 1) / kTile : 1, sms);
}

void layout(const Division& d, int n, bool weights, int64_t (&at)[5]) {
    const int64_t units = static_cast<int64_t>(d.rows) * d.tiles;
    at[0] = 0;
    at[1] = at[0] + align256(2ll * d.ctas * 2 * n * 4);
    at[2] = at[1] + align256(2ll * d.ctas * n * kLatent * 4);
    at[3] = at[2] + (weights ? align256(units * n * 4) : 0);
    at[4] = at[3] + (weights ? units * kTile * n * 2 : 0);
}

template <int kN>
int launch(cudaStream_t s, const Operands& op, void* workspace) {
    const Division d = division(op.tokens, op.heads, op.topk, asu_sm_count());
    int64_t at[5];
    layout(d, kN, op.weights != nullptr, at);
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    const Scratch scratch = {reinterpret_cast<float*>(ws + at[0]), reinterpret_cast<float*>(ws + at[1]),
                             reinterpret_cast<float*>(ws + at[2]), reinterpret_cast<__nv_bfloat16*>(ws + at[3])};
    int max_dynamic = 0;
    int rc = asu_max_dynamic_smem(reinterpret_cast<const void*>(kv4_decode_kernel<kN>), &max_dynamic);
    if (rc != ASU_OK) return rc;
    if (max_dynamic < Layout<kN>::kBytes) return ASU_ERR_ARG;
    rc = launch_pdl(kv4_decode_kernel<kN>, dim3(d.ctas), dim3(kThreads), Layout<kN>::kBytes, s, op, d, scratch);
    bool shared_rows = false;  // does any row lie in several CTAs' ranges?
    for (int i = 1; i < d.ctas && !shared_rows; ++i) shared_rows = d.start(i) % d.tiles != 0;
    if (rc != ASU_OK || (!shared_rows && op.weights == nullptr)) return rc;
    return launch_pdl(kv4_finish_kernel<kN>,
                      dim3(static_cast<unsigned>(op.tokens),
                           static_cast<unsigned>(op.heads + (op.weights != nullptr ? d.tiles : 0))),
                      dim3(128), 0, s, op, d, scratch);
}

}  // namespace

int64_t decode_workspace(int64_t tokens, int64_t heads, int64_t topk, bool weights) {
    int64_t at[5];
    layout(division(tokens, heads, topk, asu_sm_count()), columns_of(heads), weights, at);
    return at[4];
}

int launch_decode(cudaStream_t s, const Operands& op, void* workspace) {
    return columns_of(op.heads) == 16 ? launch<16>(s, op, workspace) : launch<32>(s, op, workspace);
}

}  // namespace kv4
}  // namespace asu

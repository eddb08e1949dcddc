// Sparse decode attention over the 4-bit cache for more than 64 heads, on the tcgen05 tensor cores.
#include "kv4_decode.cuh"
#include "tcgen05.cuh"

namespace asu {
namespace kv4 {
namespace {

// 128 rows of heads (padded) x 64 entries a tile.  A CTA makes 256 of the 512 output columns, since
// all 512 in 32 bits would fill the tensor memory and leave no room for the scores; the two CTAs of a
// token each compute the scores (1.5 times the products of a scheme that shares them, but no
// exchange between SMs).
//
// Tensor memory, 512 columns: output 256, scores 64, their weights as bf16 pairs 32, and q's latents
// 256..511 and rope part, bf16 pairs, 160.
// Shared memory, 221 KB: q's latents 0..255, 64 KB; two tiles of 4-bit rows, 52 KB; and dequantised rows
// as blocks of [64 entries x 64 values] in the 128-byte swizzle.  A block serves both products: entries
// x values with the values contiguous is K-major for the scores and MN-major for the output.
// "Part A", the other half's four blocks and the rope block, only the scores read; it is free again
// when its products of this tile are done, a thousand cycles before those of the next begin, and needs
// no second copy.  "Part B", the four blocks of this half, is held until the output product: two copies.
//
// 15 warps: 4 for the softmax, a thread a head (its row of scores lies in its tensor memory lane, so
// there is no exchange); 8 that dequantise; one that issues the products; two that fetch rows.  (Rows
// through registers instead made 8 KB of straight-line code and 5500 cycles a tile: the scoreboards wait
// for all loads in flight, and the instruction caches did not keep up.)
// The products of tile n's scores run while the softmax works on tile n - 1.
//
// The running maximum only moves when it grows by more than 2^8: until then the weights stay below
// 2^8, as exact in bf16 as any others, and the output needs no rescaling.
//
// The two CTAs of a pair walk the same tiles, so that the rows' second reading finds them in L2.
//
// 128 tokens x 128 heads x 2048 entries take 139 us, with weights 162 (inputs in rotation, none in L2; 120 and 150 where
// the same rows are read again).  There a tile takes 1.7 us, in which the
// issuing lane waits for the products and for nothing else: they would take 1.0 alone, but the traffic of shared
// memory is 1.3 (q read again for every tile 0.4, rows dequantised 0.3 and read 0.4, 4-bit rows in and out 0.2).
// A change of tokens takes 4 us (the next q's 147 KB, the output through the lanes), the start 5, the joining of
// the pieces 9, with the weights' way through memory and back 23.
constexpr int kTile = 64;  // entries a tile
constexpr int kWideThreads = 15 * 32;
constexpr int kBlock = kTile * 128;  // bytes of a [64 x 64] bf16 block
constexpr int kQBlock = 128 * 128;   // bytes of a [128 x 64] bf16 block
constexpr int kRawTile = kTile * kRowBytes;
constexpr int kSmemQ = 0;
constexpr int kSmemA = kSmemQ + 4 * kQBlock;
constexpr int kSmemB = kSmemA + 5 * kBlock;
constexpr int kSmemRaw = kSmemB + 2 * 4 * kBlock;
constexpr int kSmemBars = kSmemRaw + 2 * kRawTile;
constexpr int kWideSmem = kSmemBars + 128 + 1024;  // the base is rounded up to 1024
constexpr uint32_t kColO = 0, kColS = 256, kColP = 320, kColQ = 352;
constexpr float kMaxGrowth = 8.0f;

// Barriers.  One of a pair is that of the even tiles.  Where a waiter may be a phase behind the
// barrier's other users there is a pair; single ones are waited for in every phase by someone that
// the next phase depends on.
enum Bar {
    kRowsHere = 0,   // pair: the tile's 4-bit rows are in shared memory (64 threads' copies)
    kRowsRead = 2,   // pair: and have been read (8 warps)
    kFullB = 4,      // pair: part B is dequantised (8 warps)
    kOutput = 6,     // pair: the tile's output product is done: its part B and weights are free
    kFullA = 8,      // part A is dequantised (8 warps)
    kFreeA = 9,      // and its products are done
    kScores = 10,    // the tile's scores are made
    kScoresRead = 11,  // and have been read (128 threads)
    kWeights = 12,   // the tile's weights are in tensor memory (128 threads)
    kQuery = 13,     // the token's q is in place (128 threads)
    kDrain = 14,
    kBars = 15
};

struct Scratch {
    float* ml;         // [2 * pairs][2 halves][2][128] running maximum (base 2) and sum of a piece
    float* o;          // [2 * pairs][2 halves][256][128] its output, columns by heads
    float* ref;        // [tokens][tiles][128] the maximum that a tile's weights are relative to
    uint32_t* p;       // [tokens][tiles][32][128] a tile's weights, pairs of entries
};

__device__ __forceinline__ uint4 shared_load16(uint32_t at) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at));
    return v;
}
// A whole sector of a thread's own: nothing is gained by another thread's stores next to it.
__device__ __forceinline__ void store32(void* to, const uint32_t (&w)[8]) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to), "r"(w[0]), "r"(w[1]), "r"(w[2]),
                 "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
}
__device__ __forceinline__ uint32_t shared_load2(uint32_t at) {
    unsigned short v;
    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(at));
    return v;
}
__global__ void __launch_bounds__(kWideThreads, 1)
kv4_decode_wide_kernel(const Operands op, const Division div, const Scratch scratch) {
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint32_t s_tmem;
    __shared__ int s_dead;
    const uint32_t base = (tc::smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t bars = base + kSmemBars;
    auto bar = [&](int which) { return bars + 8u * which; };
    auto bar2 = [&](int which, uint32_t n) { return bars + 8u * (which + (n & 1)); };
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    volatile int* dead = &s_dead;
    // A wait that runs out sets the flag, and then no other one waits: every loop goes through to its end, on
    // whatever the buffers hold, so that each barrier is met by all; the status says that it happened.
    auto warp_wait = [&](uint32_t b, uint32_t parity) {
        tc::mbar_wait(b, parity & 1, dead);
        __syncwarp();
    };

    if (tid == 0) {
        s_dead = 0;
        for (int i = 0; i < 2; ++i) {
            tc::mbar_init(bar(kRowsHere + i), 64);
            tc::mbar_init(bar(kRowsRead + i), 8);
            tc::mbar_init(bar(kFullB + i), 8);
            tc::mbar_init(bar(kOutput + i), 1);
        }
        tc::mbar_init(bar(kFullA), 8);
        tc::mbar_init(bar(kFreeA), 1);
        tc::mbar_init(bar(kScores), 1);
        tc::mbar_init(bar(kScoresRead), 128);
        tc::mbar_init(bar(kWeights), 128);
        tc::mbar_init(bar(kQuery), 128);
        tc::mbar_init(bar(kDrain), 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 12) tc::tmem_alloc<512>(tc::smem_u32(&s_tmem));
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    // all columns are this block's: they start at 0, and the addresses below are constants
    if (tid == 0 && s_tmem != 0) *dead = 1;
    pdl_wait();

    const int half = blockIdx.x & 1;  // of the output columns
    const int32_t u0 = div.start(blockIdx.x >> 1), u1 = div.start((blockIdx.x >> 1) + 1);
    const int tiles = div.tiles;

    if (warp >= 4 && warp < 12) {
        // ---- 4-bit rows -> dequantised blocks ----
        // lane = 8 q + 2 rr + lp: row rr of four, latents 32 * (2 q + lp) .. of either half.  Eight
        // consecutive lanes read and store four rows x two chunks: all banks, on both sides (a row is 104
        // words, 8 more than a multiple of 32, and the blocks are swizzled).
        const int quarter = lane >> 3, lp = lane & 1;
        const int row0 = (warp - 4) * 4 + ((lane >> 1) & 3);  // and row0 + 32
        const uint32_t chunk = 2 * quarter + lp;
        const uint32_t raw_at = base + kSmemRaw + row0 * kRowBytes;
        const uint32_t chunk_at = quarter * kBlock + row0 * 128 + (((lp * 4) ^ (row0 & 7)) << 4);
        const uint32_t rope_chunk = lp * 4 + quarter;
        const uint32_t rope_at = base + kSmemA + 4 * kBlock + row0 * 128 + ((rope_chunk ^ (row0 & 7)) << 4);
        uint32_t n = 0;
        for (Walk at(div, u0); at.u < u1; at.next(div), ++n) {
            const uint32_t raw = raw_at + (n & 1) * kRawTile;
            const uint32_t mine = half ? 8 : 0, other = 8 - mine;  // chunks before this half's
            warp_wait(bar2(kRowsHere, n), n >> 1);
            if (n >= 1) warp_wait(bar(kFreeA), n - 1);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint32_t from = raw + i * 32 * kRowBytes;
                const uint4 code = shared_load16(from + (other + chunk) * 16);
                const uint32_t scales = shared_load2(from + kScaleOffset + (other + chunk) * 2);
                const uint4 rope = shared_load16(from + kRopeOffset + rope_chunk * 16);
                shared_store16(rope_at + i * 32 * 128, rope.x, rope.y, rope.z, rope.w);
                dequantise(code, scales, base + kSmemA + chunk_at + i * 32 * 128);
            }
            tc::fence_async_shared();
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(bar(kFullA));
            if (n >= 2) warp_wait(bar2(kOutput, n), (n >> 1) - 1);
            const uint32_t part_b = base + kSmemB + (n & 1) * 4 * kBlock;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint32_t from = raw + i * 32 * kRowBytes;
                const uint4 code = shared_load16(from + (mine + chunk) * 16);
                const uint32_t scales = shared_load2(from + kScaleOffset + (mine + chunk) * 2);
                dequantise(code, scales, part_b + chunk_at + i * 32 * 128);
            }
            tc::fence_async_shared();
            __syncwarp();
            if (lane == 0) {
                tc::mbar_arrive(bar2(kFullB, n));
                tc::mbar_arrive(bar2(kRowsRead, n));
            }
        }
    } else if (warp >= 13) {
        // ---- rows: asynchronous copies, two tiles ahead; slots three.  32 rows of a tile a warp, 26 lanes a
        // row.  (One bulk copy a row took 40 ns each and was the bound.) ----
        const int row0 = (warp - 13) * 32;
        int32_t bits = 0;
        auto slot_of = [&](const Walk& w) -> int32_t {
            const int e = w.tile * kTile + row0 + lane;
            if (w.u >= u1 || e >= op.topk) return kNotFound;
            return __ldg(op.slots + w.row * op.slots_token + e);
        };
        Walk at(div, u0);
        int32_t slot = slot_of(at);
        const uint32_t raw_at = base + kSmemRaw + row0 * kRowBytes + lane * 16;
        for (uint32_t n = 0; at.u < u1; ++n) {
            // an entry that is not there copies nothing and leaves zeros: finite values, whose weights are 0
            const bool there = slot >= 0 && slot < op.pool_rows;
            if (!there && slot != kNotFound) bits |= ASU_ST_BAD_QUERY;
            const uint64_t from = reinterpret_cast<uint64_t>(op.pool) +
                                  static_cast<uint64_t>(at.row) * op.pool_token +
                                  static_cast<uint64_t>(there ? slot : 0) * op.pool_pitch;
            const uint32_t valid = __ballot_sync(0xffffffffu, there);
            at.next(div);
            slot = slot_of(at);
            if (n >= 2) warp_wait(bar2(kRowsRead, n), (n >> 1) - 1);
            const uint32_t to = raw_at + (n & 1) * kRawTile;
#pragma unroll 8
            for (int r = 0; r < 32; ++r) {
                const uint64_t src = __shfl_sync(0xffffffffu, from, r) + lane * 16;
                if (lane < kRowBytes / 16)
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + r * kRowBytes), "l"(src),
                                 "r"((valid >> r) & 1u ? 16 : 0)
                                 : "memory");
            }
            asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar2(kRowsHere, n)) : "memory");
        }
        // no copy may land after this block has ended, whatever way the loops were left
        asm volatile("cp.async.wait_all;" ::: "memory");
        if (bits) flag_status(op.status, 0, bits);
    } else if (warp == 12) {
        // ---- the products, all by one lane.  (The branch has to be that of elect.sync itself: with a plain
        // lane number, or its result kept, the issue of a product takes 80 cycles instead of 30.) ----
        if (tc::elect_one()) {
            constexpr uint32_t kDescS = tc::instruction(128, kTile, false, false);
            constexpr uint32_t kDescO = tc::instruction(128, 256, false, true);
            const uint32_t desc_q = tc::operand(base + kSmemQ, 0);
            const uint32_t desc_a = tc::operand(base + kSmemA, 0);
            const uint32_t desc_b = tc::operand(base + kSmemB, 0);
            const uint32_t desc_v = tc::operand(base + kSmemB, kBlock);
            auto wait = [&](uint32_t b, uint32_t parity) { tc::mbar_wait(b, parity & 1, dead); };
            // four blocks of latents with q's 0..255 (shared memory) or 256..511 (tensor memory)
            auto low = [&](uint32_t rows) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        tc::mma_ss(kColS, desc_q + i * (kQBlock / 16) + 2 * k, rows + i * (kBlock / 16) + 2 * k, kDescS, 1);
            };
            auto high = [&](uint32_t rows) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        tc::mma_ts(kColS, kColQ + i * 32 + 8 * k, rows + i * (kBlock / 16) + 2 * k, kDescS, 1);
            };
            auto output = [&](uint32_t n, bool accumulate) {
                wait(bar(kWeights), n);
                tc::fence_after();
                const uint32_t v = desc_v + (n & 1) * (4 * kBlock / 16);
#pragma unroll
                for (int k = 0; k < kTile / 16; ++k)
                    tc::mma_ts(kColO, kColP + 8 * k, v + k * (2048 / 16), kDescO, accumulate || k > 0);
                tc::commit(bar2(kOutput, n));
            };
            uint32_t n = 0, segment = 0;
            bool before_first = true;  // was tile n - 1 the first of its piece?
            for (Walk at(div, u0); at.u < u1; at.next(div), ++n) {
                const bool first = at.u == u0 || at.tile == 0;
                if (first) {
                    // the token before is finished first: its weights do not depend on this one's q
                    if (n > 0) output(n - 1, !before_first);
                    wait(bar(kQuery), segment++);
                }
                if (n >= 1) wait(bar(kScoresRead), n - 1);
#pragma unroll 1
                for (int part = 0; part < 2; ++part) {
                    if (part) wait(bar2(kFullB, n), n >> 1);
                    else wait(bar(kFullA), n);
                    tc::fence_after();
                    const uint32_t rows = part ? desc_b + (n & 1) * (4 * kBlock / 16) : desc_a;
                    if (!part) {
#pragma unroll
                        for (int k = 0; k < 4; ++k)  // rope; the tile's first product overwrites
                            tc::mma_ts(kColS, kColQ + 4 * 32 + 8 * k, rows + 4 * (kBlock / 16) + 2 * k, kDescS, k > 0);
                    }
                    if ((half != 0) == (part == 0)) low(rows);
                    else high(rows);
                    tc::commit(part ? bar(kScores) : bar(kFreeA));
                }
                if (!first) output(n - 1, !before_first);
                before_first = first;
                if (at.u + 1 == u1) output(n, !first);
            }
        }
        __syncwarp();
    } else {
        // ---- softmax, a thread a head ----
        const uint32_t lanes = static_cast<uint32_t>(warp * 32) << 16;
        const int head = tid;
        auto softmax_sync = [] { asm volatile("bar.sync 1, 128;" ::: "memory"); };  // these four warps
        // A token's q, zero for heads beyond the last.  Its latents 256..511 pass through the shared blocks of
        // 0..255 on their way to tensor memory, so that every load is of whole lines: with a thread a head
        // they took 6 us a token.  Every score of the token before must have been made.
        auto load_q = [&](int32_t token) {
            const __nv_bfloat16* q = op.q + token * op.q_token;
            const bool mine_there = head < op.heads;
            const __nv_bfloat16* mine = q + (mine_there ? head : 0) * op.q_head + kLatent;
            uint4 rope[8];
            if (op.q_aligned) {
#pragma unroll
                for (int k = 0; k < 8; ++k) rope[k] = __ldg(reinterpret_cast<const uint4*>(mine) + k);
            } else {
#pragma unroll 1
                for (int k = 0; k < 8; ++k) {
                    const uint4 v = load_unaligned(mine + k * 8);
                    shared_store16(base + kSmemQ + head * 128 + k * 16, v.x, v.y, v.z, v.w);
                }
#pragma unroll
                for (int k = 0; k < 8; ++k) rope[k] = shared_load16(base + kSmemQ + head * 128 + k * 16);
                softmax_sync();
            }
            const uint32_t to0 = base + kSmemQ + (tid >> 3) * 128 + (((tid ^ (tid >> 3)) & 7) << 4);
#pragma unroll 1
            for (int first = 256; first >= 0; first -= 256) {
                const __nv_bfloat16* from = q + (tid >> 3) * op.q_head + first + (tid & 7) * 8;
#pragma unroll 1
                for (int h = tid >> 3, i = 0; i < 8; ++i, h += 16, from += 16 * op.q_head) {
                    const bool there = h < op.heads;
                    const __nv_bfloat16* src = there ? from : q;  // not read where not there
                    const uint32_t to = to0 + i * 16 * 128;
                    if (op.q_aligned || !there) {
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + k * kQBlock),
                                         "l"(src + k * 64), "r"(there ? 16 : 0)
                                         : "memory");
                    } else {
#pragma unroll 1
                        for (int k = 0; k < 4; ++k) {
                            const uint4 v = load_unaligned(from + k * 64);
                            shared_store16(to + k * kQBlock, v.x, v.y, v.z, v.w);
                        }
                    }
                }
                asm volatile("cp.async.wait_all;" ::: "memory");
                if (first == 0) break;
                softmax_sync();
#pragma unroll 1
                for (int i = 0; i < 5; ++i) {
                    uint32_t w[32];
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        uint4 v = mine_there ? rope[k] : make_uint4(0, 0, 0, 0);
                        if (i < 4) v = shared_load16(base + kSmemQ + i * kQBlock + head * 128 + ((k ^ (head & 7)) << 4));
                        w[4 * k] = v.x;
                        w[4 * k + 1] = v.y;
                        w[4 * k + 2] = v.z;
                        w[4 * k + 3] = v.w;
                    }
                    tc::tmem_store(lanes + kColQ + i * 32, w);
                }
                softmax_sync();
            }
            tc::fence_async_shared();
            tc::tmem_wait_store();
            tc::fence_before();
            tc::mbar_arrive(bar(kQuery));
        };
        float m = -INFINITY;
        uint64_t l2 = 0;  // the sum of the even and of the odd entries
        Walk at(div, u0);
        load_q(at.row);
        for (uint32_t n = 0; at.u < u1; at.next(div), ++n) {
            const int64_t token = at.row;
            const int tile = at.tile;
            const bool first = at.u == u0 || tile == 0;
            const bool last = at.u + 1 == u1 || tile + 1 == tiles;
            if (first) {
                m = -INFINITY;
                l2 = 0;
                // the next token's q to L2: its loads come between two tokens, where nothing hides them
                const int32_t next = (at.row + 1) * tiles;
                if (next < u1 && head < op.heads) {
                    const __nv_bfloat16* q = op.q + (token + 1) * op.q_token + head * op.q_head;
#pragma unroll
                    for (int k = 0; k < kDim; k += 64) asm volatile("prefetch.global.L2 [%0];" ::"l"(q + k));
                }
            }
            // which entries are there
            uint32_t there[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int e = tile * kTile + 32 * i + lane;
                const int32_t s = e < op.topk ? __ldg(op.slots + token * op.slots_token + e) : kNotFound;
                there[i] = __ballot_sync(0xffffffffu, s >= 0 && s < op.pool_rows);
            }
            warp_wait(bar(kScores), n);
            tc::fence_after();
            uint32_t s[2][32];
            tc::tmem_load(lanes + kColS, s[0]);
            tc::tmem_load(lanes + kColS + 32, s[1]);
            tc::tmem_wait_load(s[0]);
            tc::tmem_wait_load(s[1]);
            tc::fence_before();
            tc::mbar_arrive(bar(kScoresRead));
            if ((there[0] & there[1]) != 0xffffffffu) {
#pragma unroll
                for (int i = 0; i < 64; ++i)
                    if (!((there[i / 32] >> (i % 32)) & 1u)) s[i / 32][i % 32] = 0xff800000u;  // -inf
            }
            float top = -INFINITY;
#pragma unroll
            for (int i = 0; i < 64; ++i) top = fmaxf(top, __uint_as_float(s[i / 32][i % 32]));
            top *= op.scale_log2;
            float fade = 1.0f;
            if (first) {
                m = top;
            } else if (top > m + kMaxGrowth) {
                fade = exp2_fast(m - top);
                m = top;
            }
            const float from = m == -INFINITY ? 0.0f : m;
            // the output product before has read the weights there
            if (n >= 1) warp_wait(bar2(kOutput, n - 1), (n - 1) >> 1);
            tc::fence_after();
            if (__any_sync(0xffffffffu, fade != 1.0f)) {
                float a, b;
                unpair(l2, a, b);
                l2 = pair(a * fade, b * fade);
#pragma unroll 1
                for (int c = 0; c < 256; c += 32) {
                    uint32_t o[32];
                    tc::tmem_load(lanes + kColO + c, o);
                    tc::tmem_wait_load(o);
#pragma unroll
                    for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * fade);
                    tc::tmem_store(lanes + kColO + c, o);
                }
            }
            const uint64_t scale2 = pair(op.scale_log2, op.scale_log2);
            const uint64_t from2 = pair(-from, -from);
            // rounded to bf16, as the tensor cores take them beside bf16 rows (2^-8 of each at most, averaged out by the
            // sums); their sum takes them before the rounding
            uint32_t p[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) {
                const float x = __uint_as_float(s[i / 16][2 * i % 32]), y = __uint_as_float(s[i / 16][(2 * i + 1) % 32]);
                float a, b;
                unpair(fma2(pair(x, y), scale2, from2), a, b);
                a = exp2_fast(a);
                b = exp2_fast(b);
                l2 = add2(l2, pair(a, b));
                p[i] = pack_bf16(a, b);
            }
            tc::tmem_store(lanes + kColP, p);
            tc::tmem_wait_store();
            tc::fence_before();
            tc::mbar_arrive(bar(kWeights));
            if (op.weights != nullptr && half == 0) {
                const int64_t to = token * tiles + tile;
                scratch.ref[to * 128 + head] = m;
#pragma unroll
                for (int i = 0; i < 32; ++i) scratch.p[(to * 32 + i) * 128 + head] = p[i];
            }
            if (last) {
                // a token's scores are all made: the next one's q, whose first scores then run
                // beside what follows here
                if (at.u + 1 < u1) load_q(token + 1);
                float l, odd;
                unpair(l2, l, odd);
                l += odd;
                warp_wait(bar2(kOutput, n), n >> 1);
                tc::fence_after();
                const int32_t row_start = at.row * tiles;
                const bool whole = row_start >= u0 && row_start + tiles <= u1;
                if (whole) {
                    const float inv = l != 0.0f ? 1.0f / l : 0.0f;  // a NaN goes on
                    __nv_bfloat16* out = op.out + (token * op.heads + head) * kLatent + half * 256;
#pragma unroll 1
                    for (int c = 0; c < 256; c += 32) {
                        uint32_t o[32];
                        tc::tmem_load(lanes + kColO + c, o);
                        tc::tmem_wait_load(o);
                        if (head < op.heads) {
#pragma unroll
                            for (int i = 0; i < 2; ++i) {
                                uint32_t w[8];
#pragma unroll
                                for (int k = 0; k < 8; ++k)
                                    w[k] = pack_bf16(__uint_as_float(o[16 * i + 2 * k]) * inv,
                                                     __uint_as_float(o[16 * i + 2 * k + 1]) * inv);
                                store32(out + c + 16 * i, w);
                            }
                        }
                        __syncwarp();
                    }
                    if (half == 0 && head < op.heads)
                        op.lse[token * op.heads + head] =
                            l != 0.0f ? (m + log2f(l)) * 0.6931471805599453f : -INFINITY;
                } else {
                    const int piece = div.piece(blockIdx.x >> 1, row_start) * 2 + half;
                    float* to = scratch.o + static_cast<int64_t>(piece) * 256 * 128 + head;
#pragma unroll 1
                    for (int c = 0; c < 256; c += 32) {
                        uint32_t o[32];
                        tc::tmem_load(lanes + kColO + c, o);
                        tc::tmem_wait_load(o);
#pragma unroll
                        for (int i = 0; i < 32; ++i) to[(c + i) * 128] = __uint_as_float(o[i]);
                    }
                    scratch.ml[piece * 256 + head] = m;
                    scratch.ml[piece * 256 + 128 + head] = l;
                }
                tc::fence_before();
            }
        }
    }
    pdl_trigger();
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

constexpr int kFinishTiles = 4;  // tiles whose weights one block sums

// Joins the pieces of the rows that several CTAs share, and sums the weights over the heads.
//   blocks y < kJoins: a thread takes some columns of a head, of one half of a token.  kGroups 1: 16 columns,
//                  for rows of few pieces.  kGroups 8: 8 columns and every eighth piece; the groups are
//                  added up in shared memory in their order
//   other blocks:  weights_j = sum_h p_hj 2^(ref_h - lse_h) of kFinishTiles tiles, a warp two entries at a time
// Loads that do not depend on one another are issued together: the blocks are short and wait for little else.
template <int kGroups>
__global__ void __launch_bounds__(kGroups == 1 ? 256 : 128 * kGroups)
kv4_finish_wide_kernel(const Operands op, const Division div, const Scratch scratch) {
    pdl_wait();
    pdl_trigger();
    constexpr int kThreads = kGroups == 1 ? 256 : 128 * kGroups, kWarps = kThreads / 32;
    constexpr int kCols = kGroups == 1 ? 16 : 8, kBlockCols = kGroups == 1 ? 32 : 8, kJoins = 512 / kBlockCols;
    constexpr int kParts = kThreads / 128;  // of the pieces, where a block sums weights
    __shared__ float s_shared[kGroups == 1 ? kFinishTiles * 128 : 10 * kGroups * 128];
    const int64_t token = blockIdx.x;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, head = tid & 127, group = tid >> 7;
    const int y = blockIdx.y;
    const int half = y < kJoins ? y / (kJoins / 2) : 0;  // the weights are of half 0's pieces
    const int32_t first = static_cast<int32_t>(token) * div.tiles;
    const int i0 = div.cta_of(first), i1 = div.cta_of(first + div.tiles - 1);
    // running maximum (base 2) and sum of this thread's pieces, two at a time
    float m = -INFINITY, l = 0.0f;
    auto join = [&](float m0, float l0, float m1, float l1, float& old, float& f0, float& f1) {
        const float top = fmaxf(m, fmaxf(m0, m1));
        old = m == -INFINITY ? 0.0f : exp2_fast(m - top);
        f0 = m0 == -INFINITY ? 0.0f : exp2_fast(m0 - top);
        f1 = m1 == -INFINITY ? 0.0f : exp2_fast(m1 - top);
        l = fmaf(l, old, fmaf(l0, f0, l1 * f1));
        m = top;
    };
    auto load_ml = [&](int i, float& pm, float& pl) {
        const float* ml = scratch.ml + (div.piece(i, first) * 2 + half) * 256 + head;
        pm = i <= i1 ? __ldcg(ml) : -INFINITY;
        pl = i <= i1 ? __ldcg(ml + 128) : 0.0f;
    };
    if (y < kJoins) {
        if (i0 == i1) return;  // written by its one CTA
        const int c0 = y % (kJoins / 2) * kBlockCols + (kGroups == 1 ? group * kCols : 0);
        constexpr int kStep = kGroups;
        float acc[kCols] = {};
        for (int i = i0 + (kGroups == 1 ? 0 : group); i <= i1; i += 2 * kStep) {
            float m0, l0, m1, l1, old, f0, f1, a[kCols], b[kCols];
            load_ml(i, m0, l0);
            load_ml(i + kStep, m1, l1);
            auto piece = [&](int k) {
                return scratch.o + (static_cast<int64_t>(div.piece(k, first) * 2 + half) * 256 + c0) * 128 + head;
            };
            const float* o0 = piece(i);
            const float* o1 = piece(i + kStep <= i1 ? i + kStep : i);
#pragma unroll
            for (int c = 0; c < kCols; ++c) {
                a[c] = __ldcg(o0 + c * 128);
                b[c] = __ldcg(o1 + c * 128);
            }
            join(m0, l0, m1, l1, old, f0, f1);
#pragma unroll
            for (int c = 0; c < kCols; ++c) acc[c] = fmaf(acc[c], old, fmaf(a[c], f0, b[c] * f1));
        }
        if constexpr (kGroups > 1) {
            float* mine = s_shared + group * 128 + head;  // [10][kGroups][128]
            mine[8 * kGroups * 128] = m;
            mine[9 * kGroups * 128] = l;
#pragma unroll
            for (int c = 0; c < kCols; ++c) mine[c * kGroups * 128] = acc[c];
            __syncthreads();
            if (group != 0) return;
            float f[kGroups];
#pragma unroll
            for (int g = 0; g < kGroups; ++g) m = fmaxf(m, mine[(8 * kGroups + g) * 128]);
            l = 0.0f;
#pragma unroll
            for (int g = 0; g < kGroups; ++g) {
                const float mg = mine[(8 * kGroups + g) * 128];
                f[g] = mg == -INFINITY ? 0.0f : exp2_fast(mg - m);
                l = fmaf(mine[(9 * kGroups + g) * 128], f[g], l);
            }
#pragma unroll
            for (int c = 0; c < kCols; ++c) {
                acc[c] = 0.0f;
#pragma unroll
                for (int g = 0; g < kGroups; ++g) acc[c] = fmaf(mine[(c * kGroups + g) * 128], f[g], acc[c]);
            }
        }
        if (head >= op.heads) return;
        const float inv = l != 0.0f ? 1.0f / l : 0.0f;
        uint32_t w[kCols / 2];
#pragma unroll
        for (int c = 0; c < kCols; c += 2) w[c / 2] = pack_bf16(acc[c] * inv, acc[c + 1] * inv);
        __nv_bfloat16* out = op.out + (token * op.heads + head) * kLatent + half * 256 + c0;
        if constexpr (kCols == 16) store32(out, w);
        else *reinterpret_cast<uint4*>(out) = make_uint4(w[0], w[1], w[2], w[3]);
        if (y == 0 && c0 == 0)
            op.lse[token * op.heads + head] = l != 0.0f ? (m + log2f(l)) * 0.6931471805599453f : -INFINITY;
        return;
    }
    const int tile0 = (y - kJoins) * kFinishTiles, count = min(kFinishTiles, div.tiles - tile0);
    constexpr int kBatch = 128 / kWarps < 8 ? 128 / kWarps : 8;
    const uint32_t* from = scratch.p + (token * div.tiles + tile0) * 32 * 128 + lane * 4;
    uint4 p[kBatch];  // row k: two entries, the halves of the words
    auto load_rows = [&](int k0) {
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const int k = k0 + i * kWarps;
            p[i] = k < count * 32 ? __ldcg(reinterpret_cast<const uint4*>(from + k * 128)) : make_uint4(0, 0, 0, 0);
        }
    };
    load_rows(warp);
    float ref[kFinishTiles];
#pragma unroll
    for (int k = 0; k < kFinishTiles; ++k)
        ref[k] = group == 0 && k < count ? __ldcg(scratch.ref + (token * div.tiles + tile0 + k) * 128 + head) : 0.0f;
    if (i0 == i1) {
        if (group == 0 && head < op.heads) m = op.lse[token * op.heads + head] * 1.4426950408889634f, l = 1.0f;
    } else {  // the joining blocks may not have written lse yet
        for (int i = i0 + group; i <= i1; i += 2 * kParts) {
            float m0, l0, m1, l1, old, f0, f1;
            load_ml(i, m0, l0);
            load_ml(i + kParts, m1, l1);
            join(m0, l0, m1, l1, old, f0, f1);
        }
        s_shared[tid] = m;
        s_shared[kThreads + tid] = l;
        __syncthreads();
        if (group == 0) {
#pragma unroll
            for (int g = 1; g < kParts; ++g) {
                float old, f0, f1;
                join(s_shared[g * 128 + head], s_shared[kThreads + g * 128 + head], -INFINITY, 0.0f, old, f0, f1);
            }
        }
        __syncthreads();
    }
    if (group == 0) {
        const float lse = l != 0.0f && head < op.heads ? m + log2f(l) : -INFINITY;  // base 2
#pragma unroll
        for (int k = 0; k < kFinishTiles; ++k)
            s_shared[k * 128 + head] = lse == -INFINITY ? 0.0f : exp2_fast(ref[k] - lse);
    }
    __syncthreads();
    for (int k0 = warp; k0 < count * 32; k0 += kBatch * kWarps) {
        if (k0 != warp) load_rows(k0);
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const int k = k0 + i * kWarps;
            const float4 f = *reinterpret_cast<const float4*>(s_shared + k / 32 % kFinishTiles * 128 + lane * 4);
            float a = __uint_as_float(p[i].x << 16) * f.x, b = __uint_as_float(p[i].x & 0xffff0000u) * f.x;
            a = fmaf(__uint_as_float(p[i].y << 16), f.y, a), b = fmaf(__uint_as_float(p[i].y & 0xffff0000u), f.y, b);
            a = fmaf(__uint_as_float(p[i].z << 16), f.z, a), b = fmaf(__uint_as_float(p[i].z & 0xffff0000u), f.z, b);
            a = fmaf(__uint_as_float(p[i].w << 16), f.w, a), b = fmaf(__uint_as_float(p[i].w & 0xffff0000u), f.w, b);
            // the lower lanes go on with the first entry, the upper ones with the second
            float sum = (lane < 16 ? a : b) + __shfl_xor_sync(0xffffffffu, lane < 16 ? b : a, 16);
#pragma unroll
            for (int d = 8; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
            const int e = tile0 * kTile + 2 * k + (lane >> 4);
            if ((lane & 15) == 0 && k < count * 32 && e < op.topk) op.weights[token * op.topk + e] = __float2bfloat16(sum);
        }
    }
    // The factor of a head whose scores are not numbers, NaN in each tile, has made all sums NaN: entries that are not
    // there stay at 0.  (Out of the loop above, where asking each sum cost 2 us of 162 with 128 tokens.)
    const float4 f = *reinterpret_cast<const float4*>(s_shared + lane * 4);
    const float any = f.x + f.y + f.z + f.w;
    if (!__any_sync(0xffffffffu, any != any)) return;
    __syncwarp();
    for (int k = warp; k < count * 32; k += kWarps) {  // the warp's own stores
        const int e = tile0 * kTile + 2 * k + lane;
        if (lane < 2 && e < op.topk && !is_there(op, token, e))
            op.weights[token * op.topk + e] = __float2bfloat16(0.0f);
    }
}

int64_t tiles_of(int64_t topk) { return topk > 0 ? (topk + kTile - 1) / kTile : 1; }  // no entry: an empty tile

// Among pairs of CTAs, one for each half of the output columns.
Division wide_division(int64_t tokens, int64_t topk, int sms) {
    return Division(tokens, tiles_of(topk), sms > 1 ? sms / 2 : 1, 3);
}

// Byte offsets of the scratch arrays; [4] is the size.
void wide_layout(const Division& d, int64_t tokens, bool weights, int64_t (&at)[5]) {
    const int64_t pieces = d.shares() ? 4ll * d.ctas : 0;  // of halves
    at[0] = 0;
    at[1] = at[0] + align256(pieces * 256 * 4);
    at[2] = at[1] + align256(pieces * 256 * 128 * 4);
    at[3] = at[2] + (weights ? align256(tokens * d.tiles * 128 * 4) : 0);
    at[4] = at[3] + (weights ? tokens * d.tiles * 32 * 128 * 4 : 0);
}

}  // namespace

int64_t wide_workspace(int64_t tokens, int64_t topk, bool weights) {
    int64_t at[5];
    wide_layout(wide_division(tokens, topk, asu_sm_count()), tokens, weights, at);
    return at[4];
}

int64_t wide_weights(int64_t topk) { return tiles_of(topk) * 128 * (4 + 2 * kTile); }

int launch_wide(cudaStream_t s, const Operands& op, void* workspace) {
    const Division d = wide_division(op.tokens, op.topk, asu_sm_count());
    int64_t at[5];
    wide_layout(d, op.tokens, op.weights != nullptr, at);
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    const Scratch scratch = {reinterpret_cast<float*>(ws + at[0]), reinterpret_cast<float*>(ws + at[1]),
                             reinterpret_cast<float*>(ws + at[2]), reinterpret_cast<uint32_t*>(ws + at[3])};
    int max_dynamic = 0;
    int rc = asu_max_dynamic_smem(reinterpret_cast<const void*>(kv4_decode_wide_kernel), &max_dynamic);
    if (rc != ASU_OK) return rc;
    if (max_dynamic < kWideSmem) return ASU_ERR_ARG;
    rc = launch_pdl(kv4_decode_wide_kernel, dim3(2 * d.ctas), dim3(kWideThreads), kWideSmem, s, op, d, scratch);
    int most = 1;  // pieces of a row
    for (int i = 1; i < d.ctas && most < 3; ++i)
        if (d.start(i) % d.tiles != 0) most = d.start(i + 1) / d.tiles == d.start(i) / d.tiles && i + 1 < d.ctas ? 3 : 2;
    if (rc != ASU_OK || (most == 1 && op.weights == nullptr)) return rc;
    const int sums = op.weights != nullptr ? (d.tiles + kFinishTiles - 1) / kFinishTiles : 0;
    const unsigned tokens = static_cast<unsigned>(op.tokens);
    if (most > 2)
        return launch_pdl(kv4_finish_wide_kernel<8>, dim3(tokens, 64 + sums), dim3(1024), 0, s, op, d, scratch);
    return launch_pdl(kv4_finish_wide_kernel<1>, dim3(tokens, 16 + sums), dim3(256), 0, s, op, d, scratch);
}

}  // namespace kv4
}  // namespace asu

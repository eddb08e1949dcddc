// Sparse decode attention over the 4-bit cache for more than 32 heads, on the tcgen05 tensor cores.
#include "kv4_decode.cuh"
#include "tcgen05.cuh"

namespace asu {
namespace kv4 {
namespace {

// ---- many heads: tensor cores --------------------------------------------------------------------
//
// 128 rows of heads (padded) x 64 entries a tile.  A CTA makes 256 of the 512 output columns, since
// all 512 in 32 bits would fill the tensor memory and leave no room for the scores; the two CTAs of a
// token each compute the scores (1.5 times the products of a scheme that shares them, but no
// exchange between SMs).
//
// Tensor memory, 512 columns: output 256, scores 2 x 64 (their weights take the same columns,
// as bf16 pairs, once read), and q's latents 256..511, bf16 pairs, 128.
// Shared memory, 224 KB: q's other 320 values, 80 KB; two tiles of dequantised rows, 72 KB each, as nine
// blocks of [64 entries x 64 values] in the 128-byte swizzle.  A block serves both products: entries
// x values with the values contiguous is K-major for the scores and MN-major for the output.
//
// 13 warps: 4 for the softmax, a thread a head (its row of scores lies in its tensor memory lane, so
// there is no exchange); 8 that load rows, dequantise and store blocks; one whose lane 0 issues
// the products.  The running maximum only moves when it grows by more than 2^8: until then the weights
// stay below 2^8, exact enough in bf16 like any others, and the output needs no rescaling.
//
// The blocks that only the scores read ("part A": the other half's four and the rope block) are
// released after them, the four output blocks ("part B") after the output product: the next tile's
// part A is in place when the tensor cores get there, and its products hide the filling of part B.
constexpr int kWideThreads = 13 * 32;
constexpr int kBlock = kTile * 128;           // bytes of a [64 x 64] bf16 block
constexpr int kQBlock = 128 * 128;            // bytes of a [128 x 64] bf16 block
constexpr int kSmemQ = 0;
constexpr int kSmemA = 5 * kQBlock;
constexpr int kSmemB = kSmemA + 2 * 5 * kBlock;
constexpr int kSmemBars = kSmemB + 2 * 4 * kBlock;
constexpr int kWideSmem = kSmemBars + 128 + 1024;  // the base is rounded up to 1024
constexpr uint32_t kColO = 0, kColS = 256, kColQ = 384;
constexpr float kMaxGrowth = 8.0f;

enum Bar { kFullA = 0, kFullB = 2, kScores = 4, kWeights = 6, kOutput = 8, kQuery = 10, kDrain = 11, kBars = 12 };

struct Scratch {
    float* ml;         // [2 * ctas][2][128] running maximum (base 2) and sum of a piece
    float* o;          // [2 * ctas][256][128] its output, columns by heads
    float* ref;        // [tokens][tiles][128] the maximum that a tile's weights are relative to
    uint32_t* p;       // [tokens][tiles][32][128] a tile's weights, pairs of entries
};

struct RawRows {  // a thread's part of a tile before dequantising: two rows
    uint4 code[2][2], rope[2];
    uint32_t scale[2][2];
};

__device__ __forceinline__ void dequantise(const uint4& code, uint32_t scales, uint32_t block, int row, int lp) {
    const uint32_t w[4] = {code.x, code.y, code.z, code.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        __nv_bfloat162 s, c;
        scale_pair((scales >> (8 * (i / 2))) & 0xffu, s, c);
        uint32_t v[4];
        unpack_word(w[i], s, c, v);
        const uint32_t at = block + row * 128 + (((lp * 4 + i) ^ (row & 7)) << 4);
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3])
                     : "memory");
    }
}

__global__ void __launch_bounds__(kWideThreads, 1)
kv4_decode_wide_kernel(const Operands op, const Division div, const Scratch scratch) {
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint32_t s_tmem;
    __shared__ int s_dead;
    const uint32_t base = (tc::smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t bars = base + kSmemBars;
    auto bar = [&](int which, int64_t n) { return bars + 8u * (which + static_cast<int>(n & 1)); };
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    volatile int* dead = &s_dead;
    // by whole warps: all lanes go on, or none
    auto warp_wait = [&](uint32_t b, uint32_t parity) {
        return __all_sync(0xffffffffu, tc::mbar_wait(b, parity, dead)) != 0;
    };

    if (tid == 0) {
        s_dead = 0;
        for (int i = 0; i < 2; ++i) {
            tc::mbar_init(bars + 8 * (kFullA + i), 8);
            tc::mbar_init(bars + 8 * (kFullB + i), 8);
            tc::mbar_init(bars + 8 * (kScores + i), 1);
            tc::mbar_init(bars + 8 * (kWeights + i), 128);
            tc::mbar_init(bars + 8 * (kOutput + i), 1);
        }
        tc::mbar_init(bars + 8 * kQuery, 128);
        tc::mbar_init(bars + 8 * kDrain, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 12) tc::tmem_alloc<512>(tc::smem_u32(&s_tmem));
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    const uint32_t tmem = s_tmem;
    pdl_wait();

    const int64_t u0 = div.start(blockIdx.x), u1 = div.start(blockIdx.x + 1);
    const int tiles = div.tiles;

    if (warp >= 4 && warp < 12) {
        // ---- rows: global memory -> registers -> dequantised blocks ----
        // lane = 8 q + 2 rr + lp: row rr of four, 32 latents 32 * (2 q + lp) of either half.  Eight
        // consecutive lanes store to four rows x two chunks, which the swizzle spreads over all banks.
        const int quarter = lane >> 3, lp = lane & 1;
        const int row0 = (warp - 4) * 4 + ((lane >> 1) & 3);
        const int chunk = 2 * quarter + lp;
        int32_t bits = 0;
        int64_t row = u0 / tiles;
        int tile = static_cast<int>(u0 - row * tiles);
        auto slot_of = [&](int64_t r, int t, int half) -> int32_t {
            const int e = t * kTile + half * 32 + row0;
            if (e >= op.topk) return kNotFound;
            const int64_t token = r % op.tokens;
            const int32_t s = __ldg(op.slots + token * op.slots_token + e);
            if (s >= 0 && s < op.pool_rows) return s;
            if (s != kNotFound) bits |= ASU_ST_BAD_QUERY;
            return kNotFound;
        };
        auto load = [&](RawRows& raw, int64_t r, const int32_t (&slot)[2]) {
            const uint8_t* pool = op.pool + static_cast<uint64_t>(r % op.tokens) * op.pool_token;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                raw.code[i][0] = raw.code[i][1] = make_uint4(0x88888888u, 0x88888888u, 0x88888888u, 0x88888888u);
                raw.rope[i] = make_uint4(0, 0, 0, 0);
                raw.scale[i][0] = raw.scale[i][1] = 0;
                if (slot[i] < 0) continue;  // a row of zeros
                const uint8_t* p = pool + static_cast<uint64_t>(slot[i]) * op.pool_pitch;
                raw.code[i][0] = __ldg(reinterpret_cast<const uint4*>(p + chunk * 16));
                raw.code[i][1] = __ldg(reinterpret_cast<const uint4*>(p + 128 + chunk * 16));
                raw.scale[i][0] = __ldg(reinterpret_cast<const unsigned short*>(p + kScaleOffset + chunk * 2));
                raw.scale[i][1] = __ldg(reinterpret_cast<const unsigned short*>(p + kScaleOffset + 16 + chunk * 2));
                raw.rope[i] = __ldg(reinterpret_cast<const uint4*>(p + kRopeOffset + (lp * 4 + quarter) * 16));
            }
        };
        RawRows cur, nxt;
        int32_t slot[2], slot_nxt[2];
        for (int i = 0; i < 2; ++i) slot[i] = u0 < u1 ? slot_of(row, tile, i) : kNotFound;
        load(cur, row, slot);
        int64_t row_n = row;
        int tile_n = tile;
        auto advance = [&](int64_t& r, int& t) {
            if (++t == tiles) {
                t = 0;
                ++r;
            }
        };
        advance(row_n, tile_n);
        for (int i = 0; i < 2; ++i) slot_nxt[i] = u0 + 1 < u1 ? slot_of(row_n, tile_n, i) : kNotFound;
        for (int64_t u = u0, n = 0; u < u1; ++u, ++n) {
            // the next tile's rows and the slots of the one behind it are on their way meanwhile
            load(nxt, row_n, slot_nxt);
            int64_t row_nn = row_n;
            int tile_nn = tile_n;
            advance(row_nn, tile_nn);
            if (u + 2 < u1)
                for (int i = 0; i < 2; ++i) slot_nxt[i] = slot_of(row_nn, tile_nn, i);
            else
                slot_nxt[0] = slot_nxt[1] = kNotFound;
            const int half = row >= op.tokens;  // this CTA's output columns: latents 256 * half ..
            const uint32_t part_a = base + kSmemA + static_cast<int>(n & 1) * 5 * kBlock;
            const uint32_t part_b = base + kSmemB + static_cast<int>(n & 1) * 4 * kBlock;
            if (n >= 2 && !warp_wait(bar(kScores, n), ((n >> 1) - 1) & 1)) break;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int r = row0 + 32 * i;
                const uint4 c = half ? cur.code[i][0] : cur.code[i][1];
                dequantise(c, half ? cur.scale[i][0] : cur.scale[i][1], part_a + quarter * kBlock, r, lp);
                const uint32_t at = part_a + 4 * kBlock + r * 128 + (((lp * 4 + quarter) ^ (r & 7)) << 4);
                asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(cur.rope[i].x),
                             "r"(cur.rope[i].y), "r"(cur.rope[i].z), "r"(cur.rope[i].w)
                             : "memory");
            }
            tc::fence_async_shared();
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(bar(kFullA, n));
            if (n >= 2 && !warp_wait(bar(kOutput, n), ((n >> 1) - 1) & 1)) break;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint4 c = half ? cur.code[i][1] : cur.code[i][0];
                dequantise(c, half ? cur.scale[i][1] : cur.scale[i][0], part_b + quarter * kBlock, row0 + 32 * i, lp);
            }
            tc::fence_async_shared();
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(bar(kFullB, n));
            cur = nxt;
            row = row_n;
            tile = tile_n;
            row_n = row_nn;
            tile_n = tile_nn;
        }
        if (bits) flag_status(op.status, 0, bits);
    } else if (warp == 12) {
        if (lane == 0) {
            // ---- the products ----
            constexpr uint32_t kDescS = tc::instruction(128, kTile, false);
            constexpr uint32_t kDescO = tc::instruction(128, 256, true);
            auto scores = [&](int64_t n, int half) {
                const uint32_t part_a = base + kSmemA + static_cast<int>(n & 1) * 5 * kBlock;
                const uint32_t part_b = base + kSmemB + static_cast<int>(n & 1) * 4 * kBlock;
                const uint32_t d = tmem + kColS + kTile * static_cast<uint32_t>(n & 1);
                // of the two halves of the latents, q's first lies in shared and its second in tensor memory
                auto block = [&](uint32_t rows, int which, uint32_t accumulate) {  // which: 64 values of q
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const uint64_t b = tc::operand(rows + k * 32, 0, 1024);
                        if (which >= 4 && which < 8) {
                            tc::mma_ts(d, tmem + kColQ + (which - 4) * 32 + k * 8, b, kDescS, accumulate | (k > 0));
                        } else {
                            const uint32_t q = base + kSmemQ + (which < 4 ? which : 4) * kQBlock + k * 32;
                            tc::mma_ss(d, tc::operand(q, 0, 1024), b, kDescS, accumulate | (k > 0));
                        }
                    }
                };
                if (!tc::mbar_wait(bar(kFullA, n), (n >> 1) & 1, dead)) return false;
                tc::fence_after();
                block(part_a + 4 * kBlock, 8, 0);
                for (int i = 0; i < 4; ++i) block(part_a + i * kBlock, (half ? 0 : 4) + i, 1);
                if (!tc::mbar_wait(bar(kFullB, n), (n >> 1) & 1, dead)) return false;
                tc::fence_after();
                for (int i = 0; i < 4; ++i) block(part_b + i * kBlock, (half ? 4 : 0) + i, 1);
                tc::commit(bar(kScores, n));
                return true;
            };
            int64_t n = 0, segment = 0;
            bool ok = true;
            for (int64_t u = u0; ok && u < u1; ++u, ++n) {
                const int64_t row = u / tiles;
                const int half = row >= op.tokens;
                const bool first = u == u0 || u == row * tiles;
                const bool last = u + 1 == u1 || u + 1 == (row + 1) * tiles;
                if (first) {
                    ok = tc::mbar_wait(bars + 8 * kQuery, segment & 1, dead);
                    ++segment;
                    if (!ok) break;
                    tc::fence_after();
                    if (!(ok = scores(n, half))) break;
                }
                if (!last) {
                    // the other score columns hold the weights of tile n - 1 until its output product is done
                    if (!first && !(ok = tc::mbar_wait(bar(kOutput, n - 1), ((n - 1) >> 1) & 1, dead))) break;
                    tc::fence_after();
                    if (!(ok = scores(n + 1, half))) break;
                }
                if (!(ok = tc::mbar_wait(bar(kWeights, n), (n >> 1) & 1, dead))) break;
                tc::fence_after();
                const uint32_t part_b = base + kSmemB + static_cast<int>(n & 1) * 4 * kBlock;
                const uint32_t p = tmem + kColS + kTile * static_cast<uint32_t>(n & 1);
#pragma unroll
                for (int k = 0; k < kTile / 16; ++k)
                    tc::mma_ts(tmem + kColO, p + 8 * k, tc::operand(part_b + k * 2048, kBlock, 1024), kDescO,
                               !first || k > 0);
                tc::commit(bar(kOutput, n));
            }
            if (!ok) {  // nothing of this block may still run when its tensor memory is given back
                tc::commit(bars + 8 * kDrain);
                for (int i = 0; i < tc::kSpinLimit && !tc::mbar_try(bars + 8 * kDrain, 0); ++i) {
                }
            }
        }
        __syncwarp();
    } else {
        // ---- softmax, a thread a head ----
        const uint32_t lanes = tmem + (static_cast<uint32_t>(warp * 32) << 16);
        const int head = tid;
        float m = -INFINITY, l = 0.0f;
        int64_t n = 0;
        for (int64_t u = u0; u < u1; ++u, ++n) {
            const int64_t row = u / tiles;
            const int half = row >= op.tokens;
            const int64_t token = row - (half ? op.tokens : 0);
            const int tile = static_cast<int>(u - row * tiles);
            const bool first = u == u0 || tile == 0;
            const bool last = u + 1 == u1 || tile + 1 == tiles;
            if (first) {
                // this token's q: latents 0..255 and the rope part to shared memory, the rest to tensor memory
                const __nv_bfloat16* qt = op.q + token * op.q_token;
                auto chunk8 = [&](int h, int at) -> uint4 {
                    if (h >= op.heads) return make_uint4(0, 0, 0, 0);
                    const __nv_bfloat16* p = qt + h * op.q_head + at;
                    if (op.q_aligned) return __ldg(reinterpret_cast<const uint4*>(p));
                    const unsigned short* s = reinterpret_cast<const unsigned short*>(p);
                    uint32_t w[4];
                    for (int i = 0; i < 4; ++i)
                        w[i] = static_cast<uint32_t>(__ldg(s + 2 * i)) | (static_cast<uint32_t>(__ldg(s + 2 * i + 1)) << 16);
                    return make_uint4(w[0], w[1], w[2], w[3]);
                };
#pragma unroll 8
                for (int i = tid; i < 5 * 128 * 8; i += 128) {
                    const int block = i >> 10, h = (i >> 3) & 127, c = i & 7;
                    const uint4 v = chunk8(h, (block < 4 ? block * 64 : kLatent) + c * 8);
                    const uint32_t at = base + kSmemQ + block * kQBlock + h * 128 + ((c ^ (h & 7)) << 4);
                    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(v.x), "r"(v.y), "r"(v.z),
                                 "r"(v.w)
                                 : "memory");
                }
                tc::fence_async_shared();
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    uint32_t w[32];
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const uint4 v = chunk8(head, 256 + i * 64 + k * 8);
                        w[4 * k] = v.x;
                        w[4 * k + 1] = v.y;
                        w[4 * k + 2] = v.z;
                        w[4 * k + 3] = v.w;
                    }
                    tc::tmem_store32(lanes + kColQ + i * 32, w);
                }
                tc::tmem_wait_store();
                tc::fence_before();
                tc::mbar_arrive(bars + 8 * kQuery);
                m = -INFINITY;
                l = 0.0f;
            }
            // which entries are there
            uint32_t there[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int e = tile * kTile + 32 * i + lane;
                const int32_t s = e < op.topk ? __ldg(op.slots + token * op.slots_token + e) : kNotFound;
                there[i] = __ballot_sync(0xffffffffu, s >= 0 && s < op.pool_rows);
            }
            if (!warp_wait(bar(kScores, n), (n >> 1) & 1)) break;
            tc::fence_after();
            const uint32_t cols = lanes + kColS + kTile * static_cast<uint32_t>(n & 1);
            uint32_t s[2][32];
            tc::tmem_load32(cols, s[0]);
            tc::tmem_load32(cols + 32, s[1]);
            tc::tmem_wait_load(s[0]);
            tc::tmem_wait_load(s[1]);
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
            if (__any_sync(0xffffffffu, fade != 1.0f)) {
                l *= fade;
                if (!warp_wait(bar(kOutput, n - 1), ((n - 1) >> 1) & 1)) break;
                tc::fence_after();
#pragma unroll 1
                for (int c = 0; c < 256; c += 32) {
                    uint32_t o[32];
                    tc::tmem_load32(lanes + kColO + c, o);
                    tc::tmem_wait_load(o);
#pragma unroll
                    for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * fade);
                    tc::tmem_store32(lanes + kColO + c, o);
                }
                tc::tmem_wait_store();
            }
            const float from = m == -INFINITY ? 0.0f : m;
            uint32_t p[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) {
                const float a = exp2_fast(fmaf(__uint_as_float(s[i / 16][(2 * i) % 32]), op.scale_log2, -from));
                const float b = exp2_fast(fmaf(__uint_as_float(s[i / 16][(2 * i + 1) % 32]), op.scale_log2, -from));
                l += a;
                l += b;
                p[i] = pack_bf16(a, b);
            }
            tc::tmem_store32(cols, p);
            tc::tmem_wait_store();
            tc::fence_before();
            tc::mbar_arrive(bar(kWeights, n));
            if (op.weights != nullptr && half == 0) {
                const int64_t at = token * tiles + tile;
                scratch.ref[at * 128 + head] = m;
#pragma unroll
                for (int i = 0; i < 32; ++i) scratch.p[(at * 32 + i) * 128 + head] = p[i];
            }
            if (last) {
                if (!warp_wait(bar(kOutput, n), (n >> 1) & 1)) break;
                tc::fence_after();
                const bool whole = row * tiles >= u0 && (row + 1) * tiles <= u1;
                if (whole) {
                    const float inv = l > 0.0f ? 1.0f / l : 0.0f;
                    __nv_bfloat16* out = op.out + (token * op.heads + head) * kLatent + half * 256;
#pragma unroll 1
                    for (int c = 0; c < 256; c += 32) {
                        uint32_t o[32];
                        tc::tmem_load32(lanes + kColO + c, o);
                        tc::tmem_wait_load(o);
                        if (head < op.heads) {
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                uint32_t w[4];
#pragma unroll
                                for (int k = 0; k < 4; ++k)
                                    w[k] = pack_bf16(__uint_as_float(o[8 * i + 2 * k]) * inv,
                                                     __uint_as_float(o[8 * i + 2 * k + 1]) * inv);
                                reinterpret_cast<uint4*>(out + c)[i] = make_uint4(w[0], w[1], w[2], w[3]);
                            }
                        }
                    }
                    if (half == 0 && head < op.heads)
                        op.lse[token * op.heads + head] =
                            l > 0.0f ? (m + log2f(l)) * 0.6931471805599453f : -INFINITY;
                } else {
                    const int piece = div.piece(blockIdx.x, row * tiles);
                    float* to = scratch.o + static_cast<int64_t>(piece) * 256 * 128 + head;
#pragma unroll 1
                    for (int c = 0; c < 256; c += 32) {
                        uint32_t o[32];
                        tc::tmem_load32(lanes + kColO + c, o);
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
        tc::fence_after();
        tc::tmem_free<512>(tmem);
    }
}

// Joins the pieces of the rows that several CTAs share, and sums the weights over the heads.
//   blocks y < 16: output columns [16 * y, ...) ... of the token's two halves
//   other blocks:  one tile's weights: weights_j = sum_h p_hj 2^(ref_h - lse_h)
constexpr int kFinishThreads = 256;
__global__ void __launch_bounds__(kFinishThreads)
kv4_finish_wide_kernel(const Operands op, const Division div, const Scratch scratch) {
    pdl_wait();
    pdl_trigger();
    __shared__ float s_tile[32][129];
    __shared__ float s_lse[128];  // base 2
    const int64_t token = blockIdx.x;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const bool joins = blockIdx.y < 16;
    const int half = joins ? blockIdx.y >> 3 : 0;
    const int64_t first = (half * static_cast<int64_t>(op.tokens) + token) * div.tiles;
    const int i0 = div.cta_of(first), i1 = div.cta_of(first + div.tiles - 1);
    if (joins && i0 == i1) return;  // written by its one CTA
    if (joins) {
        const int c0 = (blockIdx.y & 7) * 32;
        const int head = tid & 127, part = tid >> 7;  // two threads a head, 16 columns each
        float m = -INFINITY;
        for (int i = i0; i <= i1; ++i) m = fmaxf(m, scratch.ml[div.piece(i, first) * 256 + head]);
        float l = 0.0f, acc[16] = {};
        for (int i = i0; i <= i1; ++i) {
            const int piece = div.piece(i, first);
            const float pm = scratch.ml[piece * 256 + head];
            const float f = pm == -INFINITY ? 0.0f : exp2_fast(pm - m);
            l += scratch.ml[piece * 256 + 128 + head] * f;
            const float* o = scratch.o + (static_cast<int64_t>(piece) * 256 + c0 + part * 16) * 128 + head;
#pragma unroll
            for (int c = 0; c < 16; ++c) acc[c] += o[c * 128] * f;
        }
        const float inv = l > 0.0f ? 1.0f / l : 0.0f;
#pragma unroll
        for (int c = 0; c < 16; ++c) s_tile[part * 16 + c][head] = acc[c] * inv;
        if (blockIdx.y == 0 && part == 0 && head < op.heads)
            op.lse[token * op.heads + head] = l > 0.0f ? (m + log2f(l)) * 0.6931471805599453f : -INFINITY;
        __syncthreads();
        for (int i = tid; i < op.heads * 16; i += kFinishThreads) {
            const int h = i >> 4, c = (i & 15) * 2;
            *reinterpret_cast<uint32_t*>(op.out + (token * op.heads + h) * kLatent + half * 256 + c0 + c) =
                pack_bf16(s_tile[c][h], s_tile[c + 1][h]);
        }
        return;
    }
    // the token's lse again (the joining blocks may not have written it yet)
    if (tid < 128) {
        float v = -INFINITY;
        if (tid < op.heads) {
            if (i0 == i1) {
                v = op.lse[token * op.heads + tid] * 1.4426950408889634f;
            } else {
                float m = -INFINITY, l = 0.0f;
                for (int i = i0; i <= i1; ++i) m = fmaxf(m, scratch.ml[div.piece(i, first) * 256 + tid]);
                for (int i = i0; i <= i1; ++i) {
                    const int piece = div.piece(i, first);
                    const float pm = scratch.ml[piece * 256 + tid];
                    l += scratch.ml[piece * 256 + 128 + tid] * (pm == -INFINITY ? 0.0f : exp2_fast(pm - m));
                }
                if (l > 0.0f) v = m + log2f(l);
            }
        }
        s_lse[tid] = v;
    }
    __syncthreads();
    const int tile = blockIdx.y - 16;
    const int64_t at = token * div.tiles + tile;
    float f[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int h = lane * 4 + i;
        f[i] = s_lse[h] == -INFINITY ? 0.0f : exp2_fast(scratch.ref[at * 128 + h] - s_lse[h]);
    }
    for (int k = warp; k < 32; k += kFinishThreads / 32) {  // a warp a pair of entries
        const uint4 p = *reinterpret_cast<const uint4*>(scratch.p + (at * 32 + k) * 128 + lane * 4);
        const uint32_t w[4] = {p.x, p.y, p.z, p.w};
        float a = 0.0f, b = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            a = fmaf(__uint_as_float(w[i] << 16), f[i], a);
            b = fmaf(__uint_as_float(w[i] & 0xffff0000u), f[i], b);
        }
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) {
            a += __shfl_xor_sync(0xffffffffu, a, d);
            b += __shfl_xor_sync(0xffffffffu, b, d);
        }
        const int e = tile * kTile + 2 * k;
        if (lane == 0 && e < op.topk) op.weights[token * op.topk + e] = __float2bfloat16(a);
        if (lane == 1 && e + 1 < op.topk) op.weights[token * op.topk + e + 1] = __float2bfloat16(b);
    }
}

int64_t align256(int64_t x) { return (x + 255) / 256 * 256; }

Division wide_division(int64_t tokens, int64_t topk, int sms) {
    Division d;
    d.rows = static_cast<int32_t>(2 * tokens);
    d.tiles = static_cast<int32_t>(topk > 0 ? (topk + kTile - 1) / kTile : 1);  // no entry: one empty tile
    const int64_t units = d.units();
    d.ctas = static_cast<int32_t>(units < sms ? units : sms);
    return d;
}

// Byte offsets of the scratch arrays; [4] is the size.
void wide_layout(const Division& d, int64_t tokens, bool weights, int64_t (&at)[5]) {
    at[0] = 0;
    at[1] = at[0] + align256(2ll * d.ctas * 256 * 4);
    at[2] = at[1] + align256(2ll * d.ctas * 256 * 128 * 4);
    at[3] = at[2] + (weights ? align256(tokens * d.tiles * 128 * 4) : 0);
    at[4] = at[3] + (weights ? tokens * d.tiles * 32 * 128 * 4 : 0);
}

}  // namespace

int64_t wide_workspace(int64_t tokens, int64_t topk, bool weights) {
    int64_t at[5];
    wide_layout(wide_division(tokens, topk, asu_sm_count()), tokens, weights, at);
    return at[4];
}

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
    rc = launch_pdl(kv4_decode_wide_kernel, dim3(d.ctas), dim3(kWideThreads), kWideSmem, s, op, d, scratch);
    bool shared_rows = false;  // does any row lie in several CTAs' ranges?
    for (int i = 1; i < d.ctas && !shared_rows; ++i) shared_rows = d.start(i) % d.tiles != 0;
    if (rc != ASU_OK || (!shared_rows && op.weights == nullptr)) return rc;
    return launch_pdl(kv4_finish_wide_kernel,
                      dim3(static_cast<unsigned>(op.tokens), 16 + (op.weights != nullptr ? d.tiles : 0)),
                      dim3(kFinishThreads), 0, s, op, d, scratch);
}

}  // namespace kv4
}  // namespace asu

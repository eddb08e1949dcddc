// Sparse decode attention over the 4-bit cache for few heads, on the warp-level tensor cores.
//
// With 16 heads a row of 416 bytes meets 35 KFLOP: memory bound, and the 128-row products of the
// tcgen05 kernel would be seven eighths padding.  m16n8k16 products take the heads as their 16 rows
// (kMT such groups of 16 in a CTA) and the entries (scores) or latents (output) as their columns.
//
// A CTA of 8 warps takes tiles of 32 entries: warp (d, e) has the latents 128 d .. 128 d + 127 of the entries
// 16 e .. 16 e + 15, for the scores and for the output.  It dequantises them once, into registers in the
// layout that the score products want (entry g = lane / 4 of 8, values 32 c .. 32 c + 31 with
// c = lane % 4: one 16-byte load), and turns the same registers into the output products' layout with
// movmatrix, a transposition of 8 x 8 values.  No dequantised value goes through shared memory.  The
// price: a warp's scores are partial sums over its latents, added up through shared memory by the threads
// that then do the softmax (16 threads a row with one group of heads, 8 with two); and its output is a
// partial sum over its entries, added up once a token.  (Eight warps of 64 latents and all 32 entries
// each took twice the instructions: 81 us instead of the time below.)
//
// Which 4 values of a latent row a thread's k indexes mean is free as long as both operands agree: k index
// 2c, 2c + 1, 2c + 8, 2c + 9 of step s are the values 32 c + 4 s .. 32 c + 4 s + 3.
//
// Rows come by asynchronous copies, kStages - 1 tiles ahead.  Two barriers a tile: partial scores
// written, weights written.  One group of heads: 128 registers, two CTAs on an SM, whose phases fill each
// other's waits.
#include "kv4_decode.cuh"

namespace asu {
namespace kv4 {
namespace {

constexpr int kThreads = 256;
constexpr int kKeys = 32;  // entries a tile
constexpr int kStages = 5;
constexpr int kRawRow = kRowBytes + 32;  // 16 words more than a multiple of 32: two rows' 64 bytes are all banks
constexpr int kPartRow = kKeys + 8;      // floats; 8 more than a multiple of 32: no bank conflicts
constexpr int kWeightRow = kKeys + 8;    // bf16
constexpr float kMaxGrowth = 8.0f;       // the maximum moves when it grows by more than 2^8

template <int kMT>
struct Shared {
    alignas(128) uint8_t raw[kStages][kKeys * kRawRow];
    uint4 q[kMT][32][32];                    // q's latents by product operand: [step 8 d + s][lane]
    uint4 rope[kMT][4][32];                  // and its rope part
    float part[4][16 * kMT][kPartRow];       // each d's partial scores
    __nv_bfloat16 weights[16 * kMT][kWeightRow];
    float row[16 * kMT];                     // a row's factor
    uint32_t there[kStages][8];              // four entries a warp: which are there
};

struct NarrowScratch {
    float* ml;           // [2 * ctas][2][16 * kMT]
    float* o;            // [2 * ctas][16 * kMT][512]
    float* ref;          // [tokens][tiles][heads rounded up to the group]
    __nv_bfloat16* p;    // [tokens][heads rounded up][tiles * kKeys]
};

__device__ __forceinline__ uint32_t shared_address(const void* p) {
    return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}

__device__ __forceinline__ void mma(float (&d)[4], const uint4& a, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}

// kN pairs of values of a head of q, from any element on; zeros for a head that is not there.
template <int kN>
__device__ __forceinline__ void load_q(const __nv_bfloat16* p, bool there, bool aligned, uint32_t (&w)[kN]) {
#pragma unroll
    for (int i = 0; i < kN; ++i) w[i] = 0;
    if (!there) return;
    if (aligned) {
#pragma unroll
        for (int i = 0; i < kN; i += 2) {
            const uint2 v = __ldg(reinterpret_cast<const uint2*>(p) + i / 2);
            w[i] = v.x, w[i + 1] = v.y;
        }
    } else {
        const unsigned short* s = reinterpret_cast<const unsigned short*>(p);
#pragma unroll
        for (int i = 0; i < kN; ++i)
            w[i] = static_cast<uint32_t>(__ldg(s + 2 * i)) | (static_cast<uint32_t>(__ldg(s + 2 * i + 1)) << 16);
    }
}

template <int kMT>
__global__ void __launch_bounds__(kThreads, kMT == 1 ? 2 : 1)
kv4_decode_narrow_kernel(const Operands op, const Division div, const NarrowScratch scratch) {
    extern __shared__ uint8_t smem_raw[];
    Shared<kMT>& sm = *reinterpret_cast<Shared<kMT>*>(smem_raw);
    constexpr int kRows = 16 * kMT;
    constexpr int kLanesRow = kThreads / kRows;      // softmax threads a row
    constexpr int kMine = kKeys / kLanesRow;         // entries a thread: 2 or 4
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int g = lane >> 2, c = lane & 3;
    const int d = warp >> 1, e = warp & 1;
    const int srow = tid / kLanesRow, skey = (tid % kLanesRow) * kMine;
    const int u0 = div.start(blockIdx.x), u1 = div.start(blockIdx.x + 1);
    const int padded = (op.heads + kRows - 1) / kRows * kRows;
    int32_t bits = 0;
    pdl_wait();

    // ---- copies: this warp's four rows of a tile, 26 lanes a row ----
    Walk ahead(div, u0);
    int ahead_token = ahead.row % op.tokens;
    auto slot_of_lane = [&]() -> int32_t {  // lane r < 4: the warp's row r of the tile ahead
        const int entry = ahead.tile * kKeys + warp * 4 + lane;
        if (lane >= 4 || ahead.u >= u1 || entry >= op.topk) return kNotFound;
        return __ldg(op.slots + ahead_token * op.slots_token + entry);
    };
    int32_t slot = slot_of_lane();
    const uint32_t copy_to = shared_address(sm.raw[0]) + warp * 4 * kRawRow + lane * 16;
    auto copy = [&](int stage) {
        if (ahead.u < u1) {
            const bool there = slot >= 0 && slot < op.pool_rows;
            if (!there && slot != kNotFound) bits |= ASU_ST_BAD_QUERY;
            const uint32_t valid = __ballot_sync(0xffffffffu, there);
            if (lane == 0) sm.there[stage][warp] = valid;
            const int32_t read = there ? slot : 0;  // an entry that is not there: zeros, finite values of weight 0
            const uint8_t* pool = op.pool + static_cast<uint64_t>(ahead_token) * op.pool_token + lane * 16;
            const uint32_t to = copy_to + stage * (kKeys * kRawRow);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const uint8_t* from = pool + static_cast<uint64_t>(__shfl_sync(0xffffffffu, read, r)) * op.pool_pitch;
                if (lane < kRowBytes / 16)
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + r * kRawRow), "l"(from),
                                 "r"((valid >> r) & 1u ? 16 : 0)
                                 : "memory");
            }
            const int row = ahead.row;
            ahead.next(div);
            if (ahead.row != row && ++ahead_token == op.tokens) ahead_token = 0;
            slot = slot_of_lane();
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll 1
    for (int i = 0; i < kStages - 1; ++i) copy(i);

    float o[kMT][16][4];            // [pair of latents 32 c + 2 b][heads g, g + 8]
    float m = -INFINITY, l = 0.0f;  // of row srow; l: this thread's entries
    int stage = 0;
    asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
    __syncthreads();

    for (Walk at(div, u0); at.u < u1; at.next(div)) {
        const bool first = at.u == u0 || at.tile == 0;
        const bool last = at.u + 1 == u1 || at.tile + 1 == div.tiles;
        const int token = at.row % op.tokens, head0 = at.row / op.tokens * kRows;
        if (first) {
            const __nv_bfloat16* qt = op.q + token * op.q_token;
#pragma unroll
            for (int t = 0; t < kMT; ++t) {
                const int h0 = head0 + 16 * t + g, h1 = h0 + 8;
                const __nv_bfloat16* q0 = qt + (h0 < op.heads ? h0 : 0) * op.q_head;
                const __nv_bfloat16* q1 = qt + (h1 < op.heads ? h1 : 0) * op.q_head;
                uint32_t a[8], b[8];
                load_q(q0 + d * 128 + c * 32 + e * 16, h0 < op.heads, op.q_aligned, a);
                load_q(q1 + d * 128 + c * 32 + e * 16, h1 < op.heads, op.q_aligned, b);
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    sm.q[t][8 * d + 4 * e + k][lane] = make_uint4(a[2 * k], b[2 * k], a[2 * k + 1], b[2 * k + 1]);
                if (e == 0) {
                    uint32_t x[2], y[2];
                    load_q(q0 + kLatent + d * 16 + c * 4, h0 < op.heads, op.q_aligned, x);
                    load_q(q1 + kLatent + d * 16 + c * 4, h1 < op.heads, op.q_aligned, y);
                    sm.rope[t][d][lane] = make_uint4(x[0], y[0], x[1], y[1]);
                }
            }
            __syncthreads();
#pragma unroll
            for (int t = 0; t < kMT; ++t)
#pragma unroll
                for (int b = 0; b < 16; ++b)
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[t][b][i] = 0.0f;
            m = -INFINITY;
            l = 0.0f;
        }

        // ---- dequantise, partial scores ----
        const uint8_t* raw = sm.raw[stage] + (16 * e + g) * kRawRow;
        uint32_t v[2][16];  // [8 entries][pairs of latents]
        float s[kMT][2][4];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const uint8_t* row = raw + 8 * j * kRawRow;
            const uint4 code = *reinterpret_cast<const uint4*>(row + d * 64 + c * 16);
            const uint32_t scales = *reinterpret_cast<const unsigned short*>(row + kScaleOffset + d * 8 + c * 2);
            const uint2 rope = *reinterpret_cast<const uint2*>(row + kRopeOffset + d * 32 + c * 8);
            __nv_bfloat162 sc, cc;
            scale_pair(scales, 0, sc, cc);
            unpack_word(code.x, sc, cc, &v[j][0]);
            unpack_word(code.y, sc, cc, &v[j][4]);
            scale_pair(scales, 1, sc, cc);
            unpack_word(code.z, sc, cc, &v[j][8]);
            unpack_word(code.w, sc, cc, &v[j][12]);
#pragma unroll
            for (int t = 0; t < kMT; ++t) {
#pragma unroll
                for (int i = 0; i < 4; ++i) s[t][j][i] = 0.0f;
                mma(s[t][j], sm.rope[t][d][lane], rope.x, rope.y);
            }
        }
#pragma unroll
        for (int k = 0; k < 8; ++k)
#pragma unroll
            for (int t = 0; t < kMT; ++t) {
                const uint4 a = sm.q[t][8 * d + k][lane];
#pragma unroll
                for (int j = 0; j < 2; ++j) mma(s[t][j], a, v[j][2 * k], v[j][2 * k + 1]);
            }
#pragma unroll
        for (int t = 0; t < kMT; ++t)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                float* to = &sm.part[d][16 * t + g][16 * e + 8 * j + 2 * c];
                *reinterpret_cast<float2*>(to) = make_float2(s[t][j][0], s[t][j][1]);
                *reinterpret_cast<float2*>(to + 8 * kPartRow) = make_float2(s[t][j][2], s[t][j][3]);
            }
        __syncthreads();
        copy(stage == 0 ? kStages - 1 : stage - 1);  // the tile before has been read

        // ---- softmax: kLanesRow threads a row ----
        float x[kMine];
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float* from = &sm.part[w][srow][skey];
            if constexpr (kMine == 2) {
                const float2 y = *reinterpret_cast<const float2*>(from);
                x[0] = w ? x[0] + y.x : y.x, x[1] = w ? x[1] + y.y : y.y;
            } else {
                const float4 y = *reinterpret_cast<const float4*>(from);
                x[0] = w ? x[0] + y.x : y.x, x[1] = w ? x[1] + y.y : y.y;
                x[2] = w ? x[2] + y.z : y.z, x[3] = w ? x[3] + y.w : y.w;
            }
        }
        const uint32_t there = sm.there[stage][skey >> 2] >> (skey & 3);
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < kMine; ++i) {
            x[i] = (there >> i) & 1u ? x[i] * op.scale_log2 : -INFINITY;
            top = fmaxf(top, x[i]);
        }
#pragma unroll
        for (int k = kLanesRow / 2; k > 0; k >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, k));
        float fade = 1.0f;
        if (first) {
            m = top;
        } else if (top > m + kMaxGrowth) {
            fade = exp2_fast(m - top);
            m = top;
            l *= fade;
        }
        const float from = m == -INFINITY ? 0.0f : m;
        uint32_t p[kMine / 2];
#pragma unroll
        for (int i = 0; i < kMine; i += 2) {
            const float a = exp2_fast(x[i] - from), b = exp2_fast(x[i + 1] - from);
            l += a + b;
            p[i / 2] = pack_bf16(a, b);
            *reinterpret_cast<uint32_t*>(&sm.weights[srow][skey + i]) = p[i / 2];
        }
        if (tid % kLanesRow == 0) sm.row[srow] = fade;
        if (op.weights != nullptr) {
            const int head = head0 + srow;
            uint32_t* to = reinterpret_cast<uint32_t*>(
                scratch.p + (static_cast<int64_t>(token) * padded + head) * div.tiles * kKeys + at.tile * kKeys + skey);
#pragma unroll
            for (int i = 0; i < kMine / 2; ++i) to[i] = p[i];
            if (tid % kLanesRow == 0) scratch.ref[(static_cast<int64_t>(token) * div.tiles + at.tile) * padded + head] = m;
        }
        asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");  // the next tile is here
        if (__syncthreads_or(fade != 1.0f)) {
#pragma unroll
            for (int t = 0; t < kMT; ++t) {
                const float f0 = sm.row[16 * t + g], f1 = sm.row[16 * t + g + 8];
#pragma unroll
                for (int b = 0; b < 16; ++b) o[t][b][0] *= f0, o[t][b][1] *= f0, o[t][b][2] *= f1, o[t][b][3] *= f1;
            }
        }

        // ---- output ----
        uint4 a[kMT];
#pragma unroll
        for (int t = 0; t < kMT; ++t)
            asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                         : "=r"(a[t].x), "=r"(a[t].y), "=r"(a[t].z), "=r"(a[t].w)
                         : "r"(shared_address(&sm.weights[16 * t + (lane & 15)][16 * e + (lane >> 4) * 8])));
#pragma unroll
        for (int b = 0; b < 16; ++b) {
            const uint32_t b0 = transpose8x8(v[0][b]), b1 = transpose8x8(v[1][b]);
#pragma unroll
            for (int t = 0; t < kMT; ++t) mma(o[t][b], a[t], b0, b1);
        }

        if (last) {
            // the two halves of the entries, 64 latents at a time, through q's place
            float4* half = reinterpret_cast<float4*>(sm.q);
#pragma unroll
            for (int t = 0; t < kMT; ++t)
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    __syncthreads();  // q, or the round before, has been read
                    if (e == 1)
#pragma unroll
                        for (int b = 0; b < 8; ++b) {
                            const float* x = o[t][8 * r + b];
                            half[(d * 8 + b) * 32 + lane] = make_float4(x[0], x[1], x[2], x[3]);
                        }
                    __syncthreads();
                    if (e == 0)
#pragma unroll
                        for (int b = 0; b < 8; ++b) {
                            const float4 x = half[(d * 8 + b) * 32 + lane];
                            float* y = o[t][8 * r + b];
                            y[0] += x.x, y[1] += x.y, y[2] += x.z, y[3] += x.w;
                        }
                }
#pragma unroll
            for (int k = kLanesRow / 2; k > 0; k >>= 1) l += __shfl_xor_sync(0xffffffffu, l, k);
            const int row_start = at.row * div.tiles;
            const bool whole = row_start >= u0 && row_start + div.tiles <= u1;
            const int piece = div.piece(blockIdx.x, row_start);
            if (tid % kLanesRow == 0) {
                if (whole) {
                    sm.row[srow] = l > 0.0f ? 1.0f / l : 0.0f;
                    if (head0 + srow < op.heads)
                        op.lse[static_cast<int64_t>(token) * op.heads + head0 + srow] =
                            l > 0.0f ? (m + log2f(l)) * 0.6931471805599453f : -INFINITY;
                } else {
                    scratch.ml[piece * 2 * kRows + srow] = m;
                    scratch.ml[(piece * 2 + 1) * kRows + srow] = l;
                }
            }
            __syncthreads();
            if (e == 0) {
#pragma unroll
                for (int t = 0; t < kMT; ++t)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const int r = 16 * t + 8 * i + g, h = head0 + r;
                        if (whole) {
                            if (h >= op.heads) continue;
                            const float f = sm.row[r];
                            uint4* to = reinterpret_cast<uint4*>(
                                op.out + (static_cast<int64_t>(token) * op.heads + h) * kLatent + d * 128 + c * 32);
#pragma unroll
                            for (int k = 0; k < 4; ++k) {
                                uint32_t w[4];
#pragma unroll
                                for (int b = 0; b < 4; ++b)
                                    w[b] = pack_bf16(o[t][4 * k + b][2 * i] * f, o[t][4 * k + b][2 * i + 1] * f);
                                to[k] = make_uint4(w[0], w[1], w[2], w[3]);
                            }
                        } else {
                            float4* to = reinterpret_cast<float4*>(
                                scratch.o + (static_cast<int64_t>(piece) * kRows + r) * kLatent + d * 128 + c * 32);
#pragma unroll
                            for (int b = 0; b < 8; ++b)
                                to[b] = make_float4(o[t][2 * b][2 * i], o[t][2 * b][2 * i + 1], o[t][2 * b + 1][2 * i],
                                                    o[t][2 * b + 1][2 * i + 1]);
                        }
                    }
            }
        }
        stage = stage + 1 == kStages ? 0 : stage + 1;
    }
    pdl_trigger();
    asm volatile("cp.async.wait_all;" ::: "memory");
    if (bits) flag_status(op.status, 0, bits);
}

// Joins the pieces of rows that several CTAs share, and sums the weights over the heads.
//   blocks y < heads: one head of a token, 4 latents a thread
//   other blocks:     256 entries: weights_j = sum_h p_hj 2^(ref_h - lse_h)
template <int kMT>
__global__ void __launch_bounds__(128)
kv4_finish_narrow_kernel(const Operands op, const Division div, const NarrowScratch scratch) {
    pdl_wait();
    pdl_trigger();
    constexpr int kRows = 16 * kMT;
    __shared__ float s_lse[ASU_KV4_MAX_HEADS];  // base 2
    const int token = blockIdx.x, tid = threadIdx.x;
    // maximum and sum (base 2) of a head over its pieces; the CTAs of its row
    auto total = [&](int head, int& i0, int& i1, float& m, float& l) {
        const int first = (head / kRows * op.tokens + token) * div.tiles;
        i0 = div.cta_of(first);
        i1 = div.cta_of(first + div.tiles - 1);
        if (i0 == i1) return;
        m = -INFINITY, l = 0.0f;
#pragma unroll 4
        for (int i = i0; i <= i1; ++i) m = fmaxf(m, scratch.ml[div.piece(i, first) * 2 * kRows + head % kRows]);
#pragma unroll 4
        for (int i = i0; i <= i1; ++i) {
            const float* ml = scratch.ml + div.piece(i, first) * 2 * kRows + head % kRows;
            l += ml[kRows] * (ml[0] == -INFINITY ? 0.0f : exp2_fast(ml[0] - m));
        }
    };
    if (static_cast<int>(blockIdx.y) < op.heads) {
        const int head = blockIdx.y;
        int i0, i1;
        float m, l;
        total(head, i0, i1, m, l);
        if (i0 == i1) return;  // written by its one CTA
        const int first = (head / kRows * op.tokens + token) * div.tiles;
        float4 acc = make_float4(0, 0, 0, 0);
#pragma unroll 4
        for (int i = i0; i <= i1; ++i) {
            const int piece = div.piece(i, first);
            const float pm = scratch.ml[piece * 2 * kRows + head % kRows];
            const float f = pm == -INFINITY ? 0.0f : exp2_fast(pm - m);
            const float4 v = reinterpret_cast<const float4*>(
                scratch.o + (static_cast<int64_t>(piece) * kRows + head % kRows) * kLatent)[tid];
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
    for (int head = tid; head < op.heads; head += 128) {  // the joining blocks may not have written them yet
        int i0, i1;
        float m, l;
        total(head, i0, i1, m, l);
        s_lse[head] = i0 == i1 ? op.lse[static_cast<int64_t>(token) * op.heads + head] * 1.4426950408889634f
                               : (l > 0.0f ? m + log2f(l) : -INFINITY);
    }
    __syncthreads();
    const int padded = (op.heads + kRows - 1) / kRows * kRows;
    const int e = (blockIdx.y - op.heads) * 256 + tid * 2;
    if (e >= op.topk) return;
    const float* ref = scratch.ref + (static_cast<int64_t>(token) * div.tiles + e / kKeys) * padded;
    const __nv_bfloat16* p = scratch.p + static_cast<int64_t>(token) * padded * div.tiles * kKeys + e;
    float a = 0.0f, b = 0.0f;
#pragma unroll 4
    for (int head = 0; head < op.heads; ++head) {
        const uint32_t w = *reinterpret_cast<const uint32_t*>(p + static_cast<int64_t>(head) * div.tiles * kKeys);
        const float f = s_lse[head] == -INFINITY ? 0.0f : exp2_fast(ref[head] - s_lse[head]);
        a = fmaf(__uint_as_float(w << 16), f, a);
        b = fmaf(__uint_as_float(w & 0xffff0000u), f, b);
    }
    op.weights[static_cast<int64_t>(token) * op.topk + e] = __float2bfloat16(a);
    if (e + 1 < op.topk) op.weights[static_cast<int64_t>(token) * op.topk + e + 1] = __float2bfloat16(b);
}

int64_t align256(int64_t x) { return (x + 255) / 256 * 256; }

int groups_of(int64_t heads) { return heads > 16 ? 2 : 1; }  // of 16 heads in a CTA

Division division(int64_t tokens, int64_t heads, int64_t topk, int sms) {
    const int rows = 16 * groups_of(heads);
    return Division((heads + rows - 1) / rows * tokens, topk > 0 ? (topk + kKeys - 1) / kKeys : 1,
                    rows == 16 ? 2 * sms : sms);
}

void layout(const Division& d, int64_t tokens, int64_t heads, bool weights, int64_t (&at)[5]) {
    const int64_t rows = 16 * groups_of(heads), padded = (heads + rows - 1) / rows * rows;
    at[0] = 0;
    at[1] = at[0] + align256(2ll * d.ctas * 2 * rows * 4);
    at[2] = at[1] + align256(2ll * d.ctas * rows * kLatent * 4);
    at[3] = at[2] + (weights ? align256(tokens * d.tiles * padded * 4) : 0);
    at[4] = at[3] + (weights ? tokens * padded * d.tiles * kKeys * 2 : 0);
}

template <int kMT>
int launch(cudaStream_t s, const Operands& op, void* workspace) {
    const Division d = division(op.tokens, op.heads, op.topk, asu_sm_count());
    int64_t at[5];
    layout(d, op.tokens, op.heads, op.weights != nullptr, at);
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    const NarrowScratch scratch = {reinterpret_cast<float*>(ws + at[0]), reinterpret_cast<float*>(ws + at[1]),
                                   reinterpret_cast<float*>(ws + at[2]), reinterpret_cast<__nv_bfloat16*>(ws + at[3])};
    int max_dynamic = 0;
    int rc = asu_max_dynamic_smem(reinterpret_cast<const void*>(kv4_decode_narrow_kernel<kMT>), &max_dynamic);
    if (rc != ASU_OK) return rc;
    if (max_dynamic < static_cast<int>(sizeof(Shared<kMT>))) return ASU_ERR_ARG;
    rc = launch_pdl(kv4_decode_narrow_kernel<kMT>, dim3(d.ctas), dim3(kThreads), sizeof(Shared<kMT>), s, op, d, scratch);
    bool shared_rows = false;  // does any row lie in several CTAs' ranges?
    for (int i = 1; i < d.ctas && !shared_rows; ++i) shared_rows = d.start(i) % d.tiles != 0;
    if (rc != ASU_OK || (!shared_rows && op.weights == nullptr)) return rc;
    return launch_pdl(kv4_finish_narrow_kernel<kMT>,
                      dim3(static_cast<unsigned>(op.tokens),
                           static_cast<unsigned>(op.heads + (op.weights != nullptr ? (op.topk + 255) / 256 : 0))),
                      dim3(128), 0, s, op, d, scratch);
}

}  // namespace

int64_t narrow_workspace(int64_t tokens, int64_t heads, int64_t topk, bool weights) {
    int64_t at[5];
    layout(division(tokens, heads, topk, asu_sm_count()), tokens, heads, weights, at);
    return at[4];
}

int launch_narrow(cudaStream_t s, const Operands& op, void* workspace) {
    return groups_of(op.heads) == 1 ? launch<1>(s, op, workspace) : launch<2>(s, op, workspace);
}

}  // namespace kv4
}  // namespace asu

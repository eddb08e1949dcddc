// Sparse decode attention over the 4-bit cache for few heads, on the warp-level tensor cores.
//
// With 16 heads a row of 416 bytes meets 35 KFLOP: memory bound, and the 128-row products of the
// tcgen05 kernel would be seven eighths padding.  m16n8k16 products take the heads as their 16 rows
// (kMT such groups of 16 in a CTA) and the entries (scores) or latents (output) as their columns.
//
// A CTA of 8 warps takes tiles of 32 entries.  Warp w owns the latents 64 w .. 64 w + 63, for the scores and
// for the output: it dequantises them once, into registers in the layout that the score products want
// (entry g = lane / 4 of 8, values 16 c .. 16 c + 15 with c = lane % 4: one 8-byte load and one
// scale), and turns the same registers into the output products' layout with movmatrix, a transposition
// of 8 x 8 values.  No dequantised value goes through shared memory.  The price is that each warp's
// scores are partial sums over its latents: they are added up through shared memory, by the threads
// that then do the softmax (16 threads a row with one group of heads, 8 with two).
//
// Which 16 values of a latent row a product's k index means is free as long as both operands agree: k
// index 2c, 2c + 1, 2c + 8, 2c + 9 of step s are the values 16 c + 4 s .. 16 c + 4 s + 3.
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
constexpr int kStages = 6;
constexpr int kRawTile = kKeys * kRowBytes;
constexpr int kPartRow = kKeys + 8;      // floats; 8 more than a multiple of 32: no bank conflicts
constexpr int kWeightRow = kKeys + 8;    // bf16
constexpr float kMaxGrowth = 8.0f;       // the maximum moves when it grows by more than 2^8

template <int kMT>
struct Shared {
    alignas(128) uint8_t raw[kStages][kRawTile];
    float part[8][16 * kMT][kPartRow];       // each warp's partial scores
    __nv_bfloat16 weights[16 * kMT][kWeightRow];
    uint4 rope[kMT][4][32];                  // q's rope part by product operand: [step][lane]
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

// 16 values of a head of q from any element on; zeros for a head that is not there.
__device__ __forceinline__ void load_q16(const __nv_bfloat16* p, bool there, bool aligned, uint32_t (&w)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = 0;
    if (!there) return;
    if (aligned) {
        const uint4 a = __ldg(reinterpret_cast<const uint4*>(p)), b = __ldg(reinterpret_cast<const uint4*>(p) + 1);
        w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w, w[4] = b.x, w[5] = b.y, w[6] = b.z, w[7] = b.w;
        return;
    }
    const unsigned short* s = reinterpret_cast<const unsigned short*>(p);
#pragma unroll
    for (int i = 0; i < 8; ++i)
        w[i] = static_cast<uint32_t>(__ldg(s + 2 * i)) | (static_cast<uint32_t>(__ldg(s + 2 * i + 1)) << 16);
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
    const int srow = tid / kLanesRow, skey = (tid % kLanesRow) * kMine;
    const int u0 = div.start(blockIdx.x), u1 = div.start(blockIdx.x + 1);
    const int padded = (op.heads + kRows - 1) / kRows * kRows;
    int32_t bits = 0;
    pdl_wait();

    // ---- copies: this warp's four rows of a tile, 26 lanes a row ----
    Walk ahead(div, u0);
    auto slot_of = [&](const Walk& w) -> int32_t {
        const int e = w.tile * kKeys + warp * 4 + lane;
        if (lane >= 4 || w.u >= u1 || e >= op.topk) return kNotFound;
        return __ldg(op.slots + (w.row % op.tokens) * op.slots_token + e);
    };
    int32_t slot = slot_of(ahead);
    auto copy = [&](int stage) {
        if (ahead.u < u1) {
            const bool there = slot >= 0 && slot < op.pool_rows;
            if (!there && slot != kNotFound) bits |= ASU_ST_BAD_QUERY;
            const uint32_t valid = __ballot_sync(0xffffffffu, there) & 15u;
            if (lane == 0) sm.there[stage][warp] = valid;
            const uint64_t pool = reinterpret_cast<uint64_t>(op.pool) + static_cast<uint64_t>(ahead.row % op.tokens) * op.pool_token +
                                  lane * 16;
            const uint32_t to = shared_address(sm.raw[stage]) + warp * 4 * kRowBytes + lane * 16;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int32_t s = __shfl_sync(0xffffffffu, slot, r);
                const bool t = (valid >> r) & 1u;  // an entry that is not there: zeros, finite values of weight 0
                const uint64_t from = pool + static_cast<uint64_t>(t ? s : 0) * op.pool_pitch;
                if (lane < kRowBytes / 16)
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + r * kRowBytes), "l"(from),
                                 "r"(t ? 16 : 0)
                                 : "memory");
            }
            ahead.next(div);
            slot = slot_of(ahead);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll 1
    for (int i = 0; i < kStages - 1; ++i) copy(i);

    uint32_t q[kMT][2][8];  // heads g and g + 8 of each group, this thread's 16 latents
    float o[kMT][8][4];     // [8 pairs of latents] heads g, g + 8
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
            for (int t = 0; t < kMT; ++t)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int h = head0 + 16 * t + 8 * i + g;
                    load_q16(qt + (h < op.heads ? h : 0) * op.q_head + warp * 64 + c * 16, h < op.heads, op.q_aligned, q[t][i]);
                }
            if (warp < kMT) {  // the rope part, warp t for group t; read behind the barrier below
                uint32_t r[2][8];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int h = head0 + 16 * warp + 8 * i + g;
                    load_q16(qt + (h < op.heads ? h : 0) * op.q_head + kLatent + c * 16, h < op.heads, op.q_aligned, r[i]);
                }
#pragma unroll
                for (int s = 0; s < 4; ++s)
                    sm.rope[warp][s][lane] = make_uint4(r[0][2 * s], r[1][2 * s], r[0][2 * s + 1], r[1][2 * s + 1]);
            }
            __syncthreads();
#pragma unroll
            for (int t = 0; t < kMT; ++t)
#pragma unroll
                for (int b = 0; b < 8; ++b)
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[t][b][i] = 0.0f;
            m = -INFINITY;
            l = 0.0f;
        }

        // ---- dequantise, partial scores ----
        const uint8_t* raw = sm.raw[stage];
        uint32_t v[4][8];  // [8 entries][pairs of latents]
        float s[kMT][4][4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint8_t* row = raw + (8 * j + g) * kRowBytes;
            const uint2 code = *reinterpret_cast<const uint2*>(row + warp * 32 + c * 8);
            __nv_bfloat162 sc, cc;
            scale_pair(row[kScaleOffset + warp * 4 + c], sc, cc);
            unpack_word(code.x, sc, cc, &v[j][0]);
            unpack_word(code.y, sc, cc, &v[j][4]);
#pragma unroll
            for (int t = 0; t < kMT; ++t) {
#pragma unroll
                for (int i = 0; i < 4; ++i) s[t][j][i] = 0.0f;
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    mma(s[t][j], make_uint4(q[t][0][2 * k], q[t][1][2 * k], q[t][0][2 * k + 1], q[t][1][2 * k + 1]),
                        v[j][2 * k], v[j][2 * k + 1]);
            }
        }
        {  // rope: warp w takes the entries 8 (w % 4) .. and two of the four steps
            const int j = warp & 3, k0 = (warp >> 2) * 2;
            const uint4 r = *reinterpret_cast<const uint4*>(raw + (8 * j + g) * kRowBytes + kRopeOffset + c * 32 + k0 * 8);
#pragma unroll
            for (int t = 0; t < kMT; ++t) {
                float x[4] = {};
                mma(x, sm.rope[t][k0][lane], r.x, r.y);
                mma(x, sm.rope[t][k0 + 1][lane], r.z, r.w);
#pragma unroll
                for (int jj = 0; jj < 4; ++jj)
                    if (jj == j)
#pragma unroll
                        for (int i = 0; i < 4; ++i) s[t][jj][i] += x[i];
            }
        }
#pragma unroll
        for (int t = 0; t < kMT; ++t)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                *reinterpret_cast<float2*>(&sm.part[warp][16 * t + g][8 * j + 2 * c]) = make_float2(s[t][j][0], s[t][j][1]);
                *reinterpret_cast<float2*>(&sm.part[warp][16 * t + g + 8][8 * j + 2 * c]) = make_float2(s[t][j][2], s[t][j][3]);
            }
        __syncthreads();
        copy(stage == 0 ? kStages - 1 : stage - 1);  // the tile before has been read

        // ---- softmax: kLanesRow threads a row ----
        float x[kMine];
#pragma unroll
        for (int i = 0; i < kMine; ++i) x[i] = 0.0f;
#pragma unroll
        for (int w = 0; w < 8; ++w) {
            const float* from = &sm.part[w][srow][skey];
            if constexpr (kMine == 2) {
                const float2 y = *reinterpret_cast<const float2*>(from);
                x[0] += y.x, x[1] += y.y;
            } else {
                const float4 y = *reinterpret_cast<const float4*>(from);
                x[0] += y.x, x[1] += y.y, x[2] += y.z, x[3] += y.w;
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
        for (int d = kLanesRow / 2; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
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
                for (int b = 0; b < 8; ++b) o[t][b][0] *= f0, o[t][b][1] *= f0, o[t][b][2] *= f1, o[t][b][3] *= f1;
            }
        }

        // ---- output ----
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            uint4 a[kMT];
#pragma unroll
            for (int t = 0; t < kMT; ++t)
                asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                             : "=r"(a[t].x), "=r"(a[t].y), "=r"(a[t].z), "=r"(a[t].w)
                             : "r"(shared_address(&sm.weights[16 * t + (lane & 15)][16 * k + (lane >> 4) * 8])));
#pragma unroll
            for (int b = 0; b < 8; ++b) {
                const uint32_t b0 = transpose8x8(v[2 * k][b]), b1 = transpose8x8(v[2 * k + 1][b]);
#pragma unroll
                for (int t = 0; t < kMT; ++t) mma(o[t][b], a[t], b0, b1);
            }
        }

        if (last) {
#pragma unroll
            for (int d = kLanesRow / 2; d > 0; d >>= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
            const int row_start = at.row * div.tiles;
            const bool whole = row_start >= u0 && row_start + div.tiles <= u1;
            __syncthreads();  // sm.row has been read
            if (whole) {
                if (tid % kLanesRow == 0) {
                    sm.row[srow] = l > 0.0f ? 1.0f / l : 0.0f;
                    if (head0 + srow < op.heads)
                        op.lse[static_cast<int64_t>(token) * op.heads + head0 + srow] =
                            l > 0.0f ? (m + log2f(l)) * 0.6931471805599453f : -INFINITY;
                }
                __syncthreads();
#pragma unroll
                for (int t = 0; t < kMT; ++t)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const int h = head0 + 16 * t + 8 * i + g;
                        if (h >= op.heads) continue;
                        const float f = sm.row[16 * t + 8 * i + g];
                        uint32_t w[8];
#pragma unroll
                        for (int b = 0; b < 8; ++b) w[b] = pack_bf16(o[t][b][2 * i] * f, o[t][b][2 * i + 1] * f);
                        uint4* to = reinterpret_cast<uint4*>(op.out + (static_cast<int64_t>(token) * op.heads + h) * kLatent +
                                                             warp * 64 + c * 16);
                        to[0] = make_uint4(w[0], w[1], w[2], w[3]);
                        to[1] = make_uint4(w[4], w[5], w[6], w[7]);
                    }
            } else {
                const int piece = div.piece(blockIdx.x, row_start);
                if (tid % kLanesRow == 0) {
                    scratch.ml[piece * 2 * kRows + srow] = m;
                    scratch.ml[(piece * 2 + 1) * kRows + srow] = l;
                }
#pragma unroll
                for (int t = 0; t < kMT; ++t)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        float4* to = reinterpret_cast<float4*>(
                            scratch.o + (static_cast<int64_t>(piece) * kRows + 16 * t + 8 * i + g) * kLatent + warp * 64 + c * 16);
#pragma unroll
                        for (int b = 0; b < 4; ++b)
                            to[b] = make_float4(o[t][2 * b][2 * i], o[t][2 * b][2 * i + 1], o[t][2 * b + 1][2 * i],
                                                o[t][2 * b + 1][2 * i + 1]);
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

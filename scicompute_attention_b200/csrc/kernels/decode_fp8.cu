// Paged decode attention (one query token per head) over the 8-bit KV cache of kv_fp8.cuh.
//
// Per (sequence, head): s_j = scale * q . k_j, out = sum_j exp(s_j) v_j / sum_j exp(s_j) over the sequence's tokens, with
// k_j = 2^e_j codes_j and v_j likewise. The one-launch form on clusters is that of the 16-bit cache (decode_common.cuh), the schedule
// and the merge of the parts do the same in less time; what differs is the pass over a piece of a sequence:
//
//   * bytes: 2 * (D + 1) per token and kv head, read once for all query heads of the kv head. 4 * D FLOPs per byte pair and
//     query head: at eight heads 16 FLOPs a byte, so the products run on the tensor cores and HBM stays the bound;
//   * a warp takes 32 tokens at a time (16 above D=128) - as many bytes as 16 tokens of a 16-bit cache - through its own ring of 16-byte
//     cp.async copies, no CTA barrier in the loop. The scales come with them in 4-byte copies (4 tokens of a page);
//   * the tokens are the rows of the products and the query heads their 8 columns, S^T = K Q^T and O^T = V^T P^T (m16n8k16), so
//     that a group of up to 8 heads wastes nothing (with the heads as rows half of each product would be padding). Codes go
//     from the ring to fp16 operands in registers: cvt for two codes at a time, exact. The order in which the products walk
//     along D and the rows of V^T is free, and chosen so that a lane's operands lie side by side in the ring (no ldmatrix, no
//     transposition of V: a byte permutation pairs two tokens' codes ahead of the cvt);
//   * the scale of K multiplies the scores in fp32; the scale of V multiplies V's codes in fp16, which is exact too (see
//     kv_fp8.cuh). Applied to P instead it would cost less, but P in fp16 has no range for it: 2^21 between two rows of V;
//   * bf16 queries become fp16 by a power of two per head that puts the largest at 2^14: exact but for numbers below 2^-28 of
//     it; P is rounded to fp16 (2^-11 of a weight; below 2^-14 of the largest one 2^-25 of that), V and K not at all. Sums and statistics are fp32.
//
// What bounds it: HBM where a call is long - 256 sequences of 512 to 8192 tokens (32 / 8 heads, D=128, 2.31 GB) 368 us = 6.3 TB/s, the
// slope over the length 6.9 (D=64 6.2; 4.9 with 16 heads to a kv head, where a warp's chain of products and exponentials counts: issue slots 51 % busy). Every
// other call pays 11 us that no byte moves in: 1.3 until a CTA knows its share, 1.2 until its first loads are out, 2 until they are there,
// 1 for the CTA's merge, 3 for the merge kernel, and 2 between the median CTA's end and the last one's.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "common.cuh"
#include "decode_common.cuh"
#include "decode_fp8_shares.cuh"
#include "kv_fp8.cuh"

namespace sca_b200 {
namespace {

struct Fp8Scales {
    const uint8_t* k;
    const uint8_t* v;
};

// kHi: more than 8 heads.
template <int D, bool kHi>
struct Fp8Geom {
    static constexpr int kTokens = D > 128 ? 16 : 32;  // of a warp's step
    static constexpr int kSpan = kWarps * kTokens;     // of the CTA's: the unit of the schedule (ops.py counts on it)
    // CTAs that stay on an SM: what the registers of O and Q leave room for (FP8 slots in ops.py counts on it)
    static constexpr int kCtas = D <= 64 ? 4 : kHi && D > 96 ? 2 : 3;

    static constexpr int kChunks = D / 16;  // 16-byte pieces of a row
    static constexpr int kTileBytes = kTokens * D;
    static constexpr int kStageBytes = 2 * kTileBytes + 2 * kTokens;  // K, V, scales of K, scales of V
    static constexpr int kStages = D <= 64 || kCtas == 2 ? 3 : 2;
    static constexpr int kWarpBytes = std::max(kStages * kStageBytes, MergeBytes<D>());  // a warp's ring, and then its results
    static constexpr int kSmemBytes = kWarps * kWarpBytes;
    static constexpr int kWordsK = D / 16;  // words of K (4 codes) a lane holds per row: its quarter of the row
    static constexpr int kWordsV = D / 32;  // words of V a lane holds per row: its eighth
    static_assert(D % 32 == 0 && D <= 256, "head_dim");
    static_assert(kCtas * (kSmemBytes + 1024) <= 233472, "shared memory of an SM");
};

// A phase of 8 lanes reads rows {r, r + 1} of K, 4 adjacent pieces each, or rows {r, r + 2, r + 4, r + 6} of V, 2 adjacent pieces.
template <int D>
__device__ __forceinline__ int PieceK(int row, int piece) { return D % 128 == 0 ? piece ^ ((row & 1) << 2) : piece; }
template <int D>
__device__ __forceinline__ int PieceV(int row, int piece) { return D % 128 == 0 ? piece ^ (((row >> 1) & 3) << 1) : piece; }

// The products as functions of their operands: not volatile, so that those of independent rows may overlap.
__device__ __forceinline__ void Mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// The transpose of an 8x8 matrix of 16-bit numbers spread over the warp as an operand is (row lane / 4, columns 2 * (lane % 4)).
__device__ __forceinline__ uint32_t Transpose8x8(uint32_t v) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}

// First code of word w of a lane's share of a K row (c = lane % 4): 16 codes in a row of 64, then 8 in what is left.
template <int D>
__device__ __forceinline__ int CodeK(int w, int c) { return w < 4 * (D / 64) ? (w / 4) * 64 + 16 * c + 4 * (w % 4) : (D / 64) * 64 + 8 * c + 4 * (w % 4); }
// The same of a V row (g = lane / 4): 16 codes in a row of 128, then an eighth of what is left.
template <int D>
__device__ __forceinline__ int CodeV(int w, int g) {
    return w < 4 * (D / 128) ? (w / 4) * 128 + 16 * g + 4 * (w % 4) : (D / 128) * 128 + (D % 128 / 8) * g + 4 * (w - 4 * (D / 128));
}
template <int D>
__device__ __forceinline__ void LoadK(const unsigned char* tile, int row, int c, uint32_t (&words)[D / 16]) {
#pragma unroll
    for (int i = 0; i < D / 64; ++i) {
        const uint4 v = *reinterpret_cast<const uint4*>(tile + row * D + PieceK<D>(row, 4 * i + c) * 16);
        words[4 * i] = v.x, words[4 * i + 1] = v.y, words[4 * i + 2] = v.z, words[4 * i + 3] = v.w;
    }
    if constexpr (D % 64 != 0) {
        const uint2 v = *reinterpret_cast<const uint2*>(tile + row * D + CodeK<D>(4 * (D / 64), c));
        words[4 * (D / 64)] = v.x, words[4 * (D / 64) + 1] = v.y;
    }
}
template <int D>
__device__ __forceinline__ void LoadV(const unsigned char* tile, int row, int g, uint32_t (&words)[D / 32]) {
    constexpr int kFull = D / 128;
#pragma unroll
    for (int i = 0; i < kFull; ++i) {
        const uint4 v = *reinterpret_cast<const uint4*>(tile + row * D + PieceV<D>(row, 8 * i + g) * 16);
        words[4 * i] = v.x, words[4 * i + 1] = v.y, words[4 * i + 2] = v.z, words[4 * i + 3] = v.w;
    }
    if constexpr (D % 128 == 64) {
        const uint2 v = *reinterpret_cast<const uint2*>(tile + row * D + CodeV<D>(4 * kFull, g));
        words[4 * kFull] = v.x, words[4 * kFull + 1] = v.y;
    } else {
#pragma unroll
        for (int w = 4 * kFull; w < D / 32; ++w) words[w] = *reinterpret_cast<const uint32_t*>(tile + row * D + CodeV<D>(w, g));
    }
}

// The end of a segment: MergeWarps of decode_common.cuh with the weights of the warps computed once per row and O four numbers at a
// time (at D=256 it took 6200 clocks of a segment the other way).
template <int D, int kWarpBytes, bool kToShared>
__device__ __forceinline__ void MergeFp8Warps(const ScaDecodeFwdParams& p, unsigned char* smem, const int64_t b, const int head0,
                                              const int nheads, const int slot) {
    __shared__ float weights[16][kWarps];
    __syncthreads();
    if (threadIdx.x < nheads) {
        const int row = threadIdx.x;
        float m[kWarps], m_all = -CUDART_INF_F, l_all = 0.0f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            m[w] = reinterpret_cast<const float*>(smem + w * kWarpBytes)[row];
            m_all = fmaxf(m_all, m[w]);
        }
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float weight = m[w] == -CUDART_INF_F ? 0.0f : Exp2(m[w] - m_all);
            weights[row][w] = weight;
            l_all += reinterpret_cast<const float*>(smem + w * kWarpBytes)[16 + row] * weight;
        }
        if (kToShared) {
            float* partial = CtaPartial<D>(smem);
            partial[row] = m_all;
            partial[16 + row] = l_all;
        } else {
            const int64_t flat = (b * p.num_heads + head0 + row) * p.num_splits + slot;
            p.partial_m[flat] = m_all * kLn2;  // in natural units, as the 16-bit cache's
            p.partial_l[flat] = l_all;
        }
    }
    __syncthreads();
    for (int item = threadIdx.x; item < nheads * (D / 4); item += kThreads) {
        const int row = item / (D / 4), d = item % (D / 4) * 4;
        float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float weight = weights[row][w];
            const float4 x = *reinterpret_cast<const float4*>(smem + w * kWarpBytes + (32 + row * D + d) * 4);  // zeros where a warp had no key
            acc.x = fmaf(x.x, weight, acc.x), acc.y = fmaf(x.y, weight, acc.y), acc.z = fmaf(x.z, weight, acc.z), acc.w = fmaf(x.w, weight, acc.w);
        }
        if (kToShared) *reinterpret_cast<float4*>(smem + (32 + row * D + d) * 4) = acc;
        else *reinterpret_cast<float4*>(p.partial_o + ((b * p.num_heads + head0 + row) * p.num_splits + slot) * D + d) = acc;
    }
    __syncthreads();  // the rings double as merge staging: nobody refills them before everyone has read
}

// Tokens [j_begin, j_end) of one (sequence, kv head, head chunk): see DecodeSegment in decode.cu. kHi: more than 8 heads.
template <typename T, int D, bool kHi, bool kToShared>
__device__ __forceinline__ void Fp8Segment(const ScaDecodeFwdParams& p, const Fp8Scales& scales, unsigned char* smem, const int64_t b,
                                           const int hk, const int hc, const int64_t j_begin, const int64_t j_end, const int slot) {
    using G = Fp8Geom<D, kHi>;
    constexpr int kTokens = G::kTokens, kRows = kTokens / 16;  // rows of products, 16 tokens each
    constexpr int kCols = kHi ? 2 : 1;                          // head columns of 8
    const int lane = threadIdx.x & 31;
    const int warp = threadIdx.x >> 5;
    const int g = lane >> 2;
    const int c = lane & 3;
    const int group = static_cast<int>(p.num_heads / p.num_kv_heads);
    const int head0 = hk * group + hc * 16;
    const int nheads = min(16, group - hc * 16);

    const int ntiles = j_end > j_begin ? static_cast<int>((j_end - j_begin + kTokens - 1) / kTokens) : 0;
    const int my_tiles = ntiles > warp ? (ntiles - warp + kWarps - 1) / kWarps : 0;

    const unsigned char* k_base = static_cast<const unsigned char*>(p.k) + hk * D;
    const unsigned char* v_base = static_cast<const unsigned char*>(p.v) + hk * D;
    const uint32_t row_pieces = static_cast<uint32_t>(p.num_kv_heads * G::kChunks);
    const int32_t* table_row = p.page_table + b * p.max_blocks_per_seq;
    const int block_size = static_cast<int>(p.block_size);
    const int64_t scale_row = fp8::ScaleRow(block_size);

    unsigned char* ring = smem + warp * G::kWarpBytes;
    const uint32_t ring_addr = SmemAddr(ring);

    // This lane's token of the tile whose table entry is fetched next, as (page of the sequence, offset in the page), moved on by the tokens
    // of the CTA's warps per tile without a division, and the entries of the next kAhead tiles: the first loads of a segment wait for
    // one entry, not for one after the other.
    const int token = lane % kTokens;
    constexpr int kStep = kWarps * kTokens, kAhead = G::kStages - 1;
    const int page_step = kStep / block_size, offset_step = kStep % block_size;
    const uint32_t first_token = static_cast<uint32_t>(j_begin) + warp * kTokens + token;  // lengths are below 2^31
    int page = static_cast<int>(first_token / block_size), offset = static_cast<int>(first_token) - page * block_size;
    int32_t entries[kAhead];
    auto fetch_entry = [&](int tl) -> int32_t {
        const bool in = first_token + static_cast<uint32_t>(tl) * kStep < static_cast<uint32_t>(j_end) && page < p.max_blocks_per_seq;
        const int32_t entry = in ? table_row[page] : -1;
        page += page_step;
        offset += offset_step;
        if (offset >= block_size) {
            offset -= block_size;
            ++page;
        }
        return entry;
    };
#pragma unroll
    for (int i = 0; i < kAhead; ++i) entries[i] = fetch_entry(i);

    // Issues the copies of this warp's `tl`-th tile into `stage`, tile after tile; returns which of its tokens there are.
    auto issue = [&](int tl, int stage) -> uint32_t {
        const int32_t phys = entries[0];
        const bool there = phys >= 0 && phys < p.num_kv_blocks;
        int at_offset = offset;  // in its page: `offset` is kAhead tiles ahead
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            at_offset -= offset_step;
            if (at_offset < 0) at_offset += block_size;
        }
        // place of the row in 16-byte pieces; pools stay below 2^32 of them
        const uint32_t at = there ? static_cast<uint32_t>(phys * block_size + at_offset) * row_pieces : 0u;
        const uint32_t k_stage = ring_addr + stage * G::kStageBytes;
        const uint32_t v_stage = k_stage + G::kTileBytes;
        const uint32_t mask = __ballot_sync(0xffffffffu, there);
        if (c == 0 && lane < kTokens) {
            // block_size is a multiple of 4, and so is the tile's first token: four tokens share a page and a word of scales
            const int64_t scales_at = there ? (static_cast<int64_t>(phys) * p.num_kv_heads + hk) * scale_row + at_offset : 0;
            CpAsync4(v_stage + G::kTileBytes + lane, scales.k + scales_at, there ? 4 : 0);
            CpAsync4(v_stage + G::kTileBytes + kTokens + lane, scales.v + scales_at, there ? 4 : 0);
        }
#pragma unroll
        for (int i = 0; i + 1 < kAhead; ++i) entries[i] = entries[i + 1];
        entries[kAhead - 1] = fetch_entry(tl + kAhead);
        auto copy = [&](auto whole) {
#pragma unroll
            for (int n = 0; n < kTokens * G::kChunks / 32; ++n) {
                const int item = lane + 32 * n;
                const int row = item / G::kChunks;
                const int piece = item % G::kChunks;
                const uint64_t from = static_cast<uint64_t>(__shfl_sync(0xffffffffu, at, row)) * 16u;
                const uint32_t k_dst = k_stage + row * D + PieceK<D>(row, piece) * 16, v_dst = v_stage + row * D + PieceV<D>(row, piece) * 16;
                const int bytes = decltype(whole)::value || ((mask >> row) & 1u) ? 16 : 0;
                CpAsync16(k_dst, k_base + piece * 16 + from, bytes);
                CpAsync16(v_dst, v_base + piece * 16 + from, bytes);
            }
        };
        if (mask == 0xffffffffu) copy(std::true_type{});
        else copy(std::false_type{});
        CpAsyncCommit();
        return mask;
    };

    // ---- running state of heads 8 * t + 2 * c, + 1; m_run in units of `unit`, which is positive ----
    float m_run[kCols][2], l_run[kCols][2];
    float o[kCols][2 * G::kWordsV][4];  // rows CodeV(w, g) + 2 * half, + 1 of O^T
#pragma unroll
    for (int t = 0; t < kCols; ++t) {
#pragma unroll
        for (int i = 0; i < 2; ++i) m_run[t][i] = -CUDART_INF_F, l_run[t][i] = 0.0f;
#pragma unroll
        for (int j = 0; j < 2 * G::kWordsV; ++j) {
#pragma unroll
            for (int e = 0; e < 4; ++e) o[t][j][e] = 0.0f;
        }
    }

    constexpr uint32_t kAllTokens = 0xffffffffu;  // 16 tokens to a tile: lanes 16 to 31 look at the same ones
    uint32_t masks[G::kStages - 1];
#pragma unroll
    for (int s = 0; s < G::kStages - 1; ++s) {
        masks[s] = 0;
        if (s < my_tiles) masks[s] = issue(s, s);
        else CpAsyncCommit();
    }

    // ---- queries: columns of B, heads 8 * t + g; `unit` turns a product of codes into a score in the log2 domain ----
    uint32_t qb[kCols][G::kWordsK][2];
    float unit[kCols][2];  // of heads 8 * t + 2 * c, + 1
    {
        const T* q_base = reinterpret_cast<const T*>(p.q) + b * p.q_stride.s_b;
        const float scale_log2 = p.scale * kLog2e;
#pragma unroll
        for (int t = 0; t < kCols; ++t) {
            const bool mine = 8 * t + g < nheads;
            const T* q_row = q_base + (head0 + 8 * t + g) * p.q_stride.s_h;
            float factor = 1.0f, amax = 0.0f;
#pragma unroll
            for (int w = 0; w < G::kWordsK; ++w) {
                const uint2 v = mine ? *reinterpret_cast<const uint2*>(q_row + CodeK<D>(w, c)) : make_uint2(0, 0);
                qb[t][w][0] = v.x, qb[t][w][1] = v.y;
                if constexpr (std::is_same<T, __nv_bfloat16>::value) {
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        amax = fmaxf(amax, fmaxf(fabsf(__uint_as_float(qb[t][w][i] << 16)), fabsf(__uint_as_float(qb[t][w][i] & 0xffff0000u))));
                    }
                }
            }
            if constexpr (std::is_same<T, __nv_bfloat16>::value) {
                amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
                amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
                // 2^14 over the power of two at or below amax; for numbers below 2^-112 (and rows of zeros) 2^126
                const int k = max(static_cast<int>(__float_as_uint(amax) >> 23) - 127, -112);
                const float to_half = fp8::PowerOfTwo(14 - k);
                factor = fp8::PowerOfTwo(k - 14 < -126 ? -126 : k - 14);
#pragma unroll
                for (int w = 0; w < G::kWordsK; ++w) {
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        qb[t][w][i] = Pack2<__half>(__uint_as_float(qb[t][w][i] << 16) * to_half, __uint_as_float(qb[t][w][i] & 0xffff0000u) * to_half);
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                // not 0, which would make NaN of a masked token's -inf: scores of tiny rows under a tiny scale are 0 either way
                unit[t][i] = fmaxf(__shfl_sync(0xffffffffu, factor, (2 * c + i) * 4) * scale_log2, fp8::PowerOfTwo(-126));
            }
        }
    }

    int stage = 0;
    for (int tl = 0; tl < my_tiles; ++tl) {
        CpAsyncWait<G::kStages - 2>();
        __syncwarp();
        const uint32_t cur = masks[0];
#pragma unroll
        for (int s = 0; s + 1 < G::kStages - 1; ++s) masks[s] = masks[s + 1];
        {
            const int nt = tl + G::kStages - 1;
            int nstage = stage + G::kStages - 1;
            if (nstage >= G::kStages) nstage -= G::kStages;
            uint32_t mk = 0;
            if (nt < my_tiles) mk = issue(nt, nstage);
            else CpAsyncCommit();
            masks[G::kStages - 2] = mk;
        }
        if (cur != 0) {
            const unsigned char *k_stage = ring + stage * G::kStageBytes, *v_stage = k_stage + G::kTileBytes;
            const unsigned char *k_scale = v_stage + G::kTileBytes, *v_scale = k_scale + kTokens;

            // S^T: tokens 16 * r + g (elements 0, 1: heads 2c, 2c + 1) and 16 * r + g + 8 (elements 2, 3)
            float s[kRows][kCols][4];
#pragma unroll
            for (int r = 0; r < kRows; ++r) {
                uint32_t lo[G::kWordsK], hi[G::kWordsK];
                LoadK<D>(k_stage, 16 * r + g, c, lo);
                LoadK<D>(k_stage, 16 * r + g + 8, c, hi);
#pragma unroll
                for (int t = 0; t < kCols; ++t) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[r][t][e] = 0.0f;
                }
#pragma unroll
                for (int w = 0; w < G::kWordsK; ++w) {
                    const uint32_t a0 = fp8::DecodeLow(lo[w]), a1 = fp8::DecodeLow(hi[w]), a2 = fp8::DecodeHigh(lo[w]), a3 = fp8::DecodeHigh(hi[w]);
#pragma unroll
                    for (int t = 0; t < kCols; ++t) Mma(s[r][t], a0, a1, a2, a3, qb[t][w][0], qb[t][w][1]);
                }
            }
#pragma unroll
            for (int i = 0; i < 2 * kRows; ++i) {  // tokens 8 * i + g
                const float k_unit = fp8::ScaleOf(k_scale[8 * i + g]);
#pragma unroll
                for (int t = 0; t < kCols; ++t) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) s[i / 2][t][2 * (i & 1) + h] *= k_unit;
                }
            }
            if (cur != kAllTokens) {
#pragma unroll
                for (int i = 0; i < 2 * kRows; ++i) {
                    if ((cur >> (8 * i + g)) & 1u) continue;
#pragma unroll
                    for (int t = 0; t < kCols; ++t) s[i / 2][t][2 * (i & 1)] = s[i / 2][t][2 * (i & 1) + 1] = -CUDART_INF_F;
                }
            }

            uint32_t pb[kCols][2 * kRows];  // P^T, columns of B: tokens 8 * i + 2 * c, + 1 of head 8 * t + g
#pragma unroll
            for (int t = 0; t < kCols; ++t) {
                float alpha[2];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float mx = fmaxf(s[0][t][h], s[0][t][2 + h]);
                    if constexpr (kRows == 2) mx = Max3(mx, s[kRows - 1][t][h], s[kRows - 1][t][2 + h]);
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                    const float m_new = fmaxf(m_run[t][h], mx);
                    const float shift = m_new == -CUDART_INF_F ? 0.0f : -__fmul_rn(m_new, unit[t][h]);
                    // the difference of the two shifts as they were rounded, so exactly 1 where the maximum stands still: a fused product
                    // leaves the rounding of the shift, up to 2^-24 of the score, which every tile would multiply l and O by again
                    alpha[h] = Exp2(__fadd_rn(__fmul_rn(m_run[t][h], unit[t][h]), shift));
                    m_run[t][h] = m_new;
                    float sum = 0.0f;
#pragma unroll
                    for (int i = 0; i < 2 * kRows; ++i) {
                        float& x = s[i / 2][t][2 * (i & 1) + h];
                        x = Exp2(fmaf(x, unit[t][h], shift));
                        sum += x;
                    }
                    l_run[t][h] = fmaf(l_run[t][h], alpha[h], sum);
                }
#pragma unroll
                for (int i = 0; i < 2 * kRows; ++i) pb[t][i] = Transpose8x8(Pack2<__half>(s[i / 2][t][2 * (i & 1)], s[i / 2][t][2 * (i & 1) + 1]));
                // the maximum of a long sequence hardly moves: O is touched where it does
                if (__any_sync(0xffffffffu, alpha[0] != 1.0f || alpha[1] != 1.0f)) {
#pragma unroll
                    for (int j = 0; j < 2 * G::kWordsV; ++j) {
                        o[t][j][0] *= alpha[0], o[t][j][1] *= alpha[1], o[t][j][2] *= alpha[0], o[t][j][3] *= alpha[1];
                    }
                }
            }

            // O^T += V^T P^T
#pragma unroll
            for (int r = 0; r < kRows; ++r) {
                const int row = 16 * r + 2 * c;
                uint32_t v0[G::kWordsV], v1[G::kWordsV], v8[G::kWordsV], v9[G::kWordsV];
                LoadV<D>(v_stage, row, g, v0);
                LoadV<D>(v_stage, row + 1, g, v1);
                LoadV<D>(v_stage, row + 8, g, v8);
                LoadV<D>(v_stage, row + 9, g, v9);
                uint32_t s01 = *reinterpret_cast<const uint16_t*>(v_scale + row), s89 = *reinterpret_cast<const uint16_t*>(v_scale + row + 8);
                if (cur != kAllTokens) {
                    // the scales come four at a time: those of tokens that do not count are anything, and infinity times 0 is not 0
                    const uint32_t there = cur >> row;
                    s01 &= ((there & 1u) ? 0xffu : 0u) | ((there & 2u) ? 0xff00u : 0u);
                    s89 &= ((there & 0x100u) ? 0xffu : 0u) | ((there & 0x200u) ? 0xff00u : 0u);
                }
                const uint32_t unit01 = fp8::ScalePair(s01, s01 >> 8), unit89 = fp8::ScalePair(s89, s89 >> 8);
#pragma unroll
                for (int w = 0; w < G::kWordsV; ++w) {
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        // two codes of each of two tokens, paired by code
                        const uint32_t p01 = __byte_perm(v0[w], v1[w], half ? 0x7362 : 0x5140);
                        const uint32_t p89 = __byte_perm(v8[w], v9[w], half ? 0x7362 : 0x5140);
                        const uint32_t a0 = fp8::MulHalf2(fp8::DecodeLow(p01), unit01), a1 = fp8::MulHalf2(fp8::DecodeHigh(p01), unit01);
                        const uint32_t a2 = fp8::MulHalf2(fp8::DecodeLow(p89), unit89), a3 = fp8::MulHalf2(fp8::DecodeHigh(p89), unit89);
#pragma unroll
                        for (int t = 0; t < kCols; ++t) Mma(o[t][2 * w + half], a0, a1, a2, a3, pb[t][2 * r], pb[t][2 * r + 1]);
                    }
                }
            }
        }
        __syncwarp();
        if (++stage == G::kStages) stage = 0;
    }
    CpAsyncWait<0>();
    __syncwarp();

    // ---- per-warp results -> this warp's (now idle) ring, then the CTA's merge ----
    float* stage_m = reinterpret_cast<float*>(ring);  // [16]
    float* stage_l = stage_m + 16;                    // [16]
    float* stage_o = stage_m + 32;                    // [16][D]
#pragma unroll
    for (int t = 0; t < kCols; ++t) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float l = l_run[t][h];
            l += __shfl_xor_sync(0xffffffffu, l, 4);
            l += __shfl_xor_sync(0xffffffffu, l, 8);
            l += __shfl_xor_sync(0xffffffffu, l, 16);
            const int head = 8 * t + 2 * c + h;
            // a maximum passes over NaN: where every score is NaN, so is l, and the merges must not take it for a part without a key
            const float m = m_run[t][h] != -CUDART_INF_F ? m_run[t][h] * unit[t][h] : l == l ? -CUDART_INF_F : 0.0f;
            if (g == 0) stage_m[head] = m, stage_l[head] = l;
#pragma unroll
            for (int w = 0; w < G::kWordsV; ++w) {
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    *reinterpret_cast<float2*>(stage_o + head * D + CodeV<D>(w, g) + 2 * half) = make_float2(o[t][2 * w + half][h], o[t][2 * w + half][2 + h]);
                }
            }
        }
    }
    MergeFp8Warps<D, G::kWarpBytes, kToShared>(p, smem, b, head0, nheads, slot);
}

// The schedule of decode_common.cuh (WalkSchedule: what it does and why) for lists of less than 2^31 steps, with borders that count, shares
// that differ by a step at most, lengths that are read once, and nothing divided in 64 bits. With the last two it took 3500 clocks until a
// CTA knew its share; a CTA's K/V is 30000 to 60000. Its arithmetic is in decode_fp8_shares.cuh.
template <int kSpan, typename Segment>
__device__ __forceinline__ void WalkFp8Schedule(const ScaDecodeFwdParams& p, const int head_chunks, const Segment& segment) {
    __shared__ int s_part[kWarps][2];
    __shared__ int s_found[2];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int columns = static_cast<int>(p.num_kv_heads) * head_chunks;
    const SchedulePlace place = PlaceOf(static_cast<int>(blockIdx.x), static_cast<int>(gridDim.x), columns);
    WaitForPredecessor();
    if (place.share >= place.sharers) return;  // a grid that is no multiple of the column count

    const int batch = static_cast<int>(p.batch), splits = static_cast<int>(p.num_splits);
    const int cap = static_cast<int>(p.max_blocks_per_seq * p.block_size < 0x7fffff00LL ? p.max_blocks_per_seq * p.block_size : 0x7fffff00LL);
    const int all = static_cast<int>(min(p.seq_kv, static_cast<int64_t>(cap)));  // without lengths
    auto length = [&](int i) { return max(0, min(p.seq_lens != nullptr ? p.seq_lens[i] : all, cap)); };
    // sequences [mine, end_mine) are this thread's
    const int each = (batch + kThreads - 1) / kThreads;
    const int mine = min(batch, static_cast<int>(threadIdx.x) * each), end_mine = min(batch, mine + each);
    int sum = 0, longest = 0;
    for (int i = mine; i < end_mine; ++i) {
        const int t = StepsOf(length(i), kSpan);
        sum += t;
        longest = max(longest, t);
    }
    const int border = BorderOf(__syncthreads_or(longest > 1) ? 2 : 1);
    sum += (end_mine - mine) * border;
    int up = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, up, o);
        if (lane >= o) up += x;
    }
    longest = __reduce_max_sync(0xffffffffu, longest);
    if (lane == 31) s_part[warp][0] = up, s_part[warp][1] = longest;
    __syncthreads();
    int total = 0, first = up - sum;  // steps of the list, and those ahead of this thread's sequences
    longest = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        if (w < warp) first += s_part[w][0];
        total += s_part[w][0];
        longest = max(longest, s_part[w][1]);
    }
    const Shares shares = ShareSteps(total, longest + border, splits, place.sharers);
    if (place.share >= shares.sharing) return;
    const int begin = shares.Begin(place.share);
    if (first <= begin && begin < first + sum) {
        int i = mine, before = first;
        FindSequence(begin, kSpan, border, length, &i, &before);
        s_found[0] = i;
        s_found[1] = before;
    }
    __syncthreads();
    const int b_first = s_found[0], before_first = s_found[1];
    // the merge kernel that follows on the stream may be set up while this grid streams K/V
    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");

    for (int column = place.column; column < columns; column += place.column_stride) {
        const int hk = column / head_chunks, hc = column % head_chunks;
        WalkShare(
            shares, place.share, kSpan, border, b_first, before_first, length,
            [&](int b, int64_t j_begin, int64_t j_end, int slot, bool bare) {
                if (bare) MarkUnusedSlots(p, b, hk, hc, slot, slot + 1);
                else segment(b, hk, hc, j_begin, j_end, slot);
            },
            [&](int b, int used) { MarkUnusedSlots(p, b, hk, hc, used, splits); });
    }
}

template <typename T, int D, bool kHi>
__global__ void __launch_bounds__(kThreads, Fp8Geom<D, kHi>::kCtas)
decode_fp8_partial_kernel(const ScaDecodeFwdParams p, const Fp8Scales scales, const int head_chunks) {
    extern __shared__ __align__(128) unsigned char smem[];
    WalkFp8Schedule<Fp8Geom<D, kHi>::kSpan>(p, head_chunks, [&](int64_t b, int hk, int hc, int64_t j_begin, int64_t j_end, int slot) {
        Fp8Segment<T, D, kHi, false>(p, scales, smem, b, hk, hc, j_begin, j_end, slot);
    });
}

template <typename T, int D, bool kHi>
__global__ void __launch_bounds__(kThreads, Fp8Geom<D, kHi>::kCtas)
decode_fp8_cluster_kernel(const ScaDecodeFwdParams p, const Fp8Scales scales, const int head_chunks, const int cluster) {
    extern __shared__ __align__(128) unsigned char smem[];
    ClusterDecode<T, D, true, Fp8Geom<D, kHi>::kSpan>(p, head_chunks, cluster, smem, [&](int64_t b, int hk, int hc, int64_t j_begin, int64_t j_end) {
        Fp8Segment<T, D, kHi, true>(p, scales, smem, b, hk, hc, j_begin, j_end, 0);
    });
}

// Merges the parts of a row: out = sum_s w_s O_s / sum_s w_s l_s with w_s = exp(m_s - max m). kWarps_ warps to a row, which take parts in
// turn, a lane 4 numbers of O at a time. Bound by latency: what a row takes is a chain of three loads from L2 (m, l and O), whose
// parts are all under way at once; one thread per number of O that goes through the parts one by one takes 17 us for the 54 parts of
// one sequence of 100 thousand tokens.
template <typename T, int D, int kRowWarps>
__global__ void __launch_bounds__(256)
decode_fp8_merge_kernel(const ScaDecodeFwdParams p) {
    constexpr int kLanes = D >= 128 ? 32 : D / 4;                       // that hold a row of O
    constexpr int kAtOnce = 32 % kLanes == 0 ? 32 / kLanes : 1;         // parts a warp takes in one turn
    constexpr int kVecs = (D + 127) / 128;                              // pieces of 4 numbers per lane
    __shared__ float4 others[kRowWarps > 1 ? 8 : 1][kVecs][kRowWarps > 1 ? 32 : 1];
    BeginAfterPredecessor();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * (8 / kRowWarps) + warp / kRowWarps;
    const int parts = static_cast<int>(p.num_splits);
    const bool there = row < p.batch * p.num_heads;
    const float *m = p.partial_m + row * parts, *l = p.partial_l + row * parts;
    float m_all = -CUDART_INF_F, l_all = 0.0f;
    for (int i = lane; i < parts && there; i += 32) m_all = fmaxf(m_all, m[i]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m_all = fmaxf(m_all, __shfl_xor_sync(0xffffffffu, m_all, o));
    for (int i = lane; i < parts && there; i += 32) {
        // a part without a key holds nothing but its m
        if (m[i] != -CUDART_INF_F) l_all = fmaf(l[i], Exp2((m[i] - m_all) * kLog2e), l_all);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) l_all += __shfl_xor_sync(0xffffffffu, l_all, o);
    float4 acc[kVecs];
#pragma unroll
    for (int v = 0; v < kVecs; ++v) acc[v] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    const int sub = kAtOnce > 1 ? lane / kLanes : 0, piece = kAtOnce > 1 ? lane % kLanes : lane;
#pragma unroll 4
    for (int s = (warp % kRowWarps) * kAtOnce + sub; s < parts && there; s += kRowWarps * kAtOnce) {
        const float m_part = m[s];
        const float w = m_part == -CUDART_INF_F ? 0.0f : Exp2((m_part - m_all) * kLog2e);
#pragma unroll
        for (int v = 0; v < kVecs; ++v) {
            const int d = v * 128 + piece * 4;
            if (D % 128 != 0 && d >= D) continue;
            float4 x = *reinterpret_cast<const float4*>(p.partial_o + (row * parts + s) * D + d);
            if (m_part == -CUDART_INF_F) x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);  // not written
            acc[v].x = fmaf(x.x, w, acc[v].x), acc[v].y = fmaf(x.y, w, acc[v].y), acc[v].z = fmaf(x.z, w, acc[v].z), acc[v].w = fmaf(x.w, w, acc[v].w);
        }
    }
#pragma unroll
    for (int v = 0; v < kVecs; ++v) {
#pragma unroll
        for (int o = kLanes; kAtOnce > 1 && o < 32; o <<= 1) {
            acc[v].x += __shfl_xor_sync(0xffffffffu, acc[v].x, o), acc[v].y += __shfl_xor_sync(0xffffffffu, acc[v].y, o);
            acc[v].z += __shfl_xor_sync(0xffffffffu, acc[v].z, o), acc[v].w += __shfl_xor_sync(0xffffffffu, acc[v].w, o);
        }
        if constexpr (kRowWarps > 1) others[warp][v][lane] = acc[v];
    }
    if constexpr (kRowWarps > 1) {
        __syncthreads();
        if (warp % kRowWarps != 0) return;
#pragma unroll
        for (int i = 1; i < kRowWarps; ++i) {
#pragma unroll
            for (int v = 0; v < kVecs; ++v) {
                const float4 x = others[warp + i][v][lane];
                acc[v].x += x.x, acc[v].y += x.y, acc[v].z += x.z, acc[v].w += x.w;
            }
        }
    }
    if (!there || sub != 0) return;
    const float inv = l_all > 0.0f ? 1.0f / l_all : 0.0f;
    T* out = reinterpret_cast<T*>(p.out) + row / p.num_heads * p.o_stride.s_b + row % p.num_heads * p.o_stride.s_h;
#pragma unroll
    for (int v = 0; v < kVecs; ++v) {
        const int d = v * 128 + piece * 4;
        if (d < D) *reinterpret_cast<uint2*>(out + d) = make_uint2(Pack2<T>(acc[v].x * inv, acc[v].y * inv), Pack2<T>(acc[v].z * inv, acc[v].w * inv));
    }
}

template <typename T, int D>
int LaunchFp8Merge(const ScaDecodeFwdParams& p, cudaStream_t stream) {
    const int64_t rows = p.batch * p.num_heads;
    if (p.num_splits <= 8 || rows > 8 * SmCount()) LaunchDependent(decode_fp8_merge_kernel<T, D, 1>, (rows + 7) / 8, 256, 0, stream, 1, p);
    else LaunchDependent(decode_fp8_merge_kernel<T, D, 8>, rows, 256, 0, stream, 1, p);
    return CheckLaunch("decode_fp8_merge_kernel", stream);
}

template <typename T, int D, bool kHi>
int64_t ResidentCtas() {
    static PerDevice per_sm;  // per instantiation
    const int n = per_sm.Get([] {
        int ctas = 0;
        const void* fn = reinterpret_cast<const void*>(&decode_fp8_partial_kernel<T, D, kHi>);
        if (EnsureDynamicSmem(fn, Fp8Geom<D, kHi>::kSmemBytes, "decode_fp8_partial_kernel") != SCA_OK ||
            cudaOccupancyMaxActiveBlocksPerMultiprocessor(&ctas, decode_fp8_partial_kernel<T, D, kHi>, kThreads, Fp8Geom<D, kHi>::kSmemBytes) != cudaSuccess ||
            ctas < 1) {
            cudaGetLastError();
            return -1;
        }
        return ctas;
    });
    return static_cast<int64_t>(SmCount()) * std::max(1, n);
}

template <typename T, int D, bool kHi>
int64_t ResidentClusters(int cluster) {
    static PerDevice resident[kMaxCluster + 1];  // per instantiation
    return std::max(0, resident[cluster].Get([cluster] {
        cudaLaunchAttribute attr{};
        cudaLaunchConfig_t cfg = ClusterConfig(static_cast<unsigned>(cluster), cluster, Fp8Geom<D, kHi>::kSmemBytes, nullptr, &attr);
        int n = 0;
        if (cudaOccupancyMaxActiveClusters(&n, decode_fp8_cluster_kernel<T, D, kHi>, &cfg) != cudaSuccess) {
            cudaGetLastError();
            return -1;
        }
        return n;
    }));
}

// Whether the one-launch kernel is the faster one for `units` (sequence, kv head, head chunk) columns of `steps` times 128 tokens (the
// longest) on clusters of `cluster` CTAs. Both times in us, fitted to 384 graph-timed calls on a B200 (D=64 to 256, 1 to 40 sequences of 60
// to 30 thousand tokens): a step of a CTA costs more the wider the head, the more heads share it and the more CTAs share the memory; the
// schedule works on what a ragged batch holds, a cluster waits for the longest sequence. One launch / schedule: D=128, 32 / 8 heads, B=1,
// S=800 5.6 / 9.1, S=12000 16.8 / 15.5, B=8, S=2000 12.9 / 14.3; D=256, 16 / 2, B=1, S=5000 16.5 / 14.8; D=64, 32 / 2, B=4, S=12000
// 18.0 / 15.8. The choices take 0.4 % longer than the faster of the two on average, 22 % at most (40 sequences of 60 tokens, 32 / 2 heads,
// D=128: 11.2 / 9.1).
bool OneLaunchIsFaster(int64_t units, int64_t steps, int cluster, int64_t resident, int head_dim, bool hi) {
    const double busy = static_cast<double>(units * cluster) / resident;
    const double share = static_cast<double>((steps + cluster - 1) / cluster);
    const double waves = static_cast<double>(units * steps) / resident;
    const double one_launch = 4.5 + share * (0.3 + 0.006 * head_dim + (hi ? 0.35 : 0.0) + 0.009 * head_dim * busy);
    return one_launch < 8.0 + 0.008 * head_dim + (hi ? 1.0 : 0.0) + 2.1 * std::sqrt(head_dim / 128.0) * (hi ? 1.3 : 1.0) * std::max(1.0, 0.8 * waves);
}

template <typename T, int D, bool kHi>
int LaunchFp8(const ScaDecodeFwdParams& p, const Fp8Scales& scales, int head_chunks, cudaStream_t stream, int* cluster_ctas) {
    using G = Fp8Geom<D, kHi>;
    const int64_t columns = p.num_kv_heads * head_chunks, units = p.batch * columns;
    const int64_t longest = std::max<int64_t>(1, std::min(p.seq_kv, p.max_blocks_per_seq * p.block_size));
    const int64_t resident = ResidentCtas<T, D, kHi>();
    if (int rc = EnsureDynamicSmem(reinterpret_cast<const void*>(&decode_fp8_cluster_kernel<T, D, kHi>), G::kSmemBytes, "decode_fp8_cluster_kernel")) return rc;
    // as many CTAs per cluster as let all clusters run at the same time
    int cluster = kMaxCluster;
    while (cluster >= 2 && units > ResidentClusters<T, D, kHi>(cluster)) cluster /= 2;
    if (cluster < 2 || !OneLaunchIsFaster(units, (longest + 127) / 128, cluster, resident, D, kHi)) cluster = 0;
    *cluster_ctas = cluster;
    if (cluster > 0) {
        LaunchDependent(decode_fp8_cluster_kernel<T, D, kHi>, units * cluster, kThreads, G::kSmemBytes, stream, cluster, p, scales, head_chunks, cluster);
        return CheckLaunch("decode_fp8_cluster_kernel", stream);
    }
    if (int rc = EnsureDynamicSmem(reinterpret_cast<const void*>(&decode_fp8_partial_kernel<T, D, kHi>), G::kSmemBytes, "decode_fp8_partial_kernel")) return rc;
    const int64_t blocks = ScheduleGrid(resident, columns, p.batch * ((longest + G::kSpan - 1) / G::kSpan));
    LaunchDependent(decode_fp8_partial_kernel<T, D, kHi>, blocks, kThreads, G::kSmemBytes, stream, 1, p, scales, head_chunks);
    if (int rc = CheckLaunch("decode_fp8_partial_kernel", stream)) return rc;
    return LaunchFp8Merge<T, D>(p, stream);
}

template <typename T, int D>
int LaunchFp8ForDim(const ScaDecodeFwdParams& p, const Fp8Scales& scales, cudaStream_t stream, int* cluster) {
    const int group = static_cast<int>(p.num_heads / p.num_kv_heads);
    const int head_chunks = (group + 15) / 16;
    return group > 8 ? LaunchFp8<T, D, true>(p, scales, head_chunks, stream, cluster) : LaunchFp8<T, D, false>(p, scales, head_chunks, stream, cluster);
}

template <typename T>
int LaunchFp8Typed(const ScaDecodeFwdParams& p, const Fp8Scales& scales, cudaStream_t stream, int* cluster) {
    switch (p.head_dim) {
        case 32: return LaunchFp8ForDim<T, 32>(p, scales, stream, cluster);
        case 64: return LaunchFp8ForDim<T, 64>(p, scales, stream, cluster);
        case 96: return LaunchFp8ForDim<T, 96>(p, scales, stream, cluster);
        case 128: return LaunchFp8ForDim<T, 128>(p, scales, stream, cluster);
        case 160: return LaunchFp8ForDim<T, 160>(p, scales, stream, cluster);
        case 192: return LaunchFp8ForDim<T, 192>(p, scales, stream, cluster);
        case 256: return LaunchFp8ForDim<T, 256>(p, scales, stream, cluster);
        default: break;
    }
    return Fail(SCA_INVALID_ARGUMENT, "paged attention (fp8): head_dim=" + std::to_string(p.head_dim) + " is not instantiated");
}

}  // namespace
}  // namespace sca_b200

using namespace sca_b200;

extern "C" int sca_launch_paged_attention_fp8(const ScaDecodeFwdParams* params, const uint8_t* k_scales, const uint8_t* v_scales,
                                              int32_t* cluster_ctas, void* stream) {
    ClearError();
    if (params == nullptr) return Fail(SCA_INVALID_ARGUMENT, "paged attention (fp8): null parameter block");
    const ScaDecodeFwdParams& p = *params;
    if (p.q == nullptr || p.k == nullptr || p.v == nullptr || p.out == nullptr || p.partial_m == nullptr || p.partial_l == nullptr ||
        p.partial_o == nullptr || p.page_table == nullptr || k_scales == nullptr || v_scales == nullptr) {
        return Fail(SCA_INVALID_ARGUMENT, "paged attention (fp8): null pointer");
    }
    if (p.dtype != SCA_DTYPE_F16 && p.dtype != SCA_DTYPE_BF16) {
        return Fail(SCA_INVALID_ARGUMENT, "paged attention (fp8): queries are fp16 or bf16 (dtype id " + std::to_string(p.dtype) + ")");
    }
    if (p.num_splits < 1 || p.batch < 1 || p.num_heads < 1 || p.num_kv_heads < 1 || p.num_heads % p.num_kv_heads != 0) {
        return Fail(SCA_INVALID_ARGUMENT, "paged attention (fp8): invalid geometry batch=" + std::to_string(p.batch) + " heads=" +
                                              std::to_string(p.num_heads) + " kv_heads=" + std::to_string(p.num_kv_heads));
    }
    if (!(p.scale > 0.0f) || !std::isfinite(p.scale)) {  // the kernel's `unit` is positive, and a maximum of scores one of products
        return Fail(SCA_INVALID_ARGUMENT, "paged attention (fp8): scale must be > 0 and finite");
    }
    if (p.num_kv_blocks > 0 && p.block_size > 0 && p.num_kv_heads * p.head_dim / 16 > 0xffffffffLL / std::max<int64_t>(1, p.num_kv_blocks * p.block_size)) {
        return Fail(SCA_INVALID_ARGUMENT, "paged attention (fp8): a pool of more than 64 GiB");
    }
    if (p.block_size <= 0 || p.block_size % 4 != 0 || p.max_blocks_per_seq <= 0 || p.num_kv_blocks <= 0 || p.num_kv_blocks * p.block_size > 0x7fffffffLL) {
        return Fail(SCA_INVALID_ARGUMENT, "paged attention (fp8): block_size=" + std::to_string(p.block_size) +
                                              " (a multiple of 4), and a pool and a table that are not empty nor beyond 2^31 tokens");
    }
    if (p.num_splits > 0x10000 || p.batch * (p.max_blocks_per_seq * p.block_size / 64 + 1 + kBorder) > 0x7fff0000LL || p.batch > 0x7fffff) {
        return Fail(SCA_INVALID_ARGUMENT, "paged attention (fp8): num_splits=" + std::to_string(p.num_splits) + ", batch=" + std::to_string(p.batch) +
                                              ": more work than the schedule counts");
    }
    if ((reinterpret_cast<uintptr_t>(p.out) | reinterpret_cast<uintptr_t>(p.partial_o) | static_cast<uintptr_t>(p.o_stride.s_b * 2) |
         static_cast<uintptr_t>(p.o_stride.s_h * 2)) % 8 != 0 || !Aligned16(p.partial_o)) {
        return Fail(SCA_INVALID_ARGUMENT, "paged attention (fp8): out must be 8-byte aligned with strides that are multiples of 4 elements, "
                                          "partial_o 16-byte aligned");
    }
    if (!Aligned16(p.q) || !Aligned16(p.k) || !Aligned16(p.v) || p.q_stride.s_b % 8 != 0 || p.q_stride.s_h % 8 != 0 ||
        (reinterpret_cast<uintptr_t>(k_scales) | reinterpret_cast<uintptr_t>(v_scales)) % 4 != 0) {
        return Fail(SCA_INVALID_ARGUMENT, "paged attention (fp8): q and codes must be 16-byte aligned, scales 4-byte aligned, "
                                          "strides of q multiples of 8 elements");
    }
    const Fp8Scales scales{k_scales, v_scales};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    int cluster = 0;
    const int rc = p.dtype == SCA_DTYPE_F16 ? LaunchFp8Typed<__half>(p, scales, s, &cluster) : LaunchFp8Typed<__nv_bfloat16>(p, scales, s, &cluster);
    if (cluster_ctas != nullptr) *cluster_ctas = cluster;
    return rc;
}

// What a warp of the decode kernels of a 16-bit cache does with a piece of a sequence (see decode.cu for the plan). The kernels of
// decode_weights.cu run the same lines.
#pragma once

#include <type_traits>

#include "common.cuh"
#include "decode_common.cuh"

namespace sca_b200 {
namespace {

constexpr int kTile = 16;   // tokens per warp step (k extent of the P.V product)
constexpr int kStages = 3;  // ring depth per warp

template <int D>
struct DecodeGeom {
    static constexpr int kRowBytes = D * 2;
    static constexpr int kChunksPerRow = kRowBytes / 16;
    static constexpr bool kSwizzle = (kChunksPerRow % 8) == 0;
    static constexpr int kTileBytes = kTile * kRowBytes;
    static constexpr int kStageBytes = 2 * kTileBytes;  // K tile then V tile
    static constexpr int kWarpBytes = kStages * kStageBytes;
    static constexpr int kSmemBytes = kWarps * kWarpBytes;
    static constexpr int kKRounds = D / 32;         // 16-byte K loads per lane and token tile half
    static constexpr int kVRounds = (D + 63) / 64;  // groups of eight n8 output tiles
    static_assert(D % 32 == 0, "head_dim must be a multiple of 32");
    static_assert(kWarpBytes >= MergeBytes<D>(), "merge staging and the CTA's partial must fit in a warp's ring");
};

__device__ __forceinline__ float2 Unpack2Bf16(uint32_t v) {
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}

// K fragments: a phase of 8 lanes reads rows {r, r+1} x 4 adjacent chunks -> flip bit 2 on odd rows.
template <bool kSwizzle>
__device__ __forceinline__ int SwizzleK(int row, int chunk) {
    return kSwizzle ? (chunk ^ ((row & 1) << 2)) : chunk;
}
// V fragments: a phase of 8 lanes reads rows {r, r+2, r+4, r+6} x 2 adjacent chunks.
template <bool kSwizzle>
__device__ __forceinline__ int SwizzleV(int row, int chunk) {
    return kSwizzle ? (chunk ^ (((row >> 1) & 3) << 1)) : chunk;
}

// Tokens one CTA consumes per step: every warp takes one 16-token tile.
constexpr int kSpan = kWarps * kTile;

// What else a kernel wants of a segment's scores: nothing.
struct NoTap {
    static constexpr bool kTaken = false;
};
// The scores themselves, in the log2 domain and -inf where a token does not exist: [(sequence * heads + head) * row + token], rows of a
// multiple of kTile floats.
struct ScoreTap {
    static constexpr bool kTaken = true;
    float* scores;
    int64_t row;
};

// kLog2: ends with MergeWarpsLog2.
// One segment = tokens [j_begin, j_end) of one (sequence, kv head, head chunk): streams K/V once, keeps the running
// softmax state of up to 16 query heads, and leaves one (m, l, O) partial per head: in `slot` of the partial arrays, or
// (kToShared) in this CTA's shared memory (see MergeWarps): m[16] in the log2 domain, l[16], O[16][D].
template <typename T, int D, bool kPaged, bool kHi, bool kToShared = false, typename Tap = NoTap, bool kLog2 = false>
__device__ __forceinline__ void DecodeSegment(const ScaDecodeFwdParams& p, unsigned char* smem, const int64_t b,
                                              const int hk, const int hc, const int64_t j_begin, const int64_t j_end,
                                              const int slot, const Tap& tap = Tap{}) {
    using G = DecodeGeom<D>;
    constexpr int CPR = G::kChunksPerRow;
    // bf16 keeps 8 bits of a probability: rounding P alone would cost about 1e-3 of relative L2 error in the output.
    // The kernel is bound by HBM, not by the tensor pipe, so P goes into the P V product as two bf16 terms.
    constexpr bool kSplitP = std::is_same<T, __nv_bfloat16>::value;
    const int lane = threadIdx.x & 31;
    const int warp = threadIdx.x >> 5;
    const int g = lane >> 2;  // fragment row / token slot
    const int c = lane & 3;   // fragment column pair
    const int group = static_cast<int>(p.num_heads / p.num_kv_heads);
    const int head0 = hk * group + hc * 16;
    const int nheads = min(16, group - hc * 16);

    const int ntiles = j_end > j_begin ? static_cast<int>((j_end - j_begin + kTile - 1) / kTile) : 0;
    const int my_tiles = ntiles > warp ? (ntiles - warp + kWarps - 1) / kWarps : 0;

    // ---- query fragments (A operand), rows = heads of this chunk -----------------------------
    uint32_t qa[G::kKRounds][2][4];
    {
        const T* q_base = reinterpret_cast<const T*>(p.q) + b * p.q_stride.s_b;
#pragma unroll
        for (int i = 0; i < G::kKRounds; ++i) {
            uint4 lo = make_uint4(0, 0, 0, 0), hi = make_uint4(0, 0, 0, 0);
            if (g < nheads) {
                lo = *reinterpret_cast<const uint4*>(q_base + (head0 + g) * p.q_stride.s_h + 32 * i + 8 * c);
            }
            if (kHi && g + 8 < nheads) {
                hi = *reinterpret_cast<const uint4*>(q_base + (head0 + g + 8) * p.q_stride.s_h + 32 * i + 8 * c);
            }
            qa[i][0][0] = lo.x; qa[i][0][2] = lo.y; qa[i][1][0] = lo.z; qa[i][1][2] = lo.w;
            qa[i][0][1] = hi.x; qa[i][0][3] = hi.y; qa[i][1][1] = hi.z; qa[i][1][3] = hi.w;
        }
    }

    const unsigned char* k_base = reinterpret_cast<const unsigned char*>(p.k) +
                                  ((kPaged ? 0 : b * p.k_stride.s_b) + hk * p.k_stride.s_h) * 2;
    const unsigned char* v_base = reinterpret_cast<const unsigned char*>(p.v) +
                                  ((kPaged ? 0 : b * p.v_stride.s_b) + hk * p.v_stride.s_h) * 2;
    const int64_t k_row_bytes = p.k_stride.s_s * 2;
    const int64_t v_row_bytes = p.v_stride.s_s * 2;
    const int32_t* table_row =
        kPaged ? p.page_table + b * p.max_blocks_per_seq : nullptr;

    unsigned char* ring = smem + warp * G::kWarpBytes;
    const uint32_t ring_addr = SmemAddr(ring);

    // Paged: this lane's token of the next tile to be issued, as (page of the sequence, offset in the page), moved on by
    // kSpan tokens per tile without a division, and the page's table entry, fetched one tile ahead so that the copies do
    // not wait for it.
    int64_t page = 0, page_step = 0;
    int offset = 0, offset_step = 0, block_size = 1;
    int32_t phys_next = -1;
    auto fetch_entry = [&](int64_t jt) {
        phys_next = (lane < kTile && jt < j_end && page < p.max_blocks_per_seq) ? table_row[page] : -1;
    };
    if (kPaged) {
        block_size = static_cast<int>(p.block_size);
        const int64_t jt = j_begin + warp * kTile + (lane & (kTile - 1));
        page = jt / block_size;
        offset = static_cast<int>(jt - page * block_size);
        page_step = kSpan / block_size;
        offset_step = kSpan % block_size;
        fetch_entry(jt);
    }

    uint64_t policy = 0;  // Tap: K and V leave the cache to the scores, which are read again
    if constexpr (Tap::kTaken) policy = EvictFirstPolicy();
    // Issues the copies of this warp's `tl`-th tile into `stage`, tile after tile; returns the 16-bit token validity.
    auto issue = [&](int tl, int stage) -> uint32_t {
        const int64_t jt = j_begin + static_cast<int64_t>(warp + tl * kWarps) * kTile + (lane & (kTile - 1));
        int prow = -1;  // row of the pool / the K/V slab; pools stay below 2^31 rows
        if (kPaged) {
            if (phys_next >= 0 && phys_next < p.num_kv_blocks) prow = phys_next * block_size + offset;
            page += page_step;
            offset += offset_step;
            if (offset >= block_size) {
                offset -= block_size;
                ++page;
            }
            fetch_entry(jt + kSpan);
        } else if (lane < kTile && jt < j_end) {
            prow = static_cast<int>(jt);
        }
        const uint32_t mask = __ballot_sync(0xffffffffu, prow >= 0) & 0xffffu;
        const uint32_t k_stage = ring_addr + stage * G::kStageBytes;
        const uint32_t v_stage = k_stage + G::kTileBytes;
#pragma unroll
        for (int n = 0; n < (kTile * CPR) / 32; ++n) {
            const int item = lane + 32 * n;
            const int row = item / CPR;
            const int ch = item % CPR;
            const int pr = __shfl_sync(0xffffffffu, prow, row);
            const int bytes = pr >= 0 ? 16 : 0;
            const int64_t r = pr >= 0 ? pr : 0;
            const uint32_t k_dst = k_stage + row * G::kRowBytes + SwizzleK<G::kSwizzle>(row, ch) * 16;
            const uint32_t v_dst = v_stage + row * G::kRowBytes + SwizzleV<G::kSwizzle>(row, ch) * 16;
            if constexpr (Tap::kTaken) {
                CpAsync16(k_dst, k_base + r * k_row_bytes + ch * 16, bytes, policy);
                CpAsync16(v_dst, v_base + r * v_row_bytes + ch * 16, bytes, policy);
            } else {
                CpAsync16(k_dst, k_base + r * k_row_bytes + ch * 16, bytes);
                CpAsync16(v_dst, v_base + r * v_row_bytes + ch * 16, bytes);
            }
        }
        CpAsyncCommit();
        return mask;
    };

    // ---- running state: rows g (index 0) and g + 8 (index 1); scores live in the log2 domain ----
    float m_run[2] = {-CUDART_INF_F, -CUDART_INF_F};
    float l_run[2] = {0.0f, 0.0f};
    float o[G::kVRounds][8][4];
#pragma unroll
    for (int r = 0; r < G::kVRounds; ++r)
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[r][j][e] = 0.0f;
    const float scale_log2 = p.scale * kLog2e;

    float* scores_to = nullptr;  // Tap: where this lane's scores of its next tile go, and how far up those of row g + 8 are
    int64_t scores_up = 0;
    if constexpr (Tap::kTaken) {
        scores_to = tap.scores + (b * p.num_heads + head0 + g) * tap.row + j_begin + warp * kTile + 2 * c;
        scores_up = 8 * tap.row;
    }

    uint32_t mask_queue = 0;
#pragma unroll
    for (int s = 0; s < kStages - 1; ++s) {
        uint32_t mk = 0;
        if (s < my_tiles) mk = issue(s, s);
        else CpAsyncCommit();
        mask_queue |= mk << (16 * s);
    }

    int stage = 0;
    for (int tl = 0; tl < my_tiles; ++tl) {
        CpAsyncWait<kStages - 2>();
        __syncwarp();
        {
            const int nt = tl + kStages - 1;
            int nstage = stage + kStages - 1;
            if (nstage >= kStages) nstage -= kStages;
            uint32_t mk = 0;
            if (nt < my_tiles) mk = issue(nt, nstage);
            else CpAsyncCommit();
            const uint32_t cur = mask_queue & 0xffffu;
            mask_queue = (mask_queue >> 16) | (mk << 16);
            // rows g and g + 8 of the 16 scores: a lane has tokens 2c, 2c + 1 and 8 + 2c, 9 + 2c
            auto store_scores = [&](const float (&s)[2][4]) {
                if constexpr (Tap::kTaken) {
                    if (g < nheads) {
                        *reinterpret_cast<float2*>(scores_to) = make_float2(s[0][0], s[0][1]);
                        *reinterpret_cast<float2*>(scores_to + 8) = make_float2(s[1][0], s[1][1]);
                    }
                    if (kHi && g + 8 < nheads) {
                        *reinterpret_cast<float2*>(scores_to + scores_up) = make_float2(s[0][2], s[0][3]);
                        *reinterpret_cast<float2*>(scores_to + scores_up + 8) = make_float2(s[1][2], s[1][3]);
                    }
                    scores_to += kSpan;
                }
            };
            if constexpr (Tap::kTaken) {
                if (cur == 0) {
                    const float none = -CUDART_INF_F;
                    const float hidden[2][4] = {{none, none, none, none}, {none, none, none, none}};
                    store_scores(hidden);
                }
            }
            if (cur != 0) {
                const uint32_t k_stage = ring_addr + stage * G::kStageBytes;
                const uint32_t v_stage = k_stage + G::kTileBytes;

                // S = Q K^T for 16 tokens: two n8 tiles
                float s[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
                for (int i = 0; i < G::kKRounds; ++i) {
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        const int row = 8 * t + g;
                        const uint4 kr = LdsV4(k_stage + row * G::kRowBytes +
                                               SwizzleK<G::kSwizzle>(row, 4 * i + c) * 16);
                        MmaM16N8K16<T>(s[t], qa[i][0][0], qa[i][0][1], qa[i][0][2], qa[i][0][3], kr.x, kr.y);
                        MmaM16N8K16<T>(s[t], qa[i][1][0], qa[i][1][1], qa[i][1][2], qa[i][1][3], kr.z, kr.w);
                    }
                }
                // scale, mask, online softmax
#pragma unroll
                for (int t = 0; t < 2; ++t) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const bool ok = (cur >> (8 * t + 2 * c + (e & 1))) & 1u;
                        s[t][e] = ok ? s[t][e] * scale_log2 : -CUDART_INF_F;
                    }
                }
                store_scores(s);
                uint32_t pa[4], pb[4];
                float alpha[2];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    if (h == 1 && !kHi) {
                        alpha[1] = 1.0f;
                        pa[1] = 0u;
                        pa[3] = 0u;
                        pb[1] = 0u;
                        pb[3] = 0u;
                        continue;
                    }
                    float mx = fmaxf(fmaxf(s[0][2 * h], s[0][2 * h + 1]), fmaxf(s[1][2 * h], s[1][2 * h + 1]));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                    const float m_new = fmaxf(m_run[h], mx);
                    const float m_safe = (m_new == -CUDART_INF_F) ? 0.0f : m_new;
                    alpha[h] = Exp2(m_run[h] - m_safe);
                    const float p00 = Exp2(s[0][2 * h] - m_safe);
                    const float p01 = Exp2(s[0][2 * h + 1] - m_safe);
                    const float p10 = Exp2(s[1][2 * h] - m_safe);
                    const float p11 = Exp2(s[1][2 * h + 1] - m_safe);
                    l_run[h] = l_run[h] * alpha[h] + (p00 + p01) + (p10 + p11);
                    m_run[h] = m_new;
                    pa[h] = Pack2<T>(p00, p01);      // rows g / g+8, tokens 2c, 2c+1
                    pa[2 + h] = Pack2<T>(p10, p11);  // tokens 8+2c, 8+2c+1
                    if (kSplitP) {
                        // what the 8-bit mantissa dropped, as a second bf16 operand: P = P_hi + P_lo to 2^-16
                        const float2 h0 = Unpack2Bf16(pa[h]), h1 = Unpack2Bf16(pa[2 + h]);
                        pb[h] = Pack2<T>(p00 - h0.x, p01 - h0.y);
                        pb[2 + h] = Pack2<T>(p10 - h1.x, p11 - h1.y);
                    }
                }
                // O = alpha * O + P V
#pragma unroll
                for (int r = 0; r < G::kVRounds; ++r) {
                    const int ch = 8 * r + g;
                    uint4 v0 = make_uint4(0, 0, 0, 0), v1 = v0, v2 = v0, v3 = v0;
                    if (ch < CPR) {
                        const int r0 = 2 * c;
                        v0 = LdsV4(v_stage + r0 * G::kRowBytes + SwizzleV<G::kSwizzle>(r0, ch) * 16);
                        v1 = LdsV4(v_stage + (r0 + 1) * G::kRowBytes + SwizzleV<G::kSwizzle>(r0 + 1, ch) * 16);
                        v2 = LdsV4(v_stage + (r0 + 8) * G::kRowBytes + SwizzleV<G::kSwizzle>(r0 + 8, ch) * 16);
                        v3 = LdsV4(v_stage + (r0 + 9) * G::kRowBytes + SwizzleV<G::kSwizzle>(r0 + 9, ch) * 16);
                    }
                    const uint32_t a0[4] = {v0.x, v0.y, v0.z, v0.w};
                    const uint32_t a1[4] = {v1.x, v1.y, v1.z, v1.w};
                    const uint32_t a2[4] = {v2.x, v2.y, v2.z, v2.w};
                    const uint32_t a3[4] = {v3.x, v3.y, v3.z, v3.w};
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const uint32_t sel = (j & 1) ? 0x7632u : 0x5410u;
                        const uint32_t b0 = __byte_perm(a0[j >> 1], a1[j >> 1], sel);
                        const uint32_t b1 = __byte_perm(a2[j >> 1], a3[j >> 1], sel);
                        o[r][j][0] *= alpha[0];
                        o[r][j][1] *= alpha[0];
                        if (kHi) {
                            o[r][j][2] *= alpha[1];
                            o[r][j][3] *= alpha[1];
                        }
                        MmaM16N8K16<T>(o[r][j], pa[0], pa[1], pa[2], pa[3], b0, b1);
                        if (kSplitP) MmaM16N8K16<T>(o[r][j], pb[0], pb[1], pb[2], pb[3], b0, b1);
                    }
                }
            }
        }
        __syncwarp();
        if (++stage == kStages) stage = 0;
    }
    CpAsyncWait<0>();
    __syncwarp();

    // ---- per-warp results -> this warp's (now idle) ring, then a CTA-wide merge ----------------
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        l_run[h] += __shfl_xor_sync(0xffffffffu, l_run[h], 1);
        l_run[h] += __shfl_xor_sync(0xffffffffu, l_run[h], 2);
    }
    float* stage_m = reinterpret_cast<float*>(ring);  // [16]
    float* stage_l = stage_m + 16;                    // [16]
    float* stage_o = stage_m + 32;                    // [16][D]
    if (c == 0) {
        stage_m[g] = m_run[0];
        stage_l[g] = l_run[0];
        stage_m[g + 8] = kHi ? m_run[1] : -CUDART_INF_F;
        stage_l[g + 8] = kHi ? l_run[1] : 0.0f;
    }
#pragma unroll
    for (int r = 0; r < G::kVRounds; ++r) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int d0 = 64 * r + 16 * c + j;
            const int d1 = d0 + 8;
            if (d0 < D) {
                stage_o[g * D + d0] = o[r][j][0];
                if (kHi) stage_o[(g + 8) * D + d0] = o[r][j][2];
            }
            if (d1 < D) {
                stage_o[g * D + d1] = o[r][j][1];
                if (kHi) stage_o[(g + 8) * D + d1] = o[r][j][3];
            }
        }
    }
    __syncthreads();

    if constexpr (kLog2) MergeWarpsLog2<D, G::kWarpBytes, kToShared>(p, smem, b, head0, nheads, slot);
    else MergeWarps<D, G::kWarpBytes, kToShared>(p, smem, b, head0, nheads, slot);
}

// Whether the one-launch kernel is the faster one for `units` (sequence, kv head, head chunk) columns of `steps` steps
// (the longest) on clusters of `cluster` CTAs. Both times in us, fitted to graph-timed calls of D=128 on a B200 (one-wave
// schedule with its merge / one launch): B=1, S=1000 10.9 / 6.2, S=4000 18.5 / 11.1, S=16000 27.5 / 28.5, S=60000 57 /
// 90; B=4, S=4000 21.0 / 16.5; B=16, S=2000 29.9 / 27.5, paged with lengths from 250 to 2000 25.6 / 27.7; paged B=4, 500
// to 4000 22.6 / 16.9, B=8 26.9 / 27.2. A step costs more the more CTAs share the memory; the schedule works on what a
// ragged batch holds (0.55 of the bound is assumed), a cluster waits for the longest sequence.
// Other head dims, from 1056 calls of D=32 to 256 (batch 1 to 32, 60 to 16000 tokens):
//   * above 128 one CTA fills an SM and a step is up to twice the bytes, so that clusters which leave SMs idle lose to the
//     wave: D=256, 8 kv heads, B=2, S=4000 24.2 / 20.5 (one launch / schedule), B=1, S=8000 23.1 / 21.9. Two times fitted
//     at 192 and 256, with 0.15 us per slot for the merge and 0.7 or 0.8 of the bound for a ragged batch. Groups of more than 8
//     heads pay for both row halves in the exchange; clusters of less than 8 do not make up for it in short streams,
//     unless long sequences are ragged (D=256, 16 / 1 heads, B=16, S=4000 32.8 / 24.5; B=32, S=4000 34.4 / 38.5);
//   * below 128 the memory is the limit once the stream takes 35 us, and the wave uses it better: D=64, B=32, S=8000 90 / 83.
inline bool ClusterIsFaster(int64_t units, int64_t steps, int cluster, int64_t resident, bool ragged, int head_dim, bool hi, int64_t splits) {
    const double busy = static_cast<double>(units * cluster) / resident;
    const double share = static_cast<double>((steps + cluster - 1) / cluster);
    const double waves = static_cast<double>(units * steps) / resident;
    const double stream_us = static_cast<double>(units * steps) * kSpan * head_dim * 4 / 6.5e6;
    if (head_dim > 128) {
        if (hi && cluster < kMaxCluster && steps > 1 && (!ragged || steps < 8) && stream_us < 12.0) return false;
        const double one_launch = (hi ? 3.5 + 0.027 * head_dim : 5.4) + share * (0.95 + 0.3 * busy);
        return one_launch < (hi ? 11.0 : 7.5) + 1.5 * std::max(1.0, waves * (!ragged ? 1.0 : hi ? 0.8 : 0.7)) + 0.15 * static_cast<double>(splits);
    }
    if (head_dim < 128 && stream_us > 35.0) return false;
    return 4.8 + share * (0.55 + 1.1 * busy) < 11.5 + 1.55 * std::max(1.0, waves * (ragged ? 0.55 : 1.0));
}

}  // namespace
}  // namespace sca_b200

// Decode over a paged 16-bit cache that does more than decode.cu: it adds up what each cached token weighs, and it leaves the pages that
// a group of sequences has in common to flash_shared.cu, which reads them once for all of them.
//
//   partial kernel  the segments of decode.cu over the tokens behind the common pages; where weights are wanted the scores go to scratch,
//                   4 bytes a query head and token beside the 4 * D bytes of K and V that a kv head reads;
//   finish kernel   merges the parts of every row - of its own tokens and of its prefix - and, with the row's final maximum M and sum L,
//                   weights[s, g, j] += sum over the query heads h of kv head g of 2^(score[h, j] - M[h]) / L[h]
//                   in the order of the heads: no atomics, the same bits every time.
// The scores are stored and not computed again: K once more would be half of the traffic (D=128, 4 heads to a kv head: 256 bytes a token and
// kv head against 32 written and read), and nobody knows M and L before the last key.
// A call that does not fill the machine runs in one launch, decode_step_cluster_kernel.
// Bound by memory. 192 sequences of 500 to 6000 tokens, 32 / 8 heads, D=128, bf16: 439 us for 2.6 GB, 389 without weights. Of the 50 us the stores of
// 80 MB of scores in the stream of loads cost 33, reading them back and adding 19. 96 of 200 to 6001, 32 / 2 heads, D=64, fp16: 53 us, 41.5
// without. One of 701 tokens 7.6 us in one launch, 11.1 in two.
// K and V go through the cache as what is given up first, so that the scores stay: the 96 sequences 56.0 / 52.6 us without / with it; with more scores
// than the cache holds it makes no difference. Adding the weights of whole sequences in the partial kernel, from a scratch of 128 KB a CTA, saved
// 2 % of the 192 sequences and cost the 96 a fifth: registers.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "decode_segment.cuh"
#include "shared_prefix.cuh"

namespace sca_b200 {
namespace {

struct WeightsParams {
    float* weights;    // [batch][kv_heads][row]; null: none wanted
    int64_t row;
    float* scores;     // see ScoreTap
    int64_t score_row;
    int64_t bound;     // tokens a sequence has at most
    PrefixParts prefix;
    bool behind_prefix;  // the kernel ahead is the prefix kernel of the same call
};

// Tokens of a sequence behind its common pages.
struct OwnTokens {
    const ScaDecodeFwdParams& p;
    const PrefixGroups& groups;
    int64_t bound;
    __device__ __forceinline__ int64_t First(int64_t b) const {
        const PrefixGroup* g = GroupOf(groups, b);
        return g != nullptr ? g->tokens : 0;
    }
    __device__ __forceinline__ int64_t Length(int64_t b) const { return min(SeqLen<true>(p, b), bound); }
    __device__ __forceinline__ int64_t operator()(int64_t b) const { return max(Length(b) - First(b), int64_t{0}); }
    __device__ __forceinline__ bool Regular() const { return p.seq_lens == nullptr && groups.count == 0; }
};

// kWeights: the scores go to scratch. A kernel that looks in every tile whether they are wanted takes 5 us more where they are not (96 sequences of
// 200 to 6001 tokens, 32 / 2 heads, D=64: 44 / 49).
template <bool kWeights>
using TapFor = std::conditional_t<kWeights, ScoreTap, NoTap>;
template <bool kWeights>
__device__ __forceinline__ TapFor<kWeights> MakeTap(const WeightsParams& x) {
    if constexpr (kWeights) return {x.scores, x.score_row};
    else return {};
}

template <typename T, int D, bool kHi, bool kWeights>
__global__ void __launch_bounds__(kThreads)
decode_own_kernel(const ScaDecodeFwdParams p, const int head_chunks, const WeightsParams x, const __grid_constant__ PrefixGroups groups) {
    extern __shared__ __align__(128) unsigned char smem[];
    // Behind a prefix kernel this one may run beside it: nothing here reads what that one writes, or writes what it reads, and its mark stands for the
    // kernels before it. The wait at the end makes the end of this kernel that of both. With the wait ahead of everything the two run one
    // behind the other: 128 sequences behind 8100 tokens 109 / 115 us, 14 groups of 4 to 12 behind 300 to 4000 with weights 85 / 94.
    if (!x.behind_prefix || !HasBegun(x.prefix.begun)) WaitForPredecessor();
    const OwnTokens own{p, groups, x.bound};
    const auto tap = MakeTap<kWeights>(x);
    WalkSteps<true, kSpan, true>(p, head_chunks, own, [&](int64_t b, int hk, int hc, int64_t j_begin, int64_t j_end, int slot) {
        const int64_t first = own.First(b);
        DecodeSegment<T, D, true, kHi, false, TapFor<kWeights>, true>(p, smem, b, hk, hc, first + j_begin, first + j_end, slot, tap);
    });
    if (x.behind_prefix) WaitForPredecessor();
}

// A call that does not fill the machine, in one launch (see ClusterDecode): the CTAs of a cluster share one (sequence, kv head), all of its
// tokens, those of common pages too, and weigh the tokens they have read once the row's maximum and sum are known. Up to 16 heads to a kv head.
template <typename T, int D, bool kHi, bool kWeights>
__global__ void __launch_bounds__(kThreads)
decode_step_cluster_kernel(const ScaDecodeFwdParams p, const int cluster, const WeightsParams x, const __grid_constant__ PrefixGroups groups) {
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ float s_m[16], s_inv[16];
    BeginAfterPredecessor();
    const OwnTokens own{p, groups, x.bound};
    const int rank = static_cast<int>(ClusterRank()), unit = static_cast<int>(blockIdx.x) / cluster;
    const int64_t b = unit / p.num_kv_heads;
    const int hk = static_cast<int>(unit % p.num_kv_heads), heads = static_cast<int>(p.num_heads / p.num_kv_heads), head0 = hk * heads;
    const int64_t len = own.Length(b), steps = StepsFor<kSpan>(len), share = (steps + cluster - 1) / cluster;
    const int64_t t0 = min(rank * share, steps), t1 = min(t0 + share, steps);
    const int64_t begin = t0 * kSpan, end = min(t1 * kSpan, len);
    DecodeSegment<T, D, true, kHi, true, TapFor<kWeights>, true>(p, smem, b, hk, 0, begin, end, 0, MakeTap<kWeights>(x));
    ClusterBarrier();
    const uint32_t partial = SmemAddr(CtaPartial<D>(smem)), partial_o = SmemAddr(smem) + 32 * 4;
    if (threadIdx.x < heads) {  // a thread per head; s_m: the maximum, s_inv: 1 / sum
        float m[kMaxCluster], l[kMaxCluster], m_all = -CUDART_INF_F, l_all = 0.0f;
#pragma unroll
        for (int r = 0; r < kMaxCluster; ++r) {
            m[r] = r < cluster ? LoadFromRank(partial + 4 * threadIdx.x, r) : -CUDART_INF_F;
            l[r] = r < cluster ? LoadFromRank(partial + 4 * (16 + threadIdx.x), r) : 0.0f;
            m_all = fmaxf(m_all, m[r]);
        }
#pragma unroll
        for (int r = 0; r < kMaxCluster; ++r) {
            if (m[r] != -CUDART_INF_F || l[r] != 0.0f) l_all += l[r] * Exp2(m[r] - m_all);
        }
        s_m[threadIdx.x] = m_all;
        s_inv[threadIdx.x] = l_all == 0.0f ? 0.0f : 1.0f / l_all;
    }
    __syncthreads();
    T* out = reinterpret_cast<T*>(p.out) + b * p.o_stride.s_b;
    for (int item = rank * kThreads + threadIdx.x; item < heads * D; item += cluster * kThreads) {
        const int row = item / D, d = item % D;
        float m[kMaxCluster], o[kMaxCluster], acc = 0.0f;
#pragma unroll
        for (int r = 0; r < kMaxCluster; ++r) {
            m[r] = r < cluster ? LoadFromRank(partial + 4 * row, r) : -CUDART_INF_F;
            o[r] = r < cluster ? LoadFromRank(partial_o + 4 * (row * D + d), r) : 0.0f;
        }
        // a part without a key has O = 0 beside its maximum of -inf, a part of NaN keeps it
#pragma unroll
        for (int r = 0; r < kMaxCluster; ++r) {
            if (m[r] != -CUDART_INF_F || o[r] != 0.0f) acc += o[r] * Exp2(m[r] - s_m[row]);
        }
        out[(head0 + row) * p.o_stride.s_h + d] = FromFloat<T>(acc * s_inv[row]);
    }
    if constexpr (kWeights) {
        float* w = x.weights + unit * x.row;
        const float* scores = x.scores + (b * p.num_heads + head0) * x.score_row;
        for (int64_t j = max(begin, own.First(b)) + threadIdx.x; j < end; j += kThreads) {
            float sum = 0.0f;
            for (int h = 0; h < heads; ++h) sum += Exp2(scores[h * x.score_row + j] - (s_m[h] == -CUDART_INF_F ? 0.0f : s_m[h])) * s_inv[h];
            w[j] += sum;
        }
    }
    ClusterBarrier();  // nobody leaves while its shared memory is being read
}

constexpr int kFinishThreads = 256;
constexpr int kTokens = 4 * kFinishThreads; // tokens a CTA weighs at once
constexpr int kHeadSlab = 32;               // query heads whose M and 1 / L stand in shared memory
constexpr int kTogether = 4;                // query heads whose scores a thread has on their way
constexpr int64_t kMostSplits = 64;         // parts of a sequence's own tokens
constexpr int kMostParts = 32;              // and of its prefix (PlanPrefixParts)

// Maximum and sum over the parts of a row, by a whole warp.
struct RowStats {
    float m, l;
};
__device__ __forceinline__ RowStats StatsOf(const ScaDecodeFwdParams& p, const PrefixParts& prefix, int parts, int prefix_parts, int64_t row) {
    constexpr int kOwn = kMostSplits / 32, kAll = kOwn + kMostParts / 32;
    const int lane = threadIdx.x & 31, own = static_cast<int>(p.num_splits);
    float mi[kAll], li[kAll], m = -CUDART_INF_F, l = 0.0f;
#pragma unroll
    for (int i = 0; i < kAll; ++i) {
        const int at = i < kOwn ? 32 * i + lane : 32 * (i - kOwn) + lane;
        const bool in = at < (i < kOwn ? own : prefix_parts);
        mi[i] = !in ? -CUDART_INF_F : i < kOwn ? p.partial_m[row * own + at] : prefix.m[row * parts + at];
        li[i] = !in ? 0.0f : i < kOwn ? p.partial_l[row * own + at] : prefix.l[row * parts + at];
    }
#pragma unroll
    for (int i = 0; i < kAll; ++i) m = fmaxf(m, mi[i]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
#pragma unroll
    for (int i = 0; i < kAll; ++i) {
        if (mi[i] != -CUDART_INF_F || li[i] != 0.0f) l += li[i] * Exp2(mi[i] - m);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    return {m, l};
}

// Blocks [0, merge_blocks) merge output rows, the others weigh tokens: block (s * kv_heads + g) * chunks + c of those has the c-th `chunk` tokens.
template <typename T>
__global__ void __launch_bounds__(kFinishThreads, 4)
decode_finish_kernel(const ScaDecodeFwdParams p, const WeightsParams x, const int merge_blocks, const int chunks,
                     const int64_t chunk, const __grid_constant__ PrefixGroups groups) {
    __shared__ float s_m[kHeadSlab], s_inv[kHeadSlab];
    BeginAfterPredecessor();
    if (x.behind_prefix && blockIdx.x == 0 && threadIdx.x == 0) *x.prefix.begun = 0;
    const int own = static_cast<int>(p.num_splits), parts = groups.parts;
    auto prefix_parts_of = [&](int64_t b) {
        const PrefixGroup* g = GroupOf(groups, b);
        return g != nullptr ? ((g->tokens + 127) / 128 + groups.part_tiles - 1) / groups.part_tiles : 0;
    };
    if (static_cast<int>(blockIdx.x) < merge_blocks) {
        // a thread has four numbers of a row; 32-bit divisions, 64-bit ones are what this kernel would spend its time on
        const uint32_t lanes = static_cast<uint32_t>(p.head_dim) / 4, block_rows = kFinishThreads / lanes, of_block = threadIdx.x / lanes;
        const int d = static_cast<int>(threadIdx.x - of_block * lanes) * 4;
        const uint32_t rows = static_cast<uint32_t>(p.batch * p.num_heads), heads = static_cast<uint32_t>(p.num_heads);
        for (uint32_t row32 = blockIdx.x * block_rows + of_block; of_block < block_rows && row32 < rows; row32 += merge_blocks * block_rows) {
            const int64_t row = row32, b = row32 / heads;
            const int prefix_parts = prefix_parts_of(b);
            float m = -CUDART_INF_F, l = 0.0f;
            float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            for (int i = 0; i < own; ++i) m = fmaxf(m, p.partial_m[row * own + i]);
            for (int i = 0; i < prefix_parts; ++i) m = fmaxf(m, x.prefix.m[row * parts + i]);
            auto add = [&](float mi, float li, const float* o) {
                if (mi == -CUDART_INF_F && li == 0.0f) return;
                const float w = Exp2(mi - m);
                const float4 v = *reinterpret_cast<const float4*>(o);
                l += li * w;
                acc.x += v.x * w, acc.y += v.y * w, acc.z += v.z * w, acc.w += v.w * w;
            };
            for (int i = 0; i < own; ++i) add(p.partial_m[row * own + i], p.partial_l[row * own + i], p.partial_o + (row * own + i) * p.head_dim + d);
            for (int i = 0; i < prefix_parts; ++i) add(x.prefix.m[row * parts + i], x.prefix.l[row * parts + i], x.prefix.o + (row * parts + i) * p.head_dim + d);
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
            T* out = reinterpret_cast<T*>(p.out) + b * p.o_stride.s_b + (row - b * heads) * p.o_stride.s_h + d;
            *reinterpret_cast<uint2*>(out) = make_uint2(Pack2<T>(acc.x * inv, acc.y * inv), Pack2<T>(acc.z * inv, acc.w * inv));
        }
        return;
    }
    const uint32_t block = blockIdx.x - merge_blocks, unit32 = block / static_cast<uint32_t>(chunks), seq32 = unit32 / static_cast<uint32_t>(p.num_kv_heads);
    const int64_t unit = unit32, b = seq32, g = unit32 - seq32 * static_cast<uint32_t>(p.num_kv_heads);
    const OwnTokens tokens{p, groups, x.bound};
    const int64_t chunk_begin = (block - unit32 * static_cast<uint32_t>(chunks)) * chunk;
    const int64_t first = tokens.First(b), end = min(tokens.Length(b), chunk_begin + chunk);
    if (end <= chunk_begin || first >= end) return;
    const int group = static_cast<int>(static_cast<uint32_t>(p.num_heads) / static_cast<uint32_t>(p.num_kv_heads));
    const int prefix_parts = prefix_parts_of(b);
    const int64_t row0 = b * p.num_heads + g * group;
    const float* scores = x.scores + row0 * x.score_row;
    float* weights = x.weights + unit * x.row;
    const bool aligned = (reinterpret_cast<uintptr_t>(weights) & 15u) == 0;
    // a thread has four tokens: all of them own ones of the sequence, or some, or none
    float4 s[kTogether], old;
    auto load = [&](int64_t j, int h0) {
#pragma unroll
        for (int i = 0; i < kTogether; ++i) {
            if (h0 + i < group) s[i] = *reinterpret_cast<const float4*>(scores + (h0 + i) * x.score_row + j);
        }
    };
    auto some = [&](int64_t j) { return j + 3 >= first && j < end; };
    auto whole = [&](int64_t j) { return aligned && j >= first && j + 3 < end; };  // one load and one store for all four
    auto load_tokens = [&](int64_t j) {
        if (some(j)) load(j, 0);
        if (whole(j)) old = *reinterpret_cast<const float4*>(weights + j);
    };
    const int64_t j = max(chunk_begin, first & ~static_cast<int64_t>(kTokens - 1)) + 4 * threadIdx.x;
    load_tokens(j);  // on their way while the rows' maxima and sums are made
    for (int slab = 0; slab < group; slab += kHeadSlab) {
        const int heads = min(kHeadSlab, group - slab);
        __syncthreads();  // the last slab has been read
        for (int h = threadIdx.x >> 5; h < heads; h += kFinishThreads / 32) {
            const RowStats r = StatsOf(p, x.prefix, parts, prefix_parts, row0 + slab + h);
            if ((threadIdx.x & 31) == 0) {
                s_m[h] = r.m == -CUDART_INF_F ? 0.0f : r.m;
                s_inv[h] = r.l == 0.0f ? 0.0f : 1.0f / r.l;
            }
        }
        __syncthreads();
        for (int64_t at = j; at - 4 * threadIdx.x < end; at += kTokens) {
            if (!some(at)) continue;
            if (at != j || slab > 0) {
                load(at, slab);
                if (whole(at)) old = *reinterpret_cast<const float4*>(weights + at);
            }
            float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            for (int h0 = 0; h0 < heads; h0 += kTogether) {
                if (h0 > 0) load(at, slab + h0);
#pragma unroll
                for (int i = 0; i < kTogether; ++i) {
                    if (h0 + i >= heads) continue;
                    const float m = s_m[h0 + i], inv = s_inv[h0 + i];
                    sum.x += Exp2(s[i].x - m) * inv;
                    sum.y += Exp2(s[i].y - m) * inv;
                    sum.z += Exp2(s[i].z - m) * inv;
                    sum.w += Exp2(s[i].w - m) * inv;
                }
            }
            float* w = weights + at;
            if (whole(at)) {
                *reinterpret_cast<float4*>(w) = make_float4(old.x + sum.x, old.y + sum.y, old.z + sum.z, old.w + sum.w);
            } else {
                const float add[4] = {sum.x, sum.y, sum.z, sum.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (at + i >= first && at + i < end) w[i] += add[i];
                }
            }
        }
    }
}

// What a slice of a call is made of (see SliceOf): sizes of its launches, and where its arrays lie in the scratch.
struct Plan {
    PrefixGroups groups;
    int64_t splits;
    int64_t bound;                // tokens of a sequence at most
    int64_t own_m, own_l, own_o;  // floats from the start, where the mark of the prefix kernel stands
    int64_t prefix_m, prefix_l, prefix_o;
    int64_t scores, score_row;
    int64_t floats;
};

int64_t RoundUp(int64_t x, int64_t to) { return (x + to - 1) / to * to; }

}  // namespace

// Launches the kernel that leaves the parts of the prefixes in `parts` (flash_shared.cu).
int LaunchPrefixParts(const ScaDecodeFwdParams& p, const PrefixGroups& groups, const PrefixParts& parts, cudaStream_t stream);
// Fills part_tiles, parts and the groups' first entries for the SMs at hand.
void PlanPrefixParts(const ScaDecodeFwdParams& p, PrefixGroups* groups);

namespace {

int Validate(const ScaDecodeFwdParams* params, const ScaPagedStep* step, const char* what) {
    auto invalid = [&](const std::string& why) { return Fail(SCA_INVALID_ARGUMENT, std::string(what) + ": " + why); };
    if (params == nullptr || step == nullptr) return invalid("null parameter block");
    const ScaDecodeFwdParams& p = *params;
    const ScaPagedStep& x = *step;
    if (p.dtype != SCA_DTYPE_F16 && p.dtype != SCA_DTYPE_BF16) return invalid("fp16 or bf16 only");
    if (p.batch < 1 || p.num_heads < 1 || p.num_kv_heads < 1 || p.num_heads % p.num_kv_heads != 0) {
        return invalid("invalid geometry batch=" + std::to_string(p.batch) + " heads=" + std::to_string(p.num_heads) + " kv_heads=" + std::to_string(p.num_kv_heads));
    }
    switch (p.head_dim) {
        case 32: case 64: case 96: case 128: case 160: case 192: case 256: break;
        default: return invalid("head_dim=" + std::to_string(p.head_dim) + " is not instantiated");
    }
    if (p.block_size < 1 || p.max_blocks_per_seq < 1 || p.num_kv_blocks < 1) return invalid("block_size/max_blocks_per_seq/num_kv_blocks must be positive");
    if (p.num_kv_blocks * p.block_size > 0x7fffff00LL || p.max_blocks_per_seq * p.block_size > 0x7fffff00LL || p.batch * p.num_heads > 0x7fffff00LL) {
        return invalid("more than 2^31 tokens or rows");
    }
    if (!(p.scale > 0.0f) || !std::isfinite(p.scale)) return invalid("scale must be a positive number");
    if (x.num_groups < 0 || (x.num_groups > 0 && (x.cu_groups == nullptr || x.prefix_lens == nullptr))) return invalid("null groups");
    if (x.weights != nullptr && x.weights_row < p.max_blocks_per_seq * p.block_size) {
        return invalid("rows of " + std::to_string(x.weights_row) + " weights for page-table rows of " + std::to_string(p.max_blocks_per_seq * p.block_size) + " tokens");
    }
    if (x.num_groups > 0) {
        if (p.block_size != 8 && p.block_size != 16 && p.block_size != 32 && p.block_size != 64) {
            return invalid("block_size=" + std::to_string(p.block_size) + " (pages of a prefix are loaded as boxes of 8, 16, 32 or 64 tokens)");
        }
        if (x.cu_groups[0] != 0 || x.cu_groups[x.num_groups] != p.batch) return invalid("group offsets must start at 0 and end at the number of sequences");
        int sharing = 0;
        for (int64_t g = 0; g < x.num_groups; ++g) {
            if (x.cu_groups[g + 1] < x.cu_groups[g]) return invalid("group offsets must not fall");
            if (x.prefix_lens[g] < 0 || x.prefix_lens[g] > p.max_blocks_per_seq * p.block_size) {
                return invalid("group " + std::to_string(g) + " has a prefix of " + std::to_string(x.prefix_lens[g]) + " tokens (the page-table row holds " +
                               std::to_string(p.max_blocks_per_seq * p.block_size) + ")");
            }
            if (x.cu_groups[g + 1] - x.cu_groups[g] > 1 && x.prefix_lens[g] >= p.block_size) ++sharing;
        }
        if (sharing > kMaxGroups) return invalid(std::to_string(sharing) + " groups that share a page (at most " + std::to_string(kMaxGroups) + " in one call)");
    }
    return SCA_OK;
}

// Tokens of a sequence at most, as far as the host knows.
int64_t BoundOf(const ScaDecodeFwdParams& p, const ScaPagedStep& x) {
    const int64_t capacity = p.max_blocks_per_seq * p.block_size;
    return x.longest_len > 0 ? std::min(x.longest_len, capacity) : capacity;
}
// Scores of a query head. A tile of 16 may begin at any page of a prefix, 8 tokens say, and is stored whole.
int64_t ScoreRow(const ScaDecodeFwdParams& p, const ScaPagedStep& x) { return x.weights != nullptr ? RoundUp(BoundOf(p, x), kTile) + kTile : 0; }

// Sequences that go through the kernels together. The scratch has a score for every token that a sequence may have, whatever it has, so a call
// with weights whose table is wide, or one of whose sequences is long, is taken in slices of sequences whose scores fit kMostScores, 2 GB, or of one.
// us and MB of scratch without slices / of 2 GB / of 1 GB (D=128, 32 / 8 heads unless said):
//   192 sequences of 500 to 6000 tokens, table of 131 072         456, 3848 / 473, 1924 / 487, 962
//   one of 100 000 among 191 of 200 to 1500, exact hints          235, 2987 / 241, 1518 / 245, 1030
//   2 groups, 128 sequences behind 3000 tokens, table of 131 072  110, 2580 / 117, 1291 / 139, 867
//   96 of 200 to 6001, 32 / 2 heads, D=64, table of 131 072        64, 1925 /  64, 1925 /  78, 963
constexpr int64_t kMostScores = int64_t{1} << 29;
int64_t SliceOf(const ScaDecodeFwdParams& p, const ScaPagedStep& x) {
    if (x.weights == nullptr) return p.batch;
    const int64_t most = std::max<int64_t>(1, kMostScores / (p.num_heads * ScoreRow(p, x))), slices = (p.batch + most - 1) / most;
    return (p.batch + slices - 1) / slices;
}

// Sequences [begin, end) of a validated call.
Plan MakePlan(const ScaDecodeFwdParams& p, const ScaPagedStep& x, int64_t begin, int64_t end) {
    Plan plan{};
    PrefixGroups& groups = plan.groups;
    const int64_t batch = end - begin;
    plan.bound = BoundOf(p, x);
    int64_t prefix_of_all = 0;                                  // tokens that are read for others
    int64_t least_prefix = x.num_groups > 0 ? plan.bound : 0;  // of a sequence
    for (int64_t g = 0; g < x.num_groups; ++g) {
        const int64_t tokens = std::min<int64_t>(x.prefix_lens[g], plan.bound) / p.block_size * p.block_size;
        const bool shared = x.cu_groups[g + 1] - x.cu_groups[g] > 1 && tokens > 0;  // one that a slice cuts stays a group, of one sequence too
        const int64_t from = std::max<int64_t>(x.cu_groups[g], begin), to = std::min<int64_t>(x.cu_groups[g + 1], end);
        if (from >= to) continue;
        least_prefix = std::min(least_prefix, shared ? tokens : 0);
        if (!shared) continue;
        groups.group[groups.count++] = {static_cast<int>(from - begin), static_cast<int>(to - begin), static_cast<int>(tokens), 0};
        prefix_of_all += (to - from) * tokens;
    }
    if (groups.count > 0) PlanPrefixParts(p, &groups);

    // Slots for the parts of a sequence's own tokens: enough for an even schedule (see slots_for_schedule in ops.py). The kernel takes
    // larger shares where these hold fewer.
    const int64_t typical = std::max<int64_t>(1, (x.typical_len > 0 ? std::min(x.typical_len, plan.bound) : plan.bound) - prefix_of_all / batch);
    const int64_t group_heads = p.num_heads / p.num_kv_heads;
    const int64_t columns = p.num_kv_heads * ((group_heads + 15) / 16);
    const int64_t steps = (typical + kSpan - 1) / kSpan;
    const int64_t longest = x.longest_len > 0 ? std::max<int64_t>(1, (plan.bound - least_prefix + kSpan - 1) / kSpan) : 2 * steps;
    const int64_t sharers = std::max<int64_t>(1, 2 * SmCount() / columns);
    const int64_t share = std::max<int64_t>(1, (batch * steps + sharers - 1) / sharers);
    // two at least, for sequences of one step too: with one the first CTA of a column would have all of them (256 sequences of 1 to 60 tokens, 32 / 8
    // heads, D=128: 806 us, 40.6 with two)
    plan.splits = std::max<int64_t>(2, std::min((longest + share - 1) / share + 1, kMostSplits));

    const int64_t rows = batch * p.num_heads;
    plan.own_m = 8;
    plan.own_l = plan.own_m + rows * plan.splits;
    plan.own_o = RoundUp(plan.own_l + rows * plan.splits, 4);  // an O starts on 16 bytes
    plan.prefix_m = plan.own_o + rows * plan.splits * p.head_dim;
    plan.prefix_l = plan.prefix_m + rows * groups.parts;
    plan.prefix_o = RoundUp(plan.prefix_l + rows * groups.parts, 8);  // 32
    plan.scores = RoundUp(plan.prefix_o + rows * groups.parts * p.head_dim, 8);
    plan.score_row = ScoreRow(p, x);
    plan.floats = plan.scores + rows * plan.score_row;
    return plan;
}

// f(begin, end, plan) for every slice of a validated call; a number other than 0 ends it.
template <typename F>
int ForSlices(const ScaDecodeFwdParams& p, const ScaPagedStep& x, const F& f) {
    const int64_t slice = SliceOf(p, x);
    for (int64_t begin = 0; begin < p.batch; begin += slice) {
        const int64_t end = std::min(begin + slice, p.batch);
        if (int rc = f(begin, end, MakePlan(p, x, begin, end))) return rc;
    }
    return 0;
}
// The slices follow one another on the stream and use the same scratch.
int64_t ScratchFloats(const ScaDecodeFwdParams& p, const ScaPagedStep& x) {
    int64_t most = 0;
    ForSlices(p, x, [&](int64_t, int64_t, const Plan& plan) { return most = std::max(most, plan.floats), 0; });
    return most;
}

// Where sequences share pages, the one launch reads them once for each; that pays as long as a CTA has few steps. us, one launch / with the
// prefix kernel, and the steps of a CTA: 32 / 8 heads, D=128: 5 sequences of 600 tokens 9.0 / 13.5 (2), 3 of 4100 15.1 / 17.0 (8), 12 of 1300 16.6
// / 19.8 (10), 2 of 8100 21.8 / 19.8 (16), 5 of 4200 22.9 / 21.7 (16). 32 / 2 heads, D=64: 3 of 8100 15.5 / 16.7 (16), 2 of 16100 24.7 / 19.0 (32).
// 16 / 2 heads, D=256: 16 of 400 12.5 / 17.8 (1), 8 of 1100 17.1 / 16.4 (3), 8 of 2100 23.4 / 17.4 (5).
// Launches decode_step_cluster_kernel if it is the kernel for this call; *taken = its CTAs per cluster, 0 if it is not.
template <typename T, int D, bool kHi, bool kWeights>
int LaunchStepCluster(const ScaDecodeFwdParams& p, const WeightsParams& x, const PrefixGroups& groups, cudaStream_t stream, int* taken) {
    auto kernel = decode_step_cluster_kernel<T, D, kHi, kWeights>;
    constexpr int kSmem = DecodeGeom<D>::kSmemBytes;
    if (int rc = EnsureDynamicSmem(reinterpret_cast<const void*>(kernel), kSmem, "decode_step_cluster_kernel")) return rc;
    static PerDevice resident[kMaxCluster + 1], per_sm;  // per instantiation
    auto clusters = [&](int cluster) -> int64_t {
        return std::max(0, resident[cluster].Get([&] {
            cudaLaunchAttribute attr{};
            cudaLaunchConfig_t cfg = ClusterConfig(static_cast<unsigned>(cluster), cluster, kSmem, nullptr, &attr);
            int n = 0;
            if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess) {
                cudaGetLastError();
                return -1;
            }
            return n;
        }));
    };
    const int ctas = per_sm.Get([&] {
        int n = 0;
        if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, kThreads, kSmem) != cudaSuccess || n < 1) {
            cudaGetLastError();
            return -1;
        }
        return n;
    });
    const int64_t units = p.batch * p.num_kv_heads, steps = std::max<int64_t>(1, (x.bound + kSpan - 1) / kSpan);
    int cluster = kMaxCluster;
    while (cluster >= 2 && units > clusters(cluster)) cluster /= 2;
    *taken = 0;
    const int64_t share = (steps + cluster - 1) / cluster;
    if (D > 128 && share > 6) return SCA_OK;  // one sequence of 4000 tokens, D=256, 16 / 2 heads: 8 steps a CTA 23.6 us, three kernels 18.9
    const bool pays = groups.count > 0 ? share <= (D <= 64 ? 20 : D <= 128 ? 12 : 2)
                                       : ClusterIsFaster(units, steps, cluster, static_cast<int64_t>(SmCount()) * std::max(1, ctas), p.seq_lens != nullptr, D, kHi, p.num_splits);
    if (cluster < 2 || !pays) return SCA_OK;
    *taken = cluster;
    LaunchDependent(kernel, units * cluster, kThreads, kSmem, stream, cluster, p, cluster, x, groups);
    return CheckLaunch("decode_step_cluster_kernel", stream);
}

template <typename T, int D, bool kHi, bool kWeights>
int LaunchOwn(const ScaDecodeFwdParams& p, const WeightsParams& x, const PrefixGroups& groups, cudaStream_t stream) {
    using G = DecodeGeom<D>;
    auto kernel = decode_own_kernel<T, D, kHi, kWeights>;
    if (int rc = EnsureDynamicSmem(reinterpret_cast<const void*>(kernel), G::kSmemBytes, "decode_own_kernel")) return rc;
    static PerDevice per_sm;  // per instantiation
    const int resident = per_sm.Get([&] {
        int n = 0;
        if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, kThreads, G::kSmemBytes) != cudaSuccess || n < 1) {
            cudaGetLastError();
            return -1;
        }
        return n;
    });
    const int64_t wave = static_cast<int64_t>(SmCount()) * std::max(1, resident);
    const int head_chunks = static_cast<int>((p.num_heads / p.num_kv_heads + 15) / 16);
    const int64_t columns = p.num_kv_heads * head_chunks;
    const int64_t steps = std::max<int64_t>(1, (x.bound + kSpan - 1) / kSpan);
    const int64_t useful = p.batch * steps;  // CTAs of a column that can have something to do
    const int64_t blocks = wave >= columns ? columns * std::max<int64_t>(1, std::min(wave / columns, useful)) : wave;
    LaunchDependent(kernel, blocks, kThreads, G::kSmemBytes, stream, 1, p, head_chunks, x, groups);
    return CheckLaunch("decode_own_kernel", stream);
}

// f(head dim, more than 8 heads to a kv head, weights wanted), as types
template <typename F>
int ForGeometry(const ScaDecodeFwdParams& p, bool weights, const F& f) {
    const bool hi = p.num_heads / p.num_kv_heads > 8;
    auto with = [&](auto d) {
        if (weights) return hi ? f(d, std::true_type{}, std::true_type{}) : f(d, std::false_type{}, std::true_type{});
        return hi ? f(d, std::true_type{}, std::false_type{}) : f(d, std::false_type{}, std::false_type{});
    };
    switch (p.head_dim) {
        case 32: return with(std::integral_constant<int, 32>{});
        case 64: return with(std::integral_constant<int, 64>{});
        case 96: return with(std::integral_constant<int, 96>{});
        case 128: return with(std::integral_constant<int, 128>{});
        case 160: return with(std::integral_constant<int, 160>{});
        case 192: return with(std::integral_constant<int, 192>{});
        default: return with(std::integral_constant<int, 256>{});
    }
}

template <typename T>
int LaunchStep(const ScaDecodeFwdParams& p, WeightsParams x, const PrefixGroups& groups, cudaStream_t stream) {
    const int64_t heads = p.num_heads / p.num_kv_heads;
    if (heads <= 16) {
        int taken = 0;
        if (int rc = ForGeometry(p, x.weights != nullptr, [&](auto d, auto hi, auto weights) { return LaunchStepCluster<T, decltype(d)::value, decltype(hi)::value, decltype(weights)::value>(p, x, groups, stream, &taken); })) return rc;
        if (taken > 0) return SCA_OK;
    }
    if (groups.count > 0) {
        if (int rc = LaunchPrefixParts(p, groups, x.prefix, stream)) return rc;
    }
    if (int rc = ForGeometry(p, x.weights != nullptr, [&](auto d, auto hi, auto weights) { return LaunchOwn<T, decltype(d)::value, decltype(hi)::value, decltype(weights)::value>(p, x, groups, stream); })) return rc;
    const int64_t block_rows = kFinishThreads / (p.head_dim / 4);
    const int64_t merge_blocks = std::min<int64_t>((p.batch * p.num_heads + block_rows - 1) / block_rows, 1 << 16);
    // tokens to a CTA: few enough that all SMs have some, as many as let a CTA make the maxima and sums once
    const int64_t units = p.batch * p.num_kv_heads;
    const int64_t chunk = std::min<int64_t>(8 * kTokens, std::max<int64_t>(1, units * x.bound / (8 * SmCount() * kTokens)) * kTokens);
    const int64_t chunks = x.weights != nullptr ? (x.bound + chunk - 1) / chunk : 0;
    const int64_t blocks = merge_blocks + p.batch * p.num_kv_heads * chunks;
    if (blocks > 0x7fffffffLL) return Fail(SCA_INVALID_ARGUMENT, "paged attention (weights): grid of " + std::to_string(blocks) + " blocks is out of range");
    LaunchDependent(decode_finish_kernel<T>, blocks, kFinishThreads, 0, stream, 1, p, x, static_cast<int>(merge_blocks), static_cast<int>(std::max<int64_t>(chunks, 1)), chunk, groups);
    return CheckLaunch("decode_finish_kernel", stream);
}

}  // namespace
}  // namespace sca_b200

using namespace sca_b200;

extern "C" long long sca_paged_step_scratch_floats(const ScaDecodeFwdParams* params, const ScaPagedStep* step) {
    ClearError();
    if (Validate(params, step, "paged step") != SCA_OK) return -1;
    return ScratchFloats(*params, *step);
}

extern "C" int sca_launch_paged_step(const ScaDecodeFwdParams* params, const ScaPagedStep* step, void* stream) {
    ClearError();
    if (int rc = Validate(params, step, "paged step")) return rc;
    ScaDecodeFwdParams p = *params;
    const ScaPagedStep& x = *step;
    if (p.q == nullptr || p.k == nullptr || p.v == nullptr || p.out == nullptr || p.page_table == nullptr || x.scratch == nullptr) {
        return Fail(SCA_INVALID_ARGUMENT, "paged step: null pointer");
    }
    if (!Aligned16(p.q) || !Aligned16(p.k) || !Aligned16(p.v) || !Aligned16(p.out) || p.q_stride.s_b % 8 != 0 || p.q_stride.s_h % 8 != 0 ||
        p.o_stride.s_b % 8 != 0 || p.o_stride.s_h % 8 != 0 || (reinterpret_cast<uintptr_t>(x.scratch) & 31u) != 0) {
        return Fail(SCA_INVALID_ARGUMENT, "paged step: q/k/v/out must be 16-byte aligned with strides that are multiples of 8 elements, the scratch 32-byte aligned");
    }
    auto scratch_holds = [&](int64_t need) {
        if (x.scratch_floats >= need) return static_cast<int>(SCA_OK);
        return Fail(SCA_INVALID_ARGUMENT, "paged step: scratch of " + std::to_string(x.scratch_floats) + " floats is too small (" + std::to_string(need) + " needed)");
    };
    if (SliceOf(p, x) < p.batch) {  // ahead of the first slice's launches
        if (int rc = scratch_holds(ScratchFloats(p, x))) return rc;
    }
    float* scratch = x.scratch;
    p.seq_kv = p.num_kv_blocks * p.block_size;  // of a sequence without a length: all of its row
    p.k_stride = p.v_stride = ScaDecodeStrides{0, p.head_dim, p.num_kv_heads * p.head_dim};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return ForSlices(p, x, [&](int64_t begin, int64_t end, const Plan& plan) {
        if (int rc = scratch_holds(plan.floats)) return rc;
        ScaDecodeFwdParams part = p;
        part.batch = end - begin;
        part.q = static_cast<const char*>(p.q) + begin * p.q_stride.s_b * 2;
        part.out = static_cast<char*>(p.out) + begin * p.o_stride.s_b * 2;
        part.page_table = p.page_table + begin * p.max_blocks_per_seq;
        if (p.seq_lens != nullptr) part.seq_lens = p.seq_lens + begin;
        part.num_splits = plan.splits;
        part.partial_m = scratch + plan.own_m;
        part.partial_l = scratch + plan.own_l;
        part.partial_o = scratch + plan.own_o;
        WeightsParams w{};
        w.weights = x.weights != nullptr ? x.weights + begin * p.num_kv_heads * x.weights_row : nullptr;
        w.row = x.weights_row;
        w.scores = x.weights != nullptr ? scratch + plan.scores : nullptr;
        w.score_row = plan.score_row;
        w.bound = plan.bound;
        w.prefix = PrefixParts{scratch + plan.prefix_m, scratch + plan.prefix_l, scratch + plan.prefix_o, reinterpret_cast<unsigned long long*>(scratch)};
        w.behind_prefix = plan.groups.count > 0;
        return p.dtype == SCA_DTYPE_F16 ? LaunchStep<__half>(part, w, plan.groups, s) : LaunchStep<__nv_bfloat16>(part, w, plan.groups, s);
    });
}

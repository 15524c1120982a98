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
#include <algorithm>
#include <cmath>

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

template <typename T, int D, bool kHi>
__global__ void __launch_bounds__(kThreads)
decode_own_kernel(const ScaDecodeFwdParams p, const int head_chunks, const WeightsParams x, const __grid_constant__ PrefixGroups groups) {
    extern __shared__ __align__(128) unsigned char smem[];
    // Behind a prefix kernel this one may run beside it: every CTA of that one has waited for the kernels before it, and nothing
    // here reads what it writes. The wait at the end makes the end of this kernel that of both.
    if (!x.behind_prefix) WaitForPredecessor();
    const OwnTokens own{p, groups, x.bound};
    const ScoreTap tap{x.scores, x.score_row};
    WalkSteps<true, kSpan, true>(p, head_chunks, own, [&](int64_t b, int hk, int hc, int64_t j_begin, int64_t j_end, int slot) {
        const int64_t first = own.First(b);
        DecodeSegment<T, D, true, kHi, false, ScoreTap>(p, smem, b, hk, hc, first + j_begin, first + j_end, slot, tap);
    });
    if (x.behind_prefix) WaitForPredecessor();
}

constexpr int kFinishThreads = 256;
constexpr int kChunk = 4 * kFinishThreads;  // tokens a CTA weighs at once
constexpr int kHeadSlab = 32;               // query heads whose M and 1 / L stand in shared memory

// Maximum and sum over the parts of a row, by a whole warp.
struct RowStats {
    float m, l;
};
__device__ __forceinline__ RowStats StatsOf(const ScaDecodeFwdParams& p, const PrefixParts& prefix, int parts, int prefix_parts, int64_t row) {
    const int lane = threadIdx.x & 31;
    const int own = static_cast<int>(p.num_splits);
    auto each = [&](auto f) {
        for (int i = lane; i < own; i += 32) f(p.partial_m[row * own + i], p.partial_l[row * own + i]);
        for (int i = lane; i < prefix_parts; i += 32) f(prefix.m[row * parts + i], prefix.l[row * parts + i]);
    };
    float m = -CUDART_INF_F, l = 0.0f;
    each([&](float mi, float) { m = fmaxf(m, mi); });
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    each([&](float mi, float li) {
        if (mi != -CUDART_INF_F || li != 0.0f) l += li * Exp2(mi - m);
    });
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    return {m, l};
}

// Blocks [0, merge_blocks) merge output rows, the others weigh tokens: block (s * kv_heads + g) * chunks + c of those has chunk c.
template <typename T>
__global__ void __launch_bounds__(kFinishThreads)
decode_finish_kernel(const ScaDecodeFwdParams p, const WeightsParams x, const int merge_blocks, const int chunks,
                     const __grid_constant__ PrefixGroups groups) {
    __shared__ float s_m[kHeadSlab], s_inv[kHeadSlab];
    BeginAfterPredecessor();
    const int own = static_cast<int>(p.num_splits), parts = groups.parts;
    auto prefix_parts_of = [&](int64_t b) {
        const PrefixGroup* g = GroupOf(groups, b);
        const int tiles = g != nullptr ? (g->tokens + 127) / 128 : 0;
        return groups.part_tiles > 0 ? (tiles + groups.part_tiles - 1) / groups.part_tiles : 0;
    };
    if (static_cast<int>(blockIdx.x) < merge_blocks) {
        const int lanes = static_cast<int>(p.head_dim) / 4;  // threads to a row, four numbers each
        const int64_t total = p.batch * p.num_heads * lanes;
        for (int64_t item = static_cast<int64_t>(blockIdx.x) * kFinishThreads + threadIdx.x; item < total; item += static_cast<int64_t>(merge_blocks) * kFinishThreads) {
            const int64_t row = item / lanes, b = row / p.num_heads;
            const int d = static_cast<int>(item % lanes) * 4;
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
            T* out = reinterpret_cast<T*>(p.out) + b * p.o_stride.s_b + (row % p.num_heads) * p.o_stride.s_h + d;
            *reinterpret_cast<uint2*>(out) = make_uint2(Pack2<T>(acc.x * inv, acc.y * inv), Pack2<T>(acc.z * inv, acc.w * inv));
        }
        return;
    }
    const int64_t unit = (static_cast<int64_t>(blockIdx.x) - merge_blocks) / chunks;
    const int chunk = static_cast<int>((static_cast<int64_t>(blockIdx.x) - merge_blocks) % chunks);
    const int64_t b = unit / p.num_kv_heads, g = unit % p.num_kv_heads;
    const OwnTokens tokens{p, groups, x.bound};
    const int64_t first = tokens.First(b), end = tokens.Length(b);
    if (end <= static_cast<int64_t>(chunk) * kChunk || first >= static_cast<int64_t>(chunk + 1) * kChunk) return;
    const int64_t j = static_cast<int64_t>(chunk) * kChunk + 4 * threadIdx.x;  // the first of four tokens that this thread weighs
    const int group = static_cast<int>(p.num_heads / p.num_kv_heads);
    const int prefix_parts = prefix_parts_of(b);
    const int64_t row0 = b * p.num_heads + g * group;
    const bool mine = j + 3 >= first && j < end;
    float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int h0 = 0; h0 < group; h0 += kHeadSlab) {
        const int heads = min(kHeadSlab, group - h0);
        for (int h = threadIdx.x >> 5; h < heads; h += kFinishThreads / 32) {
            const RowStats r = StatsOf(p, x.prefix, parts, prefix_parts, row0 + h0 + h);
            if ((threadIdx.x & 31) == 0) {
                s_m[h] = r.m == -CUDART_INF_F ? 0.0f : r.m;
                s_inv[h] = r.l == 0.0f ? 0.0f : 1.0f / r.l;
            }
        }
        __syncthreads();
        if (mine) {
            const float* scores = x.scores + (row0 + h0) * x.score_row + j;
            for (int h = 0; h < heads; ++h) {
                const float4 s = *reinterpret_cast<const float4*>(scores + h * x.score_row);
                const float m = s_m[h], inv = s_inv[h];
                sum.x += Exp2(s.x - m) * inv;
                sum.y += Exp2(s.y - m) * inv;
                sum.z += Exp2(s.z - m) * inv;
                sum.w += Exp2(s.w - m) * inv;
            }
        }
        __syncthreads();
    }
    if (!mine) return;
    float* w = x.weights + unit * x.row + j;
    const float add[4] = {sum.x, sum.y, sum.z, sum.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (j + i >= first && j + i < end) w[i] += add[i];
    }
}

constexpr int64_t kMostSplits = 64;

// What a call is made of: sizes of its launches, and where its arrays lie in the scratch.
struct Plan {
    PrefixGroups groups;
    int64_t splits;
    int64_t bound;                // tokens of a sequence at most
    int64_t own_l, own_o;         // floats from the start: own_m at 0
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

// A validated call.
Plan MakePlan(const ScaDecodeFwdParams& p, const ScaPagedStep& x) {
    Plan plan{};
    PrefixGroups& groups = plan.groups;
    const int64_t capacity = p.max_blocks_per_seq * p.block_size;
    plan.bound = x.longest_len > 0 ? std::min(x.longest_len, capacity) : capacity;
    int64_t prefix_of_all = 0;  // tokens that are read for others
    for (int64_t g = 0; g < x.num_groups; ++g) {
        const int64_t tokens = std::min<int64_t>(x.prefix_lens[g], plan.bound) / p.block_size * p.block_size;
        const int64_t sequences = x.cu_groups[g + 1] - x.cu_groups[g];
        if (sequences < 2 || tokens == 0) continue;
        groups.group[groups.count++] = {x.cu_groups[g], x.cu_groups[g + 1], static_cast<int>(tokens), 0};
        prefix_of_all += sequences * tokens;
    }
    if (groups.count > 0) PlanPrefixParts(p, &groups);

    // Slots for the parts of a sequence's own tokens: enough for an even schedule (see slots_for_schedule in ops.py). The kernel takes
    // larger shares where these hold fewer.
    const int64_t typical = std::max<int64_t>(1, (x.typical_len > 0 ? std::min(x.typical_len, plan.bound) : plan.bound) - prefix_of_all / p.batch);
    const int64_t group_heads = p.num_heads / p.num_kv_heads;
    const int64_t columns = p.num_kv_heads * ((group_heads + 15) / 16);
    const int64_t steps = (typical + kSpan - 1) / kSpan, longest = (x.longest_len > 0 && groups.count == 0 ? (plan.bound + kSpan - 1) / kSpan : 2 * steps);
    const int64_t sharers = std::max<int64_t>(1, 2 * SmCount() / columns);
    const int64_t share = std::max<int64_t>(1, (p.batch * steps + sharers - 1) / sharers);
    plan.splits = longest <= 1 ? 1 : std::max<int64_t>(2, std::min((longest + share - 1) / share + 1, kMostSplits));

    const int64_t rows = p.batch * p.num_heads;
    plan.own_l = rows * plan.splits;
    plan.own_o = RoundUp(2 * plan.own_l, 4);  // an O starts on 16 bytes
    plan.prefix_m = plan.own_o + rows * plan.splits * p.head_dim;
    plan.prefix_l = plan.prefix_m + rows * groups.parts;
    plan.prefix_o = RoundUp(plan.prefix_l + rows * groups.parts, 8);  // 32
    plan.scores = RoundUp(plan.prefix_o + rows * groups.parts * p.head_dim, 8);
    plan.score_row = x.weights != nullptr ? RoundUp(plan.bound, kTile) : 0;
    plan.floats = plan.scores + rows * plan.score_row;
    return plan;
}

template <typename T, int D, bool kHi>
int LaunchOwn(const ScaDecodeFwdParams& p, const WeightsParams& x, const PrefixGroups& groups, cudaStream_t stream) {
    using G = DecodeGeom<D>;
    auto kernel = decode_own_kernel<T, D, kHi>;
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
    const int64_t useful = p.num_splits == 1 ? p.batch : p.batch * steps;  // CTAs of a column that can have something to do
    const int64_t blocks = wave >= columns ? columns * std::max<int64_t>(1, std::min(wave / columns, useful)) : wave;
    LaunchDependent(kernel, blocks, kThreads, G::kSmemBytes, stream, 1, p, head_chunks, x, groups);
    return CheckLaunch("decode_own_kernel", stream);
}

template <typename T>
int LaunchStep(const ScaDecodeFwdParams& p, const WeightsParams& x, const PrefixGroups& groups, cudaStream_t stream) {
    const bool hi = p.num_heads / p.num_kv_heads > 8;
    int rc = SCA_OK;
    switch (p.head_dim) {
        case 32: rc = hi ? LaunchOwn<T, 32, true>(p, x, groups, stream) : LaunchOwn<T, 32, false>(p, x, groups, stream); break;
        case 64: rc = hi ? LaunchOwn<T, 64, true>(p, x, groups, stream) : LaunchOwn<T, 64, false>(p, x, groups, stream); break;
        case 96: rc = hi ? LaunchOwn<T, 96, true>(p, x, groups, stream) : LaunchOwn<T, 96, false>(p, x, groups, stream); break;
        case 128: rc = hi ? LaunchOwn<T, 128, true>(p, x, groups, stream) : LaunchOwn<T, 128, false>(p, x, groups, stream); break;
        case 160: rc = hi ? LaunchOwn<T, 160, true>(p, x, groups, stream) : LaunchOwn<T, 160, false>(p, x, groups, stream); break;
        case 192: rc = hi ? LaunchOwn<T, 192, true>(p, x, groups, stream) : LaunchOwn<T, 192, false>(p, x, groups, stream); break;
        default: rc = hi ? LaunchOwn<T, 256, true>(p, x, groups, stream) : LaunchOwn<T, 256, false>(p, x, groups, stream); break;
    }
    if (rc != SCA_OK) return rc;
    const int64_t merge_items = p.batch * p.num_heads * (p.head_dim / 4);
    const int64_t merge_blocks = std::min<int64_t>((merge_items + kFinishThreads - 1) / kFinishThreads, 1 << 16);
    const int64_t chunks = x.weights != nullptr ? (x.bound + kChunk - 1) / kChunk : 0;
    const int64_t blocks = merge_blocks + p.batch * p.num_kv_heads * chunks;
    if (blocks > 0x7fffffffLL) return Fail(SCA_INVALID_ARGUMENT, "paged attention (weights): grid of " + std::to_string(blocks) + " blocks is out of range");
    LaunchDependent(decode_finish_kernel<T>, blocks, kFinishThreads, 0, stream, 1, p, x, static_cast<int>(merge_blocks), static_cast<int>(std::max<int64_t>(chunks, 1)), groups);
    return CheckLaunch("decode_finish_kernel", stream);
}

}  // namespace
}  // namespace sca_b200

using namespace sca_b200;

extern "C" long long sca_paged_step_scratch_floats(const ScaDecodeFwdParams* params, const ScaPagedStep* step) {
    ClearError();
    if (Validate(params, step, "paged step") != SCA_OK) return -1;
    return MakePlan(*params, *step).floats;
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
    const Plan plan = MakePlan(p, x);
    if (x.scratch_floats < plan.floats) {
        return Fail(SCA_INVALID_ARGUMENT, "paged step: scratch of " + std::to_string(x.scratch_floats) + " floats is too small (" + std::to_string(plan.floats) + " needed)");
    }
    float* scratch = x.scratch;
    p.num_splits = plan.splits;
    p.partial_m = scratch;
    p.partial_l = scratch + plan.own_l;
    p.partial_o = scratch + plan.own_o;
    p.seq_kv = p.num_kv_blocks * p.block_size;  // of a sequence without a length: all of its row
    p.k_stride = p.v_stride = ScaDecodeStrides{0, p.head_dim, p.num_kv_heads * p.head_dim};
    WeightsParams w{};
    w.weights = x.weights;
    w.row = x.weights_row;
    w.scores = x.weights != nullptr ? scratch + plan.scores : nullptr;
    w.score_row = plan.score_row;
    w.bound = plan.bound;
    w.prefix = PrefixParts{scratch + plan.prefix_m, scratch + plan.prefix_l, scratch + plan.prefix_o};
    w.behind_prefix = plan.groups.count > 0;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (plan.groups.count > 0) {
        if (int rc = LaunchPrefixParts(p, plan.groups, w.prefix, s)) return rc;
    }
    return p.dtype == SCA_DTYPE_F16 ? LaunchStep<__half>(p, w, plan.groups, s) : LaunchStep<__nv_bfloat16>(p, w, plan.groups, s);
}

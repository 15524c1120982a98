// Eviction from a paged cache by accumulated weight: every kv head of a sequence that is longer than its limit m keeps its first tokens, its
// last ones, and of those in between the heaviest, in place.
//
// What is kept stays where it is if it can. With n tokens, `first` and `recent` protected and stay = m - first - recent, the places are
//   [0, first)               the first tokens, untouched
//   [first, m - recent)      `stay` of those in between: the kept ones that are here already, and in the places that come free, lowest
//                            first, the kept ones from behind m - recent, lowest first
//   [m - recent, m)          the last `recent` tokens in their order
// so that a row moves once at most, and of the places in between only those whose token goes. Attention does not depend on the order of the
// keys; what does, the last tokens and a causal mask over new ones, keeps its order.
//
// A cluster of CTAs takes one (sequence, kv head). The `stay`-th largest weight is found digit by digit (8 bits of a key that orders
// like the numbers at a time) from histograms in shared memory, which the CTAs read from one another; ties go to the lower place by counting.
// Free places and rows that move are listed by rank in scratch, then all CTAs copy. No free place is the source of a move, so that these
// copies need no order. The last tokens move down behind them, all rows of a wave read before the first one of it is written: the
// destination of a row is never behind its source, so that later waves read what no earlier one has written.
// Bound by memory where there are many sequences: 192 of 500 to 6000 tokens, 8 kv heads, D=128, down to 2000: 246 us, 5.2 TB/s. One sequence is
// a chain of phases: of 100 thousand tokens 49 us, of which 19 are the copies, 16 the digits, 9 the lists; of 1100 13 us.
// Algorithmic traffic: 8 bytes a token and kv head of weights, and 4 * row bytes a moved row (K and V, read and written).
#include <algorithm>
#include <type_traits>

#include "common.cuh"

namespace sca_b200 {
namespace {

constexpr int kEvictThreads = 256;
constexpr int kEvictWarps = kEvictThreads / 32;
constexpr int kDigits = 4;
constexpr int kBins = 256;
static_assert(kBins == kEvictThreads, "a bin to a thread");
constexpr int kEvictCluster = 16;  // CTAs to a (sequence, kv head) at most
constexpr int kEvictCtas = 4;      // CTAs to an SM that there are registers for; shared memory for, where a CTA keeps up to 13 thousand keys
// Pieces that a thread has on their way at once; 16, with registers for one CTA to an SM, take 53.7 us for 49.2 (100 thousand tokens).
constexpr int kHeld = 8;
constexpr int kLoads = 8;          // weights that a thread has on their way at once

struct EvictParams {
    void *k, *v;
    float* weights;            // [num_seqs][kv_heads][weights_row]
    const int32_t* page_table; // [num_seqs][max_blocks]
    const int32_t* seq_lens;
    const int32_t* first;      // [num_seqs]; null: first_of_all
    int32_t* new_lens;
    int32_t* lists;            // [num_seqs * kv_heads][2][list]: free places, sources
    int64_t weights_row, list;
    int32_t max_blocks, block_size, num_blocks, kv_heads;
    int32_t first_of_all, keep, recent;
    int32_t cached;            // keys that a CTA keeps in shared memory
    int32_t cluster;
    int32_t row_pieces;        // of K: pieces of sizeof(V) bytes to a token of one kv head
};

// Orders like the numbers: NaN above all, both zeros alike.
__device__ __forceinline__ uint32_t KeyOf(float w) {
    if (w != w) return 0xffffffffu;
    const uint32_t bits = __float_as_uint(w == 0.0f ? 0.0f : w);
    return (bits >> 31) ? ~bits : bits | 0x80000000u;
}

template <typename V>
__global__ void __launch_bounds__(kEvictThreads, kEvictCtas)
kv_evict_kernel(const EvictParams p) {
    extern __shared__ __align__(16) uint32_t smem[];
    uint32_t(*hist)[kBins] = reinterpret_cast<uint32_t(*)[kBins]>(smem);
    uint32_t* cache = smem + kDigits * kBins;
    __shared__ int s_ties[kEvictWarps], s_free[kEvictWarps], s_late[kEvictWarps];
    __shared__ int s_counts[2];            // free places and late rows of this CTA's slice
    __shared__ uint32_t s_warp[2][kEvictWarps], s_found[2][3];
    BeginAfterPredecessor();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = static_cast<int>(ClusterRank()), cluster = p.cluster;
    const int64_t unit = static_cast<int64_t>(blockIdx.x) / cluster;
    const int64_t seq = unit / p.kv_heads;
    const int head = static_cast<int>(unit % p.kv_heads);
    const int64_t capacity = static_cast<int64_t>(p.max_blocks) * p.block_size;
    const int n = static_cast<int>(min(max(static_cast<int64_t>(p.seq_lens[seq]), int64_t{0}), capacity));
    const int64_t first64 = max(p.first != nullptr ? p.first[seq] : p.first_of_all, 0);
    const int64_t m64 = max(static_cast<int64_t>(p.keep), first64 + p.recent);
    if (head == 0 && rank == 0 && threadIdx.x == 0) p.new_lens[seq] = static_cast<int32_t>(min(static_cast<int64_t>(n), m64));
    if (n <= m64) return;  // all CTAs of the cluster
    const int first = static_cast<int>(first64), m = static_cast<int>(m64), recent = p.recent;
    const int stay = m - first - recent, between = n - recent - first, keep_end = m - recent;
    float* w = p.weights + unit * p.weights_row;
    int32_t* free_places = p.lists + unit * 2 * p.list;
    int32_t* sources = free_places + p.list;
    const int32_t* table = p.page_table + seq * p.max_blocks;
    int moves = 0;

    const int slice = (between + cluster - 1) / cluster;
    const int begin = first + min(rank * slice, between), count = first + min((rank + 1) * slice, between) - begin;
    auto select = [&](auto all_cached) {
        constexpr bool kAllCached = decltype(all_cached)::value;  // a look at every key costs half of the phases' time otherwise
        // ---- the stay-th largest key -------------------------------------------------------------------------
        for (int i = threadIdx.x; i < kDigits * kBins; i += kEvictThreads) smem[i] = 0;
        __syncthreads();
        auto key_at = [&](int i) { return kAllCached || i < p.cached ? cache[i] : KeyOf(w[begin + i]); };
        uint32_t prefix = 0, border = 0, need = static_cast<uint32_t>(stay), equal = 0;
#pragma unroll
        for (int digit = 0; digit < kDigits; ++digit) {
            const int shift = 24 - 8 * digit;
            if (digit == 0) {
                // Few values are possible here, a sign and seven bits of exponent, but a warp that adds up equal ones by itself (__match_any_sync)
                // is slower: 100 thousand tokens, one CTA, 817 us for 780.
                for (int i0 = 0; i0 < count; i0 += kLoads * kEvictThreads) {
                    float x[kLoads];
#pragma unroll
                    for (int e = 0; e < kLoads; ++e) {
                        const int i = i0 + e * kEvictThreads + threadIdx.x;
                        if (i < count) x[e] = w[begin + i];
                    }
#pragma unroll
                    for (int e = 0; e < kLoads; ++e) {
                        const int i = i0 + e * kEvictThreads + threadIdx.x;
                        if (i >= count) continue;
                        const uint32_t key = KeyOf(x[e]);
                        if (i < p.cached) cache[i] = key;
                        atomicAdd(&hist[0][key >> shift], 1u);
                    }
                }
            } else {
#pragma unroll 4
                for (int i = threadIdx.x; i < count; i += kEvictThreads) {
                    const uint32_t key = key_at(i);
                    if ((key >> (shift + 8)) == prefix) atomicAdd(&hist[digit][(key >> shift) & 255u], 1u);
                }
            }
            ClusterBarrier();
            // a bin a thread, the highest first, of all CTAs; each begins with its own, so that they do not all read from one
            const int bin = kBins - 1 - static_cast<int>(threadIdx.x);
            uint32_t mine = 0;
            for (int i0 = 0; i0 < cluster; i0 += kLoads) {
                uint32_t x[kLoads];
#pragma unroll
                for (int e = 0; e < kLoads; ++e) {
                    const int i = rank + i0 + e;
                    x[e] = i0 + e < cluster ? __float_as_uint(LoadFromRank(SmemAddr(&hist[digit][bin]), i < cluster ? i : i - cluster)) : 0u;
                }
#pragma unroll
                for (int e = 0; e < kLoads; ++e) mine += x[e];
            }
            uint32_t incl = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t up = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += up;
            }
            if (lane == 31) s_warp[digit & 1][warp] = incl;
            __syncthreads();
            uint32_t above = incl - mine;
            for (int i = 0; i < warp; ++i) above += s_warp[digit & 1][i];
            if (above < need && need <= above + mine) {
                s_found[digit & 1][0] = static_cast<uint32_t>(bin);
                s_found[digit & 1][1] = above;
                s_found[digit & 1][2] = mine;
            }
            __syncthreads();
            prefix = (prefix << 8) | s_found[digit & 1][0];
            need -= s_found[digit & 1][1];
            equal = s_found[digit & 1][2];
            border = prefix << shift;
            if (equal == need) break;  // all keys that begin like this stay
        }
        // keys above the border stay, and `need` of those equal to it, the lowest places first
        // ---- ranks: every warp walks a piece of the slice --------------------------------------------------------
        const int piece = ((count + kEvictWarps - 1) / kEvictWarps + 31) / 32 * 32;
        const int piece_begin = min(warp * piece, count), piece_end = min(piece_begin + piece, count);
        int ties_before = 0;
        if (equal != need) {  // some of the equal ones go
            for (int r = 0; r < rank; ++r) ties_before += __float_as_int(LoadFromRank(SmemAddr(&hist[kDigits - 1][border & 255u]), r));
            int ties = 0;
            for (int i = piece_begin; i < piece_end; i += 32) {
                const bool tie = i + lane < piece_end && key_at(i + lane) == border;
                ties += __popc(__ballot_sync(0xffffffffu, tie));
            }
            if (lane == 0) s_ties[warp] = ties;
            __syncthreads();
            for (int i = 0; i < warp; ++i) ties_before += s_ties[i];
        }
        const uint32_t below = (1u << lane) - 1u;
        // f(place, is free, is late, ballots of both)
        auto walk = [&](auto f) {
            if (equal == need) {
#pragma unroll 4
                for (int i = piece_begin; i < piece_end; i += 32) {
                    const bool in = i + lane < piece_end, kept = in && key_at(i + lane) >= border;
                    const int place = begin + i + lane;
                    const bool is_free = in && !kept && place < keep_end, is_late = kept && place >= keep_end;
                    f(place, is_free, is_late, __ballot_sync(0xffffffffu, is_free), __ballot_sync(0xffffffffu, is_late));
                }
                return;
            }
            int tie_rank = ties_before;
            for (int i = piece_begin; i < piece_end; i += 32) {
                const bool in = i + lane < piece_end;
                const uint32_t key = in ? key_at(i + lane) : 0u;
                const uint32_t tie = __ballot_sync(0xffffffffu, in && key == border);
                const bool kept = in && (key > border || (key == border && tie_rank + __popc(tie & below) < static_cast<int>(need)));
                tie_rank += __popc(tie);
                const int place = begin + i + lane;
                const bool is_free = in && !kept && place < keep_end, is_late = kept && place >= keep_end;
                f(place, is_free, is_late, __ballot_sync(0xffffffffu, is_free), __ballot_sync(0xffffffffu, is_late));
            }
        };
        int free_count = 0, late_count = 0;
        walk([&](int, bool, bool, uint32_t free_lanes, uint32_t late_lanes) {
            free_count += __popc(free_lanes);
            late_count += __popc(late_lanes);
        });
        if (lane == 0) {
            s_free[warp] = free_count;
            s_late[warp] = late_count;
        }
        __syncthreads();
        if (threadIdx.x < 2) {
            const int* counts = threadIdx.x == 0 ? s_free : s_late;
            int sum = 0;
            for (int i = 0; i < kEvictWarps; ++i) sum += counts[i];
            s_counts[threadIdx.x] = sum;
        }
        ClusterBarrier();
        int free_rank = 0, late_rank = 0;
        for (int r = 0; r < cluster; ++r) {
            const float2 x = make_float2(LoadFromRank(SmemAddr(&s_counts[0]), r), LoadFromRank(SmemAddr(&s_counts[1]), r));
            moves += __float_as_int(x.x);
            if (r < rank) {
                free_rank += __float_as_int(x.x);
                late_rank += __float_as_int(x.y);
            }
        }
        for (int i = 0; i < warp; ++i) {
            free_rank += s_free[i];
            late_rank += s_late[i];
        }
        walk([&](int place, bool is_free, bool is_late, uint32_t free_lanes, uint32_t late_lanes) {
            if (is_free) free_places[free_rank + __popc(free_lanes & below)] = place;
            if (is_late) sources[late_rank + __popc(late_lanes & below)] = place;
            free_rank += __popc(free_lanes);
            late_rank += __popc(late_lanes);
        });
        ClusterBarrier();
    };
    if (stay > 0) {
        if (count <= p.cached) select(std::true_type{});
        else select(std::false_type{});
    }

    // ---- copies: a warp looks up as many moves as it has lanes, one each, and copies their rows together ---------------
    // A step copies `moves_a_step` of them, or one in several steps where its pieces are more than a warp's lanes.
    const int row_pieces = p.row_pieces, move_pieces = 2 * row_pieces;  // K, then V
    const int moves_a_step = max(1, 32 / move_pieces), steps_a_move = (move_pieces + 31) / 32;
    const int lane_move = steps_a_move > 1 ? 0 : lane / move_pieces, lane_part = lane - lane_move * move_pieces;
    const bool lane_works = lane_move < moves_a_step;
    const int64_t token_pieces = static_cast<int64_t>(p.kv_heads) * row_pieces;
    auto row_of = [&](int place) {  // of the pool; negative: its page is not mapped
        const int page = place / p.block_size;
        const int32_t id = table[page];
        return id >= 0 && id < p.num_blocks ? id * p.block_size + (place - page * p.block_size) : -1;
    };
    // where piece `part` of this head's row 0 of the pool is
    auto piece_of = [&](int part) {
        return (part < row_pieces ? static_cast<V*>(p.k) + part : static_cast<V*>(p.v) + (part - row_pieces)) + static_cast<int64_t>(head) * row_pieces;
    };
    V* const lane_base = piece_of(lane_part);
    // step `s` of the moves whose rows the lanes hold in `row`: this lane's piece; null: none
    auto piece_at = [&](int s, int row, int count) -> V* {
        const int first = steps_a_move == 1 ? s * moves_a_step : s / steps_a_move;
        const int at = __shfl_sync(0xffffffffu, row, (first + lane_move) & 31);
        if (first + lane_move >= count || at < 0 || !lane_works) return nullptr;
        if (steps_a_move == 1) return lane_base + at * token_pieces;
        const int part = (s - first * steps_a_move) * 32 + lane;
        return part < move_pieces ? piece_of(part) + at * token_pieces : nullptr;
    };
    const int warps = cluster * kEvictWarps, my_warp = rank * kEvictWarps + warp;
    // few moves are spread over all warps
    const int batch = min(32, max(4, (moves + warps - 1) / warps));
    for (int move0 = batch * my_warp; move0 < moves; move0 += batch * warps) {
        const int count = min(batch, moves - move0);
        int from = -1, into = -1;
        if (lane < count) {
            const int src = sources[move0 + lane], dst = free_places[move0 + lane];
            const float weight = w[src];
            from = row_of(src);
            into = row_of(dst);
            if (from < 0 || into < 0) from = into = -1;
            w[dst] = weight;
        }
        const int steps = (count + moves_a_step - 1) / moves_a_step * steps_a_move;
        for (int s0 = 0; s0 < steps; s0 += kHeld) {
            V held[kHeld];
#pragma unroll
            for (int i = 0; i < kHeld; ++i) {
                const V* at = piece_at(s0 + i, from, count);
                if (at != nullptr) held[i] = *at;
            }
#pragma unroll
            for (int i = 0; i < kHeld; ++i) {
                V* at = piece_at(s0 + i, into, count);
                if (at != nullptr) *at = held[i];
            }
        }
    }
    // The last tokens: a warp has kHeld steps at a time. A row of more steps takes several turns, of other columns each.
    const int wave_rows = steps_a_move == 1 ? min(32, kHeld * moves_a_step) : max(1, kHeld / steps_a_move);  // of a warp
    const int turns = (steps_a_move + kHeld - 1) / kHeld;
    for (int row0 = 0; row0 < recent || row0 == 0; row0 += wave_rows * warps) {
        const int mine = row0 + my_warp * wave_rows, count = min(max(recent - mine, 0), wave_rows);
        int from = -1, into = -1;
        float weight = 0.0f;
        if (lane < count) {
            weight = w[n - recent + mine + lane];
            from = row_of(n - recent + mine + lane);
            into = row_of(keep_end + mine + lane);
            if (from < 0 || into < 0) from = into = -1;
        }
        for (int turn = 0; turn < turns; ++turn) {
            V held[kHeld];
#pragma unroll
            for (int i = 0; i < kHeld; ++i) {
                const V* at = piece_at(turn * kHeld + i, from, count);
                if (at != nullptr) held[i] = *at;
            }
            ClusterBarrier();
            if (turn == 0 && lane < count) w[keep_end + mine + lane] = weight;
#pragma unroll
            for (int i = 0; i < kHeld; ++i) {
                V* at = piece_at(turn * kHeld + i, into, count);
                if (at != nullptr) *at = held[i];
            }
        }
    }
    const int threads = cluster * kEvictThreads, me = rank * kEvictThreads + threadIdx.x;
    for (int j = m + me; j < n; j += threads) w[j] = 0.0f;  // every weight has been read by now
}

// Keys that stay in shared memory between the digits; what a CTA has beyond them is read again. So many leave three CTAs to an SM; with 12 800, which leave
// four, 192 sequences of up to 6000 tokens in a table of 131 072 take 263 us for 277, but 100 of 15 000 tokens 664 for 485 and 20 of 30 000 306 for 223.
constexpr int kCachedKeys = 16384;

template <typename V>
int LaunchEvict(const EvictParams& p, int64_t units, cudaStream_t stream) {
    constexpr size_t kHistograms = kDigits * kBins * sizeof(uint32_t);
    const size_t smem = kHistograms + static_cast<size_t>(p.cached) * sizeof(uint32_t);
    auto kernel = kv_evict_kernel<V>;
    if (int rc = EnsureDynamicSmem(reinterpret_cast<const void*>(kernel), kHistograms + kCachedKeys * sizeof(uint32_t), "kv_evict_kernel")) return rc;
    static PerDevice allowed;  // per instantiation: clusters of more than 8 CTAs have to be asked for
    if (p.cluster > 8 && allowed.Get([&] { return cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) == cudaSuccess ? 1 : -1; }) < 1) {
        return FailCuda(cudaGetLastError(), "kv_evict_kernel: clusters of more than 8 CTAs");
    }
    LaunchDependent(kernel, units * p.cluster, kEvictThreads, smem, stream, p.cluster, p);
    return CheckLaunch("kv_evict_kernel", stream);
}

// CTAs to a (sequence, kv head). More of them shorten the chain of phases of a long one and cost barriers in a short one; up to 8 as long as
// all CTAs are resident (counted as 4 to an SM), 16 where that leaves one to an SM. The lengths are on the device: the width of the table stands for
// them here and for the keys that a CTA keeps, and one that is much wider than its sequences costs (one of 1100 tokens in a table of 1104 / 131 072: 11.8 /
// 15.7 us, 192 of 500 to 6000 in one of 6016 / 131 072: 220 / 276). us for 8 kv heads, D=128, 16 bits, 1 / 2 / 4 / 8 / 16 CTAs:
//   one sequence of 1100 tokens down to 1024   12.5 / 13.6 / 13.4 / 13.7 / 17.7     4 of 8192 to 4096    101 / 58 / 35 / 30 / 49
//   of 2200 to 1024                            32.4 / 26.1 / 16.8 / 15.4 / 18.1     8 of 16000 to 4000   160 / 89 / 60 / 61 / 95
//   of 8192 to 4096                            85.6 / 48.8 / 30.0 / 21.8 / 22.2     16 of 4096 to 2048    62 / 46 / 44 / 56 / 115
//   of 16000 to 8000                            168 / 90 / 50 / 31.6 / 26.9         32 of 8192 to 4096   142 / 138 / 133 / 154 / 254
//   of 33000 to 4000                            248 / 91 / 53 / 33.8 / 28.2         64 of 2200 to 1024    80 / 90 / 101 / 161 / 367
int ClusterFor(int64_t units, int64_t capacity) {
    if (units * 16 <= SmCount() && capacity >= 12000) return 16;
    int cluster = 8;
    while (cluster > 1 && (units * cluster > kEvictCtas * SmCount() || capacity / cluster < 256)) cluster /= 2;
    return cluster;
}

int64_t ListLength(int64_t keep, int64_t capacity) { return std::max<int64_t>(1, std::min(keep, capacity)); }

}  // namespace
}  // namespace sca_b200

using namespace sca_b200;

extern "C" long long sca_kv_evict_scratch_ints(int64_t num_seqs, int64_t num_kv_heads, int64_t keep, int64_t max_tokens) {
    if (num_seqs < 1 || num_kv_heads < 1 || keep < 0 || max_tokens < 1) return -1;
    return num_seqs * num_kv_heads * 2 * ListLength(keep, max_tokens);
}

extern "C" int sca_launch_kv_evict(const ScaKvEvict* params, const ScaKvCacheShape* shape, int64_t elem_bytes, void* stream) {
    ClearError();
    auto invalid = [](const std::string& why) { return Fail(SCA_INVALID_ARGUMENT, "kv evict: " + why); };
    if (params == nullptr || shape == nullptr) return invalid("null parameter block");
    const ScaKvEvict& x = *params;
    if (x.layer_k == nullptr || x.layer_v == nullptr || x.weights == nullptr || x.page_table == nullptr || x.seq_lens == nullptr || x.new_lens == nullptr ||
        x.scratch == nullptr) {
        return invalid("null pointer");
    }
    if (x.new_lens == x.seq_lens) return invalid("the new lengths go to memory of their own");
    if (shape->num_blocks < 1 || shape->block_size < 1 || shape->num_kv_heads < 1 || shape->head_dim < 1 || elem_bytes < 1 || x.num_seqs < 1 || x.max_blocks_per_seq < 1) {
        return invalid("sizes must be positive");
    }
    const int64_t capacity = x.max_blocks_per_seq * shape->block_size, units = x.num_seqs * shape->num_kv_heads;
    const int64_t row_bytes = shape->head_dim * elem_bytes;
    if (capacity > 0x7fffff00LL || shape->num_blocks > 0x7fffff00LL / shape->block_size || row_bytes > (1 << 20) || units > 0x7fffffffLL / kEvictCluster) return invalid("sizes are out of range");
    if (x.keep < 0 || x.recent < 0 || x.first < 0) return invalid("keep, recent and first must not be negative");
    if (x.weights_row < capacity) {
        return invalid("rows of " + std::to_string(x.weights_row) + " weights for page-table rows of " + std::to_string(capacity) + " tokens");
    }
    const int64_t need = sca_kv_evict_scratch_ints(x.num_seqs, shape->num_kv_heads, x.keep, capacity);
    if (x.scratch_ints < need) return invalid("scratch of " + std::to_string(x.scratch_ints) + " int32 is too small (" + std::to_string(need) + " needed)");
    EvictParams p{};
    p.k = x.layer_k;
    p.v = x.layer_v;
    p.weights = x.weights;
    p.page_table = x.page_table;
    p.seq_lens = x.seq_lens;
    p.first = x.first_lens;
    p.new_lens = x.new_lens;
    p.lists = x.scratch;
    p.weights_row = x.weights_row;
    p.list = ListLength(x.keep, capacity);
    p.max_blocks = static_cast<int32_t>(x.max_blocks_per_seq);
    p.block_size = static_cast<int32_t>(shape->block_size);
    p.num_blocks = static_cast<int32_t>(shape->num_blocks);
    p.kv_heads = static_cast<int32_t>(shape->num_kv_heads);
    // no sequence is longer than `capacity`: protected tokens beyond it are as good as that
    p.first_of_all = static_cast<int32_t>(std::min(x.first, capacity));
    p.keep = static_cast<int32_t>(std::min(x.keep, capacity));
    p.recent = static_cast<int32_t>(std::min(x.recent, capacity));
    p.cluster = ClusterFor(units, capacity);
    p.cached = static_cast<int32_t>(std::min<int64_t>((capacity + p.cluster - 1) / p.cluster, kCachedKeys));
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (row_bytes % 16 == 0 && Aligned16(x.layer_k) && Aligned16(x.layer_v)) {
        p.row_pieces = static_cast<int32_t>(row_bytes / 16);
        return LaunchEvict<uint4>(p, units, s);
    }
    p.row_pieces = static_cast<int32_t>(row_bytes);
    return LaunchEvict<unsigned char>(p, units, s);
}

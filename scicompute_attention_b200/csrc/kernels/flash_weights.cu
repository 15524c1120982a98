// What the tokens of a paged cache weigh in the attention of a chunk: weights[s, g, j] += the sum over the chunk's counted tokens i and the
// query heads h of kv head g of exp(scale q[i, h] . k[j] - lse[i, h]). It follows the prefill kernel, which leaves lse, the logarithm of each
// row's sum.
//
// An item is one tile of 128 keys of one (sequence, kv head): a CTA takes it and walks the query tiles that see it. Nobody else adds to its
// weights, so there are no atomics and the same call gives the same bits. The scores are computed with the keys as rows, S = K Q^T (tcgen05,
// M = 128 keys, N = 128 queries, into one of four buffers of tensor memory): a thread then has one key, and its sum over the queries needs no
// other thread until the end of the item. lse of the 128 queries lies in shared memory, where all threads read the same number at a time.
//   warps 0 - 15   two groups, which take the query tiles in turn; in a group two warps to 32 keys, with half of the columns each:
//                  2^(score * scale - lse), summed up
//   warp 16        TMA: tiles of keys, page by page, then their query tiles into a ring, and the queries' lse
//   warp 17        issues the products
// Items are dealt tile after tile, to the sequences that have it: with a place for every sequence up to the longest one's last tile a CTA walks what is not
// there (one sequence of 100 000 tokens among 255 of 500, 16 new ones each: 4.4 ms of 6.2).
// One CTA to an SM walks the list of items, those that most queries see first, and loads the next tile of keys under the current one: with a
// CTA to an item its start - barriers, tensor memory, the look-up of sequence and pages, the first loads - took 6 us (4 prompts of 2000, 32 / 8
// heads, D=128: 512 items 126 us; 9 sequences of which the last 64 tokens count, D=64: 2016 items 40 us).
// A query tile is 128 / P tokens of P query heads, as in the prefill, and starts with the first token that sees the tile's first key, so
// that a causal mask cuts 128 / P tokens' rows at most.
// No unit is at its limit: while an SM has work its special-function unit is busy 71 % of the time (16384 exponentials a tile take 1024 clocks, the
// products 540), and a quarter of the exponentials by a polynomial of degree 5 on the multipliers instead gained next to nothing (260 -> 256 us, half
// of them 266). A warp waits on the chain of its own tile and on shared memory, from which every thread reads 64 numbers of lse beside its 64 exponentials (stalls per issue:
// MIO throttle 2.4, wait 2.3, long scoreboard 2.2), and items do not come out even: the SMs have work 87 % of the time. 4 prompts of 1900 to 2048
// tokens, 32 / 8 heads, D=128: 112 us alone, 257 us with the prefill.
#include <algorithm>
#include <vector>

#include "flash_kernel.cuh"

namespace sca_b200 {
namespace flash {
namespace {

constexpr int kKeys = 128;     // keys of an item
constexpr int kColumns = 128;  // (token, head) rows of a query tile
constexpr int kGroups = 2, kGroupWarps = 8, kSumWarps = kGroups * kGroupWarps;
constexpr int kLoadWarp = kSumWarps, kMmaWarp = kSumWarps + 1;
constexpr int kWeightThreads = 32 * (kSumWarps + 2);
constexpr int kBuffers = 4;    // of scores in tensor memory

template <int DP>
struct WeightsGeom {
    static constexpr int kBlocks = DP / 64;              // 128-byte column blocks
    static constexpr int kTileBytes = kBlocks * kKeys * 128;
    static constexpr int kKeySlots = DP == 256 ? 1 : 2;  // tiles of keys
    static constexpr int kSlots = DP == 64 ? 8 : DP == 128 ? 4 : 2;  // query tiles
    static constexpr int kLse = (kKeySlots + kSlots) * kTileBytes;
    static constexpr int kSums = kLse + kSlots * kColumns * 4;        // [2][2 * kGroups][kKeys], items in turn
    static constexpr int kBars = kSums + 2 * 2 * kGroups * kKeys * 4;
    static constexpr int kSmemBytes = 1024 + kBars + 256;
    static_assert(kSmemBytes <= 232448, "exceeds the 227 KiB per-CTA limit");
};

// The sequences of a launch, as a parameter of the kernel, so that nothing is sent ahead: {first query token, place in the batch, S_q, S_kv}, those of
// the most tiles of keys first, and how many items there are up to the last tile of each; behind the last one a sequence of no tiles. A call of more of
// them takes several launches.
constexpr int kImageSeqs = 160;
struct SeqImage {
    int4 seqs[kImageSeqs + 1];
    int ends[kImageSeqs + 1];
};
__host__ __device__ inline int TilesOf(const int4& seq) { return (seq.w + kKeys - 1) / kKeys; }

struct ChunkParams {
    const float* lse;  // [heads][total_q], natural logarithm; -inf: the row sees nothing
    float* weights;
    int64_t weights_row, total_q;
    const int32_t* page_table;
    int* error_word;
    int max_blocks, num_blocks, block_size, block_shift;
    int heads, kv_heads, pack_shift, last, causal;
    int seqs, items;   // in the image, and the tiles of keys that they have, times the kv heads
    float scale_log2;
};

// A barrier of the warps that add up; whether all of them say so.
__device__ __forceinline__ bool AllSumWarps(bool mine) {
    uint32_t all;
    asm volatile(
        "{\n"
        ".reg .pred in, out;\n"
        "setp.ne.u32 in, %1, 0;\n"
        "barrier.cta.red.and.pred out, 1, %2, in;\n"
        "selp.u32 %0, 1, 0, out;\n"
        "}\n"
        : "=r"(all)
        : "r"(mine ? 1u : 0u), "n"(32 * kSumWarps)
        : "memory");
    return all != 0;
}

template <typename T, int DP>
__global__ void __launch_bounds__(kWeightThreads, 1)
chunk_weights_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const ChunkParams p,
                     const __grid_constant__ SeqImage image) {
    using G = WeightsGeom<DP>;
    extern __shared__ unsigned char smem_raw[];
    const uint32_t base = (SmemAddr(smem_raw) + 1023u) & ~1023u;
    unsigned char* smem = smem_raw + (base - SmemAddr(smem_raw));
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t k_smem = base, q_smem = base + G::kKeySlots * G::kTileBytes;
    float* lse_ring = reinterpret_cast<float*>(smem + G::kLse);
    auto bar = [&](int i) { return base + G::kBars + 8u * i; };
    constexpr int kKFull = 0, kKEmpty = kKFull + G::kKeySlots, kQFull = kKEmpty + G::kKeySlots, kQEmpty = kQFull + G::kSlots, kSFull = kQEmpty + G::kSlots,
                  kSEmpty = kSFull + kBuffers, kNumBars = kSEmpty + kBuffers;
    static_assert(kNumBars * 8 + 8 <= 256, "barrier area too small");
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + G::kBars + kNumBars * 8);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    if (threadIdx.x == 0) {
        for (int i = 0; i < G::kKeySlots; ++i) {
            MbarInit<1>(bar(kKFull + i));
            MbarInit<1>(bar(kKEmpty + i));
        }
        for (int i = 0; i < G::kSlots; ++i) {
            MbarInit<1 + 32>(bar(kQFull + i));            // the tile, and each lane's part of lse
            MbarInit<1 + kGroupWarps>(bar(kQEmpty + i));  // the products and the sums are done with it
        }
        for (int i = 0; i < kBuffers; ++i) {
            MbarInit<1>(bar(kSFull + i));
            MbarInit<kGroupWarps>(bar(kSEmpty + i));
        }
        *abort_flag = 0;
        FenceBarrierInit();
    }
    BeginAfterPredecessor();
    if (warp == kMmaWarp) {
        TmemAlloc(SmemAddr(tmem_slot), kBuffers * kColumns);
        TmemRelinquish();
    }
    TcFenceBefore();
    __syncthreads();
    TcFenceAfter();
    const uint32_t tmem = *tmem_slot;

    // ---- items: tile after tile of all sequences that have it and their kv heads, dealt in rounds of gridDim.x, every other one in reverse order ----
    const int heads_tile = 1 << p.pack_shift, tile_tokens = kColumns >> p.pack_shift;
    const int group = p.heads / p.kv_heads, packs = group >> p.pack_shift;
    const int rounds = (p.items + static_cast<int>(gridDim.x) - 1) / static_cast<int>(gridDim.x);  // at most 2^30 items
    struct Item {
        int seq, head_kv, key0, keys, new_tokens, q0;
        int first_token;  // that sees the first key and counts
        int tiles;        // 0: the sequence has no such keys
        int diagonal;     // token t sees keys up to t + diagonal
    };
    // what an item is, in two steps, so that the look-up in memory is made an item ahead
    struct Look {
        int seq, head_kv, key0;
        int4 s;
    };
    int active = p.seqs;  // those that have the tile: the first so many. Rounds go upwards, so this goes down
    auto look = [&](int round) {
        Look l;
        const int ctas = static_cast<int>(gridDim.x), me = static_cast<int>(blockIdx.x), index = round * ctas + ((round & 1) ? ctas - 1 - me : me);
        l.s = make_int4(0, 0, 0, 0);
        l.seq = l.head_kv = l.key0 = 0;
        if (round < rounds && index < p.items) {
            while (index >= image.ends[active - 1]) --active;
            // from the tile on at which the next shorter sequence ends
            const uint32_t units = static_cast<uint32_t>(active * p.kv_heads), at = static_cast<uint32_t>(index - image.ends[active]);
            const uint32_t tile = at / units, unit = at - tile * units, place = unit / static_cast<uint32_t>(p.kv_heads);
            l.s = image.seqs[place];
            l.seq = l.s.y;
            l.head_kv = static_cast<int>(unit - place * static_cast<uint32_t>(p.kv_heads));
            l.key0 = (TilesOf(image.seqs[active]) + static_cast<int>(tile)) * kKeys;
        }
        return l;
    };
    auto item_of = [&](const Look& l) {
        Item w;
        w.seq = l.seq, w.head_kv = l.head_kv, w.key0 = l.key0;
        w.q0 = l.s.x, w.new_tokens = l.s.z, w.keys = l.s.w;
        w.diagonal = p.causal ? w.keys - w.new_tokens : w.keys;
        w.first_token = max(p.last > 0 ? max(0, w.new_tokens - p.last) : 0, w.key0 - w.diagonal);
        w.tiles = w.key0 < w.keys ? (w.new_tokens - w.first_token + tile_tokens - 1) / tile_tokens * packs : 0;  // the last token sees every key
        return w;
    };
    auto token_of = [&](const Item& w, int tile) { return w.first_token + tile / packs * tile_tokens; };
    auto head_of = [&](const Item& w, int tile) { return w.head_kv * group + (tile % packs << p.pack_shift); };
    bool ok = true;

    if (warp == kLoadWarp) {
        // ---- loads ----
        if (lane == 0) {
            PrefetchTensorMap(&map_q);
            PrefetchTensorMap(&map_k);
        }
        const int pages = kKeys >> p.block_shift;
        uint32_t items = 0, loads = 0;
        auto page_of = [&](const Look& l) {  // of this lane, in the pool
            const int page = (l.key0 >> p.block_shift) + lane;
            const bool in = lane < pages && page < p.max_blocks && (static_cast<int64_t>(page) << p.block_shift) < l.s.w;
            return in ? p.page_table[static_cast<int64_t>(l.seq) * p.max_blocks + page] : -1;
        };
        Look next = look(0);
        int32_t next_id = page_of(next);
        for (int r = 0; r < rounds && ok; ++r) {
            const Item w = item_of(next);
            const int32_t id = next_id;
            next = look(r + 1);
            next_id = page_of(next);
            if (w.tiles == 0) continue;
            const int first_row = id >= 0 && id < p.num_blocks ? id << p.block_shift : p.num_blocks << p.block_shift;  // behind the pool: zeros
            const uint32_t k_slot = items % G::kKeySlots;
            ok = __all_sync(0xffffffffu, MbarWait(bar(kKEmpty + k_slot), ((items / G::kKeySlots) & 1u) ^ 1u, abort_flag));
            if (!ok) break;
            ++items;
            if (lane == 0) MbarExpectTx(bar(kKFull + k_slot), G::kTileBytes);
            __syncwarp();
            for (int i = 0; i < pages; ++i) {
                const int row = __shfl_sync(0xffffffffu, first_row, i);
                if (ElectOne()) {
#pragma unroll
                    for (int kb = 0; kb < G::kBlocks; ++kb) {
                        TmaLoad4D(k_smem + k_slot * G::kTileBytes + kb * (kKeys * 128) + i * p.block_size * 128, &map_k, bar(kKFull + k_slot), kb * 64, row, w.head_kv, 0);
                    }
                }
            }
            auto lse_of = [&](int tile, float (&v)[4]) {
                const int token0 = token_of(w, tile), head0 = head_of(w, tile);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int c = lane + 32 * i, token = token0 + (c >> p.pack_shift), head = head0 + (c & (heads_tile - 1));
                    v[i] = tile < w.tiles && token < w.new_tokens ? p.lse[static_cast<int64_t>(head) * p.total_q + w.q0 + token] : -CUDART_INF_F;
                }
            };
            float ahead[4];
            lse_of(0, ahead);
            for (int tile = 0; tile < w.tiles && ok; ++tile, ++loads) {
                const uint32_t slot = loads % G::kSlots;
                float v[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] = ahead[i];
                lse_of(tile + 1, ahead);
                ok = __all_sync(0xffffffffu, MbarWait(bar(kQEmpty + slot), ((loads / G::kSlots) & 1u) ^ 1u, abort_flag));
                if (!ok) break;
                if (ElectOne()) {
                    MbarExpectTx(bar(kQFull + slot), G::kTileBytes);
#pragma unroll
                    for (int kb = 0; kb < G::kBlocks; ++kb) {
                        TmaLoad4D(q_smem + slot * G::kTileBytes + kb * (kColumns * 128), &map_q, bar(kQFull + slot), kb * 64, head_of(w, tile), w.q0 + token_of(w, tile), 0);
                    }
                }
                __syncwarp();
                // a row that sees nothing has no sum: 2^-inf
#pragma unroll
                for (int i = 0; i < 4; ++i) lse_ring[slot * kColumns + lane + 32 * i] = v[i] == -CUDART_INF_F ? v[i] : -v[i] * kLog2e;
                MbarArrive(bar(kQFull + slot));
            }
        }
    } else if (warp == kMmaWarp) {
        // ---- products ----
        if (ElectOne()) {
            constexpr uint32_t fmt = std::is_same<T, __half>::value ? kFmtF16 : kFmtBf16;
            constexpr uint32_t idesc = MakeInstrDesc(fmt, fmt, 0, 0, kKeys, kColumns);
            const uint64_t major = MakeSmemDesc(0, 16, 1024);  // both K-major
            uint32_t items = 0, count = 0;
            Look next = look(0);
            for (int r = 0; r < rounds && ok; ++r) {
                const Item w = item_of(next);
                next = look(r + 1);
                if (w.tiles == 0) continue;
                const uint32_t k_slot = items % G::kKeySlots;
                const uint64_t a0 = major | (((k_smem + k_slot * G::kTileBytes) & 0x3FFFFu) >> 4);
                ok = MbarWait(bar(kKFull + k_slot), (items / G::kKeySlots) & 1u, abort_flag);
                ++items;
                for (int tile = 0; tile < w.tiles && ok; ++tile, ++count) {
                    const uint32_t slot = count % G::kSlots, buffer = count % kBuffers;
                    ok = MbarWait(bar(kQFull + slot), (count / G::kSlots) & 1u, abort_flag) && MbarWait(bar(kSEmpty + buffer), ((count / kBuffers) & 1u) ^ 1u, abort_flag);
                    if (!ok) break;
                    TcFenceAfter();
                    const uint64_t b0 = major | (((q_smem + slot * G::kTileBytes) & 0x3FFFFu) >> 4);
#pragma unroll
                    for (int ks = 0; ks < DP / 16; ++ks) {
                        const uint32_t at = ((ks >> 2) * (kKeys * 128) + (ks & 3) * 32) >> 4;
                        if (ks == 0) MmaSS<false>(tmem + buffer * kColumns, a0 + at, b0 + at, idesc);
                        else MmaSS<true>(tmem + buffer * kColumns, a0 + at, b0 + at, idesc);
                    }
                    MmaCommit(bar(kQEmpty + slot));
                    MmaCommit(bar(kSFull + buffer));
                }
                if (ok) MmaCommit(bar(kKEmpty + k_slot));
            }
        }
    } else {
        // ---- sums ----
        const int mine = warp / kGroupWarps, half = warp / 4 % 2, row = 32 * (warp & 3) + lane;
        const uint32_t scores = tmem + (static_cast<uint32_t>(32 * (warp & 3)) << 16) + half * 64;
        float* sums = reinterpret_cast<float*>(smem + G::kSums);
        const float2 scale = make_float2(p.scale_log2, p.scale_log2);
        uint32_t count = 0, items = 0;  // tiles before this item
        Look next = look(0);
        for (int r = 0; r < rounds && ok; ++r) {
            const Item w = item_of(next);
            next = look(r + 1);
            if (w.tiles == 0) continue;
            const int key = w.key0 + row;
            float* weight = nullptr;  // the threads of the first four warps add up and store
            float before = 0.0f;
            if (warp < 4 && key < w.keys) {
                const int32_t id = p.page_table[static_cast<int64_t>(w.seq) * p.max_blocks + (key >> p.block_shift)];
                if (id >= 0 && id < p.num_blocks) {
                    weight = p.weights + (static_cast<int64_t>(w.seq) * p.kv_heads + w.head_kv) * p.weights_row + key;
                    before = *weight;
                }
            }
            const int sees_from = p.causal ? key - w.diagonal : 0;  // first token that sees the key
            float sum = 0.0f;
            for (int tile = static_cast<int>((count ^ mine) & 1u); tile < w.tiles && ok; tile += kGroups) {
                const uint32_t n = count + tile, slot = n % G::kSlots, buffer = n % kBuffers;
                ok = __all_sync(0xffffffffu, MbarWait(bar(kSFull + buffer), (n / kBuffers) & 1u, abort_flag) && MbarWait(bar(kQFull + slot), (n / G::kSlots) & 1u, abort_flag));
                if (!ok) break;
                TcFenceAfter();
                // columns [first, end) of this half count and see the key
                const int token0 = token_of(w, tile);
                const int first = (max(sees_from - token0, 0) << p.pack_shift) - half * 64, end = (min(w.new_tokens - token0, tile_tokens) << p.pack_shift) - half * 64;
                const float4* lse = reinterpret_cast<const float4*>(lse_ring + slot * kColumns + half * 64);
                uint32_t sc[2][32];
                TmemLd32(scores + buffer * kColumns, sc[0]);
                TmemLd32(scores + buffer * kColumns + 32, sc[1]);
                TmemWaitLd();
                TcFenceBefore();
                __syncwarp();
                if (lane == 0) MbarArrive(bar(kSEmpty + buffer));
                if (first > 0 || end < 64) {
#pragma unroll
                    for (int b = 0; b < 2; ++b) {
                        const int c0 = b * 32;
                        const uint32_t below_end = end - c0 >= 32 ? 0xffffffffu : end <= c0 ? 0u : (1u << (end - c0)) - 1u;
                        const uint32_t below_first = first - c0 >= 32 ? 0xffffffffu : first <= c0 ? 0u : (1u << (first - c0)) - 1u;
                        const uint32_t visible = below_end & ~below_first;
#pragma unroll
                        for (int i = 0; i < 32; ++i) {
                            if (!(visible & (1u << i))) sc[b][i] = 0xff800000u;  // -inf
                        }
                    }
                }
                float2 acc[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[e] = make_float2(0.0f, 0.0f);
#pragma unroll
                for (int b = 0; b < 2; ++b) {
#pragma unroll
                    for (int i = 0; i < 32; i += 4) {
                        const float4 l = lse[b * 8 + i / 4];
                        const float2 x = Fma2(make_float2(__uint_as_float(sc[b][i]), __uint_as_float(sc[b][i + 1])), scale, make_float2(l.x, l.y));
                        const float2 y = Fma2(make_float2(__uint_as_float(sc[b][i + 2]), __uint_as_float(sc[b][i + 3])), scale, make_float2(l.z, l.w));
                        acc[(i / 4) % 2 * 2] = Add2(acc[(i / 4) % 2 * 2], make_float2(Exp2(x.x), Exp2(x.y)));
                        acc[(i / 4) % 2 * 2 + 1] = Add2(acc[(i / 4) % 2 * 2 + 1], make_float2(Exp2(y.x), Exp2(y.y)));
                    }
                }
                __syncwarp();
                if (lane == 0) MbarArrive(bar(kQEmpty + slot));
                sum += ((acc[0].x + acc[0].y) + (acc[1].x + acc[1].y)) + ((acc[2].x + acc[2].y) + (acc[3].x + acc[3].y));
            }
            count += w.tiles;
            // Items take turns with two sets of sums: the next barrier is behind the reads of this set.
            float* set = sums + (items++ & 1u) * (2 * kGroups * kKeys) + row;
            set[(2 * mine + half) * kKeys] = sum;
            ok = AllSumWarps(ok);  // one that gave up takes all along: none may wait here for one that has left
            if (weight != nullptr && ok) *weight = before + ((set[0] + set[kKeys]) + (set[2 * kKeys] + set[3 * kKeys]));
        }
    }
    if (!ok && p.error_word != nullptr) *p.error_word = 1 + warp;
    __syncwarp();
    TcFenceBefore();
    __syncthreads();
    if (warp == kMmaWarp) {
        __syncwarp();
        TcFenceAfter();
        TmemDealloc(tmem, kBuffers * kColumns);
    }
}

template <typename T, int DP>
int Launch(const ScaFlashPagedParams& x, ChunkParams p, const std::vector<int4>& seqs, cudaStream_t stream) {
    using G = WeightsGeom<DP>;
    CUtensorMap map_q, map_k;
    const int64_t rows = x.num_blocks * x.block_size, row = x.num_kv_heads * x.head_dim;
    if (int rc = MakeRowsMap(&map_q, x.q, x.dtype_id, x.head_dim, x.num_heads, x.total_q, x.head_dim, x.num_heads * x.head_dim, 1 << p.pack_shift,
                             kColumns >> p.pack_shift, "q")) return rc;
    if (int rc = MakeRowsMap(&map_k, x.k_pool, x.dtype_id, x.head_dim, rows, x.num_kv_heads, row, x.head_dim, static_cast<int>(x.block_size), 1, "k pool")) return rc;
    auto kernel = chunk_weights_kernel<T, DP>;
    if (int rc = EnsureDynamicSmem(reinterpret_cast<const void*>(kernel), G::kSmemBytes, "chunk_weights_kernel")) return rc;
    const size_t launches = (seqs.size() + kImageSeqs - 1) / kImageSeqs, share = (seqs.size() + launches - 1) / launches;
    for (size_t first = 0; first < seqs.size(); first += share) {
        SeqImage image;
        p.seqs = static_cast<int>(std::min(share, seqs.size() - first));
        image.seqs[p.seqs] = make_int4(0, 0, 0, 0);
        image.ends[p.seqs] = 0;
        for (int i = p.seqs - 1; i >= 0; --i) {  // from the tile on at which i + 1 ends, i + 1 sequences go on to where i does
            image.seqs[i] = seqs[first + i];
            image.ends[i] = image.ends[i + 1] + (TilesOf(image.seqs[i]) - TilesOf(image.seqs[i + 1])) * (i + 1) * p.kv_heads;
        }
        p.items = image.ends[0];
        LaunchDependent(kernel, std::min(p.items, SmCount()), kWeightThreads, G::kSmemBytes, stream, 1, map_q, map_k, p, image);
        if (int rc = CheckFlashLaunch(stream)) return rc;
    }
    return SCA_OK;
}

template <typename T>
int LaunchTyped(const ScaFlashPagedParams& x, const ChunkParams& p, const std::vector<int4>& seqs, cudaStream_t stream) {
    if (x.head_dim <= 64) return Launch<T, 64>(x, p, seqs, stream);
    if (x.head_dim <= 128) return Launch<T, 128>(x, p, seqs, stream);
    return Launch<T, 256>(x, p, seqs, stream);
}

}  // namespace

// Tiles of keys of a call, as many as 32-bit arithmetic on them holds. 2^30 of them have 512 GB of weights.
int CheckChunkTiles(const ScaFlashPagedParams& x) {
    if (x.seq_lens_kv == nullptr) return SCA_OK;  // the prefill refuses it
    int64_t tiles = 0;
    for (int64_t i = 0; i < x.num_seqs; ++i) tiles += (std::max<int64_t>(x.seq_lens_kv[i], 0) + kKeys - 1) / kKeys * std::max<int64_t>(x.num_kv_heads, 0);
    if (tiles <= int64_t{1} << 30) return SCA_OK;
    return Fail(SCA_INVALID_ARGUMENT, "flash paged (weights): " + std::to_string(tiles) + " tiles of keys are out of range");
}

// Behind the prefill of the same validated call, which has left `lse`.
int LaunchChunkWeights(const ScaFlashPagedParams& x, const ScaChunkWeights& w, cudaStream_t stream) {
    ChunkParams p{};
    p.lse = w.lse;
    p.weights = w.weights;
    p.weights_row = w.weights_row;
    p.total_q = x.total_q;
    p.page_table = x.page_table;
    p.error_word = ErrorWord();
    p.max_blocks = static_cast<int>(x.max_blocks_per_seq);
    p.num_blocks = static_cast<int>(x.num_blocks);
    p.block_size = static_cast<int>(x.block_size);
    while ((1 << p.block_shift) < p.block_size) ++p.block_shift;
    p.heads = static_cast<int>(x.num_heads);
    p.kv_heads = static_cast<int>(x.num_kv_heads);
    const int64_t group = x.num_heads / x.num_kv_heads;
    while (p.pack_shift < 4 && group % (2ll << p.pack_shift) == 0) ++p.pack_shift;
    p.last = static_cast<int>(w.last < x.total_q ? w.last : 0);
    p.causal = x.causal ? 1 : 0;
    p.scale_log2 = x.scale * kLog2e;
    std::vector<int4> seqs(static_cast<size_t>(x.num_seqs));
    for (int i = 0; i < x.num_seqs; ++i) seqs[static_cast<size_t>(i)] = make_int4(x.cu_seqlens_q[i], i, x.cu_seqlens_q[i + 1] - x.cu_seqlens_q[i], x.seq_lens_kv[i]);
    std::stable_sort(seqs.begin(), seqs.end(), [](const int4& a, const int4& b) { return TilesOf(a) > TilesOf(b); });
    return x.dtype_id == SCA_DTYPE_F16 ? LaunchTyped<__half>(x, p, seqs, stream) : LaunchTyped<__nv_bfloat16>(x, p, seqs, stream);
}

}  // namespace flash
}  // namespace sca_b200

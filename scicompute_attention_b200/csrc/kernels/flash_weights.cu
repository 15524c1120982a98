// What the tokens of a paged cache weigh in the attention of a chunk: weights[s, g, j] += the sum over the chunk's counted tokens i and the
// query heads h of kv head g of exp(scale q[i, h] . k[j] - lse[i, h]). It follows the prefill kernel, which leaves lse, the logarithm of each
// row's sum.
//
// A CTA has one tile of 128 keys of one (sequence, kv head) and walks the query tiles that see it; nobody else adds to its weights, so there are
// no atomics and the same call gives the same bits. The scores are computed with the keys as rows, S = K Q^T (tcgen05, M = 128 keys, N = 128
// queries, into one of two buffers of tensor memory): a thread then has one key, and its sum over the queries needs no other thread. lse of
// the 128 queries lies in shared memory, where all threads read the same number at the same time.
//   warps 0 - 3  a key each thread: 2^(score * scale - lse), summed up
//   warp 4       TMA: the tile of keys once, page by page, then query tiles into a ring, and their lse
//   warp 5       issues the products
// A query tile is 128 / P tokens of P query heads, as in the prefill, and starts with the first token that sees the tile's first key, so
// that a causal mask cuts 128 / P tokens' rows at most.
// Bound by the special-function unit: 16384 exponentials a tile take 1024 clocks of an SM, the products 540.
#include "flash_kernel.cuh"

namespace sca_b200 {
namespace flash {
namespace {

constexpr int kKeys = 128;     // keys of a CTA
constexpr int kColumns = 128;  // (token, head) rows of a query tile
constexpr int kSumWarps = 4;
constexpr int kWeightThreads = 32 * (kSumWarps + 2);
constexpr int kBuffers = 2;    // of scores in tensor memory

template <int DP>
struct WeightsGeom {
    static constexpr int kBlocks = DP / 64;              // 128-byte column blocks
    static constexpr int kTileBytes = kBlocks * kKeys * 128;
    static constexpr int kSlots = DP == 64 ? 4 : 2;      // query tiles in flight; two CTAs to an SM up to D=128
    static constexpr int kLse = (1 + kSlots) * kTileBytes;
    static constexpr int kBars = kLse + kSlots * kColumns * 4;
    static constexpr int kSmemBytes = 1024 + kBars + 256;
    static constexpr int kCtas = DP == 256 ? 1 : 2;
};

struct ChunkParams {
    const int4* seqs;  // {first query token, -, S_q, S_kv}
    const float* lse;  // [heads][total_q], natural logarithm; -inf: the row sees nothing
    float* weights;
    int64_t weights_row, total_q;
    const int32_t* page_table;
    int* error_word;
    int max_blocks, num_blocks, block_size, block_shift;
    int heads, kv_heads, pack_shift, last, causal;
    float scale_log2;
};

template <typename T, int DP>
__global__ void __launch_bounds__(kWeightThreads, WeightsGeom<DP>::kCtas)
chunk_weights_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const ChunkParams p) {
    using G = WeightsGeom<DP>;
    extern __shared__ unsigned char smem_raw[];
    const uint32_t base = (SmemAddr(smem_raw) + 1023u) & ~1023u;
    unsigned char* smem = smem_raw + (base - SmemAddr(smem_raw));
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    BeginAfterPredecessor();
    const int seq = static_cast<int>(blockIdx.x) / p.kv_heads, head_kv = static_cast<int>(blockIdx.x) % p.kv_heads;
    const int4 s = p.seqs[seq];
    const int new_tokens = s.z, keys = s.w, key0 = static_cast<int>(blockIdx.y) * kKeys;
    if (key0 >= keys) return;
    // token t of the chunk sees keys up to t + diagonal; counted are tokens from `counted` on
    const int diagonal = p.causal ? keys - new_tokens : keys;
    const int counted = p.last > 0 ? max(0, new_tokens - p.last) : 0;
    const int first_token = max(counted, key0 - diagonal);
    const int heads_tile = 1 << p.pack_shift, tile_tokens = kColumns >> p.pack_shift;
    const int group = p.heads / p.kv_heads, packs = group >> p.pack_shift;
    const int tiles = (new_tokens - first_token + tile_tokens - 1) / tile_tokens * packs;  // one at least: the last token sees every key

    const uint32_t k_smem = base, q_smem = base + G::kTileBytes;
    float* lse_ring = reinterpret_cast<float*>(smem + G::kLse);
    auto bar = [&](int i) { return base + G::kBars + 8u * i; };
    constexpr int kKFull = 0, kQFull = 1, kQEmpty = kQFull + G::kSlots, kSFull = kQEmpty + G::kSlots, kSEmpty = kSFull + kBuffers,
                  kNumBars = kSEmpty + kBuffers;
    static_assert(kNumBars * 8 + 8 <= 256, "barrier area too small");
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + G::kBars + kNumBars * 8);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    if (threadIdx.x == 0) {
        MbarInit<1>(bar(kKFull));
        for (int i = 0; i < G::kSlots; ++i) {
            MbarInit<1 + 32>(bar(kQFull + i));         // the tile, and each lane's part of lse
            MbarInit<1 + kSumWarps>(bar(kQEmpty + i)); // the products and the sums are done with it
        }
        for (int i = 0; i < kBuffers; ++i) {
            MbarInit<1>(bar(kSFull + i));
            MbarInit<kSumWarps>(bar(kSEmpty + i));
        }
        *abort_flag = 0;
        FenceBarrierInit();
    }
    if (warp == 5) {
        TmemAlloc(SmemAddr(tmem_slot), kBuffers * kColumns);
        TmemRelinquish();
    }
    TcFenceBefore();
    __syncthreads();
    TcFenceAfter();
    const uint32_t tmem = *tmem_slot;
    const int32_t* table = p.page_table + static_cast<int64_t>(seq) * p.max_blocks;
    auto token_of = [&](int tile) { return first_token + tile / packs * tile_tokens; };
    bool ok = true;

    if (warp == 4) {
        // ---- loads ----
        const int pages = kKeys >> p.block_shift, page = (key0 >> p.block_shift) + lane;
        const bool in = lane < pages && page < p.max_blocks && (static_cast<int64_t>(page) << p.block_shift) < keys;
        const int32_t id = in ? table[page] : -1;
        const int first_row = id >= 0 && id < p.num_blocks ? id << p.block_shift : p.num_blocks << p.block_shift;  // behind the pool: zeros
        if (lane == 0) {
            PrefetchTensorMap(&map_q);
            PrefetchTensorMap(&map_k);
            MbarExpectTx(bar(kKFull), G::kTileBytes);
        }
        __syncwarp();
        for (int i = 0; i < pages; ++i) {
            const int row = __shfl_sync(0xffffffffu, first_row, i);
            if (ElectOne()) {
#pragma unroll
                for (int kb = 0; kb < G::kBlocks; ++kb) {
                    TmaLoad4D(k_smem + kb * (kKeys * 128) + i * p.block_size * 128, &map_k, bar(kKFull), kb * 64, row, head_kv, 0);
                }
            }
        }
        auto lse_of = [&](int tile, float (&v)[4]) {
            const int token0 = token_of(tile), head0 = head_kv * group + (tile % packs << p.pack_shift);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int c = lane + 32 * i, token = token0 + (c >> p.pack_shift), head = head0 + (c & (heads_tile - 1));
                v[i] = tile < tiles && token < new_tokens ? p.lse[static_cast<int64_t>(head) * p.total_q + s.x + token] : -CUDART_INF_F;
            }
        };
        float next[4];
        lse_of(0, next);
        for (int tile = 0; tile < tiles && ok; ++tile) {
            const int slot = tile % G::kSlots;
            float v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = next[i];
            lse_of(tile + 1, next);
            ok = __all_sync(0xffffffffu, MbarWait(bar(kQEmpty + slot), ((tile / G::kSlots) & 1u) ^ 1u, abort_flag));
            if (!ok) break;
            if (ElectOne()) {
                MbarExpectTx(bar(kQFull + slot), G::kTileBytes);
#pragma unroll
                for (int kb = 0; kb < G::kBlocks; ++kb) {
                    TmaLoad4D(q_smem + slot * G::kTileBytes + kb * (kColumns * 128), &map_q, bar(kQFull + slot), kb * 64,
                              head_kv * group + (tile % packs << p.pack_shift), s.x + token_of(tile), 0);
                }
            }
            __syncwarp();
            // a row that sees nothing has no sum: 2^-inf
#pragma unroll
            for (int i = 0; i < 4; ++i) lse_ring[slot * kColumns + lane + 32 * i] = v[i] == -CUDART_INF_F ? v[i] : -v[i] * kLog2e;
            MbarArrive(bar(kQFull + slot));
        }
    } else if (warp == 5) {
        // ---- products ----
        if (ElectOne()) {
            constexpr uint32_t fmt = std::is_same<T, __half>::value ? kFmtF16 : kFmtBf16;
            constexpr uint32_t idesc = MakeInstrDesc(fmt, fmt, 0, 0, kKeys, kColumns);
            const uint64_t major = MakeSmemDesc(0, 16, 1024);  // both K-major
            const uint64_t a0 = major | ((k_smem & 0x3FFFFu) >> 4);
            ok = MbarWait(bar(kKFull), 0, abort_flag);
            for (int tile = 0; tile < tiles && ok; ++tile) {
                const int slot = tile % G::kSlots, buffer = tile % kBuffers;
                ok = MbarWait(bar(kQFull + slot), (tile / G::kSlots) & 1u, abort_flag) &&
                     MbarWait(bar(kSEmpty + buffer), ((tile / kBuffers) & 1u) ^ 1u, abort_flag);
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
        }
    } else {
        // ---- sums ----
        const int key = key0 + 32 * warp + lane;
        const uint32_t lanes = static_cast<uint32_t>(32 * warp) << 16;
        // a column that the key is visible to and that counts: [first, end) below; the same in every tile but the first and last tokens'
        const int sees_from = p.causal ? key - diagonal : 0;  // first token that sees the key
        float sum = 0.0f;
        for (int tile = 0; tile < tiles && ok; ++tile) {
            const int slot = tile % G::kSlots, buffer = tile % kBuffers;
            ok = __all_sync(0xffffffffu, MbarWait(bar(kSFull + buffer), (tile / kBuffers) & 1u, abort_flag) &&
                                             MbarWait(bar(kQFull + slot), (tile / G::kSlots) & 1u, abort_flag));
            if (!ok) break;
            TcFenceAfter();
            const int token0 = token_of(tile);
            const int first = max(sees_from - token0, 0) << p.pack_shift, end = min(new_tokens - token0, tile_tokens) << p.pack_shift;
            const bool ragged = first > 0 || end < kColumns;
            const float4* lse = reinterpret_cast<const float4*>(lse_ring + slot * kColumns);
            const float2 scale = make_float2(p.scale_log2, p.scale_log2);
            float2 acc[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[e] = make_float2(0.0f, 0.0f);
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                uint32_t sc[2][32];
                TmemLd32(tmem + lanes + buffer * kColumns + half * 64, sc[0]);
                TmemLd32(tmem + lanes + buffer * kColumns + half * 64 + 32, sc[1]);
                TmemWaitLd();
                if (half == 1) {
                    TcFenceBefore();
                    __syncwarp();
                    if (lane == 0) MbarArrive(bar(kSEmpty + buffer));
                }
                if (ragged) {
#pragma unroll
                    for (int b = 0; b < 2; ++b) {
                        const int c0 = half * 64 + b * 32;
                        const uint32_t below_end = end - c0 >= 32 ? 0xffffffffu : end <= c0 ? 0u : (1u << (end - c0)) - 1u;
                        const uint32_t below_first = first - c0 >= 32 ? 0xffffffffu : first <= c0 ? 0u : (1u << (first - c0)) - 1u;
                        const uint32_t visible = below_end & ~below_first;
#pragma unroll
                        for (int i = 0; i < 32; ++i) {
                            if (!(visible & (1u << i))) sc[b][i] = 0xff800000u;  // -inf
                        }
                    }
                }
#pragma unroll
                for (int b = 0; b < 2; ++b) {
#pragma unroll
                    for (int i = 0; i < 32; i += 4) {
                        const float4 l = lse[half * 16 + b * 8 + i / 4];
                        const float2 x = Fma2(make_float2(__uint_as_float(sc[b][i]), __uint_as_float(sc[b][i + 1])), scale, make_float2(l.x, l.y));
                        const float2 y = Fma2(make_float2(__uint_as_float(sc[b][i + 2]), __uint_as_float(sc[b][i + 3])), scale, make_float2(l.z, l.w));
                        acc[(i / 4) % 2 * 2] = Add2(acc[(i / 4) % 2 * 2], make_float2(Exp2(x.x), Exp2(x.y)));
                        acc[(i / 4) % 2 * 2 + 1] = Add2(acc[(i / 4) % 2 * 2 + 1], make_float2(Exp2(y.x), Exp2(y.y)));
                    }
                }
            }
            __syncwarp();
            if (lane == 0) MbarArrive(bar(kQEmpty + slot));
            sum += ((acc[0].x + acc[0].y) + (acc[1].x + acc[1].y)) + ((acc[2].x + acc[2].y) + (acc[3].x + acc[3].y));
        }
        if (ok && key < keys) {
            const int32_t id = table[key >> p.block_shift];
            if (id >= 0 && id < p.num_blocks) p.weights[(static_cast<int64_t>(seq) * p.kv_heads + head_kv) * p.weights_row + key] += sum;
        }
    }
    if (!ok && p.error_word != nullptr) *p.error_word = 1 + warp;
    __syncwarp();
    TcFenceBefore();
    __syncthreads();
    if (warp == 5) {
        __syncwarp();
        TcFenceAfter();
        TmemDealloc(tmem, kBuffers * kColumns);
    }
}

template <typename T, int DP>
int Launch(const ScaFlashPagedParams& x, const ChunkParams& p, int64_t most_keys, cudaStream_t stream) {
    using G = WeightsGeom<DP>;
    CUtensorMap map_q, map_k;
    const int64_t rows = x.num_blocks * x.block_size, row = x.num_kv_heads * x.head_dim;
    if (int rc = MakeRowsMap(&map_q, x.q, x.dtype_id, x.head_dim, x.num_heads, x.total_q, x.head_dim, x.num_heads * x.head_dim, 1 << p.pack_shift,
                             kColumns >> p.pack_shift, "q")) return rc;
    if (int rc = MakeRowsMap(&map_k, x.k_pool, x.dtype_id, x.head_dim, rows, x.num_kv_heads, row, x.head_dim, static_cast<int>(x.block_size), 1, "k pool")) return rc;
    auto kernel = chunk_weights_kernel<T, DP>;
    if (int rc = EnsureDynamicSmem(reinterpret_cast<const void*>(kernel), G::kSmemBytes, "chunk_weights_kernel")) return rc;
    // the tiles of the first keys, which most tokens see, go first
    const dim3 grid(static_cast<unsigned>(x.num_seqs * x.num_kv_heads), static_cast<unsigned>((most_keys + kKeys - 1) / kKeys));
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(kWeightThreads);
    cfg.dynamicSmemBytes = G::kSmemBytes;
    cfg.stream = stream;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    cudaLaunchKernelEx(&cfg, kernel, map_q, map_k, p);
    return CheckFlashLaunch(stream);
}

template <typename T>
int LaunchTyped(const ScaFlashPagedParams& x, const ChunkParams& p, int64_t most_keys, cudaStream_t stream) {
    if (x.head_dim <= 64) return Launch<T, 64>(x, p, most_keys, stream);
    if (x.head_dim <= 128) return Launch<T, 128>(x, p, most_keys, stream);
    return Launch<T, 256>(x, p, most_keys, stream);
}

}  // namespace

// Behind the prefill of the same validated call, which has left `seqs` and `lse`.
int LaunchChunkWeights(const ScaFlashPagedParams& x, const ScaChunkWeights& w, const int4* seqs, cudaStream_t stream) {
    ChunkParams p{};
    p.seqs = seqs;
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
    int64_t most_keys = 0;
    for (int64_t i = 0; i < x.num_seqs; ++i) most_keys = most_keys < x.seq_lens_kv[i] ? x.seq_lens_kv[i] : most_keys;
    return x.dtype_id == SCA_DTYPE_F16 ? LaunchTyped<__half>(x, p, most_keys, stream) : LaunchTyped<__nv_bfloat16>(x, p, most_keys, stream);
}

}  // namespace flash
}  // namespace sca_b200

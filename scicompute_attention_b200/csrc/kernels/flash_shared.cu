// Decode of groups of sequences over the pages they have in common: the prefill kernel (kShared in flash_kernel.cuh) with the query tokens of
// a group as the rows of its tiles. The pages are read once per group instead of once per sequence, and the products run on the tensor cores.
//
// An item is 256 rows (one token of up to 16 query heads of a kv head, as many sequences as fill it up) against `part_tiles` tiles of 128
// keys of the prefix. It leaves {m, l, O} of each of its rows in fp32; the finish kernel of decode_weights.cu merges them with the parts of
// the sequence's own tokens.
// Bound by the chain of a tile's scores, softmax and products where a prefix is long and many share it, 128 sequences behind 8100 tokens (32 / 8 heads,
// D=128): 32 us, 550 TFLOP/s, of which 4 are the O of 9 parts in fp32. 14 groups of 4 to 12 behind 300 to 4000 tokens, 123 MB: 39 us; a quarter of
// the rows are filled, and a step of one tile takes 1.8 us whatever it holds.
#include <algorithm>

#include "flash_kernel.cuh"

namespace sca_b200 {
namespace flash {
namespace {

constexpr int kTileKeys = 128;

// log2 of the query heads that share a tile: the largest power of two that divides the group of a kv head, up to 16. The rows of a tile are a
// group's sequences times these heads, and a kv head's keys are read once for all of them.
int PackShift(int64_t group) {
    int shift = 0;
    while (shift < 4 && group % (2ll << shift) == 0) ++shift;
    return shift;
}
int QueryTiles(int64_t head_dim) { return head_dim > 128 ? 1 : 2; }

template <typename T, int DP, int QT>
int Launch(const ScaDecodeFwdParams& d, const PrefixGroups& groups, const PrefixParts& parts, cudaStream_t stream) {
    using G = FlashGeom<DP, QT, kTileKeys>;
    const int pack_shift = PackShift(d.num_heads / d.num_kv_heads);
    CUtensorMap map_q, map_k, map_v;
    if (int rc = MakeRowsMap(&map_q, d.q, d.dtype, d.head_dim, d.num_heads, d.batch, d.q_stride.s_h, d.q_stride.s_b, 1 << pack_shift, kBlockM >> pack_shift, "q")) return rc;
    const int64_t rows = d.num_kv_blocks * d.block_size, row = d.num_kv_heads * d.head_dim;
    auto pool_map = [&](CUtensorMap* map, const void* pool, const char* what) {  // one box = one page of one kv head and column block
        return MakeRowsMap(map, pool, d.dtype, d.head_dim, rows, d.num_kv_heads, row, d.head_dim, static_cast<int>(d.block_size), 1, what);
    };
    if (int rc = pool_map(&map_k, d.k, "k pool")) return rc;
    if (int rc = pool_map(&map_v, d.v, "v pool")) return rc;
    FlashKernelParams p{};
    p.error_word = ErrorWord();
    p.heads = static_cast<int>(d.num_heads);
    p.kv_heads = static_cast<int>(d.num_kv_heads);
    p.head_dim = static_cast<int>(d.head_dim);
    p.batch = 1;
    p.scale_log2 = d.scale * kLog2e;
    p.pack_shift = pack_shift;
    p.tiles_per_item = QT;
    p.page_table = d.page_table;
    p.max_blocks_per_seq = static_cast<int>(d.max_blocks_per_seq);
    p.num_kv_blocks = static_cast<int>(d.num_kv_blocks);
    p.block_size = static_cast<int>(d.block_size);
    while ((1 << p.block_shift) < p.block_size) ++p.block_shift;
    const int item_tokens = (QT * kBlockM) >> pack_shift;
    for (int g = 0; g < groups.count; ++g) {
        const PrefixGroup& x = groups.group[g];
        const int tiles = (x.tokens + kTileKeys - 1) / kTileKeys;
        p.num_entries = x.first_entry + (x.end - x.first + item_tokens - 1) / item_tokens * ((tiles + groups.part_tiles - 1) / groups.part_tiles);
    }
    const int64_t items = static_cast<int64_t>(p.num_entries) * (p.heads >> pack_shift);
    if (items > 0x7fffffffLL) return Fail(SCA_INVALID_ARGUMENT, "shared prefix: grid of " + std::to_string(items) + " blocks is out of range");
    SharedImage image{groups, parts, d.seq_lens};
    auto kernel = flash_fwd_sm100_kernel<T, DP, QT, kTileKeys, true, true, false, true>;
    if (int rc = EnsureDynamicSmem(reinterpret_cast<const void*>(kernel), G::kSmemBytes, "flash_fwd_sm100_kernel")) return rc;
    LaunchDependent(kernel, std::min<int64_t>(items, SmCount()), FlashThreads<T, DP, QT>(), G::kSmemBytes, stream, 1, map_q, map_k, map_v, p, image);
    return CheckFlashLaunch(stream);
}

template <typename T>
int LaunchTyped(const ScaDecodeFwdParams& p, const PrefixGroups& groups, const PrefixParts& parts, cudaStream_t stream) {
    if (p.head_dim <= 64) return Launch<T, 64, 2>(p, groups, parts, stream);
    if (p.head_dim <= 128) return Launch<T, 128, 2>(p, groups, parts, stream);
    return Launch<T, 256, 1>(p, groups, parts, stream);
}

}  // namespace
}  // namespace flash

int LaunchPrefixParts(const ScaDecodeFwdParams& p, const PrefixGroups& groups, const PrefixParts& parts, cudaStream_t stream) {
    return p.dtype == SCA_DTYPE_F16 ? flash::LaunchTyped<__half>(p, groups, parts, stream) : flash::LaunchTyped<__nv_bfloat16>(p, groups, parts, stream);
}

// Parts that fill the SMs: with more of them an SM has fewer tiles to walk, but each costs its start, 4 bytes a number and row for its O, and
// its share of the merge. The cost of an item is its tiles and three more, that of a part in the merge half a tile. us of a call by the tiles of a
// part (32 / 8 heads, D=128; taken: 5, 8, 21):
//   32 sequences, prefix of 4000    2: 26.5  3: 27.3  4: 23.7  5: 24.0  6: 25.2  8: 28.4  16: 42
//   128, 8100, 20 to 1500 of their own   4: 121  6: 119  7: 110.5  8: 109.2  9: 109.1  12: 111  16: 117  32: 145
//   300, 8000                       4: 143  6: 126  8: 126.5  9: 116.2  10: 120  16: 129  21: 116.8  32: 138
void PlanPrefixParts(const ScaDecodeFwdParams& p, PrefixGroups* groups) {
    const int pack_shift = flash::PackShift(p.num_heads / p.num_kv_heads);
    const int64_t packed_heads = p.num_heads >> pack_shift;
    const int item_tokens = (flash::QueryTiles(p.head_dim) * flash::kBlockM) >> pack_shift;
    const int sms = SmCount();
    int longest = 1;
    for (int g = 0; g < groups->count; ++g) longest = std::max(longest, (groups->group[g].tokens + flash::kTileKeys - 1) / flash::kTileKeys);
    auto items_of = [&](const PrefixGroup& x, int part_tiles) -> int64_t {
        const int tiles = (x.tokens + flash::kTileKeys - 1) / flash::kTileKeys;
        return static_cast<int64_t>((x.end - x.first + item_tokens - 1) / item_tokens) * ((tiles + part_tiles - 1) / part_tiles);
    };
    double best = 0.0;
    int last = 0;
    for (int parts = 1; parts <= 32 && parts <= longest; ++parts) {
        const int part_tiles = (longest + parts - 1) / parts;
        if (part_tiles == last) continue;
        last = part_tiles;
        int64_t items = 0;
        for (int g = 0; g < groups->count; ++g) items += items_of(groups->group[g], part_tiles);
        const double rounds = static_cast<double>((items * packed_heads + sms - 1) / sms), cost = rounds * (part_tiles + 3) + 0.5 * parts;
        if (groups->part_tiles == 0 || cost < best) {
            best = cost;
            groups->part_tiles = part_tiles;
        }
    }
    groups->parts = (longest + groups->part_tiles - 1) / groups->part_tiles;
    int64_t entries = 0;
    for (int g = 0; g < groups->count; ++g) {
        groups->group[g].first_entry = static_cast<int>(entries);
        entries += items_of(groups->group[g], groups->part_tiles);
    }
}

}  // namespace sca_b200

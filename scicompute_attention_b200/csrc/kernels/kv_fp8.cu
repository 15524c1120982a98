// The 8-bit KV cache (kv_fp8.cuh): rows are quantised as they are written, blocks are read back as 16- or 32-bit numbers.
//
// Both kernels move every byte once: a row of D numbers of w bytes is read, D + 1 bytes are written, or the other way round. Both are bound
// by HBM: 50 thousand tokens of 8 heads, D=128, appended at 6.5 TB/s from bf16 and 6.85 from fp32 (47 us, 91), 1500 blocks of 16 tokens read
// back at 6.5 TB/s as bf16 and 5.9 as fp32; a call of a few rows is its launch, 1.7 us.
#include <algorithm>
#include <string>

#include "common.cuh"
#include "kv_fp8.cuh"

namespace sca_b200 {
namespace {

constexpr int kFp8Threads = 256;

constexpr int kPiece = 16;  // numbers a lane takes

// kPiece consecutive numbers of a row as they come, by 32-byte loads where `aligned` says that rows start on a 32-byte boundary.
template <typename T>
struct Piece {
    static constexpr int kWords = kPiece * sizeof(T) / 4;
    uint32_t w[kWords];
    __device__ __forceinline__ void Load(const T* src, bool aligned) {
        if (aligned) {
#pragma unroll
            for (int i = 0; i < kWords; i += 8) {
                asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                             : "=r"(w[i]), "=r"(w[i + 1]), "=r"(w[i + 2]), "=r"(w[i + 3]), "=r"(w[i + 4]), "=r"(w[i + 5]), "=r"(w[i + 6]), "=r"(w[i + 7])
                             : "l"(reinterpret_cast<const uint32_t*>(src) + i)
                             : "memory");
            }
        } else {
#pragma unroll
            for (int i = 0; i < kPiece; ++i) reinterpret_cast<T*>(w)[i] = src[i];
        }
    }
    __device__ __forceinline__ float operator[](int i) const { return ToFloat(reinterpret_cast<const T*>(w)[i]); }
    // The largest number; NaN is passed over.
    __device__ __forceinline__ float Largest() const {
        float m = 0.0f;  // fmaxf passes over NaN
#pragma unroll
        for (int i = 0; i < kPiece; ++i) m = fmaxf(m, fabsf((*this)[i]));
        return m;
    }
    // 16 bits: the same as its bits without the sign, which compare as whole numbers do - with a NaN above all numbers.
    __device__ __forceinline__ uint32_t LargestBits() const {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < kWords; ++i) m = __vmaxu2(m, w[i] & 0x7fff7fffu);
        return max(m >> 16, m & 0xffffu);
    }
};

// Where rows go: `slots` (one per token), or the page table at position seq_lens[token] - 1 (one token per sequence).
struct AppendTarget {
    uint8_t *k_codes, *v_codes, *k_scales, *v_scales;
    const int32_t* slots;
    const int32_t* page_table;
    const int32_t* seq_lens;
    int64_t max_blocks_per_seq;
    int64_t num_blocks;
    int block_size, heads, head_dim;
    bool aligned;  // the new rows start on 32-byte boundaries
};

// Slot of a token, -1 where it is not stored. Pools have less than 2^31 slots.
template <bool kBatched>
__device__ __forceinline__ int SlotOf(const AppendTarget& a, int64_t token) {
    if constexpr (!kBatched) {
        const int slot = a.slots[token];
        return slot < a.num_blocks * a.block_size ? slot : -1;
    } else {
        const int pos = a.seq_lens[token] - 1;
        if (pos < 0) return -1;
        const int logical = pos / a.block_size;
        if (logical >= a.max_blocks_per_seq) return -1;
        const int phys = a.page_table[token * a.max_blocks_per_seq + logical];
        if (phys < 0 || phys >= a.num_blocks) return -1;
        return phys * a.block_size + (pos - logical * a.block_size);
    }
}

// kLanes lanes of a warp (the smallest power of two that covers D / 16) take a row of K and the same row of V: 16 numbers each, the
// largest by shuffles, 16 codes each. I: type of a row's number. Bound by HBM, and by how much of it is under way: each lane has 64 bytes
// of K and V on their way (128 of fp32) before it looks at the first.
template <typename T, int kLanes, bool kBatched, typename I>
__global__ void __launch_bounds__(kFp8Threads)
kv_append_fp8_kernel(const T* k_new, const T* v_new, const I rows, const AppendTarget a) {
    BeginAfterPredecessor();
    constexpr int kRows = kFp8Threads / kLanes;  // of a CTA
    const int piece = threadIdx.x % kLanes;
    const bool in_row = piece * kPiece < a.head_dim;
    for (I base = static_cast<I>(blockIdx.x) * kRows; base < rows; base += static_cast<I>(gridDim.x) * kRows) {
        const I row = base + threadIdx.x / kLanes;
        const bool mine = row < rows && in_row;
        Piece<T> x[2];
        if (mine) {
            x[0].Load(k_new + static_cast<int64_t>(row) * a.head_dim + piece * kPiece, a.aligned);
            x[1].Load(v_new + static_cast<int64_t>(row) * a.head_dim + piece * kPiece, a.aligned);
        } else {
#pragma unroll
            for (int i = 0; i < Piece<T>::kWords; ++i) x[0].w[i] = x[1].w[i] = 0;
        }
        const I token = row / a.heads;
        const int head = static_cast<int>(row - token * a.heads);
        const int slot = row < rows ? SlotOf<kBatched>(a, token) : -1;
        float amax[2];
        bool by_value = sizeof(T) == 4;
        if constexpr (sizeof(T) == 2) {
            uint32_t most = x[0].LargestBits() << 16 | x[1].LargestBits();  // K and V in one
#pragma unroll
            for (int o = 1; o < kLanes; o <<= 1) most = __vmaxu2(most, __shfl_xor_sync(0xffffffffu, most, o));
            amax[0] = fminf(ToFloat(*(reinterpret_cast<const T*>(&most) + 1)), fp8::kLargest);
            amax[1] = fminf(ToFloat(*reinterpret_cast<const T*>(&most)), fp8::kLargest);
            constexpr uint32_t kInf = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
            by_value = __any_sync(0xffffffffu, (most >> 16) > kInf || (most & 0xffffu) > kInf);
        }
        if (by_value) {
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                float m = x[s].Largest();
#pragma unroll
                for (int o = 1; o < kLanes; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
                amax[s] = fminf(m, fp8::kLargest);
            }
        }
        if (!mine || slot < 0) continue;
        const int block = slot / a.block_size, offset = slot - block * a.block_size;
        const int64_t code_at = (static_cast<int64_t>(slot) * a.heads + head) * a.head_dim + piece * kPiece;
        const int64_t scale_at = (static_cast<int64_t>(block) * a.heads + head) * fp8::ScaleRow(a.block_size) + offset;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const int e = fp8::ExponentFor(amax[s]);
            const float inv = fp8::PowerOfTwo(-e);
            uint32_t words[4];
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                words[w] = fp8::Encode2(x[s][4 * w] * inv, x[s][4 * w + 1] * inv) | fp8::Encode2(x[s][4 * w + 2] * inv, x[s][4 * w + 3] * inv) << 16;
            }
            *reinterpret_cast<uint4*>((s == 0 ? a.k_codes : a.v_codes) + code_at) = make_uint4(words[0], words[1], words[2], words[3]);
            if (piece == 0) (s == 0 ? a.k_scales : a.v_scales)[scale_at] = static_cast<uint8_t>(e + 15);
        }
    }
}

// 32 bytes, in one store where `wide` says that they start on a 32-byte boundary.
__device__ __forceinline__ void Store32(void* dst, const uint32_t (&v)[8], bool wide) {
    if (wide) {
        asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]),
                     "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                     : "memory");
    } else {
        static_cast<uint4*>(dst)[0] = make_uint4(v[0], v[1], v[2], v[3]);
        static_cast<uint4*>(dst)[1] = make_uint4(v[4], v[5], v[6], v[7]);
    }
}

// 16 codes per thread and turn: a thread's numbers are 32 or 64 bytes, whole sectors of their own.
template <typename T, typename I>
__global__ void __launch_bounds__(kFp8Threads)
kv_gather_fp8_kernel(const uint8_t* codes, const uint8_t* scales, const int32_t* ids, const I total, T* out, const int64_t num_blocks,
                     const int block_size, const int heads, const int head_dim, const bool wide) {
    BeginAfterPredecessor();
    const int pieces = head_dim / 16;
    const I block_pieces = static_cast<I>(block_size) * heads * pieces;
    for (I idx = static_cast<I>(blockIdx.x) * kFp8Threads + threadIdx.x; idx < total; idx += static_cast<I>(gridDim.x) * kFp8Threads) {
        const I i = idx / block_pieces;
        const int within = static_cast<int>(idx - i * block_pieces);
        const int32_t phys = ids[i];
        uint4 c = make_uint4(0, 0, 0, 0);
        uint32_t byte = 15;
        if (phys >= 0 && phys < num_blocks) {
            const int row = within / pieces;
            const int token = row / heads, head = row - token * heads;
            c = reinterpret_cast<const uint4*>(codes)[static_cast<int64_t>(phys) * block_pieces + within];
            byte = scales[(static_cast<int64_t>(phys) * heads + head) * fp8::ScaleRow(block_size) + token];
        }
        const uint32_t words[4] = {c.x, c.y, c.z, c.w};
        uint32_t h[8];
#pragma unroll
        for (int w = 0; w < 4; ++w) h[2 * w] = fp8::DecodeLow(words[w]), h[2 * w + 1] = fp8::DecodeHigh(words[w]);
        T* dst = out + static_cast<int64_t>(idx) * 16;
        if constexpr (sizeof(T) == 4) {
            const float s = fp8::ScaleOf(byte);
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                uint32_t f[8];
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    const float2 x = fp8::UnpackHalf2(h[4 * half + w]);
                    f[2 * w] = __float_as_uint(x.x * s), f[2 * w + 1] = __float_as_uint(x.y * s);
                }
                Store32(dst + 8 * half, f, wide);
            }
        } else {
            const uint32_t pair = fp8::ScalePair(byte, byte);
            const float s = fp8::ScaleOf(byte);
#pragma unroll
            for (int w = 0; w < 8; ++w) {
                if constexpr (std::is_same<T, __half>::value) {
                    h[w] = fp8::MulHalf2(h[w], pair);
                } else {
                    const float2 f = fp8::UnpackHalf2(h[w]);
                    h[w] = Pack2<T>(f.x * s, f.y * s);
                }
            }
            Store32(dst, h, wide);
        }
    }
}

// A grid that covers the work once, at most a few waves of the machine: the loops are grid-stride.
int64_t Fp8Grid(int64_t ctas) { return std::max<int64_t>(1, std::min(ctas, static_cast<int64_t>(SmCount()) * 32)); }

int CheckFp8Shape(const ScaKvCacheShape* shape, const char* what) {
    if (shape == nullptr) return Fail(SCA_INVALID_ARGUMENT, std::string(what) + ": null shape");
    if (shape->num_blocks <= 0 || shape->block_size <= 0 || shape->num_kv_heads <= 0) {
        return Fail(SCA_INVALID_ARGUMENT, std::string(what) + ": non-positive geometry");
    }
    if (shape->head_dim <= 0 || shape->head_dim > 256 || shape->head_dim % 16 != 0) {
        return Fail(SCA_INVALID_ARGUMENT, std::string(what) + ": head_dim=" + std::to_string(shape->head_dim) +
                                              " (rows of an 8-bit cache are multiples of 16 up to 256)");
    }
    if (shape->num_blocks * shape->block_size > 0x7fffffffLL || shape->block_size * shape->num_kv_heads > 0x3fffffLL) {
        return Fail(SCA_INVALID_ARGUMENT, std::string(what) + ": slots beyond 32 bits");
    }
    return SCA_OK;
}

template <typename T, bool kBatched, typename I>
void LaunchAppend(const void* k_new, const void* v_new, I rows, const AppendTarget& a, cudaStream_t stream) {
    auto go = [&](auto lanes) {
        constexpr int kLanes = decltype(lanes)::value;
        constexpr int kRows = kFp8Threads / kLanes;
        LaunchDependent(kv_append_fp8_kernel<T, kLanes, kBatched, I>, Fp8Grid((static_cast<int64_t>(rows) + kRows - 1) / kRows), kFp8Threads, 0,
                        stream, 1, static_cast<const T*>(k_new), static_cast<const T*>(v_new), rows, a);
    };
    const int pieces = a.head_dim / kPiece;
    if (pieces <= 2) go(std::integral_constant<int, 2>{});
    else if (pieces <= 4) go(std::integral_constant<int, 4>{});
    else if (pieces <= 8) go(std::integral_constant<int, 8>{});
    else go(std::integral_constant<int, 16>{});
}

template <bool kBatched>
int AppendRows(const ScaFp8Layer& l, const void* k_new, const void* v_new, int64_t tokens, const ScaKvCacheShape& shape, AppendTarget a,
               int32_t dtype_id, cudaStream_t stream, const char* what) {
    a.k_codes = static_cast<uint8_t*>(l.k_codes);
    a.v_codes = static_cast<uint8_t*>(l.v_codes);
    a.k_scales = static_cast<uint8_t*>(l.k_scales);
    a.v_scales = static_cast<uint8_t*>(l.v_scales);
    a.num_blocks = shape.num_blocks;
    a.block_size = static_cast<int>(shape.block_size);
    a.heads = static_cast<int>(shape.num_kv_heads);
    a.head_dim = static_cast<int>(shape.head_dim);
    a.aligned = ((reinterpret_cast<uintptr_t>(k_new) | reinterpret_cast<uintptr_t>(v_new)) & 31u) == 0;
    if (!Aligned16(a.k_codes) || !Aligned16(a.v_codes)) return Fail(SCA_INVALID_ARGUMENT, std::string(what) + ": the codes must be 16-byte aligned");
    const int64_t rows = tokens * shape.num_kv_heads;
    auto typed = [&](auto* type) {
        using T = std::remove_pointer_t<decltype(type)>;
        // what the loop may step past `rows` fits the narrow counter too
        if (rows < (1ll << 31)) LaunchAppend<T, kBatched, uint32_t>(k_new, v_new, static_cast<uint32_t>(rows), a, stream);
        else LaunchAppend<T, kBatched, int64_t>(k_new, v_new, rows, a, stream);
    };
    switch (dtype_id) {
        case SCA_DTYPE_F32: typed(static_cast<float*>(nullptr)); break;
        case SCA_DTYPE_F16: typed(static_cast<__half*>(nullptr)); break;
        case SCA_DTYPE_BF16: typed(static_cast<__nv_bfloat16*>(nullptr)); break;
        default: return Fail(SCA_INVALID_ARGUMENT, std::string(what) + ": unsupported dtype id");
    }
    return CheckLaunch("kv_append_fp8_kernel", stream);
}

bool AnyNull(const ScaFp8Layer* l) {
    return l == nullptr || l->k_codes == nullptr || l->v_codes == nullptr || l->k_scales == nullptr || l->v_scales == nullptr;
}

}  // namespace
}  // namespace sca_b200

using namespace sca_b200;

extern "C" int sca_launch_kv_append_fp8(const ScaFp8Layer* layer, const void* k_new, const void* v_new, const int32_t* slot_mapping,
                                        int64_t num_tokens, const ScaKvCacheShape* shape, int32_t dtype_id, void* stream) {
    ClearError();
    if (AnyNull(layer) || k_new == nullptr || v_new == nullptr || slot_mapping == nullptr) {
        return Fail(SCA_INVALID_ARGUMENT, "kv append (fp8): null pointer");
    }
    if (num_tokens <= 0) return Fail(SCA_INVALID_ARGUMENT, "kv append (fp8): num_tokens <= 0");
    if (int rc = CheckFp8Shape(shape, "kv append (fp8)")) return rc;
    AppendTarget a{};
    a.slots = slot_mapping;
    return AppendRows<false>(*layer, k_new, v_new, num_tokens, *shape, a, dtype_id, static_cast<cudaStream_t>(stream), "kv append (fp8)");
}

extern "C" int sca_launch_kv_append_batched_fp8(const ScaFp8Layer* layer, const void* k_new, const void* v_new, const int32_t* page_table,
                                                const int32_t* seq_lens, int64_t num_seqs, int64_t max_blocks_per_seq,
                                                const ScaKvCacheShape* shape, int32_t dtype_id, void* stream) {
    ClearError();
    if (AnyNull(layer) || k_new == nullptr || v_new == nullptr || page_table == nullptr || seq_lens == nullptr) {
        return Fail(SCA_INVALID_ARGUMENT, "kv append (batched, fp8): null pointer");
    }
    if (num_seqs <= 0 || max_blocks_per_seq <= 0) {
        return Fail(SCA_INVALID_ARGUMENT, "kv append (batched, fp8): num_seqs/max_blocks_per_seq <= 0");
    }
    if (int rc = CheckFp8Shape(shape, "kv append (batched, fp8)")) return rc;
    AppendTarget a{};
    a.page_table = page_table;
    a.seq_lens = seq_lens;
    a.max_blocks_per_seq = max_blocks_per_seq;
    return AppendRows<true>(*layer, k_new, v_new, num_seqs, *shape, a, dtype_id, static_cast<cudaStream_t>(stream), "kv append (batched, fp8)");
}

extern "C" int sca_launch_kv_gather_fp8(const void* codes, const uint8_t* scales, const int32_t* block_ids, int64_t num_blocks, void* out,
                                        const ScaKvCacheShape* shape, int32_t dtype_id, void* stream) {
    ClearError();
    if (codes == nullptr || scales == nullptr || block_ids == nullptr || out == nullptr) {
        return Fail(SCA_INVALID_ARGUMENT, "kv gather (fp8): null pointer");
    }
    if (num_blocks <= 0) return SCA_OK;
    if (int rc = CheckFp8Shape(shape, "kv gather (fp8)")) return rc;
    if (!Aligned16(codes) || !Aligned16(out)) return Fail(SCA_INVALID_ARGUMENT, "kv gather (fp8): codes and output must be 16-byte aligned");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const int64_t total = num_blocks * shape->block_size * shape->num_kv_heads * (shape->head_dim / 16);
    const int64_t grid = Fp8Grid((total + kFp8Threads - 1) / kFp8Threads);
    auto typed = [&](auto* type) {
        using T = std::remove_pointer_t<decltype(type)>;
        auto go = [&](auto count) {
            LaunchDependent(kv_gather_fp8_kernel<T, decltype(count)>, grid, kFp8Threads, 0, s, 1, static_cast<const uint8_t*>(codes), scales,
                            block_ids, count, static_cast<T*>(out), shape->num_blocks, static_cast<int>(shape->block_size),
                            static_cast<int>(shape->num_kv_heads), static_cast<int>(shape->head_dim),
                            (reinterpret_cast<uintptr_t>(out) & 31u) == 0);
        };
        if (total < (1ll << 31)) go(static_cast<uint32_t>(total));
        else go(total);
    };
    switch (dtype_id) {
        case SCA_DTYPE_F32: typed(static_cast<float*>(nullptr)); break;
        case SCA_DTYPE_F16: typed(static_cast<__half*>(nullptr)); break;
        case SCA_DTYPE_BF16: typed(static_cast<__nv_bfloat16*>(nullptr)); break;
        default: return Fail(SCA_INVALID_ARGUMENT, "kv gather (fp8): unsupported dtype id");
    }
    return CheckLaunch("kv_gather_fp8_kernel", s);
}

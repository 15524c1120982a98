// Chunks of new tokens over a paged cache of 8 bits: the prefill kernels whose converters rewrite codes of K and V as fp16 (kKv8 in
// flash_kernel.cuh), so that the scores and the products run on the tensor cores as they do over a 16-bit cache, from half the bytes.
//
// What bounds it, D=128: the chain of scores, softmax and products of a tile, as over a 16-bit cache (20 chunks of 5140 tokens, 32 / 8 heads:
// tensor pipe 47 % of the time, special-function unit 47 %, issue slots 45 %): 770 to 910 TFLOP/s, where products alone sustain 1390 under the
// same power cap, so that the cap is the smaller part of a lasting load's 440 us against 375 in a burst. The converters take
// issue slots from the softmax: 5 instructions for 4 codes, K as well as V, where the 16-bit kernel rewrites V only. 373 us against 332
// over the 16-bit cache; D=64 3 % to 10 % more; D=256, where the bytes in shared memory are what counts, 404 us, a sixth less. Shared
// memory sees as much as with 16 bits: codes in and out, numbers in, against numbers in, out and in for V.
#include "flash_kernel.cuh"

namespace sca_b200 {
namespace flash {
namespace {

template <typename T, int DP, int QT, int BN, bool kSplit>
int Launch(int64_t ctas, int cluster, cudaStream_t stream, const CUtensorMap& map_q, const CUtensorMap& map_k, const CUtensorMap& map_v,
           const FlashKernelParams& p, const WorkImage& image) {
    auto kernel = flash_fwd_sm100_kernel<T, DP, QT, BN, true, true, true, false, kSplit>;
    constexpr int kSmem = FlashGeom<DP, QT, BN, true>::kSmemBytes;
    if (int rc = EnsureDynamicSmem(reinterpret_cast<const void*>(kernel), kSmem, "flash_fwd_sm100_kernel")) return rc;
    constexpr int kThreads = FlashThreads<T, DP, QT, true>();
    if constexpr (TakesWorkImage(DP, true, kSplit, true)) LaunchDependent(kernel, ctas, kThreads, kSmem, stream, cluster, map_q, map_k, map_v, p, image);
    else LaunchDependent(kernel, ctas, kThreads, kSmem, stream, cluster, map_q, map_k, map_v, p, NoWorkImage{});
    return SCA_OK;
}

}  // namespace

template <typename T, int DP, int QT, int BN>
int LaunchKv8(int64_t items, unsigned grid, cudaStream_t stream, const CUtensorMap& map_q, const CUtensorMap& map_k, const CUtensorMap& map_v,
              const FlashKernelParams& p, const WorkImage& image) {
    if (p.cluster > 1) return Launch<T, DP, QT, BN, true>(items * p.cluster, p.cluster, stream, map_q, map_k, map_v, p, image);
    return Launch<T, DP, QT, BN, false>(grid, 1, stream, map_q, map_k, map_v, p, image);
}

#define SCA_KV8(T, DP, QT)                                                                                                          \
    template int LaunchKv8<T, DP, QT, 128>(int64_t, unsigned, cudaStream_t, const CUtensorMap&, const CUtensorMap&, const CUtensorMap&, \
                                           const FlashKernelParams&, const WorkImage&);
SCA_KV8(__half, 64, 2)
SCA_KV8(__half, 128, 2)
SCA_KV8(__half, 256, 1)
SCA_KV8(__nv_bfloat16, 64, 2)
SCA_KV8(__nv_bfloat16, 128, 2)
SCA_KV8(__nv_bfloat16, 256, 1)
#undef SCA_KV8

}  // namespace flash
}  // namespace sca_b200

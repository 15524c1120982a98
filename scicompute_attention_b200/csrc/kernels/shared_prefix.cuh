// What the kernels of a decode over shared prefixes know about the groups: a parameter of the launch, so that nothing is copied ahead of it
// and a captured graph keeps it.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

namespace sca_b200 {

constexpr int kMaxGroups = 128;

// Sequences [first, end) whose first `tokens` tokens (whole pages) are read through the page-table row of the first of them.
struct PrefixGroup {
    int first, end, tokens;
    int first_entry;  // in the work list of the prefix kernel
};
struct PrefixGroups {
    int count;       // groups that share something, in the order of their sequences
    int part_tiles;  // tiles of 128 keys to a part of a prefix
    int parts;       // parts of the longest prefix: a row's parts in the arrays below
    PrefixGroup group[kMaxGroups];
};

// The group of sequence b; null where it shares nothing.
__device__ __forceinline__ const PrefixGroup* GroupOf(const PrefixGroups& groups, int64_t b) {
    int lo = 0, hi = groups.count;  // the last one that begins at b or before is below hi
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (groups.group[mid].first <= b) lo = mid + 1;
        else hi = mid;
    }
    return lo > 0 && b < groups.group[lo - 1].end ? &groups.group[lo - 1] : nullptr;
}

// Where the parts of the prefixes are left, fp32: m (log2 domain) and l [rows][parts], O [rows][parts][D]; a row is sequence * heads + head.
struct PrefixParts {
    float *m, *l, *o;
    unsigned long long* begun;  // see SayBegun; 0 between two calls
};

// The kernel that takes the sequences' own tokens may run beside the prefix kernel ahead of it, but the order of a launch says nothing about what that
// one has waited for. So the prefix kernel, which has, releases this mark (the pattern of two signalling NaN: no kernel leaves these numbers in
// scratch), and who acquires it stands behind all kernels ahead of the call, as the prefix kernel does. The finish kernel takes the mark away.
constexpr unsigned long long kBegun = 0xff8b4d277f9a3c51ull;
// One thread, behind its wait for the kernel ahead.
__device__ __forceinline__ void SayBegun(unsigned long long* begun) { asm volatile("st.release.gpu.global.u64 [%0], %1;\n" ::"l"(begun), "l"(kBegun) : "memory"); }
// All threads of a CTA; the barrier passes on what the first thread has acquired.
__device__ __forceinline__ bool HasBegun(const unsigned long long* begun) {
    unsigned long long seen = 0;
    if (threadIdx.x == 0) asm volatile("ld.acquire.gpu.global.u64 %0, [%1];\n" : "=l"(seen) : "l"(begun) : "memory");
    return __syncthreads_or(seen == kBegun) != 0;
}

}  // namespace sca_b200

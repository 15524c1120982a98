// What the decode kernels of a 16-bit and of an 8-bit cache share: the schedule, the merge of a CTA's warps, the one-launch form on
// clusters and its merge.
#pragma once

#include <algorithm>

#include "common.cuh"

namespace sca_b200 {

// Merges the partials of p into p.out; directly behind the kernel that writes them (decode.cu).
int LaunchMergeOut(const ScaDecodeFwdParams& p, cudaStream_t stream);

namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kMaxCluster = 8;  // CTAs that may share one (sequence, kv head, head chunk) in the one-launch kernel

// Length of sequence b as the kernel sees it (never past the K/V extent / the page table) and the number of
// kSpan-token steps it takes. An empty sequence still counts one (empty) step so that somebody writes its partial.
template <bool kPaged>
__device__ __forceinline__ int64_t SeqLen(const ScaDecodeFwdParams& p, int64_t b) {
    int64_t len = p.seq_lens != nullptr ? static_cast<int64_t>(p.seq_lens[b]) : p.seq_kv;
    if (len < 0) len = 0;
    const int64_t cap = kPaged ? p.max_blocks_per_seq * p.block_size : p.seq_kv;
    return len < cap ? len : cap;
}
template <int kSpan>
__device__ __forceinline__ int64_t StepsFor(int64_t len) {
    const int64_t t = (len + kSpan - 1) / kSpan;
    return t > 0 ? t : 1;
}

// Bytes of a warp's ring that the end of a segment takes: {m[16], l[16], O[16][D]} of the warp, {m[16], l[16]} of the CTA.
template <int D>
constexpr int MergeBytes() { return (64 + 16 * D) * 4; }
template <int D>
__device__ __forceinline__ float* CtaPartial(unsigned char* smem) {
    return reinterpret_cast<float*>(smem) + 32 + 16 * D;  // behind warp 0's staging area, inside its ring
}
// The end of a segment: the warps' results, each in its ring as {m[16], l[16], O[16][D]}, become the CTA's: in `slot` of the
// partial arrays, or (kToShared) m and l at CtaPartial<D>(smem) and O in the place of warp 0's, each number written by the thread
// that alone has read it.
template <int D, int kWarpBytes, bool kToShared>
__device__ __forceinline__ void MergeWarps(const ScaDecodeFwdParams& p, unsigned char* smem, const int64_t b, const int head0,
                                           const int nheads, const int slot) {
    for (int item = threadIdx.x; item < nheads * D; item += kThreads) {
        const int row = item / D;
        const int d = item % D;
        float m_all = -CUDART_INF_F;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            m_all = fmaxf(m_all, reinterpret_cast<const float*>(smem + w * kWarpBytes)[row]);
        }
        float acc = 0.0f, l_all = 0.0f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float* wm = reinterpret_cast<const float*>(smem + w * kWarpBytes);
            const float mw = wm[row];
            if (mw == -CUDART_INF_F) continue;
            const float wgt = Exp2(mw - m_all);
            acc += wm[32 + row * D + d] * wgt;
            l_all += wm[16 + row] * wgt;
        }
        if (kToShared) {
            reinterpret_cast<float*>(smem)[32 + row * D + d] = acc;
            float* partial = CtaPartial<D>(smem);
            if (d == 0) {
                partial[row] = m_all;
                partial[16 + row] = l_all;
            }
            continue;
        }
        const int64_t flat = (b * p.num_heads + head0 + row) * p.num_splits + slot;
        p.partial_o[flat * D + d] = acc;
        if (d == 0) {
            p.partial_m[flat] = m_all * kLn2;  // stored in natural units like the reference workspace
            p.partial_l[flat] = l_all;
        }
    }
    __syncthreads();  // the rings double as merge staging: nobody refills them before everyone has read
}

// Marks slots [first, end) of every head of one (sequence, kv head, head chunk) as empty (m = -inf; the merge
// skips such entries without reading l or O).
__device__ __forceinline__ void MarkUnusedSlots(const ScaDecodeFwdParams& p, int64_t b, int hk, int hc, int first, int end) {
    const int group = static_cast<int>(p.num_heads / p.num_kv_heads);
    const int head0 = hk * group + hc * 16;
    const int nheads = min(16, group - hc * 16);
    const int unused = end - first;
    for (int item = threadIdx.x; item < nheads * unused; item += kThreads) {
        const int row = item / unused;
        const int slot = first + item % unused;
        p.partial_m[(b * p.num_heads + head0 + row) * p.num_splits + slot] = -CUDART_INF_F;
    }
}

// A split-K partial kernel, scheduled for an equal share of the K/V stream per CTA; segment(b, hk, hc, j_begin, j_end, slot)
// is what it does with a piece of a sequence.
//
// The grid is one wave of resident CTAs, a multiple of the number of (kv head, head chunk) columns. CTA c works on
// column c % columns for its whole life; the CTAs of one column split that column's list of kSpan-token steps
// (sequence after sequence) into equal contiguous shares. Neighbouring CTAs therefore read the same tokens of
// neighbouring kv heads at about the same time - in a paged pool those are adjacent 2*D-byte pieces of one token row.
// A share may start and end in the middle of a sequence and may cover several short ones; every piece of a sequence
// a CTA holds is one "segment" and yields one partial. The pieces of one sequence sit in consecutive CTAs of the
// column, so a segment's slot in the [rows, num_splits] partial arrays is the distance to the first CTA that touches
// the sequence. A share is never smaller than longest_sequence / (num_splits - 1) steps, which bounds the pieces of
// any sequence by num_splits (with num_splits == 1 shares are made of whole sequences); slots that stay unused are
// marked empty by the CTA that holds the sequence's first step.
// Sequence lengths are read on the device (seq_lens), so the schedule needs no host knowledge of a ragged batch.
template <bool kPaged, int kSpan, typename Segment>
__device__ __forceinline__ void WalkSchedule(const ScaDecodeFwdParams& p, const int head_chunks, const Segment& segment) {
    __shared__ int64_t s_part[kWarps][2];
    __shared__ int64_t s_found[2];
    WaitForPredecessor();
    const int lane = threadIdx.x & 31;
    const int warp = threadIdx.x >> 5;
    const int columns = static_cast<int>(p.num_kv_heads) * head_chunks;
    // grids smaller than the number of columns let every CTA walk several columns, each as its only CTA
    const int sharers = gridDim.x >= static_cast<unsigned>(columns) ? static_cast<int>(gridDim.x) / columns : 1;
    const int share = gridDim.x >= static_cast<unsigned>(columns) ? static_cast<int>(blockIdx.x) / columns : 0;
    const int first_column = gridDim.x >= static_cast<unsigned>(columns) ? static_cast<int>(blockIdx.x) % columns
                                                                         : static_cast<int>(blockIdx.x);
    const int column_stride = gridDim.x >= static_cast<unsigned>(columns) ? columns : static_cast<int>(gridDim.x);
    if (share >= sharers) return;  // a grid that is no multiple of the column count

    // ---- this CTA's share [begin, end) of a column's step list, and the sequence that holds `begin` ----------
    int64_t b, before, len, steps, per_cta, begin, end;
    if (p.seq_lens == nullptr) {
        // every sequence has the same length: the list is regular and needs no look at device memory
        len = SeqLen<kPaged>(p, 0);
        steps = StepsFor<kSpan>(len);
        const int64_t total = p.batch * steps;
        per_cta = (total + sharers - 1) / sharers;
        const int64_t floor_steps = p.num_splits > 1 ? (steps + p.num_splits - 2) / (p.num_splits - 1) : total;
        if (per_cta < floor_steps) per_cta = floor_steps;
        if (p.num_splits == 1) per_cta = ((per_cta + steps - 1) / steps) * steps;  // whole sequences only
        begin = share * per_cta;
        if (begin >= total) return;
        end = begin + per_cta < total ? begin + per_cta : total;
        b = begin / steps;
        before = b * steps;
    } else {
        // pass 1: total steps and the longest sequence
        int64_t sum = 0, longest = 0;
        for (int64_t i = threadIdx.x; i < p.batch; i += kThreads) {
            const int64_t t = StepsFor<kSpan>(SeqLen<kPaged>(p, i));
            sum += t;
            longest = t > longest ? t : longest;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            sum += __shfl_xor_sync(0xffffffffu, sum, o);
            const int64_t other = __shfl_xor_sync(0xffffffffu, longest, o);
            longest = other > longest ? other : longest;
        }
        if (lane == 0) {
            s_part[warp][0] = sum;
            s_part[warp][1] = longest;
        }
        __syncthreads();
        sum = 0;
        longest = 0;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            sum += s_part[w][0];
            longest = s_part[w][1] > longest ? s_part[w][1] : longest;
        }
        const int64_t total = sum;
        per_cta = (total + sharers - 1) / sharers;
        // with one slot a share must end where a sequence ends: the whole column then goes to its first CTA
        const int64_t floor_steps = p.num_splits > 1 ? (longest + p.num_splits - 2) / (p.num_splits - 1) : total;
        if (per_cta < floor_steps) per_cta = floor_steps;
        begin = share * per_cta;
        if (begin >= total) return;
        end = begin + per_cta < total ? begin + per_cta : total;

        // pass 2: find i with before[i] <= begin < before[i] + steps[i]
        int64_t running = 0;
        __syncthreads();
        for (int64_t base = 0; base < p.batch && running <= begin; base += kThreads) {
            const int64_t i = base + threadIdx.x;
            const int64_t t = i < p.batch ? StepsFor<kSpan>(SeqLen<kPaged>(p, i)) : 0;
            int64_t incl = t;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int64_t up = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += up;
            }
            if (lane == 31) s_part[warp][0] = incl;
            __syncthreads();
            int64_t mine = running + incl - t;
            int64_t chunk_total = 0;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                if (w < warp) mine += s_part[w][0];
                chunk_total += s_part[w][0];
            }
            if (t > 0 && mine <= begin && begin < mine + t) {
                s_found[0] = i;
                s_found[1] = mine;
            }
            running += chunk_total;
            __syncthreads();
        }
        b = s_found[0];
        before = s_found[1];  // steps of this column before sequence b
        len = SeqLen<kPaged>(p, b);
        steps = StepsFor<kSpan>(len);
    }
    // the merge kernel that follows on the stream may be set up while this grid streams K/V
    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");

    // ---- walk the share segment by segment, in every column this CTA serves -----------------------------
    const int64_t b_first = b, before_first = before, len_first = len, steps_first = steps;
    for (int column = first_column; column < columns; column += column_stride) {
        const int hk = column / head_chunks, hc = column % head_chunks;
        b = b_first;
        before = before_first;
        len = len_first;
        steps = steps_first;
        int64_t pos = begin;
        while (pos < end) {
            const int64_t t0 = pos - before;
            int64_t t1 = t0 + (end - pos);
            if (t1 > steps) t1 = steps;
            const int slot = static_cast<int>(share - before / per_cta);
            if (t0 == 0) {
                const int used = static_cast<int>((before + steps - 1) / per_cta - before / per_cta) + 1;
                MarkUnusedSlots(p, b, hk, hc, used, static_cast<int>(p.num_splits));
            }
            const int64_t j_end = t1 * kSpan < len ? t1 * kSpan : len;
            segment(b, hk, hc, t0 * kSpan, j_end, slot);
            pos += t1 - t0;
            if (t1 == steps && pos < end) {
                before += steps;
                ++b;
                len = SeqLen<kPaged>(p, b);
                steps = StepsFor<kSpan>(len);
            }
        }
    }
}

// Decode of a problem that does not fill the machine, in one launch: the CTAs of a cluster split one (sequence, kv head,
// head chunk) and merge their partials through distributed shared memory. Bound by latency - a step or two of K/V per
// CTA, then the exchange - so what counts is that there is no second kernel and no trip through memory in between.
template <typename T, int D, bool kPaged, int kSpan, typename Segment>
__device__ __forceinline__ void ClusterDecode(const ScaDecodeFwdParams& p, const int head_chunks, const int cluster, unsigned char* smem,
                                              const Segment& segment) {
    BeginAfterPredecessor();
    const int columns = static_cast<int>(p.num_kv_heads) * head_chunks;
    const int rank = static_cast<int>(ClusterRank());
    const int unit = static_cast<int>(blockIdx.x) / cluster;
    const int64_t b = unit / columns;
    const int hk = (unit % columns) / head_chunks, hc = (unit % columns) % head_chunks;
    const int64_t len = SeqLen<kPaged>(p, b);
    const int64_t steps = StepsFor<kSpan>(len);
    const int64_t share = (steps + cluster - 1) / cluster;
    const int64_t t0 = rank * share < steps ? rank * share : steps;
    const int64_t t1 = t0 + share < steps ? t0 + share : steps;
    const int64_t j_end = t1 * kSpan < len ? t1 * kSpan : len;
    segment(b, hk, hc, t0 * kSpan, j_end);
    ClusterBarrier();
    const int group = static_cast<int>(p.num_heads / p.num_kv_heads);
    const int head0 = hk * group + hc * 16;
    const int total = min(16, group - hc * 16) * D;
    const uint32_t partial = SmemAddr(CtaPartial<D>(smem)), partial_o = SmemAddr(smem) + 32 * 4;
    T* out = reinterpret_cast<T*>(p.out) + b * p.o_stride.s_b;
    for (int item = rank * kThreads + threadIdx.x; item < total; item += cluster * kThreads) {
        const int row = item / D, d = item % D;
        float m[kMaxCluster], l_all = 0.0f, acc = 0.0f, m_all = -CUDART_INF_F;
#pragma unroll
        for (int r = 0; r < kMaxCluster; ++r) {
            m[r] = r < cluster ? LoadFromRank(partial + 4 * row, r) : -CUDART_INF_F;
            m_all = fmaxf(m_all, m[r]);
        }
#pragma unroll
        for (int r = 0; r < kMaxCluster; ++r) {
            if (m[r] == -CUDART_INF_F) continue;
            const float weight = Exp2(m[r] - m_all);
            l_all += LoadFromRank(partial + 4 * (16 + row), r) * weight;
            acc += LoadFromRank(partial_o + 4 * (row * D + d), r) * weight;
        }
        const float inv = l_all > 0.0f ? 1.0f / l_all : 0.0f;
        out[(head0 + row) * p.o_stride.s_h + d] = FromFloat<T>(acc * inv);
    }
    ClusterBarrier();  // nobody leaves while its shared memory is being read
}

inline cudaLaunchConfig_t ClusterConfig(unsigned grid, int cluster, int smem_bytes, cudaStream_t stream, cudaLaunchAttribute* attr) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = static_cast<size_t>(smem_bytes);
    cfg.stream = stream;
    attr->id = cudaLaunchAttributeClusterDimension;
    attr->val.clusterDim.x = static_cast<unsigned>(cluster);
    attr->val.clusterDim.y = 1;
    attr->val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cfg;
}

}  // namespace
}  // namespace sca_b200

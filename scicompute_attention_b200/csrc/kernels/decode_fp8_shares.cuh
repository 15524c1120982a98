// The arithmetic of the schedule of the 8-bit decode kernel (WalkFp8Schedule in decode_fp8.cu): how many CTAs are launched, which steps of
// a column's list a CTA takes, and which pieces of which sequences these are. Plain C++, so that the host tests run the same lines.
#pragma once

#include <cstdint>

#ifdef __CUDACC__
#define SCA_SHARES_FN __host__ __device__ __forceinline__
#define SCA_SHARES_WALK __device__ __forceinline__
#else
#define SCA_SHARES_FN inline
#define SCA_SHARES_WALK inline
#endif

namespace sca_b200 {

// What the border between two sequences of a CTA - the end of one segment, the first loads of the next - counts for in its share, in steps.
// Without it the CTAs with a border end 7 us after the others (96 sequences of 200 to 6000 tokens, 32 / 2 heads, D=64 34.3 / 30.5 us; 64 of
// 300 to 3000, 32 / 8 heads 34.4 / 32.6). One step or three 31.5.
constexpr int kBorder = 2;
// CTAs of a wave that are left out, at least: with every place of the machine taken a call takes up to 9 us more, as if a CTA found its place
// still held (the merge kernel of the call before is the one that could) and ran when the others had. With 0, 2, 4, 6, 8 left out, us: 96
// sequences of 200 to 6001 tokens, D=64, 32 / 2 heads 34.8, 32.2, 30.6, 30.2, 30.2; 32 / 1 33.7, 31.1, 28.9, 28.5, 28.6; 16 / 2 25.4, 23.5, 23.4,
// 23.4, 23.4; D=256, 40 of 100 to 5000, 16 / 2 32.7, 30.2, 30.1, 30.1, 30.1. By whole columns: 64 of 300 to 3000, D=64, 32 / 8 with 0, 8, 16 left
// out 37.8, 31.4, 31.6; 32 / 16 with 0, 16, 32 61.4, 52.3, 52.8. Other calls take the same with and without (two CTAs to an SM; 32 / 4 heads
// 21.1). Columns of few sharers keep them all: one in sixteen costs as much (40 / 40 heads, D=128, 11 sharers or 10: 110, 116).
constexpr int kLeftOut = 4;

// CTAs to launch: of `resident` that stay on the machine as many for every one of `columns` lists, never more than a list has steps.
SCA_SHARES_FN int64_t ScheduleGrid(int64_t resident, int64_t columns, int64_t steps) {
    if (resident < columns) return resident;
    int64_t sharers = resident / columns;
    if (sharers > 16 && sharers > (resident - kLeftOut) / columns) sharers = (resident - kLeftOut) / columns;
    if (sharers > steps) sharers = steps;
    return columns * (sharers > 1 ? sharers : 1);
}

// A CTA's place in the grid. Grids smaller than the number of columns let every CTA walk several columns, each as its only CTA.
struct SchedulePlace {
    int sharers;  // CTAs of a column
    int share;    // this one among them; not below `sharers`: it has nothing to do
    int column, column_stride;
};
SCA_SHARES_FN SchedulePlace PlaceOf(int cta, int grid, int columns) {
    if (grid >= columns) return SchedulePlace{grid / columns, cta / columns, cta % columns, columns};
    return SchedulePlace{1, 0, cta, grid};
}

// Steps of `span` tokens that a sequence takes; an empty one still takes one, so that somebody marks its slots.
SCA_SHARES_FN int StepsOf(int len, int span) {
    const int t = static_cast<int>((static_cast<uint32_t>(len) + span - 1) / span);
    return t > 1 ? t : 1;
}
// What a border counts for in a list whose longest sequence takes so many steps.
SCA_SHARES_FN int BorderOf(int longest) { return longest > 1 ? kBorder : 0; }

// A column's list - its sequences' steps, borders included, one sequence behind the other - among its CTAs.
struct Shares {
    int sharing;  // CTAs that take a share
    int each;     // steps of a share, one more for the first `more`
    int more;
    SCA_SHARES_FN int Begin(int share) const { return share * each + (share < more ? share : more); }
    SCA_SHARES_FN int SharerOf(int step) const {
        const int left = step - more * (each + 1);
        return left < 0 ? step / (each + 1) : more + left / each;
    }
};
// `total` steps, `longest` those of the longest sequence, borders included. A share holds at least so many that no sequence falls into more than
// `splits` pieces; with one slot a column goes to its first CTA, unless no sequence can be cut.
SCA_SHARES_FN Shares ShareSteps(int total, int longest, int splits, int sharers) {
    const int least = splits > 1 ? (longest + splits - 2) / (splits - 1) : longest == 1 ? 1 : total;
    int sharing = total / least;
    if (sharing > sharers) sharing = sharers;
    if (sharing < 1) sharing = 1;
    const int each = total / sharing;
    return Shares{sharing, each, total - sharing * each};
}

// The sequence that holds step `begin`, among those from `*b` on, which start at step `*before` of the list.
template <typename Length>
SCA_SHARES_WALK void FindSequence(int begin, int span, int border, const Length& length, int* b, int* before) {
    while (true) {
        const int t = StepsOf(length(*b), span) + border;
        if (begin < *before + t) return;
        *before += t;
        ++*b;
    }
}

// The pieces of a share: segment(b, first token, end, slot, bare) for every one of them - `bare`: of the border alone, its slot stays empty -
// and unused(b, slots) for every sequence that begins in the share, with the slots that its pieces take. Sequence `b` begins at step `before`
// and holds the share's first step.
template <typename Length, typename Segment, typename Unused>
SCA_SHARES_WALK void WalkShare(const Shares& shares, int share, int span, int border, int b, int before, const Length& length, const Segment& segment,
                               const Unused& unused) {
    const int end = shares.Begin(share + 1);
    int len = length(b), steps = StepsOf(len, span) + border;
    for (int pos = shares.Begin(share); pos < end;) {
        const int t0 = pos - before, rest = t0 + (end - pos), t1 = rest < steps ? rest : steps;
        const int slot = t0 == 0 ? 0 : share - shares.SharerOf(before);
        if (t0 == 0) unused(b, shares.SharerOf(before + steps - 1) - share + 1);
        const int64_t first = static_cast<int64_t>(t0 > border ? t0 - border : 0) * span, last = static_cast<int64_t>(t1 - border) * span;
        segment(b, first, last < len ? last : static_cast<int64_t>(len), slot, t1 <= border);
        pos += t1 - t0;
        if (t1 == steps && pos < end) {
            before += steps;
            ++b;
            len = length(b);
            steps = StepsOf(len, span) + border;
        }
    }
}

}  // namespace sca_b200

// The schedule of the 8-bit decode kernel on the CPU, through the lines that the kernel and its launch run. Reads cases, one to a line,
//   span splits resident columns useful sequences length ...
// and prints for each "grid <CTAs>" and, for every piece of every CTA, "<column> <share> <sequence> <slot> <first token> <end> <bare>" and
// "used <column> <sequence> <slots>", then "end".
#include <algorithm>
#include <cstdio>
#include <vector>

#include "decode_fp8_shares.cuh"

using namespace sca_b200;

int main() {
    int span, splits, columns, sequences;
    long long resident, useful;
    while (std::scanf("%d %d %lld %d %lld %d", &span, &splits, &resident, &columns, &useful, &sequences) == 6) {
        std::vector<int> lens(sequences);
        for (int& n : lens) {
            if (std::scanf("%d", &n) != 1) return 1;
        }
        auto length = [&](int b) { return lens[b]; };
        int total = 0, longest = 0;
        for (int n : lens) total += StepsOf(n, span), longest = std::max(longest, StepsOf(n, span));
        const int border = BorderOf(longest);
        total += sequences * border;
        const int grid = static_cast<int>(ScheduleGrid(resident, columns, useful));
        std::printf("grid %d\n", grid);
        for (int cta = 0; cta < grid; ++cta) {
            const SchedulePlace place = PlaceOf(cta, grid, columns);
            if (place.share >= place.sharers) continue;
            const Shares shares = ShareSteps(total, longest + border, splits, place.sharers);
            if (place.share >= shares.sharing) continue;
            const int begin = shares.Begin(place.share);
            if (shares.SharerOf(begin) != place.share || shares.SharerOf(shares.Begin(place.share + 1) - 1) != place.share) return 2;
            int first = 0, before = 0;
            FindSequence(begin, span, border, length, &first, &before);
            for (int column = place.column; column < columns; column += place.column_stride) {
                WalkShare(
                    shares, place.share, span, border, first, before, length,
                    [&](int b, long long from, long long to, int slot, bool bare) { std::printf("%d %d %d %d %lld %lld %d\n", column, place.share, b, slot, from, to, bare); },
                    [&](int b, int used) { std::printf("used %d %d %d\n", column, b, used); });
            }
        }
        std::printf("end\n");
    }
    return 0;
}

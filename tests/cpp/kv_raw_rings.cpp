// The rings of the prefill kernel over an 8-bit cache, each as RingOf and RawRingOf describe it, on the CPU: two producers that take the
// loads in turn, loads that land in any order, converters that carry them from a raw slot to a slot, and the thread that issues the
// products; every role runs at any speed. Prints, per ring and plan, how many runs read or overwrote a slot at the wrong time ("early")
// and how many came to a stop ("stuck"). Plan 0 is the kernel's; the others are mistakes: 1, the converters do not wait for a free slot;
// 2, they hand a raw slot back when one of them has read it.
#include <cstdio>
#include <random>
#include <vector>

#include "kv_ring.cuh"

using namespace sca_b200;

struct Barrier {  // mbarrier as a waiter sees it: the phase of the given parity is over, or it is not
    int arrivals = 0, need = 1, phases = 0;
    void Arrive() {
        if (++arrivals == need) arrivals = 0, ++phases;
    }
    bool Over(uint32_t parity) const { return (phases & 1u) != parity; }
};

// 0 = sound, 1 = early, 2 = stuck
int Run(int plan, const RingShape& ring, const RawRingShape& raw_ring, unsigned seed) {
    std::mt19937 rng(seed);
    const int slots = raw_ring.slots, raw_slots = raw_ring.raw_slots, converters = raw_ring.converters;
    std::vector<char> frees;  // whether the products free what they have waited for behind this load
    for (int item = 0; item < 3; ++item) {
        const int count = 2 * (1 + static_cast<int>(rng() % 9)) * ring.parts, first = static_cast<int>(frees.size());
        frees.resize(frees.size() + count, 1);
        // one query tile: a slot at a time; two: K_0 alone, the two loads of a step together, V_n-1 alone
        if (ring.parts == 1) {
            for (int it = 1; it + 1 < count; it += 2) frees[first + it] = 0;
        }
    }
    const int total = static_cast<int>(frees.size());
    std::vector<Barrier> raw_full(raw_slots), raw_empty(raw_slots), ready(slots), empty(slots);
    for (Barrier& b : raw_empty) b.need = plan == 2 ? 1 : converters;
    for (Barrier& b : ready) b.need = converters;
    std::vector<int> raw_content(raw_slots, -1), read_by(total, 0), written_by(total, 0), next(2), walked(converters, 0), flying;
    next[0] = 0, next[1] = 1;
    int waited = 0, freed = 0;
    RingPhases phases;
    std::vector<int> weight(4 + converters);  // producers, memory, products, converters
    for (int& w : weight) w = 1 << (rng() % 8);
    std::discrete_distribution<int> pick(weight.begin(), weight.end());
    for (int idle = 0; freed < total;) {
        if (++idle > 200000) return 2;
        const int role = pick(rng);
        if (role < 2) {
            const int i = next[role], raw = i % raw_slots;
            if (i >= total || !raw_empty[raw].Over(static_cast<uint32_t>(i / raw_slots & 1) ^ 1u)) continue;
            if (raw_content[raw] >= 0 && read_by[raw_content[raw]] < converters) return 1;  // overwritten ahead of a reader
            raw_content[raw] = -2;
            flying.push_back(i);
            next[role] += 2;
        } else if (role == 2) {
            if (flying.empty()) continue;
            const size_t at = rng() % flying.size();
            const int i = flying[at];
            flying.erase(flying.begin() + static_cast<long>(at));
            raw_content[i % raw_slots] = i;
            raw_full[i % raw_slots].Arrive();
        } else if (role == 3) {
            const int i = waited, slot = i % slots;
            if (i >= total || !ready[slot].Over(phases.bits >> slot & 1u)) continue;
            phases.Take(static_cast<uint32_t>(slot));
            if (written_by[i] < converters) return 1;
            ++waited;
            if (frees[i]) {
                for (; freed < waited; ++freed) empty[freed % slots].Arrive();
            }
        } else {
            const int c = role - 4, i = walked[c];
            if (i >= total) continue;
            const int raw = i % raw_slots, slot = i % slots;
            if (!raw_full[raw].Over(static_cast<uint32_t>(i / raw_slots & 1))) continue;
            if (plan != 1 && !empty[slot].Over(static_cast<uint32_t>(i / slots & 1) ^ 1u)) continue;
            if (raw_content[raw] != i || i - slots >= freed) return 1;
            ++read_by[i], ++written_by[i], ++walked[c];
            ready[slot].Arrive();
            if (plan != 2 || c == 0) raw_empty[raw].Arrive();
        }
        idle = 0;
    }
    return 0;
}

int main() {
    for (int dim : {64, 128, 256}) {
        for (int plan = 0; plan < 3; ++plan) {
            int early = 0, stuck = 0;
            for (unsigned seed = 0; seed < 2000; ++seed) {
                const int r = Run(plan, RingOf(dim), RawRingOf(dim), seed);
                early += r == 1;
                stuck += r == 2;
            }
            std::printf("%d %d %d %d\n", dim, plan, early, stuck);
        }
    }
    return 0;
}

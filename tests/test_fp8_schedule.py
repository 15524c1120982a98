"""The schedule of the 8-bit decode kernel, restated: every token of every sequence is in one segment, every segment has a slot of its own among those
the caller gave, and the CTAs' shares differ by a step at most."""
import random

import pytest

from scicompute_attention_b200 import ops


def shares(lens, span, splits, sharers, border_steps):
    """(sequence, slot, first token, end) of every segment that holds tokens, and (sequence, slot) of all that are written."""
    real = [max(1, -(-n // span)) for n in lens]
    border = border_steps if max(real) > 1 else 0
    steps = [n + border for n in real]
    total, longest = sum(steps), max(steps)
    least = -(-longest // (splits - 1)) if splits > 1 else 1 if longest == 1 else total
    sharing = max(1, min(sharers, total // least))
    each, more = total // sharing, total % sharing
    begin = [s * each + min(s, more) for s in range(sharing + 1)]

    def sharer_of(step):
        left = step - more * (each + 1)
        return step // (each + 1) if left < 0 else more + left // each

    starts = [sum(steps[:b]) for b in range(len(lens))]
    segments, written, held = [], [], []
    for s in range(sharing):
        assert all(sharer_of(p) == s for p in (begin[s], begin[s + 1] - 1))
        held.append(begin[s + 1] - begin[s])
        for b, at in enumerate(starts):
            t0, t1 = max(begin[s], at) - at, min(begin[s + 1], at + steps[b]) - at
            if t0 >= t1:
                continue
            slot = s - sharer_of(at)
            written.append((b, slot))
            if t0 == 0:
                written += [(b, unused) for unused in range(sharer_of(at + steps[b] - 1) - s + 1, splits)]
            if t1 > border:
                segments.append((b, slot, max(t0 - border, 0) * span, min((t1 - border) * span, lens[b])))
    return segments, written, held


@pytest.mark.parametrize("seed", range(30))
def test_every_token_once_and_every_slot_once(seed):
    rng = random.Random(seed)
    d = rng.choice((64, 128, 256))
    span = ops.fp8_step_tokens(d)
    lens = [rng.choice((0, 1, rng.randint(1, 127), rng.randint(1, 20000), rng.randint(100, 3000))) for _ in range(rng.choice((1, 2, 7, 96, 300)))]
    hkv, group, sms = rng.choice((1, 2, 8, 40)), rng.choice((1, 4, 8, 16, 40)), 148
    typical, longest = rng.choice(((sum(lens) // len(lens), max(lens)), (0, 0), (1, 1), (5000, 0)))
    splits = ops.paged_splits_for(typical or 4096, len(lens), hkv, group, sms, longest, span, ops.fp8_ctas_per_sm(d, group), ops.FP8_MAX_SPLITS,
                                  ops.FP8_BORDER_STEPS)
    columns = hkv * -(-group // 16)
    sharers = max(1, (ops.fp8_ctas_per_sm(d, group) * sms - 4) // columns)
    segments, written, held = shares(lens, span, splits, sharers, ops.FP8_BORDER_STEPS)
    assert sorted(written) == [(b, slot) for b in range(len(lens)) for slot in range(splits)]
    assert max(held) - min(held) <= 1
    for b, n in enumerate(lens):
        pieces = sorted((lo, hi) for s, _, lo, hi in segments if s == b)
        assert pieces[0][0] == 0 and pieces[-1][1] == n and all(x[1] == y[0] for x, y in zip(pieces, pieces[1:]))


def test_good_hints_leave_no_cta_out():
    """Slots from the true mean and maximum do not make the shares larger than the balance wants."""
    for d, lens in ((64, [200 + 61 * i for i in range(96)]), (128, [512 + 30 * i for i in range(256)]), (256, [100 + 125 * i for i in range(40)])):
        span, ctas = ops.fp8_step_tokens(d), ops.fp8_ctas_per_sm(d, 8)
        splits = ops.paged_splits_for(sum(lens) // len(lens), len(lens), 2, 8, 148, max(lens), span, ctas, ops.FP8_MAX_SPLITS, ops.FP8_BORDER_STEPS)
        sharers = (148 * ctas - 4) // 2
        assert len(shares(lens, span, splits, sharers, ops.FP8_BORDER_STEPS)[2]) >= 0.97 * sharers

"""The schedule of the 8-bit decode kernel: the kernel's own arithmetic, compiled for the CPU. Every token of every sequence is in one piece of every
column, every slot is written once, and no CTA has much more to do than another."""
import os
import random
import subprocess

import pytest

from scicompute_attention_b200 import ops

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SMS = 148


@pytest.fixture(scope="module")
def schedule(tmp_path_factory):
    exe = str(tmp_path_factory.mktemp("fp8_shares") / "fp8_shares")
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-fsanitize=undefined", "-fno-sanitize-recover=undefined", "-I",
                    os.path.join(ROOT, "scicompute_attention_b200", "csrc", "kernels"), os.path.join(ROOT, "tests", "cpp", "fp8_shares.cpp"), "-o", exe], check=True)

    def run(span, splits, resident, columns, useful, lens):
        """(CTAs launched, pieces, slots used by (column, sequence))."""
        given = " ".join(map(str, (span, splits, resident, columns, useful, len(lens), *lens)))
        out = subprocess.run([exe], input=given, check=True, capture_output=True, text=True, timeout=120).stdout.split("\n")
        assert out[-2] == "end"
        rows = [line.split() for line in out[1:-2]]
        used = [tuple(map(int, r[1:])) for r in rows if r[0] == "used"]
        assert len({u[:2] for u in used}) == len(used)  # said once
        return int(out[0].split()[1]), [tuple(map(int, r)) for r in rows if r[0] != "used"], {u[:2]: u[2] for u in used}
    return run


def check(lens, splits, columns, pieces, used):
    written = {}
    for column, _, b, slot, lo, hi, bare in pieces:
        of = written.setdefault((column, b), [])
        of.append((slot, lo, hi, bare))
    assert set(written) == set(used) == {(c, b) for c in range(columns) for b in range(len(lens))}
    for (column, b), of in written.items():
        assert sorted(slot for slot, *_ in of) == list(range(used[column, b])) and used[column, b] <= splits
        at = 0
        for _, lo, hi, bare in sorted(of):
            if not bare:
                assert lo == at and lo <= hi
                at = hi
        assert at == lens[b]


@pytest.mark.parametrize("seed", range(60))
def test_every_token_once_and_every_slot_once(schedule, seed):
    rng = random.Random(seed)
    d, group = rng.choice((32, 64, 128, 256)), rng.choice((1, 4, 8, 16, 40))
    span, ctas = ops.fp8_step_tokens(d), ops.fp8_ctas_per_sm(d, group)
    lens = [rng.choice((0, 1, span, span + 1, rng.randint(1, 127), rng.randint(1, 20000), rng.randint(100, 3000))) for _ in range(rng.choice((1, 2, 7, 96, 300)))]
    if seed % 7 == 0:
        lens = [min(n, span) for n in lens]  # nothing that could be cut
    hkv, sms = rng.choice((1, 2, 8, 40)), rng.choice((SMS, SMS, 20, 1))
    typical, longest = rng.choice(((sum(lens) // len(lens), max(lens)), (0, 0), (1, 1), (5000, 0)))
    splits = ops.paged_splits_for(typical or 4096, len(lens), hkv, group, sms, longest, span, ctas, ops.FP8_MAX_SPLITS, ops.FP8_BORDER_STEPS)
    columns, resident = hkv * -(-group // 16), ctas * sms
    useful = len(lens) * max(1, -(-(longest or 100000) // span))
    grid, pieces, used = schedule(span, splits, resident, columns, useful, lens)
    assert 1 <= grid <= resident and (grid % columns == 0 or grid == resident < columns)
    check(lens, splits, columns, pieces, used)
    if grid >= columns:
        steps = {}
        border = ops.FP8_BORDER_STEPS if max(lens) > span else 0
        for column, share, b, slot, lo, hi, bare in pieces:
            # the border counts where the sequence begins; a piece that ends in it, or begins in it, holds a part of it
            steps.setdefault(share, []).append(max(0 if bare else -(-(hi - lo) // span), 0))
        total = sum(max(1, -(-n // span)) + border for n in lens)
        sharing = len(steps)
        assert max(sum(s) // columns for s in steps.values()) <= -(-total // sharing)


@pytest.mark.parametrize("splits", [1, 2, 3, 8])
def test_few_slots(schedule, splits):
    """However few slots a caller gives, no sequence falls into more pieces."""
    for lens in ([5000], [0], [128] * 9, [1, 4000, 0, 129, 900, 128]):
        grid, pieces, used = schedule(128, splits, 444, 2, 1000, lens)
        check(lens, splits, 2, pieces, used)


def test_good_hints_leave_no_cta_out(schedule):
    """Slots from the true mean and maximum do not make the shares larger than the balance wants: every CTA that is launched has one."""
    for d, lens in ((64, [200 + 61 * i for i in range(96)]), (128, [512 + 30 * i for i in range(256)]), (256, [100 + 125 * i for i in range(40)])):
        span, ctas = ops.fp8_step_tokens(d), ops.fp8_ctas_per_sm(d, 8)
        splits = ops.paged_splits_for(sum(lens) // len(lens), len(lens), 2, 8, SMS, max(lens), span, ctas, ops.FP8_MAX_SPLITS, ops.FP8_BORDER_STEPS)
        grid, pieces, used = schedule(span, splits, SMS * ctas, 2, len(lens) * -(-max(lens) // span), lens)
        check(lens, splits, 2, pieces, used)
        assert len({share for _, share, *_ in pieces}) >= 0.97 * grid / 2


@pytest.mark.parametrize("ctas", [2, 3, 4])
@pytest.mark.parametrize("columns", [1, 2, 3, 4, 5, 8, 12, 16, 20, 40, 74, 200, 1000])
def test_size_of_the_wave(schedule, ctas, columns):
    """Four CTAs of the wave at least are left out where a column has more than sixteen, and no more than whole columns ask for; never a CTA per column too
    many for the machine, nor more than a list has steps."""
    resident = ctas * SMS
    grid, *_ = schedule(128, 8, resident, columns, 10 ** 6, [1000])
    if resident // columns > 16:
        assert grid % columns == 0 and resident - 4 - columns < grid <= resident - 4
    else:
        assert grid == max(1, resident // columns) * columns if resident >= columns else grid == resident
    assert schedule(128, 8, resident, columns, 3, [300])[0] == min(grid, 3 * columns)

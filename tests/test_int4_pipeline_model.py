"""The hand-overs of the 4-bit tile kernel (moe_gemm_int4.cuh) on the CPU.

A wait on an mbarrier sees only the parity of its phase, so a role that may be
two uses of a slot behind another reads the wrong one. The model runs the
kernel's roles (words, scales and rows in, decoding sets, MMA issue) on
random schedules, with copies and MMAs that complete later, and checks that
every role finds in a slot the block it expects. It covers each shape that the
kernel is built with and each number of slots that the host may choose."""
import os
import random
import re

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


class Barrier:
    def __init__(self, count):
        self.count = self.pending = count
        self.copies = self.phase = 0

    def arrive(self, copies=0):
        self.pending -= 1
        self.copies += copies
        assert self.pending >= 0, "more arrivals than the barrier counts"
        self._complete()

    def copy_done(self):
        self.copies -= 1
        self._complete()

    def _complete(self):
        if self.pending == 0 and self.copies == 0:
            self.phase += 1
            self.pending = self.count

    def passed(self, parity):
        return (self.phase & 1) != parity


def run(stages, raw, sets, raw_blocks, seed):
    """raw_blocks blocks of words (128 k), two MMA blocks each."""
    rnd = random.Random(seed)
    blocks = 2 * raw_blocks
    full, empty = [Barrier(2) for _ in range(stages)], [Barrier(1) for _ in range(stages)]
    raw_full, raw_empty = [Barrier(2) for _ in range(raw)], [Barrier(2) for _ in range(raw)]
    weights, rows = [None] * stages, [None] * stages
    words, scales = [None] * raw, [None] * raw
    copies, mmas, used = [], [], [-1]

    def ring(n, size):
        for i in range(n):
            yield i, i % size, (i // size) & 1

    def rows_in():
        for i, st, phase in ring(blocks, stages):
            while not empty[st].passed(phase ^ 1):
                yield
            assert used[0] >= i - stages, "rows over a block in use"
            full[st].arrive(copies=1)
            copies.append((rows, st, i, full[st]))
            yield

    def words_in():
        for i, slot, phase in ring(raw_blocks, raw):
            while not raw_empty[slot].passed(phase ^ 1):
                yield
            raw_full[slot].arrive(copies=1)
            copies.append((words, slot, i, raw_full[slot]))
            yield

    def scales_in():
        for i, slot, phase in ring(raw_blocks, raw):
            while not raw_empty[slot].passed(phase ^ 1):
                yield
            scales[slot] = i
            yield
            raw_full[slot].arrive()
            yield

    def decode(s):  # stages and slots in the steps that the kernel takes
        st, phase, slot, raw_phase = s, 0, s // 2, 0
        for i in range(s, blocks, sets):
            while not raw_full[slot].passed(raw_phase):
                yield
            assert words[slot] == scales[slot] == i // 2, "words of another block"
            yield
            while not empty[st].passed(phase ^ 1):
                yield
            assert used[0] >= i - stages, "weights over a block in use"
            weights[st] = i
            yield
            assert words[slot] == scales[slot] == i // 2, "words replaced while read"
            full[st].arrive()
            yield
            raw_empty[slot].arrive()
            st += sets
            if st >= stages:
                st, phase = s, phase ^ 1
            slot += (i + sets) // 2 - i // 2
            if slot >= raw:
                slot, raw_phase = slot - raw, raw_phase ^ 1
            yield

    def issue():
        for i, st, phase in ring(blocks, stages):
            while not full[st].passed(phase):
                yield
            assert weights[st] == rows[st] == i, "operands of another block"
            mmas.append((st, i))
            yield

    roles = [rows_in(), words_in(), scales_in(), issue()] + [decode(s) for s in range(sets)]
    speed = [rnd.choice([1, 1, 5, 30]) for _ in roles]
    for _ in range(200_000):
        if not (roles or copies or mmas):
            return
        pick = rnd.random()
        if copies and pick < 0.2:
            place, slot, i, bar = copies.pop(rnd.randrange(len(copies)))
            place[slot] = i
            bar.copy_done()
        elif mmas and pick < 0.3:
            st, i = mmas.pop(0)
            assert weights[st] == rows[st] == i, "operands replaced under an MMA"
            used[0] = i
            empty[st].arrive()
        elif roles:
            r = rnd.choices(range(len(roles)), speed)[0]
            if next(roles[r], roles) is roles:
                del roles[r], speed[r]
    raise AssertionError("the roles wait for one another")


def shapes():
    """(stages, slots of words, sets) of both shapes, for every number of slots
    that the host may choose, read from the kernel's source."""
    with open(os.path.join(ROOT, "mail_b200", "csrc", "moe_gemm_int4.cuh")) as f:
        src = f.read()

    def pair(name):
        m = re.search(name + r" = NARROW \? (\d+) : (\d+)", src)
        return int(m[1]), int(m[2])

    sets, stages, most, least, step = map(pair, ("kSets", "kStages", "kMaxRaw", "kMinRaw", "kRawStep"))
    return [(stages[i], raw, sets[i]) for i in range(2) for raw in range(most[i], least[i] - 1, -step[i])]


@pytest.mark.parametrize("stages,raw,sets", shapes())
def test_every_role_finds_its_block(stages, raw, sets):
    for seed in range(40):
        run(stages, raw, sets, raw_blocks=3 + seed, seed=seed)


def test_the_model_finds_stages_that_the_sets_do_not_divide():
    """A set keeps to stages of its own, so their number is a multiple of the
    sets': three sets on four stages write over one another's blocks."""
    with pytest.raises(AssertionError):
        for seed in range(40):
            run(4, 6, 3, raw_blocks=3 + seed, seed=seed)

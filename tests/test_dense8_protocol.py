"""Model check of the weight gradient kernel's mbarrier hand-offs on the CPU: every role as a coroutine over
mbarriers with the hardware's parity semantics, run in random order. A wait that its parity lets through although
the phase it means is not the last completed one (a role two phases away from another), an arrival that a phase has
no room for, a place of a ring or an accumulator that is overwritten while it is in use, or a run in which nobody
can go on is an error."""
from __future__ import annotations

import random
import re
from pathlib import Path

import pytest

SOURCE = Path(__file__).resolve().parent.parent / "tcc_spmm_b200" / "csrc" / "weight_grad.cu"


class Bar:
    def __init__(self, name, count):
        self.name, self.count, self.pending, self.done = name, count, count, 0

    def arrive(self):
        assert self.pending > 0, f"{self.name}: arrival beyond the phase's count"
        self.pending -= 1
        if self.pending == 0:
            self.done, self.pending = self.done + 1, self.count

    def ready(self, phase):
        """Whether try_wait.parity(phase & 1) passes; `phase` is the phase that the waiter means (-1: before the first)."""
        passes = (self.done & 1) != (phase & 1)
        if passes:
            assert self.done - 1 == phase, f"{self.name}: a wait for phase {phase} passed after {self.done} phases"
        return passes


def simulate(cg, raw, ring, flush, stages, seed):
    rng = random.Random(seed)
    pending = []  # asynchronous completions: per queue in order ("mma"), or free (copies)
    raw_full = [[Bar(f"rawFull{c}.{i}", 2) for i in range(raw)] for c in range(cg)]
    raw_empty = [[Bar(f"rawEmpty{c}.{i}", 2) for i in range(raw)] for c in range(cg)]   # one per set of warps: A, B
    full = [[Bar(f"full{c}.{i}", 2) for i in range(ring)] for c in range(cg)]
    empty = [[Bar(f"empty{c}.{i}", 1) for i in range(ring)] for c in range(cg)]
    peer_full = [Bar(f"peerFull.{i}", 1) for i in range(ring)]
    acc_full = [Bar(f"accFull{c}", 1) for c in range(cg)]
    acc_empty = Bar("accEmpty", 2 * cg)  # the warps of either half of the columns
    raw_data = [[[None, None] for _ in range(raw)] for _ in range(cg)]  # stage in the place: copy, scales
    op_data = [[[None, None] for _ in range(ring)] for _ in range(cg)]  # stage in the place: A, B
    acc_use, acc_seen = [0] * cg, [0] * cg                              # sums since the last read, and reads
    read = [[0] * cg for _ in range(2)]
    finished = []

    def tma(c):
        for x in range(stages):
            s = x % raw
            while not raw_empty[c][s].ready(x // raw - 1):
                yield
            pending.append(("copy", c, x))
            yield
        finished.append("tma")

    def scales(c, w):
        for x in range(w, stages, 2):
            s = x % raw
            while not raw_empty[c][s].ready(x // raw - 1):
                yield
            raw_data[c][s][1] = x
            raw_full[c][s].arrive()
            yield
        finished.append("scales")

    def convert(c, kind, w):
        for x in range(w, stages, 2):
            s, o = x % raw, x % ring
            while not raw_full[c][s].ready(x // raw):
                yield
            while not empty[c][o].ready(x // ring - 1):
                yield
            assert raw_data[c][s] == [x, x], f"stage {x} reads {raw_data[c][s]}"
            yield
            assert raw_data[c][s] == [x, x], f"stage {x} overwritten"
            op_data[c][o][kind] = x
            raw_empty[c][s].arrive()
            yield
            full[c][o].arrive()
        finished.append("convert")

    def forward():
        for x in range(stages):
            while not full[1][x % ring].ready(x // ring):
                yield
            peer_full[x % ring].arrive()
            yield
        finished.append("forward")

    def mma():
        flushes = 0
        for x in range(stages):
            while not full[0][x % ring].ready(x // ring):
                yield
            while cg == 2 and not peer_full[x % ring].ready(x // ring):
                yield
            if x % flush == 0 and flushes:
                while not acc_empty.ready(flushes - 1):
                    yield
            pending.append(("mma", x, None))
            pending.append(("empty", x % ring, x))
            if (x + 1) % flush == 0 or x + 1 == stages:
                pending.append(("accFull", None, None))
                flushes += 1
            yield
        finished.append("mma")

    def epilogue(c, h):
        for e in range(-(-stages // flush)):
            while not acc_full[c].ready(e):
                yield
            taken = acc_use[c]
            yield
            assert acc_use[c] == taken, "an accumulator grew while it was read"
            read[h][c] += taken
            acc_seen[c] += 1
            if acc_seen[c] % 2 == 0:  # both halves' warps have read it
                acc_use[c] = 0
            acc_empty.arrive()
            yield
        finished.append("epilogue")

    def complete():
        """One asynchronous completion: any copy, or the oldest tensor-core operation."""
        ops = [i for i, p in enumerate(pending) if p[0] == "copy"]
        first = next((i for i, p in enumerate(pending) if p[0] != "copy"), None)
        if first is not None:
            ops.append(first)
        kind, a, b = pending.pop(rng.choice(ops))
        if kind == "copy":
            raw_data[a][b % raw][0] = b
            raw_full[a][b % raw].arrive()
        elif kind == "mma":
            for c in range(cg):
                assert op_data[c][a % ring] == [a, a], f"MMA of stage {a} reads {op_data[c][a % ring]}"
                acc_use[c] += 1
        elif kind == "empty":
            for c in range(cg):
                empty[c][a].arrive()
        else:
            for c in range(cg):
                acc_full[c].arrive()

    roles = [mma()]
    for c in range(cg):
        roles += [tma(c), scales(c, 0), scales(c, 1), *(convert(c, k, w) for k in (0, 1) for w in (0, 1)),
                  epilogue(c, 0), epilogue(c, 1)]
    if cg == 2:
        roles.append(forward())
    speed = [rng.choice((1, 1, 4, 16)) for _ in roles]
    idle = 0
    while roles or pending:
        assert idle < 20000, f"nobody can go on; finished {finished}"
        i = rng.randrange(len(roles) + 1) if roles else 0
        idle += 1
        if i == len(roles):
            if pending and rng.random() < 0.5:
                complete()
                idle = 0
            continue
        if rng.random() > 1 / speed[i]:
            continue
        before = (len(pending), len(finished))
        try:
            next(roles[i])
        except StopIteration:
            roles.pop(i), speed.pop(i)
            idle = 0
        if before != (len(pending), len(finished)):
            idle = 0
    assert all(read[h][c] == stages for h in range(2) for c in range(cg))


# (CTAs, raw ring, operand ring, stages per flush) of the kernel's configurations
CONFIGS = [(1, 6, 6, 30), (2, 4, 6, 15), (1, 6, 6, 15), (2, 6, 4, 7), (1, 6, 4, 10), (2, 8, 4, 10)]


@pytest.mark.parametrize("config", CONFIGS)
def test_hand_offs(config):
    for seed in range(12):
        for stages in (1, 2, 3, 7, 31, 64):
            simulate(*config, stages, 100 * seed + stages)


def test_odd_rings_are_caught():
    """A set of warps on an odd ring can be two phases ahead of the other's: the model finds it."""
    with pytest.raises(AssertionError):
        for seed in range(200):
            simulate(1, 3, 4, 14, 40, seed)


def test_rings_in_the_source():
    """The configurations above are the kernel's: its rings are even and these."""
    text = SOURCE.read_text()
    assert 'static_assert(kRaw % 2 == 0 && kStages % 2 == 0, "even rings");' in text
    assert re.search(r"kRaw = kP == 3 \? \(CG == 1 \? 6 : 8\) : CG == 1 \|\| kP == 2 \? 6 : 4;", text)
    assert re.search(r"kStages = kP == 3 \|\| \(kP == 2 && CG == 2\) \? 4 : 6;", text)

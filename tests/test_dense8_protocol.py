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


def simulate(cg, raw, ring, turn, flush, stages, seed):
    rng = random.Random(seed)
    pending = []  # asynchronous completions: per queue in order ("mma"), or free (copies)
    raw_full = [[Bar(f"rawFull{c}.{i}", 2) for i in range(raw)] for c in range(cg)]
    raw_empty = [[Bar(f"rawEmpty{c}.{i}", 2) for i in range(raw)] for c in range(cg)]   # one per set of warps: A, B
    full = [[Bar(f"full{c}.{i}", 2) for i in range(ring)] for c in range(cg)]
    empty = [[Bar(f"empty{c}.{i}", 1) for i in range(ring)] for c in range(cg)]
    peer_full = [Bar(f"peerFull.{i}", 1) for i in range(ring)]
    acc_full = [[Bar(f"accFull{c}.{h}", 1) for h in range(2)] for c in range(cg)]
    acc_empty = [Bar(f"accEmpty.{h}", cg) for h in range(2)]
    raw_data = [[[None, None] for _ in range(raw)] for _ in range(cg)]  # stage in the place: copy, scales
    op_data = [[[None, None] for _ in range(ring)] for _ in range(cg)]  # stage in the place: A, B
    acc_use = [[0] * cg for _ in range(2)]                              # sums since the last read, per half
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
        nxt, end, until = [0, 0], [turn // 2, turn], [turn // 2 + flush, flush]
        drained, flushes, seen = [None, None], [0, 0], 0
        while nxt[0] < stages or nxt[1] < stages:
            for h in range(2):
                if drained[h] is not None and nxt[h] < stages:
                    while not acc_empty[h].ready(drained[h]):
                        yield
                    drained[h] = None
                while nxt[h] < min(end[h], stages):
                    x = nxt[h]
                    if x == seen:
                        while not full[0][x % ring].ready(x // ring):
                            yield
                        while cg == 2 and not peer_full[x % ring].ready(x // ring):
                            yield
                        seen += 1
                    pending.append(("mma", h, x))
                    if nxt[1 - h] > x:
                        pending.append(("empty", x % ring, x))
                    nxt[h] += 1
                    until[h] -= 1
                    if until[h] == 0 or nxt[h] == stages:
                        pending.append(("accFull", h, flushes[h]))
                        until[h], drained[h] = flush, flushes[h]
                        flushes[h] += 1
                    yield
                end[h] += turn
        finished.append("mma")

    def epilogue(c, h):
        offset = turn // 2 if h == 0 else 0
        count = 1 + ((stages - 1 - offset) // flush if stages - 1 > offset else 0)
        for e in range(count):
            while not acc_full[c][h].ready(e):
                yield
            taken = acc_use[h][c]
            yield
            assert acc_use[h][c] == taken, "an accumulator grew while it was read"
            read[h][c] += taken
            acc_use[h][c] = 0
            acc_empty[h].arrive()
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
                assert op_data[c][b % ring] == [b, b], f"MMA of stage {b} reads {op_data[c][b % ring]}"
                acc_use[a][c] += 1
        elif kind == "empty":
            for c in range(cg):
                empty[c][a].arrive()
        else:
            for c in range(cg):
                acc_full[c][a].arrive()

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


# (CTAs, raw ring, operand ring, stages per turn, stages per flush) of the kernel's configurations
CONFIGS = [(1, 6, 6, 4, 28), (2, 4, 6, 4, 12), (1, 6, 6, 4, 12), (2, 6, 4, 2, 6), (1, 6, 4, 2, 10), (2, 8, 4, 2, 10)]


@pytest.mark.parametrize("config", CONFIGS)
def test_hand_offs(config):
    for seed in range(12):
        for stages in (1, 2, 3, 7, 31, 64):
            simulate(*config, stages, 100 * seed + stages)


def test_odd_rings_are_caught():
    """A set of warps on an odd ring can be two phases ahead of the other's: the model finds it."""
    with pytest.raises(AssertionError):
        for seed in range(200):
            simulate(1, 3, 4, 2, 14, 40, seed)


def test_rings_in_the_source():
    """The configurations above are the kernel's: its rings are even and these."""
    text = SOURCE.read_text()
    assert 'static_assert(kRaw % 2 == 0 && kStages % 2 == 0, "even rings");' in text
    assert re.search(r"kRaw = kP == 3 \? \(CG == 1 \? 6 : 8\) : CG == 1 \|\| kP == 2 \? 6 : 4;", text)
    assert re.search(r"kStages = kP == 3 \|\| \(kP == 2 && CG == 2\) \? 4 : 6;", text)

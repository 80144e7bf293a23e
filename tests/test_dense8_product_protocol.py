"""Model check of the tensor-core product's mbarrier hand-offs on the CPU, as for the weight gradient's: every role as
a coroutine over mbarriers with the hardware's parity semantics, run in random order. Copies complete in any order,
tensor-core operations in theirs."""
from __future__ import annotations

import random
import re

import pytest

from tests.test_dense8_protocol import SOURCE, Bar

PRODUCT = SOURCE.parent / "matmul_fp8.cu"


def simulate(cg, ring, accs, slots, scale_warps, tiles, first, last, per_pass, seed):
    """tiles of blocks [first, last) of k (first a multiple of 4), an accumulator for every `per_pass` blocks."""
    rng = random.Random(seed)
    blocks = last - first
    groups, passes = -(-blocks // 4), -(-blocks // per_pass)
    full = [[Bar(f"full{c}.{i}", 1) for i in range(ring)] for c in range(cg)]
    empty = [[Bar(f"empty{c}.{i}", 1) for i in range(ring)] for c in range(cg)]
    peer = [Bar(f"peerFull.{i}", 1) for i in range(ring)]
    scale_full = [[Bar(f"scaleFull{c}.{i}", 1) for i in range(slots)] for c in range(cg)]
    scale_empty = [[Bar(f"scaleEmpty{c}.{i}", 1) for i in range(slots)] for c in range(cg)]
    acc_full = [[Bar(f"accFull{c}.{i}", 1) for i in range(accs)] for c in range(cg)]
    acc_empty = [Bar(f"accEmpty.{i}", 2 * cg) for i in range(accs)]  # two of the epilogue's warps stand for eight
    stage = [[None] * ring for _ in range(cg)]
    slot_data = [[None] * slots for _ in range(cg)]
    acc = [dict(use=None, count=0, readers=2 * cg) for _ in range(accs)]
    queue, flying = [], []

    def tma(c):
        it = 0
        for t in range(tiles):
            for kb in range(first, last):
                s = it % ring
                while not empty[c][s].ready(it // ring - 1):
                    yield
                flying.append((c, s, (t, kb)))
                it += 1
                yield

    def scales(c, w):
        for i in range(w, tiles * groups, scale_warps):
            s = i % slots
            while not scale_empty[c][s].ready(i // slots - 1):
                yield
            slot_data[c][s] = divmod(i, groups)
            yield
            scale_full[c][s].arrive()
            yield

    def forward():
        it = slot = 0
        for _ in range(tiles):
            for kb in range(blocks):
                if kb % 4 == 0:
                    while not scale_full[1][slot % slots].ready(slot // slots):
                        yield
                while not full[1][it % ring].ready(it // ring):
                    yield
                peer[it % ring].arrive()
                it += 1
                if kb % 4 == 3 or kb + 1 == blocks:
                    slot += 1
                yield

    def mma():
        it = slot = a = 0
        for t in range(tiles):
            for kb in range(first, last):
                fresh = (kb - first) % per_pass == 0
                if fresh:
                    while not acc_empty[a % accs].ready(a // accs - 1):
                        yield
                if kb % 4 == 0:
                    while not scale_full[0][slot % slots].ready(slot // slots):
                        yield
                while not full[0][it % ring].ready(it // ring):
                    yield
                while cg == 2 and not peer[it % ring].ready(it // ring):
                    yield
                if kb % 4 == 0:
                    queue.append(("scales", slot % slots, (t, (kb - first) // 4)))
                queue.append(("mma", it % ring, (t, kb), a % accs, fresh))
                queue.append(("commit", empty, it % ring))
                it += 1
                if kb % 4 == 3 or kb + 1 == last:
                    queue.append(("commit", scale_empty, slot % slots))
                    slot += 1
                if (kb - first + 1) % per_pass == 0 or kb + 1 == last:
                    queue.append(("commit", acc_full, a % accs))
                    a += 1
                yield

    def epilogue(c):
        for use in range(tiles * passes):
            a = use % accs
            while not acc_full[c][a].ready(use // accs):
                yield
            want = min(per_pass, blocks - use % passes * per_pass)
            for _ in range(2):
                assert acc[a]["use"] == use and acc[a]["count"] == want, f"pass {use} reads {acc[a]}"
                yield
            acc[a]["readers"] += 1
            acc_empty[a].arrive()
            yield

    uses = iter(range(tiles * passes))

    def complete():
        n = len(flying) + bool(queue)
        i = rng.randrange(n)
        if i < len(flying):
            c, s, what = flying.pop(i)
            stage[c][s] = what
            full[c][s].arrive()
            return
        op = queue.pop(0)
        if op[0] == "scales":
            assert all(slot_data[c][op[1]] == op[2] for c in range(cg)), f"scales of {op[2]}: {slot_data}"
        elif op[0] == "mma":
            _, s, what, a, fresh = op
            assert all(stage[c][s] == what for c in range(cg)), f"MMA of {what} reads {[x[s] for x in stage]}"
            if fresh:
                assert acc[a]["readers"] == 2 * cg, "an accumulator is overwritten before it was read"
                acc[a].update(use=next(uses), count=0, readers=0)
            acc[a]["count"] += 1
        else:
            for c in range(cg):
                op[1][c][op[2]].arrive()

    roles = [mma()]
    for c in range(cg):
        roles += [tma(c), epilogue(c), epilogue(c), *(scales(c, w) for w in range(scale_warps))]
    if cg == 2:
        roles.append(forward())
    speed = [rng.choice((1, 1, 4, 16)) for _ in roles]
    idle = 0
    while roles or queue or flying:
        assert idle < 20000, "nobody can go on"
        idle += 1
        i = rng.randrange(len(roles) + 1)
        if i == len(roles):
            if (queue or flying) and rng.random() < 0.7:
                complete()
                idle = 0
        elif rng.random() <= 1 / speed[i]:
            try:
                next(roles[i])
            except StopIteration:
                roles.pop(i), speed.pop(i)
                idle = 0
    assert next(uses, None) is None


# (CTAs, stages, accumulators, scale slots, scale warps) of the kernel's tiles: 256, 128, 64 and 32 columns
CONFIGS = [(2, 5, 1, 6, 2), (1, 5, 1, 6, 2), (1, 4, 2, 6, 3), (1, 6, 2, 6, 3)]


@pytest.mark.parametrize("config", CONFIGS)
@pytest.mark.parametrize("first,last,per_pass", [(0, 1, 1), (0, 2, 2), (0, 5, 5), (0, 9, 9), (0, 33, 16), (0, 16, 16), (4, 9, 5), (8, 41, 16)])
def test_hand_offs(config, first, last, per_pass):
    for seed in range(8):
        for tiles in (1, 2, 5):
            simulate(*config, tiles, first, last, per_pass, 100 * seed + tiles)


def test_unshared_slots_are_caught():
    """Scale warps that take slots in turn need the number of slots to be a multiple of theirs: otherwise a slot's
    phases belong to different warps, and one can be two phases ahead of the other."""
    with pytest.raises(AssertionError):
        for seed in range(300):
            simulate(1, 6, 2, 2, 3, 12, 0, 4, 4, seed)


def test_configurations_in_the_source():
    text = PRODUCT.read_text()
    for line in (r"kStages = BN == 256 \? 5 : BN == 128 \? 4 : 6;", r"kAcc = BN == 256 \? 1 : 2;", r"kSlots = 6;",
                 r"kScaleWarps = BN == 256 \? 2 : 3;", r"kPass = 16;", r"static_assert\(kSlots % kScaleWarps == 0,"):
        assert re.search(line, text), line

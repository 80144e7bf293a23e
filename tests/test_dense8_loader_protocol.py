"""Model check of the weight gradient's loader for rows off 16 bytes: three warps fill a raw stage by asynchronous
copies and by ordinary stores. An arrival that waits for copies says nothing about the thread's stores; only an
arrival after them does. Stores that no such arrival follows become visible at any later time here."""
from __future__ import annotations

import random
import re

import pytest

from tests.test_dense8_protocol import SOURCE, Bar

WARPS = 3


def simulate(ring, stages, seed, copies=True, released=True):
    """copies: the warps use asynchronous copies at all (rows on 4 bytes do). released: they arrive after their
    ordinary stores."""
    rng = random.Random(seed)
    full = [Bar(f"rawFull.{i}", WARPS * (2 if released else 1)) for i in range(ring)]
    empty = [Bar(f"rawEmpty.{i}", 2) for i in range(ring)]  # the readers of dy and of q
    copied = [[None] * WARPS for _ in range(ring)]
    stored = [[None] * WARPS for _ in range(ring)]
    flying, hidden = [], []  # copies on their way, stores that nobody else sees yet

    def show(w):
        """Warp w's stores become visible, in their order."""
        for item in [h for h in hidden if h[0] == w]:
            hidden.remove(item)
            stored[item[1]][w] = item[2]

    def loader(w):
        for x in range(stages):
            s = x % ring
            while not empty[s].ready(x // ring - 1):
                yield
            hidden.append((w, s, x))
            if copies:
                flying.append((w, s, x))
            else:
                full[s].arrive()
            yield
            if released:
                show(w)
                full[s].arrive()
                yield

    def reader(set_, kind):
        for x in range(set_, stages, 2):
            s = x % ring
            while not full[s].ready(x // ring):
                yield
            for _ in range(2):
                assert stored[s] == [x] * WARPS, f"stage {x} reads stores of {stored[s]}"
                assert not copies or copied[s] == [x] * WARPS, f"stage {x} reads copies of {copied[s]}"
                yield
            empty[s].arrive()
            yield

    roles = [loader(w) for w in range(WARPS)] + [reader(i, kind) for i in range(2) for kind in range(2)]
    idle = 0
    while roles:
        assert idle < 20000, "nobody can go on"
        idle += 1
        i = rng.randrange(len(roles) + 2)
        if i == len(roles):
            if flying:
                w, s, x = flying.pop(rng.randrange(len(flying)))
                copied[s][w] = x
                full[s].arrive()
                idle = 0
        elif i == len(roles) + 1:
            if hidden and rng.random() < 0.2:
                show(rng.choice(hidden)[0])
        else:
            try:
                next(roles[i])
            except StopIteration:
                roles.pop(i)
                idle = 0


@pytest.mark.parametrize("copies", [True, False])
@pytest.mark.parametrize("ring", [4, 6, 8])
def test_loader_publishes_its_stores(ring, copies):
    for seed in range(20):
        for stages in (1, 2, 7, 33):
            simulate(ring, stages, 100 * seed + stages, copies)


@pytest.mark.parametrize("copies", [True, False])
def test_arrivals_of_copies_alone_are_caught(copies):
    with pytest.raises(AssertionError, match="reads stores"):
        for seed in range(50):
            simulate(6, 20, seed, copies, released=False)


def test_arrivals_in_the_source():
    """The loader arrives after its stores, and the barrier counts the copies' arrivals and these."""
    text = SOURCE.read_text()
    assert "mbarInit(rawFull + 8 * i, TMA ? 2 : 3 * (32 + 1))" in text
    loader = text[text.index("void loadRaw("):text.index("gradTiles(")]
    stores = loader.index("stsU32(scales")
    assert re.search(r"cpAsyncArriveNoinc\(rawFull \+ 8 \* raw\);\s*__syncwarp\(\);\s*if \(lane == 0\)\s*"
                     r"dev::mbarArrive\(rawFull \+ 8 \* raw\);", loader[stores:])

"""CPU model of the attention kernel's warps, restated from rope_attend.cu: the
rings of K and V, Q, the TMEM columns that S and P share, O, and every barrier
with the parity that each wait uses.  Warps, copies and products run in random
order.  No wait may take an older phase of its barrier for its own, and nothing
may be read before it is there or overwritten while it is in use.  The sizes are
read from the source, so that the model cannot fall behind them."""

from __future__ import annotations

import random
import re
from pathlib import Path

import pytest

from test_attend_plan import COST
from testfiles_b200 import build

SOURCE = (Path(build.CSRC) / "rope_attend.cu").read_text()


def constant(name):
    return int(re.search(rf"\b{name} = (\d+)", SOURCE)[1])


STAGES_K, STAGES_V, PIECES = constant("kStagesK"), constant("kStagesV"), constant("kPieces")
WARPS = constant("kSoftmaxWarps")


def columns(name):
    """First TMEM column of S or P of a tile by its number modulo three."""
    a, b, c = re.search(rf"{name}\(uint32_t third\) {{ return third == 0 \? (\d+) : third == 1 \? (\d+) : (\d+);",
                        SOURCE).groups()
    return [int(a), int(b), int(c)]


COL_S, COL_P = columns("col_s"), columns("col_p")


class Barrier:
    def __init__(self, count):
        self.count = self.pending = count
        self.tx = self.done = 0  # bytes to come; phases that are over

    def arrive(self, tx=0):
        self.pending -= 1
        self.tx += tx
        assert self.pending >= 0
        self.settle()

    def land(self):
        self.tx -= 1
        self.settle()

    def settle(self):
        if self.pending == 0 and self.tx == 0:
            self.done += 1
            self.pending = self.count

    def over(self, phase):
        """What a parity wait for `phase` (-1: the one before the first) answers."""
        if (self.done - 1) & 1 != phase & 1:
            return False
        assert self.done > phase, "took an older phase for its own"
        return True


class Cta:
    """pieces: (tiles, warps of 32 rows, {tile: halves of V whose rows behind the keys are cleared})."""

    def __init__(self, pieces, rng, without=()):
        self.pieces, self.rng, self.without = pieces, rng, without
        bars = lambda n, count: [Barrier(count) for _ in range(n)]  # noqa: E731
        self.full_k, self.empty_k = bars(STAGES_K, 1), bars(STAGES_K, 1)
        self.full_v, self.empty_v = bars(STAGES_V, 1), bars(STAGES_V, 1)
        self.s_full, self.s_read = bars(2, 1), bars(2, WARPS)
        self.p_full, self.pv_done = bars(4, WARPS), bars(4, 1)
        self.q_first, self.q_full, self.q_empty = Barrier(WARPS), Barrier(1), Barrier(1)
        self.o_free, self.swap = Barrier(WARPS), bars(4, 2)
        self.piece_full, self.piece_empty = bars(PIECES, 1), bars(PIECES, 3 + WARPS)
        # what is where
        self.k, self.v = [None] * STAGES_K, [None] * STAGES_V     # entry that has landed
        self.k_used, self.v_used = [0] * STAGES_K, [0] * STAGES_V  # products that read the stage now
        self.cleared = {}                                         # V entry -> warps that cleared it
        self.q = {}                                               # piece -> shares of its rows that have landed
        self.q_used = 0
        # of 64 columns, and of the lanes of each two warps' 32 rows: ("S", tile) or ("P", tile)
        self.column = [[None] * 4 for _ in range(4)]
        self.writing = [0] * 4                                    # products that write S there now
        self.p_used = [0] * 4                                     # products that read P there now
        self.s_halves = {}                                        # (tile, warp of 32 rows) -> halves read
        self.p_written = {}                                       # tile -> warps
        self.o_tile, self.o_used, self.o_readers = -1, 0, 0
        self.copies = []                                          # in flight, in any order
        self.products = {"scores": [], "values": []}              # in flight, in the order of issue
        self.starts = [sum(p[0] for p in pieces[:i]) for i in range(len(pieces))]

    # --- warps, as generators of (barrier, phase) waits -------------------------------------------------------
    def read_piece(self, n):
        yield self.piece_full[n % PIECES], n // PIECES
        assert self.piece[n % PIECES] == n
        self.piece_empty[n % PIECES].arrive()

    def lister(self):
        self.piece = [None] * PIECES
        for n in range(len(self.pieces) + 1):
            yield self.piece_empty[n % PIECES], n // PIECES - 1
            self.piece[n % PIECES] = n
            self.piece_full[n % PIECES].arrive()
            if 0 < n < len(self.pieces):
                yield self.q_empty, n - 1
                assert self.q_used == 0, "Q rows overwritten while products read them"
                self.q = {n: 0}
                self.copies.append(lambda n=n: (self.q.update({n: WARPS}), self.q_full.arrive()))

    def producer(self):
        nk = nv = 0
        for n, (tiles, _, _) in enumerate(self.pieces):
            yield from self.read_piece(n)
            for j in range(tiles + 1):
                for half in range(2) if j < tiles else ():
                    s = nk % STAGES_K
                    yield self.empty_k[s], nk // STAGES_K - 1
                    assert self.k_used[s] == 0, "K stage overwritten while products read it"
                    self.k[s] = None
                    self.full_k[s].arrive(tx=1)
                    self.copies.append(lambda s=s, e=nk: (self.k.__setitem__(s, e), self.full_k[s].land()))
                    nk += 1
                for half in range(2) if j > 0 else ():
                    s = nv % STAGES_V
                    yield self.empty_v[s], nv // STAGES_V - 1
                    assert self.v_used[s] == 0, "V stage overwritten while products read it"
                    self.v[s] = None
                    self.full_v[s].arrive(tx=1)
                    self.copies.append(lambda s=s, e=nv: (self.v.__setitem__(s, e), self.full_v[s].land()))
                    nv += 1
        yield from self.read_piece(len(self.pieces))

    def scores(self):
        t = n = 0
        fifo = self.products["scores"]
        for np, (tiles, _, _) in enumerate(self.pieces):
            yield from self.read_piece(np)
            for j in range(tiles):
                third = t % 3
                mine = [COL_S[third] // 64, COL_S[third] // 64 + 1]
                if j == 0:
                    yield (self.q_first, 0) if np == 0 else (self.q_full, np - 1)
                for half in range(2):
                    s = n % STAGES_K
                    yield self.full_k[s], n // STAGES_K
                    if half == 0:
                        used = t - (2 if third == 1 else 3)
                        if third < 2 and t >= 3 and "columns" not in self.without:
                            yield self.pv_done[used & 3], used >> 2
                        if third != 1 and t >= 2:
                            yield self.s_read[(t - 1) & 1], (t - 1) >> 1
                        for c in mine:
                            for warp, held in enumerate(self.column[c]):
                                if held is None:
                                    continue
                                kind, old = held
                                if kind == "P":
                                    assert old in self.pv_over, "P overwritten before it was used"
                                elif warp < self.busy_of(old):
                                    assert c - COL_S[old % 3] // 64 in self.s_halves.get((old, warp), ()), \
                                        "S overwritten before it was read"
                            assert self.p_used[c] == 0
                            self.column[c] = [("S", t)] * 4
                    assert self.k[s] == n, "K read before it was there"
                    assert self.q.get(np) == WARPS, "Q read before it was there"
                    self.k_used[s] += 1
                    self.q_used += 1
                    for c in mine:
                        self.writing[c] += 1

                    def done(s=s, n=n, mine=tuple(mine), np=np):
                        assert self.k[s] == n and np in self.q
                        self.k_used[s] -= 1
                        self.q_used -= 1
                        for c in mine:
                            self.writing[c] -= 1

                    fifo.append(done)
                    if half == 1:
                        fifo.append(self.s_full[t & 1].arrive)
                    fifo.append(self.empty_k[s].arrive)
                    if half == 1 and j == tiles - 1:
                        fifo.append(self.q_empty.arrive)
                    n += 1
                t += 1
        yield from self.read_piece(len(self.pieces))

    def busy_of(self, t):
        return next(p[1] for p, first in zip(self.pieces, self.starts) if first <= t < first + p[0])

    def values(self):
        t = n = 0
        fifo = self.products["values"]
        for np, (tiles, busy, clears) in enumerate(self.pieces):
            yield from self.read_piece(np)
            for j in range(tiles):
                at = COL_P[t % 3] // 64
                for half in range(2):
                    s = n % STAGES_V
                    yield self.full_v[s], n // STAGES_V
                    if half == 0:
                        if j == 0:
                            yield self.o_free, np - 1
                            assert self.o_readers == 0, "O overwritten before it was read"
                        yield self.p_full[t & 3], t >> 2
                        assert self.p_written.get(t, 0) == 2 * busy, "P read before it was there"
                    assert self.column[at][:busy] == [("P", t)] * busy and self.writing[at] == 0
                    assert self.v[s] == n, "V read before it was there"
                    assert half not in clears.get(j, ()) or self.cleared.get(n) == 4, "V read before it was cleared"
                    self.v_used[s] += 1
                    self.p_used[at] += 1
                    self.o_used += 1
                    if half == 1 and j == tiles - 1:
                        self.o_readers = 2 * busy

                    def done(s=s, n=n, at=at, t=t, half=half, busy=busy):
                        assert self.v[s] == n and self.column[at][:busy] == [("P", t)] * busy
                        self.v_used[s] -= 1
                        self.p_used[at] -= 1
                        self.o_used -= 1
                        if half == 1:
                            self.pv_over.add(t)
                            self.o_tile = t

                    fifo.append(done)
                    if half == 1:
                        fifo.append(self.pv_done[t & 3].arrive)
                    fifo.append(self.empty_v[s].arrive)
                    n += 1
                t += 1
        yield from self.read_piece(len(self.pieces))

    def softmax(self, index):
        warp, half = index & 3, index >> 2
        swaps = t = 0
        for np, (tiles, rows, clears) in enumerate(self.pieces):
            yield from self.read_piece(np)
            if np == 0:
                self.copies.append(lambda: (self.q.update({0: self.q.get(0, 0) + 1}), self.q_first.arrive()))
            busy = warp < rows
            for j in range(tiles):
                yield self.s_full[t & 1], t >> 1
                if busy:
                    c = COL_S[t % 3] // 64 + half
                    assert self.column[c][warp] == ("S", t) and self.writing[c] == 0, "S read before it was there"
                    self.s_halves.setdefault((t, warp), set()).add(half)
                self.s_read[t & 1].arrive()
                if busy:
                    self.swap[warp].arrive()
                    yield self.swap[warp], swaps
                    swaps += 1
                    if j > 0 and self.rng.random() < 0.3:  # rescale
                        yield self.pv_done[(t - 1) & 3], (t - 1) >> 2
                        assert self.o_tile == t - 1 and self.o_used == 0, "O rescaled while products add to it"
                    at = COL_P[t % 3] // 64
                    assert len(self.s_halves[t, warp]) == 2, "P written over S that was not read"
                    assert self.column[at][warp] in (("S", t), ("P", t)) and self.writing[at] == 0
                    self.column[at][warp] = ("P", t)
                    self.p_written[t] = self.p_written.get(t, 0) + 1
                if half in clears.get(j, ()):
                    if t > 0 and "clear" not in self.without:
                        yield self.pv_done[(t - 1) & 3], (t - 1) >> 2
                    n = 2 * t + half
                    yield self.full_v[n % STAGES_V], n // STAGES_V
                    assert self.v[n % STAGES_V] == n, "V cleared before it was there"
                    assert self.v_used[n % STAGES_V] == 0
                    self.cleared[n] = self.cleared.get(n, 0) + 1
                self.p_full[t & 3].arrive()
                t += 1
            yield self.pv_done[(t - 1) & 3], (t - 1) >> 2
            assert self.o_tile == t - 1 and self.o_used == 0, "O read before it was there"
            if busy:
                self.swap[warp].arrive()
                yield self.swap[warp], swaps
                swaps += 1
                self.o_readers -= 1
            self.o_free.arrive()
        yield from self.read_piece(len(self.pieces))

    def run(self):
        self.pv_over = set()
        agents = [self.lister(), self.producer(), self.scores(), self.values(), *map(self.softmax, range(WARPS))]
        waits = {a: None for a in agents}
        # some of all that runs is slow this time
        speed = {a: self.rng.choice([1, 1, 1, 0.05]) for a in agents}
        pace = {x: self.rng.choice([1, 1, 0.05]) for x in ("copies", "scores", "values")}
        idle = 0
        while waits or self.copies or any(self.products.values()):
            moved = False
            for a in self.rng.sample(list(waits), len(waits)):
                if self.rng.random() > speed[a]:
                    moved = True  # it may yet
                    continue
                if waits[a] is not None and not waits[a][0].over(waits[a][1]):
                    continue
                moved = True
                try:
                    waits[a] = next(a)
                except StopIteration:
                    del waits[a]
            if self.copies:
                moved = True
                if self.rng.random() < pace["copies"]:
                    self.copies.pop(self.rng.randrange(len(self.copies)))()
            for name, fifo in self.products.items():
                if fifo:
                    moved = True
                    if self.rng.random() < pace[name]:
                        fifo.pop(0)()
            idle = 0 if moved else idle + 1
            assert idle < 2, "nothing can go on"


def random_pieces(rng):
    pieces = []
    for _ in range(rng.randint(1, 7)):
        tiles = rng.choice([1, 1, 2, 3, 4, rng.randint(1, 9)])
        clears = {}
        for j in {tiles - 1, rng.randrange(tiles)}:  # the last tile, and the prefix's last one inside the piece
            if rng.random() < 0.7:
                clears[j] = rng.choice([(1,), (0, 1)])
        pieces.append((tiles, rng.randint(1, 4), clears))
    return pieces


def test_sizes_of_the_source():
    assert (STAGES_K, STAGES_V, PIECES, WARPS) == (3, 2, 4, 8)
    assert constant("kItemCost") == COST
    assert "kPieceReaders = 3 + kSoftmaxWarps" in SOURCE
    for name, count in (("s_read", "kSoftmaxWarps"), ("p_full", "kSoftmaxWarps"), ("o_free", "kSoftmaxWarps"),
                        ("pv_done", "1"), ("s_full", "1"), ("swap", "2"), ("q_empty", "1"), ("full_k", "1"),
                        ("full_v", "1"), ("empty_k", "1"), ("empty_v", "1")):
        assert re.search(rf"mbar_init\(&ctl\.{name}(\[\w\])?, {count}\)", SOURCE), name


@pytest.mark.parametrize("seed", range(8))
def test_every_wait_is_for_its_own_phase_and_nothing_is_used_too_early(seed):
    rng = random.Random(seed)
    for _ in range(60):
        Cta(random_pieces(rng), rng).run()


@pytest.mark.parametrize("without", ["clear", "columns"])
def test_the_model_finds_waits_that_are_missing(without):
    """The softmax warps' wait before they look at V, and that of the scores for their columns."""
    rng = random.Random(1)
    with pytest.raises(AssertionError):
        for _ in range(300):
            Cta(random_pieces(rng), rng, without=(without,)).run()

"""CPU checks of the attention kernels' work division, restated from
rope_attend.cu: the pieces that the CTAs list cover every 128-key tile of every
item once, every workspace index lies inside its array, and the join kernel
finds exactly the pieces that hold a row's partial results."""

from __future__ import annotations

import random

import pytest

ROWS = KEYS = 128
COST = 2  # kItemCost


def div_up(a, b):
    return (a + b - 1) // b


class Plan:
    def __init__(self, counts, lens, prefix, q_heads, k_heads, grid):
        self.counts, self.lens, self.prefix = counts, lens, prefix
        self.q_heads, self.k_heads, self.group = q_heads, k_heads, q_heads // k_heads
        self.starts = [0]
        for n in counts:
            self.starts.append(self.starts[-1] + n)
        self.tokens = self.starts[-1]
        self.row_tiles = div_up(self.tokens * self.group, ROWS)
        self.key_tiles = div_up(prefix, KEYS)
        self.pre = self.row_tiles * k_heads * (self.key_tiles + COST) if prefix else 0
        # the shorter line: requests' items with the prefix in them, or apart from it
        self.joint = -1
        alone = sum(self.own_tiles(b) for b in range(len(counts)))
        seeing = sum(self.tiles(b, rt) > 0 for b in range(len(counts)) for rt in range(self.own_tiles(b)))
        if prefix and (alone * (self.key_tiles + COST) - seeing * COST) * k_heads <= self.pre:
            self.joint, self.pre = self.key_tiles, 0
        self.before = [0]
        for b in range(len(counts)):
            self.before.append(self.before[-1] + k_heads * sum(self.cost(b, rt) for rt in range(self.own_tiles(b))))
        self.units = self.pre + self.before[-1]
        self.grid = min(grid, self.units)
        self.slot_rows = min(ROWS, self.tokens * self.group)

    def own_tiles(self, b):
        return div_up(self.counts[b] * self.group, ROWS)

    def seen(self, b, rt):
        last = min((rt * ROWS + ROWS - 1) // self.group, self.counts[b] - 1)
        return max(0, self.lens[b] - self.counts[b] + last + 1)

    def tiles(self, b, rt):
        return div_up(self.seen(b, rt), KEYS)

    def cost(self, b, rt):
        t = self.tiles(b, rt)
        return self.joint + t + COST if self.joint >= 0 else t + COST if t else 0

    def seeing_before(self, b, rt):
        if rt == 0:
            return 0
        c = (127 + self.group * (self.lens[b] - self.counts[b] + 128)) >> 7
        return rt - min(max(self.group - c, 0), rt)

    def units_before(self, b, rt):
        return self.tiles_before(b, rt) + (
            rt * (self.joint + COST) if self.joint >= 0 else self.seeing_before(b, rt) * COST)

    def tiles_before(self, b, rt):
        """The closed form of sum(tiles(b, x) for x < rt), rt below own_tiles(b)."""
        if rt == 0:
            return 0
        c = (127 + self.group * (self.lens[b] - self.counts[b] + 128)) >> 7

        def total(x):
            if x <= 0:
                return 0
            q, r = divmod(x, self.group)
            return self.group * q * (q - 1) // 2 + q * r

        return total(rt + c) - total(c)

    def begin(self, c):
        each, more = divmod(self.units, self.grid)
        return each * c + min(c, more)

    def cta_of(self, u):
        each, more = divmod(self.units, self.grid)
        longer = more * (each + 1)
        return u // (each + 1) if u < longer else more + (u - longer) // each

    def pieces(self, cta):
        """(item, first tile, tiles, destination) in the order of list_pieces."""
        u, end = self.begin(cta), self.begin(cta + 1)
        key_tiles = self.key_tiles
        while u < end and u < self.pre:
            item, at = divmod(u, key_tiles + COST)
            step = min(end - u, key_tiles + COST - at)
            u += step
            first = max(at - COST, 0)
            n = at + step - COST - first
            if n <= 0:
                continue
            head, tile = divmod(item, self.row_tiles)
            to = ("part", 0) if n == key_tiles else ("slot", 2 * cta + (0 if first > 0 else 1))
            yield ("prefix", head, tile), first, n, to
        want = max(0, min(self.begin(cta) - self.pre, self.before[-1]))
        start = next((b for b in range(len(self.counts)) if self.before[b] <= want < self.before[b + 1]),
                     len(self.counts))
        base = self.pre + (self.before[start] if start < len(self.counts) else 0)
        for b in range(start, len(self.counts)):
            for rt in range(self.own_tiles(b)):
                cost = self.cost(b, rt)
                for h in range(self.k_heads):
                    if u < end and u < base + cost:
                        at = u - base
                        assert at >= 0
                        step = min(end - u, cost - at)
                        u += step
                        first = max(at - COST, 0)
                        n = at + step - COST - first
                        to = ("slot", 2 * cta + (0 if first > 0 else 1)) if n < cost - COST else (
                            ("part", 1) if self.pre else ("out", 0))
                        if n > 0:
                            yield ("own", b, rt, h), first, n, to
                    base += cost
        assert u == end

    def join(self, token, hq):
        """The places of a row's partial results in the order of the keys, or None where the first kernel wrote it."""
        h, g = divmod(hq, self.group)
        b = max(i for i in range(len(self.counts)) if self.starts[i] <= token and self.counts[i])
        found = []
        ranges = []
        if self.pre:
            packed = token * self.group + g
            key_tiles = self.key_tiles
            lo = (h * self.row_tiles + packed // ROWS) * (key_tiles + COST) + COST
            ranges.append((0, lo, lo + key_tiles, packed % ROWS))
        packed = (token - self.starts[b]) * self.group + g
        rt = packed // ROWS
        cost = self.cost(b, rt)
        lo = self.pre + self.before[b] + self.k_heads * self.units_before(b, rt) + h * cost + COST
        ranges.append((1, lo, lo + max(cost - COST, 0), packed % ROWS))
        for x, lo, hi, row in ranges:
            if lo == hi:
                continue
            c0, c1 = self.cta_of(lo), self.cta_of(hi - 1)
            if c0 == c1:
                found.append(("part", x, token * self.q_heads + hq) if self.pre else None)
            else:
                found += [("slot", 2 * c + (c == c0), row) for c in range(c0, c1 + 1)]
        return None if found == [None] else found


def check(plan):
    held = {}  # (token, query head) -> places in the order of the pieces' CTAs
    covered = {}
    if plan.units:
        for cta in range(plan.grid):
            used = set()
            for item, first, n, to in plan.pieces(cta):
                assert n > 0
                covered.setdefault(item, []).append((first, n))
                if to[0] == "slot":
                    assert 0 <= to[1] < 2 * plan.grid and to[1] not in used
                    used.add(to[1])
                if item[0] == "prefix":
                    _, head, tile = item
                    first_token, row0, limit = 0, tile * ROWS, plan.tokens * plan.group
                else:
                    _, b, rt, head = item
                    first_token, row0, limit = plan.starts[b], rt * ROWS, plan.counts[b] * plan.group
                for row in range(min(ROWS, limit - row0)):
                    tok, g = divmod(row0 + row, plan.group)
                    key = (first_token + tok, head * plan.group + g)
                    assert row < plan.slot_rows and key[0] < plan.tokens
                    place = None if to[0] == "out" else ("slot", to[1], row) if to[0] == "slot" else (
                        "part", to[1], key[0] * plan.q_heads + key[1])
                    held.setdefault(key, []).append(place)
    expected = {}
    if plan.pre:
        for h in range(plan.k_heads):
            for t in range(plan.row_tiles):
                expected["prefix", h, t] = plan.key_tiles
    for b in range(len(plan.counts)):
        for rt in range(plan.own_tiles(b)):
            for h in range(plan.k_heads):
                if plan.cost(b, rt):
                    expected["own", b, rt, h] = plan.cost(b, rt) - COST
    assert covered.keys() == expected.keys()
    for item, runs in covered.items():
        runs.sort()
        at = 0
        for first, n in runs:
            assert first == at
            at += n
        assert at == expected[item]
    for token in range(plan.tokens):
        for hq in range(plan.q_heads):
            want = held.get((token, hq), [])
            assert plan.join(token, hq) == (None if want == [None] else want), (token, hq)


@pytest.mark.parametrize("counts,lens,prefix,heads,grid", [
    ([1], [300], 0, (6, 1), 148), ([1], [0], 0, (6, 1), 148), ([1], [0], 1, (6, 1), 148),
    ([1] * 40, [50] * 40, 1000, (6, 1), 148), ([5, 0, 3], [7, 9, 1], 65, (8, 2), 148),
    ([100, 40], [100, 300], 200, (6, 1), 16), ([100, 41], [100, 0], 900, (12, 2), 16), ([3], [3], 5000, (6, 1), 7),
    ([64, 0, 128], [0, 70, 500], 128, (4, 2), 11), ([3], [5000], 0, (130, 1), 7), ([1] * 300, [1] * 300, 0, (6, 1), 148),
])
def test_pieces_cover_every_tile_and_the_join_finds_them(counts, lens, prefix, heads, grid):
    check(Plan(counts, lens, prefix, *heads, grid))


def test_random_batches():
    rng, joint = random.Random(5), set()
    for _ in range(60):
        batch = rng.randint(1, 20)
        counts = [rng.choice([0, 1, 1, rng.randint(1, 60)]) for _ in range(batch)]
        lens = [rng.choice([0, 1, 63, 64, 65, rng.randint(0, 2000)]) for _ in range(batch)]
        prefix = rng.choice([0, 1, 64, rng.randint(1, 3000)])
        heads = rng.choice([(6, 1), (8, 2), (4, 4), (12, 2)])
        plan = Plan(counts, lens, prefix, *heads, rng.choice([1, 5, 20, 148]))
        joint.add(plan.joint >= 0)
        check(plan)
    assert joint == {False, True}


def test_ring_order_names_every_entry_once():
    """K0, K1, V0, K2, V1, ...: what the producer loads at each entry is what the issuer looks for there."""
    ring_k = lambda j: 0 if j == 0 else 2 * j - 1  # noqa: E731
    ring_v = lambda j, n: 2 * j + 2 if j + 1 < n else 2 * n - 1  # noqa: E731
    for n in range(1, 40):
        produced = {}
        for i in range(2 * n):
            is_v = i == 2 * n - 1 or (i >= 2 and i % 2 == 0)
            j = (n - 1 if i == 2 * n - 1 else i // 2 - 1) if is_v else (i + 1) // 2
            produced[i] = (is_v, j)
        assert sorted(produced.values()) == [(v, j) for v in (False, True) for j in range(n)]
        for j in range(n):
            assert produced[ring_k(j)] == (False, j) and produced[ring_v(j, n)] == (True, j)
        # the order in which the products take them
        taken = []
        for j in range(n + 1):
            if j < n:
                taken.append(ring_k(j))
            if j > 0:
                taken.append(ring_v(j - 1, n))
        assert taken == list(range(2 * n))


def test_closed_form_of_a_requests_tiles():
    rng = random.Random(11)
    for _ in range(400):
        count, length = rng.randint(1, 2000), rng.choice([0, 1, rng.randint(0, 3000)])
        group = rng.choice([1, 2, 3, 5, 6, 7, 8, 12, 64, 127, 128, 129, 200])
        plan = Plan([count], [length], 0, group, 1, 148)
        n = plan.own_tiles(0)
        for rt in sorted({0, 1, n // 2, n - 1, rng.randrange(n)} & set(range(n))):
            assert plan.tiles_before(0, rt) == sum(plan.tiles(0, x) for x in range(rt)), (count, length, group, rt)
            assert plan.units_before(0, rt) == sum(plan.cost(0, x) for x in range(rt)), (count, length, group, rt)
            assert plan.seeing_before(0, rt) == sum(plan.tiles(0, x) > 0 for x in range(rt))
        last = div_up(length, KEYS) + COST if length else 0
        assert plan.units_before(0, n - 1) + last == plan.units
        plan = Plan([count], [length], 1000, group, 1, 148)  # one request: the prefix in its items
        assert plan.joint == 8 and plan.units_before(0, n - 1) + plan.cost(0, n - 1) == plan.units


def test_division_by_multiplication():
    for d in list(range(1, 300)) + [1000, 4095, 4096, 4097, 2 ** 20 + 1, 2 ** 30 - 1, 2 ** 30]:
        log = (d - 1).bit_length()
        mul = ((1 << (31 + log)) + d - 1) // d
        assert mul < 2 ** 32
        for x in [0, 1, d - 1, d, d + 1, 2 ** 31 - 1, (2 ** 31 - 1) // d * d - 1, (2 ** 31 - 1) // d * d]:
            if 0 <= x < 2 ** 31:
                assert (x * mul) >> (31 + log) == x // d


def test_a_stage_is_looked_at_only_when_its_last_contents_are_known_to_have_landed():
    """A parity wait returns at once while the phase before the one it is meant for is still open.  For every order of
    pieces: what the waits before prove covers the last entry in each stage that an issuer, or a softmax warp that
    clears V rows, looks at."""
    stages, per_tile = 5, 2
    rng = random.Random(3)
    for _ in range(300):
        pieces = [rng.choice([1, 1, 2, 3, rng.randint(1, 9)]) for _ in range(rng.randint(1, 8))]
        order = []  # (is V, tile counted over all pieces) of each entry
        first = 0
        for n in pieces:
            entries = {}
            for j in range(n):
                entries[0 if j == 0 else 2 * j - 1] = (False, first + j)
                entries[2 * j + 2 if j + 1 < n else 2 * n - 1] = (True, first + j)
            order += [entries[i] for i in range(2 * n)]
            first += n
        where = {entry: i for i, entry in enumerate(order)}
        starts = {sum(pieces[:i]) for i in range(len(pieces))}
        for (is_v, t), i in where.items():
            for part in range(per_tile):
                before = i * per_tile + part - stages
                if before < 0:
                    continue
                last_v, last_t = order[before // per_tile]
                if is_v:  # behind p_full(t): S(t) and so K(t) are done; the issuer itself took V before t
                    assert last_t < t if last_v else last_t <= t
                    # a softmax warp at tile t: K(t) used, V up to t - 2 used, at a piece's start V(t - 1) too
                    if t + 1 in starts or t + 1 == first:  # the piece's last tile may be short
                        assert last_t <= (t - 1 if t in starts else t - 2) if last_v else last_t <= t
                else:  # behind pv_done(t - 2); the issuer itself took K before t
                    assert last_t <= t - 2 if last_v else last_t < t


def test_scores_wait_for_all_that_their_columns_held():
    """S(t) and P(t) lie in quarters of 256 TMEM columns.  What issue_scores waits for before S(t), with what those
    waits prove, covers every S that was to be read and every P that was to be used where S(t) goes; P(t) lies in S(t).
    No barrier is waited for that may be a phase ahead or behind."""
    s_at, p_at = [{0, 1}, {2, 3}, {1, 2}], [0, 3, 2]
    read, used = {}, {}  # issue_scores(t): S read and P used up to these tiles
    for t in range(60):
        third = t % 3
        assert p_at[third] in s_at[third]
        read[t], used[t] = read.get(t - 1, -1), used.get(t - 1, -1)
        if third < 2 and t >= 3:
            wait = t - (2 if third == 1 else 3)
            assert wait - 4 <= used[t] and wait + 4 >= t  # pv_done, four phases
            used[t] = max(used[t], wait)
            read[t] = max(read[t], wait)
        if third != 1 and t >= 2:
            assert t - 3 <= read[t] and t + 1 >= t  # s_read, two phases
            read[t] = max(read[t], t - 1)
            used[t] = max(used[t], used[t - 1])
        for u in range(t):
            if s_at[u % 3] & s_at[third]:
                assert u <= read[t], (t, u)
            if p_at[u % 3] in s_at[third]:
                assert u <= used[t], (t, u)
        # S(t) is there: the softmax warps look at pv_done(t - 1), and their next phases of s_full and p_full
        assert t - 5 <= used[t]
        assert t - 2 <= read[t], "s_full(t) must not complete before every warp has seen s_full(t - 2)"
        assert t - 4 <= used[t], "p_full(t) must not complete before its last phase has been used"

"""GPU tests of the paged attention where a CTA walks many key tiles of an item:
scores that rise while it does, so that what has been summed is rescaled; many
rows to join; whole prompts; long contexts.  The restated division of the work
says that each test reaches what it is for."""

from __future__ import annotations

import math

import pytest
import torch

import testfiles_b200 as welm
from test_attend_plan import KEYS, ROWS, Plan
from test_gpu_attend import DEV, Batch, agree

pytestmark = pytest.mark.gpu

LN2 = math.log(2.0)


def plan_of(batch, heads):
    counts = [b - a for a, b in zip(batch.starts, batch.starts[1:])]
    sms = torch.cuda.get_device_properties(DEV).multi_processor_count
    return Plan(counts, batch.lens, batch.prefix, *heads, sms)


def longest_piece(plan):
    return max(n for cta in range(plan.grid) for _, _, n, _ in plan.pieces(cta))


def levels(n, g):
    """Scores of n keys in powers of two: flat for two to five tiles, then one key more than 2^8 above all before it,
    whose level the next tiles have; what lies below such a key weighs as much as it."""
    out, level, at = torch.zeros(n), 0.0, 0
    while at < n:
        run = KEYS * int(torch.randint(2, 6, (), generator=g))
        out[at:at + run] = level
        at += run
        level += 8.5 + 1.5 * float(torch.rand((), generator=g))
        if at < n:
            spike = at + int(torch.randint(0, KEYS, (), generator=g))
            out[at:at + KEYS] = out[at - 1]
            if spike < n:
                out[spike] = level
            at += KEYS
    if n > 2 * KEYS:  # at the end too, where both sides weigh as much
        out[n - 1 - int(torch.randint(0, KEYS, (), generator=g))] = level
    return out


def put(cache, table, rows):
    block = cache.shape[1]
    for i in range(0, rows.shape[0], block):
        here = rows[i:i + block]
        cache[int(table[i // block]), :here.shape[0], 0] = here


def rising(lens, counts=None, prefix=0, share=(1.0, 1.0, 0.0, -1.0, 0.5, 0.25), seed=0, **more):
    """A batch of one KV head whose scores are share x levels: a row's share is its query head's, turned by its token."""
    batch = Batch(lens, counts=counts, prefix=prefix, seed=seed, **more)
    g = torch.Generator().manual_seed(seed)
    unit = (torch.randint(0, 2, (256,), generator=g) * 2 - 1).float() / 16  # of length 1
    tokens, heads = batch.q.shape[:2]
    place = torch.arange(tokens)[:, None] + torch.arange(heads)
    of_row = torch.tensor(share)[place % len(share)][..., None]
    batch.q = (64 * of_row * unit + 0.1 * torch.randn(batch.q.shape, generator=g)).to(torch.bfloat16).to(DEV)

    def fill(table, level, block):
        n = level.shape[0]
        k = unit * (level * LN2 / (64 * batch.scale))[:, None] + 0.05 * torch.randn((n, 256), generator=g)
        # values that tell tiles apart, so that a wrong weight shows
        v = (torch.randint(0, 2, (n // KEYS + 1, 256), generator=g) * 2.0 - 1).repeat_interleave(KEYS, 0)[:n]
        v = v + 0.25 * torch.randn((n, 256), generator=g)
        put(batch.keys, table, k.to(torch.bfloat16).to(DEV))
        put(batch.values, table, v.to(torch.bfloat16).to(DEV))

    shared = levels(prefix, g)
    if prefix:
        fill(batch.prefix_table, shared, batch.block)
    for b, n in enumerate(lens):
        if n:
            own = levels(n, g) + (float(shared[-KEYS:].max()) if prefix else 0.0)
            fill(batch.table[b], own, batch.block)
    return batch


def rescales(batch, plan):
    """How often a row's maximum grows past 2^8 in the middle of a piece, with the kernel's rule: (rows in pieces of the
    prefix, of own keys, of own keys before which the piece has the prefix's)."""
    block, group = batch.block, plan.group
    gather = lambda table, n: batch.keys[table[:-(-n // block)].long(), :, 0].flatten(0, 1)[:n].double()  # noqa: E731
    pad = lambda s, tiles: torch.nn.functional.pad(s, (0, tiles * KEYS - s.shape[1]), value=-math.inf)  # noqa: E731
    tops = lambda s: s.unflatten(1, (-1, KEYS)).amax(2) * (batch.scale / LN2)  # noqa: E731
    rows = batch.q[:batch.tokens].double().flatten(0, 1)
    prefix = tops(pad(rows @ gather(batch.prefix_table, batch.prefix).t(), plan.key_tiles)) if batch.prefix else None
    own = {}
    for b, n in enumerate(batch.lens):
        first, last = batch.starts[b], batch.starts[b + 1]
        if n and last > first:
            s = rows[first * group:last * group] @ gather(batch.table[b], n).t()
            seen = n - (last - first) + 1 + torch.arange(last - first, device=DEV).repeat_interleave(group)
            s = s.masked_fill(torch.arange(n, device=DEV) >= seen[:, None], -math.inf)
            own[b] = tops(pad(s, -(-n // KEYS)))
    found = [0, 0, 0]
    for cta in range(plan.grid):
        for item, first, n, _ in plan.pieces(cta):
            if item[0] == "prefix":
                top, before = prefix[item[2] * ROWS:(item[2] + 1) * ROWS], 0
            else:
                _, b, rt, _ = item
                at = slice(rt * ROWS, (rt + 1) * ROWS)
                top, before = own.get(b, torch.empty((0, 0), device=DEV))[at], 0
                if plan.joint >= 0:
                    start = batch.starts[b] * group
                    end = batch.starts[b + 1] * group
                    top = torch.cat((prefix[start:end][at], top), dim=1)
                    before = plan.joint
            m = top[:, first].clone()
            for t in range(first + 1, first + n):
                grown = top[:, t] - m > 8
                m = torch.where(grown, top[:, t], m)
                kind = 0 if item[0] == "prefix" else 2 if first < before <= t else 1
                found[kind] += int(grown.sum())
    return found


def test_rising_scores_of_own_keys():
    lens = [1300 + 37 * b % 700 for b in range(160)]
    batch = rising(lens, seed=1)
    plan = plan_of(batch, (6, 1))
    assert longest_piece(plan) >= 8 and rescales(batch, plan)[1] > 500
    agree(batch, batch.run())


def test_rising_scores_of_a_prefix():
    batch = rising([100 + b % 90 for b in range(200)], prefix=8192, seed=2)
    plan = plan_of(batch, (6, 1))
    assert plan.pre and longest_piece(plan) >= 8 and rescales(batch, plan)[0] > 500
    agree(batch, batch.run())


@pytest.mark.parametrize("block", [8, 64])
def test_rising_scores_from_a_prefix_on_to_own_keys(block):
    """The prefix and a request's own keys in one item; rows of one warp rise by different amounts or fall."""
    batch = rising([1500, 1111], counts=[700, 640], prefix=1900, seed=3, block=block)
    plan = plan_of(batch, (6, 1))
    assert plan.joint >= 0 and longest_piece(plan) >= 8
    found = rescales(batch, plan)
    assert found[1] > 500 and found[2] > 500
    agree(batch, batch.run())


def test_rows_that_do_not_rise_are_left_alone():
    """One row in eight of a warp's rises."""
    batch = rising([2000], counts=[900], prefix=0, share=(0.0,) * 7 + (1.0,), seed=4)
    plan = plan_of(batch, (6, 1))
    assert rescales(batch, plan)[1] > 100
    agree(batch, batch.run())


@pytest.mark.parametrize("requests", [701, 1003, 1501])
def test_many_rows_with_a_prefix_are_joined(requests):
    """More than 4096 rows, or than 40 an SM, some in whole items and some in cut ones, of requests with own keys and without."""
    lens = [[0, 1, 64, 129, 300][b % 5] for b in range(requests)]
    batch = Batch(lens, prefix=4000)
    plan = plan_of(batch, (6, 1))
    assert plan.pre and requests * 6 > 4096 and requests * 6 % 32
    kinds = {(item[0], to[0]) for cta in range(plan.grid) for item, _, _, to in plan.pieces(cta)}
    assert kinds >= {("prefix", "slot"), ("own", "slot"), ("own", "part")}
    agree(batch, batch.run())
    assert batch.status.item() == 0


@pytest.mark.parametrize("counts,lens,heads", [
    ([2048], [2048], (6, 1)), ([4097, 300, 1], [4097, 300, 1], (6, 1)), ([9001], [9001], (2, 1)),
    ([1000] * 8, [1000] * 8, (8, 2)), ([16384], [16384], (1, 1)),
])
def test_whole_prompts_without_a_prefix(counts, lens, heads):
    batch = Batch(lens, counts=counts, heads=heads)
    agree(batch, batch.run())
    assert batch.status.item() == 0


@pytest.mark.parametrize("counts,lens,prefix", [([2000, 700], [5000, 4000], 0), ([2048], [2100], 6000)])
def test_chunks_of_a_prompt(counts, lens, prefix):
    batch = Batch(lens, counts=counts, prefix=prefix)
    agree(batch, batch.run())


@pytest.mark.parametrize("lens,counts", [
    ([32768], None), ([131077], None), ([40000, 33000, 1], None), ([33000 + 999 * b for b in range(8)], None),
    ([65537, 50000], [4, 3]),
])
@pytest.mark.parametrize("prefix", [0, 20001])
def test_long_contexts(lens, counts, prefix):
    batch = Batch(lens, counts=counts, prefix=prefix)
    agree(batch, batch.run())
    assert batch.status.item() == 0


def test_long_calls_repeat_themselves():
    batch = Batch([5000 + 700 * b for b in range(24)], counts=[5] * 24, prefix=9000)
    first = batch.run()
    for _ in range(5):
        again = batch.run()
        assert torch.equal(again[0], first[0]) and torch.equal(again[1], first[1])
    space = torch.full((welm.attend_workspace_bytes(batch.tokens, 24, 6, 1, 9000, DEV),), 255, dtype=torch.uint8,
                       device=DEV)
    again = batch.run(workspace=space)
    assert torch.equal(again[0], first[0]) and torch.equal(again[1], first[1])


@pytest.mark.parametrize("lens,counts,prefix,heads", [
    ([131077], None, 0, (6, 1)), ([33000 + 999 * b for b in range(8)], None, 20001, (6, 1)),
    ([8193], [8193], 0, (6, 1)), ([5000, 4000], [2000, 700], 333, (8, 2)), ([300] * 701, None, 4000, (6, 1)),
    ([0, 1, 127, 128, 129, 4000] * 9, None, 1, (12, 2)),
])
def test_equal_weights_count_every_key_once(lens, counts, prefix, heads):
    """With Q zero every p is 1 and, for values of -1, 0 and 1, every sum exact: what is left is the division, a product
    and the rounding to BF16."""
    batch = Batch(lens, counts=counts, prefix=prefix, heads=heads)
    batch.q.zero_()
    batch.values = torch.where(batch.values.isnan(), batch.values, batch.values.sign() * (batch.values.abs() > 0.4))
    out, lse = batch.run()
    want, want_lse, _, _ = batch.oracle()
    assert ((out.double() - want).abs() <= want.abs() * (2.0 ** -8 + 2.0 ** -22)).all()
    none = want_lse == -math.inf
    assert torch.equal(lse == -math.inf, none)
    assert ((lse.double() - want_lse).abs()[~none] <= want_lse.abs()[~none] * 2.0 ** -21 + 2.0 ** -21).all()

"""GPU tests of the rotating append to the paged KV cache against the 64-bit
oracle, and of one layer's decode step: rotate, append, attend."""

from __future__ import annotations

import pytest
import torch

import paged_oracle
import testfiles_b200 as welm
from testfiles_b200 import _native, workloads

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
ROWS = 4096
FILL = -3.0


def make(tokens, heads, blocks, block, axes=0, seed=0):
    g = torch.Generator().manual_seed(seed + tokens)
    qkv = torch.randn((tokens, heads[0] + 2 * heads[1], 256), generator=g).to(torch.bfloat16)
    positions = torch.randint(0, ROWS, (axes, tokens) if axes else (tokens,), generator=g)
    slots = torch.randperm(blocks * block, generator=g)[:tokens]
    return qkv, positions, slots, workloads.make_cos_sin_cache(ROWS, 10000.0)


def views(qkv, heads):
    return qkv[:, :heads[0]], qkv[:, heads[0]:sum(heads)], qkv[:, sum(heads):]


def check(q, key_cache, value_cache, qkv, heads, positions, slots, cos_sin, sections=None, interleaved=False, block=64):
    """Results against the oracle; tokens that may not be written are those of `slots` < 0 or positions out of range."""
    want_q, want_k, want_v = views(qkv, heads)
    rows = positions if positions.dim() == 2 else positions[None]
    sections = sections or (32,)
    live = (slots >= 0) & (slots < key_cache.shape[0] * block)
    for a in set(paged_oracle.pair_axes(sections, interleaved)):
        live &= (rows[a] >= 0) & (rows[a] < ROWS)
    if q is not None:
        exact = paged_oracle.rotate(want_q, rows, cos_sin, sections, interleaved)
        off = (q.cpu().double() - exact).abs()
        assert (off <= paged_oracle.rotate_bound(want_q, exact))[live].all()
        assert torch.equal(q.cpu()[~live], want_q[~live])
        assert torch.equal(q.cpu()[..., :192], want_q[..., :192])
    exact = paged_oracle.rotate(want_k, rows, cos_sin, sections, interleaved)
    bound = paged_oracle.rotate_bound(want_k, exact)
    page, place = slots[live] // block, slots[live] % block
    got = key_cache.cpu()[page, place]
    assert ((got.double() - exact[live]).abs() <= bound[live]).all()
    assert torch.equal(got[..., :192], want_k[live][..., :192])
    assert torch.equal(value_cache.cpu()[page, place], want_v[live])
    rest = torch.ones(key_cache.shape[:2], dtype=torch.bool)
    rest[page, place] = False
    assert (key_cache.cpu()[rest] == FILL).all() and (value_cache.cpu()[rest] == FILL).all()


@pytest.mark.parametrize("tokens,heads,blocks,block,sections,interleaved", [
    (1, (6, 1), 2, 64, None, False), (32, (6, 1), 3, 16, None, False), (3001, (6, 1), 60, 64, None, False),
    (500, (8, 2), 40, 16, (16, 8, 8), False), (77, (4, 4), 90, 1, (12, 10, 10), True), (65, (12, 2), 11, 7, (0, 32), False),
])
@pytest.mark.parametrize("layout", ["nhd", "hnd"])
def test_append_matches_oracle(tokens, heads, blocks, block, sections, interleaved, layout):
    qkv, positions, slots, cos_sin = make(tokens, heads, blocks, block, len(sections or ()))
    slots[::9] = -1 - slots[::9]  # padding
    shape = (blocks, block, heads[1], 256) if layout == "nhd" else (blocks, heads[1], block, 256)
    caches = [torch.full(shape, FILL, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    keys, values = caches if layout == "nhd" else [c.transpose(1, 2) for c in caches]
    d = qkv.to(DEV)
    q, k, v = views(d, heads)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    welm.rope_kv_append(q, k, v, positions.to(DEV), cos_sin.to(DEV), slots.to(DEV), keys, values, sections, interleaved,
                        status)
    assert status.item() == 0
    check(q, keys, values, qkv, heads, positions, slots, cos_sin, sections, interleaved, block)
    assert torch.equal(d[:, heads[0]:].cpu(), qkv[:, heads[0]:])  # K and V are read only


def test_bad_slots_and_positions_leave_the_token():
    heads = (6, 1)
    qkv, positions, slots, cos_sin = make(100, heads, 4, 64)
    slots[5], slots[77] = 256, 2 ** 40
    positions[9], positions[10] = -1, ROWS
    slots[11], positions[11] = -2, -7  # padding is not looked at any further
    d = qkv.to(DEV)
    q, k, v = views(d, heads)
    keys, values = (torch.full((4, 64, 1, 256), FILL, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    welm.rope_kv_append(q, k, v, positions.to(DEV), cos_sin.to(DEV), slots.to(DEV), keys, values, status=status)
    assert status.item() == _native.DEV_BAD_SLOT | _native.DEV_BAD_POSITION
    check(q, keys, values, qkv, heads, positions, slots, cos_sin)


def test_without_q_equals_the_mirror_write():
    heads = (6, 1)
    qkv, positions, slots, cos_sin = make(900, heads, 20, 64)
    d = qkv.to(DEV)
    q, k, v = views(d, heads)
    got = [torch.full((20, 64, 1, 256), FILL, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    welm.rope_kv_append(None, k, v, positions.to(DEV), cos_sin.to(DEV), slots.to(DEV), *got)
    want = [torch.full((20, 64, 1, 256), FILL, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    q_out = torch.empty((1, 6, 256), dtype=torch.bfloat16, device=DEV)
    welm.rope_mirror_kv_write(q, q_out, k, v, positions.to(DEV), cos_sin.to(DEV), torch.tensor([899], device=DEV),
                              slots.to(DEV), *want)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert torch.equal(d.cpu(), qkv)


def test_caches_inside_one_tensor_and_far_slots():
    """K and V pages interleaved in one allocation, and pages past 2^31 elements."""
    heads, block = (6, 1), 64
    blocks = 2 ** 31 // (2 * block * 256) + 40
    whole = torch.full((blocks, 2, block, 1, 256), FILL, dtype=torch.bfloat16, device=DEV)
    qkv, positions, slots, cos_sin = make(200, heads, 30, block)
    far = slots + (blocks - 30) * block
    d = qkv.to(DEV)
    q, k, v = views(d, heads)
    welm.rope_kv_append(q, k, v, positions.to(DEV), cos_sin.to(DEV), far.to(DEV), whole[:, 0], whole[:, 1])
    tail = whole[blocks - 30:]
    check(q, tail[:, 0], tail[:, 1], qkv, heads, positions, slots, cos_sin)
    assert (whole[:blocks - 30] == FILL).all()


def test_captured_append_follows_slots_and_positions():
    heads = (6, 1)
    qkv, positions, slots, cos_sin = make(40, heads, 4, 64)
    source = qkv.to(DEV)
    d, pos, to, cache = source.clone(), positions.to(DEV), slots.to(DEV), cos_sin.to(DEV)
    keys, values = (torch.full((4, 64, 1, 256), FILL, dtype=torch.bfloat16, device=DEV) for _ in range(2))

    def step():
        d.copy_(source)
        keys.fill_(FILL)
        values.fill_(FILL)
        welm.rope_kv_append(*views(d, heads), pos, cache, to, keys, values)

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for seed in (1, 2):
        g = torch.Generator().manual_seed(seed)
        new_pos, new_slots = torch.randint(0, ROWS, (40,), generator=g), torch.randperm(256, generator=g)[:40]
        new_slots[30:] = -1  # a smaller batch in the captured one
        pos.copy_(new_pos)
        to.copy_(new_slots)
        graph.replay()
        check(d[:, :6], keys, values, qkv, heads, new_pos, new_slots, cos_sin)


@pytest.mark.parametrize("heads", [(6, 1), (8, 2)])
def test_decode_steps_of_a_layer(heads):
    """Prefill a shared prefix and three requests, then decode two tokens each: every call is the package's own, and
    the attention's results are compared with the oracle on the caches that the appends filled."""
    block, prefix, scale = 16, 83, 1 / 16
    cos_sin = workloads.make_cos_sin_cache(ROWS, 10000.0).to(DEV)
    keys, values = (torch.full((64, block, heads[1], 256), float("nan"), dtype=torch.bfloat16, device=DEV)
                    for _ in range(2))
    g = torch.Generator().manual_seed(3)
    order = torch.randperm(64, generator=g).to(torch.int32)
    prefix_table = order[:6].to(DEV)
    table = order[6:6 + 3 * 8].view(3, 8).to(DEV)
    lens = [0, 0, 0]

    def append(counts, pages, start):
        """counts[i] new tokens for each page list, the first at start[i]; returns Q."""
        n = sum(counts)
        x = torch.randn((n, heads[0] + 2 * heads[1], 256), generator=g).to(torch.bfloat16).to(DEV)
        place = torch.cat([torch.arange(s, s + c) for s, c in zip(start, counts)])
        slot = torch.cat([pages[i].cpu().long()[torch.arange(s, s + c) // block] * block + torch.arange(s, s + c) % block
                          for i, (s, c) in enumerate(zip(start, counts))])
        offset = 0 if pages[0] is prefix_table else prefix
        q, k, v = views(x, heads)
        welm.rope_kv_append(q, k, v, (place + offset).to(DEV), cos_sin, slot.to(DEV), keys, values)
        return q

    append([prefix], [prefix_table], [0])
    for counts in ([40, 7, 90], [1, 1, 1], [1, 1, 1]):
        q = append(counts, [table[0], table[1], table[2]], lens)
        lens = [a + b for a, b in zip(lens, counts)]
        starts = [0]
        for c in counts:
            starts.append(starts[-1] + c)
        ragged = torch.tensor(starts, device=DEV) if max(counts) > 1 else None
        out, lse = welm.attend_shared_prefix(q, keys, values, table, torch.tensor(lens, device=DEV), ragged,
                                             prefix_table, prefix, return_lse=True)
        want, want_lse, bound, lse_bound = paged_oracle.attend(q, keys, values, table, lens, starts, prefix_table,
                                                               prefix, scale)
        assert ((out.double() - want).abs() <= bound).all()
        assert ((lse.double() - want_lse).abs() <= lse_bound).all()

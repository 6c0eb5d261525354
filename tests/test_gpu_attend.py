"""GPU tests of the paged attention with a shared prefix against the 64-bit
oracle, at the sizes, layouts and masks where it can go wrong."""

from __future__ import annotations

import math

import pytest
import torch

import paged_oracle
import testfiles_b200 as welm
from testfiles_b200 import _native

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")


class Batch:
    """A paged batch: every page that no request names, and what a page holds behind the last key, is no number."""

    def __init__(self, lens, counts=None, prefix=0, heads=(6, 1), block=64, seed=0, spare=0, scale=None, spread=1.0):
        g = torch.Generator().manual_seed(seed + 1000 * prefix + sum(lens))
        q_heads, k_heads = heads
        self.lens, self.prefix, self.block, self.k_heads = lens, prefix, block, k_heads
        counts = [1] * len(lens) if counts is None else counts
        self.starts = [0]
        for n in counts:
            self.starts.append(self.starts[-1] + n)
        self.ragged = any(n != 1 for n in counts) or spare > 0
        self.tokens = self.starts[-1]
        self.scale = 1 / 16 if scale is None else scale
        blocks_of = [-(-n // block) for n in [prefix] + lens]
        total = sum(blocks_of) + 3
        shape = (total, block, k_heads, 256)
        keys = torch.full(shape, math.nan, dtype=torch.bfloat16)
        values = torch.full(shape, math.nan, dtype=torch.bfloat16)
        order = torch.randperm(total, generator=g).to(torch.int32)
        width = max(1, max(blocks_of[1:], default=0) + 1)
        table = torch.full((len(lens), width), -7, dtype=torch.int32)  # never read behind a request's keys
        at = 0
        for i, (n, blocks) in enumerate(zip([prefix] + lens, blocks_of)):
            pages = order[at:at + blocks]
            at += blocks
            for j, page in enumerate(pages.tolist()):
                here = min(block, n - j * block)
                keys[page, :here] = torch.randn((here, k_heads, 256), generator=g).to(torch.bfloat16) * spread
                values[page, :here] = torch.randn((here, k_heads, 256), generator=g).to(torch.bfloat16)
            if i == 0:
                self.prefix_table = pages.clone().to(DEV) if prefix else None
            else:
                table[i - 1, :blocks] = pages
        self.table = table.to(DEV)
        self.keys, self.values = keys.to(DEV), values.to(DEV)
        self.q = torch.randn((self.tokens + spare, q_heads, 256), generator=g).to(torch.bfloat16).to(DEV)
        self.status = torch.zeros(1, dtype=torch.int32, device=DEV)

    def args(self):
        return dict(block_table=self.table, seq_lens=torch.tensor(self.lens, dtype=torch.int64, device=DEV),
                    query_starts=torch.tensor(self.starts, dtype=torch.int64, device=DEV) if self.ragged else None,
                    prefix_table=self.prefix_table, prefix_len=self.prefix, scale=self.scale, status=self.status)

    def run(self, **more):
        return welm.attend_shared_prefix(more.pop("q", self.q), more.pop("keys", self.keys),
                                         more.pop("values", self.values), **{**self.args(), "return_lse": True, **more})

    def oracle(self):
        return paged_oracle.attend(self.q[:self.tokens], self.keys, self.values, self.table, self.lens, self.starts,
                                   self.prefix_table, self.prefix, self.scale)


def agree(batch, got, want=None):
    out, lse = got
    o, s, bound, lse_bound = batch.oracle() if want is None else want
    n = batch.tokens
    off = (out[:n].double() - o).abs()
    assert torch.isfinite(out).all()
    assert (off <= bound).all(), f"{(off / bound.clamp_min(1e-30)).max().item():.3g} of the bound"
    none = s == -math.inf
    assert torch.equal(lse[:n] == -math.inf, none)
    assert ((lse[:n].double() - s).abs()[~none] <= lse_bound[~none]).all()
    assert (out[:n][none] == 0).all()


@pytest.mark.parametrize("lens", [[1], [63], [64], [65], [127], [128], [129], [300], [0], [5000], [0, 1, 64, 129, 1000], [17] * 150])
def test_decode_without_prefix(lens):
    batch = Batch(lens)
    agree(batch, batch.run())
    assert batch.status.item() == 0


@pytest.mark.parametrize("prefix", [1, 63, 64, 65, 127, 128, 129, 1000, 4097])
@pytest.mark.parametrize("lens", [[1], [0], [0, 1, 64, 129, 700], [30] * 40])
def test_decode_with_prefix(prefix, lens):
    batch = Batch(lens, prefix=prefix)
    agree(batch, batch.run())
    assert batch.status.item() == 0


@pytest.mark.parametrize("prefix", [0, 70])
@pytest.mark.parametrize("batch_size", [32, 33, 288, 289, 400])
def test_batches_around_the_shares_of_the_warps(batch_size, prefix):
    batch = Batch([1 + 37 * b % 150 for b in range(batch_size)], prefix=prefix)
    agree(batch, batch.run())


@pytest.mark.parametrize("heads", [(6, 1), (8, 2), (4, 4), (12, 2), (1, 1), (130, 1), (256, 2)])
@pytest.mark.parametrize("block", [8, 16, 24, 64, 128, 192])
def test_heads_and_pages(heads, block):
    batch = Batch([70, 3, 200], counts=[1, 3, 2], prefix=130, heads=heads, block=block)
    agree(batch, batch.run())


@pytest.mark.parametrize("counts,lens,prefix", [
    ([5, 0, 3], [7, 0, 3], 0), ([5, 2, 3], [3, 0, 1], 0),  # more query tokens than keys: empty rows
    ([5, 2, 3], [3, 0, 1], 70), ([200], [200], 0), ([200, 33], [500, 40], 300), ([0, 0], [4, 5], 10),
    ([22, 21], [22, 300], 64), ([700], [900], 1500),
])
def test_query_runs(counts, lens, prefix):
    batch = Batch(lens, counts=counts, prefix=prefix)
    agree(batch, batch.run())


@pytest.mark.parametrize("block", [8, 48, 64])
@pytest.mark.parametrize("counts,lens,prefix", [
    ([64, 0, 128], [64, 70, 500], 130), ([64, 64], [0, 1], 1), ([128, 64], [100, 600], 1000), ([192], [300], 127),
    ([3], [0], 300), ([2], [200], 5000), ([1], [1], 129),
])
def test_requests_that_fill_their_row_tiles(counts, lens, prefix, block):
    """The prefix and a request's own keys in one item: its tiles end inside the prefix and inside the own keys."""
    batch = Batch(lens, counts=counts, prefix=prefix, heads=(4, 2), block=block)
    agree(batch, batch.run())
    assert batch.status.item() == 0


def test_captured_call_follows_query_starts():
    """The same launch with the prefix in the requests' items and apart from them."""
    batch = Batch([300, 400], counts=[64, 128], prefix=700, heads=(4, 2))
    starts = torch.tensor(batch.starts, dtype=torch.int64, device=DEV)
    args = {**batch.args(), "query_starts": starts, "return_lse": True}
    call = lambda: welm.attend_shared_prefix(batch.q, batch.keys, batch.values, **args)  # noqa: E731
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = call()
    for new in ([0, 64, 192], [0, 65, 192], [0, 0, 192], [0, 191, 192]):
        starts.copy_(torch.tensor(new))
        graph.replay()
        batch.starts = new
        agree(batch, (out, lse))


@pytest.mark.parametrize("scale,spread", [(1.0, 1.0), (1 / 16, 8.0), (1e-3, 1.0), (0.25, 3.0)])
def test_scales(scale, spread):
    """Peaked and flat rows; with peaked ones the running maximum moves often."""
    batch = Batch([900, 30], prefix=700, scale=scale, spread=spread)
    agree(batch, batch.run())


def test_rising_scores_rescale_every_tile():
    batch = Batch([1500], prefix=0)
    rise = torch.arange(24, dtype=torch.float32, device=DEV).repeat_interleave(64)[:1500]
    flat = batch.keys[batch.table[0, :24].long()].flatten(0, 1)[:1500]
    flat = (batch.q[0, :1].float() * rise[:, None] / 16).to(torch.bfloat16)[:, None] + flat * 0.1
    pages = batch.table[0, :24].long()
    for i, page in enumerate(pages.tolist()):
        here = flat[i * 64:(i + 1) * 64]
        batch.keys[page, :len(here)] = here
    agree(batch, batch.run())


def test_rows_of_no_request():
    batch = Batch([70, 20], counts=[2, 1], prefix=100, spare=4)
    out, lse = batch.run()
    agree(batch, (out[:3], lse[:3]))
    assert (out[3:] == 0).all() and (lse[3:] == -math.inf).all()
    given = torch.full_like(batch.q, 7.0)
    out, _ = batch.run(out=given)
    assert out is given and (given[3:] == 7.0).all()
    agree(batch, (out[:3], lse[:3]))


def test_rows_of_no_request_in_a_given_out_keep_their_values_but_have_an_lse():
    batch = Batch([70, 20], counts=[2, 1], prefix=100, spare=400)
    for prefix_len in (0, 100):
        given = torch.full_like(batch.q, 7.0)
        torch.full((403, 6), math.nan, dtype=torch.float32, device=DEV)  # what the allocator may hand out next
        _, lse = batch.run(out=given, prefix_len=prefix_len, prefix_table=batch.prefix_table if prefix_len else None)
        assert (given[3:] == 7.0).all() and (lse[3:] == -math.inf).all() and torch.isfinite(lse[:3]).all()


@pytest.mark.parametrize("batch_size,at", [(3, 1), (100, 70)])
@pytest.mark.parametrize("prefix", [0, 200])
def test_with_starts_that_decrease_no_row_belongs_to_a_request(batch_size, at, prefix):
    """Else the requests could claim the same tokens again and again."""
    batch = Batch([64] * batch_size, counts=[2] * batch_size, prefix=prefix)
    starts = torch.tensor(batch.starts, device=DEV)
    starts[at] = batch.tokens
    out, lse = batch.run(query_starts=starts)
    assert batch.status.item() == _native.DEV_BAD_LENGTH
    assert (out == 0).all() and (lse == -math.inf).all()
    given = torch.full_like(batch.q, 7.0)
    batch.run(query_starts=starts, out=given)
    assert (given == 7.0).all()


def test_strides():
    """q and out inside wider tensors, a head-major cache, pages with room between them."""
    batch = Batch([70, 3, 200], counts=[1, 3, 2], prefix=130, heads=(8, 2))
    want = batch.oracle()
    plain = batch.run()
    wide = torch.full((batch.tokens, 14, 256), math.nan, dtype=torch.bfloat16, device=DEV)
    wide[:, 2:10] = batch.q
    agree(batch, batch.run(q=wide[:, 2:10]), want)
    turned = batch.q.transpose(0, 1).contiguous().transpose(0, 1)
    to = torch.full((batch.tokens, 9, 264), 3.0, dtype=torch.bfloat16, device=DEV)
    out, lse = batch.run(q=turned, out=to[:, :8, :256])
    assert torch.equal(out, plain[0]) and torch.equal(lse, plain[1])
    assert (to[:, 8] == 3.0).all() and (to[:, :, 256:] == 3.0).all()
    hnd = lambda c: c.transpose(1, 2).contiguous().transpose(1, 2)  # noqa: E731
    assert torch.equal(batch.run(keys=hnd(batch.keys), values=hnd(batch.values))[0], plain[0])
    both = torch.full((batch.keys.shape[0], 2, 64, 2, 256), math.nan, dtype=torch.bfloat16, device=DEV)
    both[:, 0], both[:, 1] = batch.keys, batch.values
    assert torch.equal(batch.run(keys=both[:, 0], values=both[:, 1])[0], plain[0])
    one = Batch([40])
    assert torch.equal(one.run(q=one.q.expand(1, 6, 256))[0], one.run()[0])


def test_bad_pages_read_as_zeros():
    batch = Batch([70, 200], prefix=130)
    table, prefix_table = batch.table.clone(), batch.prefix_table.clone()
    table[0, 0], table[1, 2], prefix_table[1] = -1, batch.keys.shape[0], 2 ** 31 - 1
    out, lse = batch.run(block_table=table, prefix_table=prefix_table)
    assert batch.status.item() == _native.DEV_BAD_PAGE
    zero = batch.keys.shape[0] - 1  # a page of zeros in their place
    used = set(batch.table[0, :2].tolist() + batch.table[1, :4].tolist() + batch.prefix_table.tolist())
    zero = next(i for i in range(batch.keys.shape[0]) if i not in used)
    batch.keys[zero] = 0
    batch.values[zero] = 0
    batch.table[0, 0], batch.table[1, 2], batch.prefix_table[1] = zero, zero, zero
    agree(batch, (out, lse))


def test_lengths_out_of_range_are_clamped_and_flagged():
    batch = Batch([64, 64])
    room = batch.table.shape[1] * 64
    batch.table[:] = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32, device=DEV)
    batch.keys.nan_to_num_(0.5)
    batch.values.nan_to_num_(0.5)
    out, lse = batch.run(seq_lens=torch.tensor([-5, 10 ** 12], device=DEV))
    assert batch.status.item() == _native.DEV_BAD_LENGTH
    batch.lens = [0, room]
    agree(batch, (out, lse))
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    batch.run(query_starts=torch.tensor([0, 5, 1], device=DEV), seq_lens=torch.tensor([3, 3], device=DEV),
              status=status)
    assert status.item() == _native.DEV_BAD_LENGTH


def test_workspace_contents_do_not_matter_and_results_repeat():
    batch = Batch([0, 1, 64, 129, 700], prefix=1000)
    need = welm.attend_workspace_bytes(5, 5, 6, 1, 1000, DEV)
    first = batch.run()
    for fill in (0, 255):
        space = torch.full((need,), fill, dtype=torch.uint8, device=DEV)
        out, lse = batch.run(workspace=space)
        assert torch.equal(out, first[0]) and torch.equal(lse, first[1])


def test_offsets_past_32_bits():
    """Pages whose elements lie more than 2^32 bytes and 2^31 elements into the cache."""
    batch = Batch([300, 64], prefix=200)
    blocks = 2 ** 32 // (64 * 256) // 2 + 64
    far = [torch.zeros((blocks, 64, 1, 256), dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    shift = blocks - batch.keys.shape[0]
    far[0][shift:], far[1][shift:] = batch.keys, batch.values
    table = torch.where(batch.table >= 0, batch.table + shift, batch.table)
    got = batch.run(keys=far[0], values=far[1], block_table=table, prefix_table=batch.prefix_table + shift)
    assert torch.equal(got[0], batch.run()[0])


def test_captured_call_follows_lengths_and_tables():
    batch = Batch([300, 64, 5], prefix=200)
    lens = torch.tensor(batch.lens, dtype=torch.int64, device=DEV)
    args = {**batch.args(), "seq_lens": lens, "return_lse": True}
    call = lambda: welm.attend_shared_prefix(batch.q, batch.keys, batch.values, **args)  # noqa: E731
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = call()
    for new in ([300, 64, 5], [1, 0, 2], [257, 33, 5]):
        lens.copy_(torch.tensor(new))
        graph.replay()
        batch.lens = new
        agree(batch, (out, lse))


@pytest.mark.parametrize("capture", [False, True])
@pytest.mark.parametrize("name,new,old", [
    ("seq_lens", [300, 200], [7, 200]), ("seq_lens", [130, 0], [300, 500]), ("seq_lens", [130, 500], [300, 500]),
    ("query_starts", [0, 130, 384], [0, 256, 384]), ("query_starts", [0, 256, 384], [0, 1, 2]),
    ("query_starts", [0, 384, 384], [0, 0, 384]), ("query_starts", [0, 130, 384], [9, 5, 1]),
    ("seq_lens", list(range(130, 180)), [500] * 50), ("seq_lens", [500] * 49 + [0], [500] * 50),
])
def test_lengths_and_starts_that_the_call_before_writes(name, new, old, capture):
    """A call may look at them while the one before still runs: what counts is what that one leaves there.  Here its
    output, the value of the only key with any weight, is what the next call reads."""
    first = Batch([1, 1], prefix=1)
    second = Batch([500] * len(new)) if name == "seq_lens" else Batch([300, 400], counts=[130, 254], prefix=200)
    first.keys[first.prefix_table[0], 0] = -30 * first.q[0, 0]
    first.keys[first.table[0, 0], 0] = 30 * first.q[0, 0]
    first.q[:] = first.q[:1, :1]
    first.values[first.prefix_table[0], 0] = 1.0
    first.values[first.table[0, 0], 0] = 0.0
    n = len(new)
    first.values[first.table[0, 0], 0, 0, :4 * n] = torch.tensor(new, device=DEV).view(torch.bfloat16)
    out = torch.empty_like(first.q)
    stale = torch.tensor(old, device=DEV).view(torch.bfloat16)
    want = second.run(**{name: torch.tensor(new, device=DEV)})
    args = {**first.args(), "out": out}
    later = {**second.args(), name: out.view(torch.int64).flatten()[:n], "return_lse": True}

    def both():
        out[0, 0, :4 * n] = stale
        welm.attend_shared_prefix(first.q, first.keys, first.values, **args)
        return welm.attend_shared_prefix(second.q, second.keys, second.values, **later)

    got = both()
    assert out.view(torch.int64).flatten()[:n].tolist() == new
    if capture:
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = both()
    for _ in range(30):
        if capture:
            graph.replay()
        else:
            got = both()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert second.status.item() == 0


def test_two_streams_at_once():
    batches = [Batch([400, 64, 5] * 9, prefix=2000, seed=s) for s in (1, 2)]
    want = [b.run() for b in batches]
    streams = [torch.cuda.Stream() for _ in batches]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, b in enumerate(batches):
            with torch.cuda.stream(streams[i]):
                got[i].append(b.run())
    torch.cuda.synchronize()
    for i in range(2):
        for out, lse in got[i]:
            assert torch.equal(out, want[i][0]) and torch.equal(lse, want[i][1])


def test_nothing_to_do():
    batch = Batch([5, 6])
    empty = torch.zeros((0, 6, 256), dtype=torch.bfloat16, device=DEV)
    out, lse = welm.attend_shared_prefix(empty, batch.keys, batch.values, batch.table[:0],
                                         torch.zeros(0, dtype=torch.int64, device=DEV), return_lse=True)
    assert out.shape == (0, 6, 256) and lse.shape == (0, 6)
    out = welm.attend_shared_prefix(batch.q, batch.keys, batch.values, batch.table[:0],
                                    torch.zeros(0, dtype=torch.int64, device=DEV),
                                    query_starts=torch.zeros(1, dtype=torch.int64, device=DEV))
    assert (out == 0).all()

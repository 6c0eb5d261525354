"""64-bit oracles of the multi-axis rotary embedding, the rotating cache append
and the paged attention, written from their definitions (test infrastructure),
with the error bounds of the kernels' arithmetic."""

from __future__ import annotations

import math

import torch

HALF = 32
LANE0 = 192


def pair_axes(sections, interleaved):
    """The axis of each of the 32 pairs."""
    if not interleaved:
        return [a for a, n in enumerate(sections) for _ in range(n)]
    left, axes = list(sections), []
    while len(axes) < HALF:
        for a in range(len(left)):
            if left[a]:
                left[a] -= 1
                axes.append(a)
    return axes


def rotate(x, positions, cos_sin, sections, interleaved=False, inverse=False):
    """x [tokens, heads, 256] rotated in 64 bits; tokens with a position outside the cache stay as they are."""
    out = x.double().clone()
    axes = pair_axes(sections, interleaved)
    good = torch.ones(x.shape[0], dtype=torch.bool)
    for a in set(axes):
        good &= (positions[a] >= 0) & (positions[a] < cos_sin.shape[0])
    for pair, a in enumerate(axes):
        row = cos_sin.double()[positions[a].clamp(0, cos_sin.shape[0] - 1)]
        c, s = row[:, pair, None], row[:, HALF + pair, None] * (-1 if inverse else 1)
        x1, x2 = out[..., LANE0 + pair].clone(), out[..., LANE0 + HALF + pair].clone()
        out[..., LANE0 + pair] = torch.where(good[:, None], x1 * c - x2 * s, x1)
        out[..., LANE0 + HALF + pair] = torch.where(good[:, None], x1 * s + x2 * c, x2)
    return out


def rotate_bound(x, exact):
    """Largest error of a rotated lane: two FP32 products and their sum, at most |x1| + |x2| each in size, three
    roundings of 2^-24 in relation to it, then one rounding to BF16 (2^-8 of the result)."""
    size = torch.zeros_like(exact)
    x = x.double().abs()
    both = x[..., LANE0:LANE0 + HALF] + x[..., LANE0 + HALF:]
    size[..., LANE0:] = torch.cat((both, both), dim=-1)
    return size * 3 * 2.0 ** -24 * (1 + 2.0 ** -8) + exact.abs() * 2.0 ** -8


def attend(q, key_cache, value_cache, block_table, lens, starts, prefix_table, prefix, scale):
    """(out, lse, bound of out's error, bound of lse's error) in 64 bits, on the inputs' device.

    Bounds.  A score is a sum of 256 exact products of BF16 values in FP32, whatever the order and with each
    addition off by at most 2^-23 of the sum of sizes (truncation allowed), then scaled and moved by the maximum
    in use with roundings of 2^-24 of the score's and the maximum's size: |error of log p| <= e.  The exponential
    is off by 2^-22, so p is off by a factor of 1 +- w with w = e + 2^-22 (first order; twice that is allowed for the
    rest).  p is rounded to BF16 for the product with the values: 2^-8 more.  Sums over the n keys and the joins add
    2 n 2^-23.  out = O / l is rounded once to BF16.
    """
    tokens, q_heads, dim = q.shape
    k_heads = key_cache.shape[2]
    group = q_heads // k_heads
    dev = q.device
    out = torch.zeros((tokens, q_heads, dim), dtype=torch.float64, device=dev)
    lse = torch.full((tokens, q_heads), -math.inf, dtype=torch.float64, device=dev)
    bound, lse_bound = torch.zeros_like(out), torch.zeros_like(lse)

    def gather(cache, table, n):
        return cache[table[:-(-n // cache.shape[1])].long()].flatten(0, 1)[:n].double()

    pk = gather(key_cache, prefix_table, prefix) if prefix else key_cache.new_zeros((0, k_heads, dim)).double()
    pv = gather(value_cache, prefix_table, prefix) if prefix else key_cache.new_zeros((0, k_heads, dim)).double()
    for b, length in enumerate(lens):
        first, last = starts[b], starts[b + 1]
        n = last - first
        keys = torch.cat((pk, gather(key_cache, block_table[b], length)))
        values = torch.cat((pv, gather(value_cache, block_table[b], length)))
        for h in range(q_heads):
            k, v = keys[:, h // group], values[:, h // group]
            rows = q[first:last, h].double()
            s = rows @ k.t() * scale
            seen = torch.arange(keys.shape[0], device=dev)[None] < (
                prefix + (length - n + 1 + torch.arange(n, device=dev)).clamp(0, length))[:, None]
            some = seen.any(dim=1)
            s = s.masked_fill(~seen, -math.inf)
            if not keys.shape[0]:
                continue
            top = s.amax(dim=1, keepdim=True).masked_fill(~some[:, None], 0)
            p = (s - top).exp()
            total = p.sum(dim=1, keepdim=True)
            safe = total.masked_fill(total == 0, 1)
            o = p @ v / safe
            # The largest score of a visible key, and the sizes it was summed from.
            size = (rows.abs() @ k.abs().t() * scale).masked_fill(~seen, 0)
            e = 256 * 2.0 ** -23 * size.amax(dim=1, keepdim=True)
            e = e + 4 * 2.0 ** -24 * (s.abs().masked_fill(~seen, 0).amax(dim=1, keepdim=True) + 12)
            w = 2 * (e + 2.0 ** -22) + 2 * keys.shape[0] * 2.0 ** -23
            mass = p @ v.abs() / safe
            out[first:last, h] = o
            bound[first:last, h] = (2 * w + 2.0 ** -8) * mass * (1 + 2.0 ** -8) + o.abs() * 2.0 ** -8
            lse[first:last, h] = torch.where(some, (top + safe.log())[:, 0], -math.inf)
            lse_bound[first:last, h] = (2 * w[:, 0] + 2.0 ** -22 *
                                        (1 + lse[first:last, h].abs().masked_fill(~some, 0) + top[:, 0].abs()))
    return out, lse, bound, lse_bound

"""Rotary embedding with several axes, and the paged KV cache's append and
attention, on the sm_100a library.

* :func:`rope_multi_axis_inplace` / :func:`rope_multi_axis` — rotary embedding
  with one position per axis (time, height, width, ...), in place, or as a
  differentiable function that returns rotated copies.
* :func:`rope_kv_append` — ordinary prefill / decode: Q rotated in place, the
  rotated K and the V written to their cache slots, in one pass.
* :func:`attend_shared_prefix` — attention over the paged cache for a batch
  whose requests share a prefix, which is read once for all of them.

Heads are this package's: 256 lanes, the last 64 rotated (pair i is lanes
192 + i and 224 + i); the number of heads is free.  Like the other entries,
every call only enqueues work on the current stream of the tensors' device,
checks its arguments on the host (``ValueError`` / ``TypeError``) and reports
out-of-range indices through ``status`` (an int32 tensor that receives
``WELM_ROPE_DEV_*`` bits).  The reference has no counterpart of these
operators.
"""

from __future__ import annotations

import importlib
from typing import Optional, Sequence

import torch

from . import build

__all__ = [
    "attend_shared_prefix",
    "attend_workspace_bytes",
    "rope_kv_append",
    "rope_multi_axis",
    "rope_multi_axis_inplace",
]

_module = None


def _binding():
    """The compiled module that checks the arguments and calls the library (csrc/torch_binding.cpp)."""
    global _module
    if _module is None:
        if not build.BINDING.exists():
            raise RuntimeError(f"{build.BINDING.name} is not built: run `python -m testfiles_b200.build` (there is no "
                               "fallback)")
        _module = importlib.import_module("._welm_torch", __package__)
    return _module


def rope_multi_axis_inplace(
    q: torch.Tensor,
    k: torch.Tensor,
    positions: torch.Tensor,
    cos_sin_cache: torch.Tensor,
    sections: Sequence[int],
    interleaved: bool = False,
    inverse: bool = False,
    status: Optional[torch.Tensor] = None,
) -> None:
    """Rotates Q ``[tokens, q_heads, 256]`` and K ``[tokens, k_heads, 256]`` in
    place with one position per axis.

    ``positions`` is int64 ``[axes, tokens]`` and ``sections`` gives the pairs
    of each axis, 32 in all, e.g. ``(16, 8, 8)`` for time, height and width.
    With ``interleaved=False`` axis 0 has the first ``sections[0]`` pairs, axis
    1 the next; with ``interleaved=True`` the pairs are dealt out in turn over
    the axes that still have some left.  Pair i of axis a is rotated by columns
    i and 32 + i of ``cos_sin_cache[positions[a, t]]``; ``inverse=True`` turns
    the other way.  A token with a position outside the cache is left as it is
    and flagged.  q and k must not overlap.  For tensors that require gradients
    use :func:`rope_multi_axis`.
    """
    (_module or _binding()).multi_axis_inplace(q, k, positions, cos_sin_cache, sections, interleaved, inverse, status)


def rope_multi_axis(
    q: torch.Tensor,
    k: torch.Tensor,
    positions: torch.Tensor,
    cos_sin_cache: torch.Tensor,
    sections: Sequence[int],
    interleaved: bool = False,
    inverse: bool = False,
    status: Optional[torch.Tensor] = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Rotated copies of Q and K, differentiable in both (any number of times)
    and in nothing else: a cos_sin_cache that requires a gradient is refused.

    Arguments as for :func:`rope_multi_axis_inplace`; q and k keep their values
    and may have any strides, the results are contiguous.  A token with a
    position outside the cache is copied as it is, its gradient too.  A backward
    pass can be captured into a graph where torch's own can: while no eager graph
    of the same leaves is alive.
    """
    return (_module or _binding()).multi_axis(q, k, positions, cos_sin_cache, sections, interleaved, inverse, status)


# ---------------------------------------------------------------------------
# Append to the paged cache.
# ---------------------------------------------------------------------------
def rope_kv_append(
    q: Optional[torch.Tensor],
    k: torch.Tensor,
    v: torch.Tensor,
    positions: torch.Tensor,
    cos_sin_cache: torch.Tensor,
    slot_mapping: torch.Tensor,
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    sections: Optional[Sequence[int]] = None,
    interleaved: bool = False,
    status: Optional[torch.Tensor] = None,
) -> None:
    """Ordinary prefill / decode fused with the append to the paged cache:

    * ``q[t] = rope(q[t])`` in place (``q`` may be None: only K and V);
    * ``key_cache[slot] = rope(k[t])`` and ``value_cache[slot] = v[t]`` for
      ``slot = slot_mapping[t] >= 0``.

    q is ``[tokens, q_heads, 256]``, k and v ``[tokens, k_heads, 256]`` (read
    only), the caches ``[num_blocks, block_size, k_heads, 256]`` (slot = block *
    block_size + place; pass ``cache.transpose(1, 2)`` of a ``[num_blocks,
    k_heads, block_size, 256]`` cache).  ``positions`` is int64 ``[tokens]``, or
    ``[axes, tokens]`` with ``sections`` (see :func:`rope_multi_axis_inplace`).
    A negative slot marks a padding token, which is left alone, its q row too;
    so is a token whose slot or position is out of range, and it is flagged.
    The slots of one call must differ.  q and the two caches must not overlap,
    nor q and k or v; k and v may lie in the caches where no token's slot holds
    a row of another token's k or v.
    """
    (_module or _binding()).kv_append(q, k, v, positions, cos_sin_cache, slot_mapping, key_cache, value_cache, sections,
                                      interleaved, status)


# ---------------------------------------------------------------------------
# Attention with a shared prefix.
# ---------------------------------------------------------------------------
def attend_workspace_bytes(tokens: int, batch: int, q_heads: int, k_heads: int, prefix_len: int,
                           device: torch.device | str = "cuda") -> int:
    """Bytes of the workspace that :func:`attend_shared_prefix` needs for these sizes."""
    device = torch.device(device)
    index = torch.cuda.current_device() if device.index is None else device.index
    return (_module or _binding()).attend_workspace_bytes(tokens, batch, q_heads, k_heads, prefix_len, index)


def attend_shared_prefix(
    q: torch.Tensor,
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    block_table: torch.Tensor,
    seq_lens: torch.Tensor,
    query_starts: Optional[torch.Tensor] = None,
    prefix_table: Optional[torch.Tensor] = None,
    prefix_len: int = 0,
    scale: Optional[float] = None,
    out: Optional[torch.Tensor] = None,
    return_lse: bool = False,
    workspace: Optional[torch.Tensor] = None,
    status: Optional[torch.Tensor] = None,
) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
    """Attention over the paged cache for a batch that shares a prefix.

    q is ``[tokens, q_heads, 256]``, already rotated; the caches are
    ``[num_blocks, block_size, k_heads, 256]`` as :func:`rope_kv_append` fills
    them (block_size a multiple of 8; q_heads a multiple of k_heads, query head
    h reads KV head ``h // (q_heads // k_heads)``).  The shared prefix is the
    first ``prefix_len`` keys of the blocks in ``prefix_table`` (int32), request
    b's own keys the first ``seq_lens[b]`` (int64) of the blocks in
    ``block_table[b]`` (int32 ``[batch, width]``).  Request b's query tokens are
    rows ``query_starts[b]`` to ``query_starts[b + 1]`` of q (int64 ``[batch +
    1]``), at its last own keys, causal; without ``query_starts`` every request
    has one.  ``scale`` is 1/16 unless given.

    Returns ``out``, and with ``return_lse`` also the logarithm of each row's
    sum of exponentials (float32 ``[tokens, q_heads]``).  A row that sees no key
    is zeros, its logarithm minus infinity; so are rows of no request, but that
    a given ``out``, which must not overlap q or a cache, keeps them as they were.

    ``workspace``: device memory of :func:`attend_workspace_bytes`, 32-byte
    aligned, for one call at a time; by default the call takes it from torch's
    allocator.  Lengths, starts and tables are read on the device, so a captured
    call follows them; ``prefix_len`` is part of the capture.  What a page holds
    behind the last key does not matter; a key that some rows of a request do
    not see yet must be finite.  There is no backward pass.

    The kernel waits for its own copies and products, each time for about two
    seconds at most.  Should a wait not end, every row of a request, and its
    logarithm, becomes NaN, and ``status`` receives
    ``WELM_ROPE_DEV_WAIT_TIMEOUT`` (``WELM_ROPE_GIVE_UP=1`` in the environment
    makes every call end so, to test a program's answer to it).
    """
    return (_module or _binding()).attend(q, key_cache, value_cache, block_table, seq_lens, query_starts, prefix_table,
                                          prefix_len, scale, out, return_lse, workspace, status)

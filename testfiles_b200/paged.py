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

import ctypes
from functools import lru_cache
from typing import Optional, Sequence

import torch

from . import _native
from .ops import HEAD_DIM, ROPE_DIM, _require

__all__ = [
    "attend_shared_prefix",
    "attend_workspace_bytes",
    "rope_kv_append",
    "rope_multi_axis",
    "rope_multi_axis_inplace",
]

_HALF = ROPE_DIM // 2


# ---------------------------------------------------------------------------
# Argument checks (host only).  Small launches take about as long as their
# checks, so each attribute is read once.
# ---------------------------------------------------------------------------
def _check(t: Optional[torch.Tensor], name: str, dtype: torch.dtype, index: int) -> None:
    if not isinstance(t, torch.Tensor) or t.dtype != dtype or t.get_device() != index:
        _require(t, name, dtype, torch.device("cuda", index))  # says what is wrong


def _index(q: torch.Tensor) -> int:
    if not isinstance(q, torch.Tensor) or not q.is_cuda:
        raise ValueError("query must be a CUDA tensor (the op runs only on the sm_100a library)")
    return q.get_device()


def _rows(t: torch.Tensor, name: str) -> tuple[int, int, int, int]:
    """Tokens, heads, token stride and head stride of a [tokens, heads, 256] tensor."""
    shape = t.shape
    if len(shape) != 3 or shape[2] != HEAD_DIM:
        raise ValueError(f"{name} must have shape [tokens, heads, {HEAD_DIM}], got {tuple(shape)}")
    token, head, lane = t.stride()
    if not shape[0] * shape[1]:
        return shape[0], shape[1], 0, 0
    if lane != 1 or (token | head) & 7 or t.data_ptr() & 15:
        raise ValueError(f"{name} must have lane stride 1, other strides that are multiples of 8, and a 16-byte "
                         "aligned start")
    return shape[0], shape[1], token, head


def _vector(t: torch.Tensor, name: str, size: int) -> None:
    if t.dim() != 1 or t.shape[0] != size or (size > 1 and t.stride(0) != 1):
        raise ValueError(f"{name} must be a contiguous 1-D tensor of {size} entries, got {tuple(t.shape)}")


@lru_cache(maxsize=256)
def _sections(sections: tuple[int, ...]) -> tuple[ctypes.Array, int]:
    """The pairs of each axis as the library takes them."""
    if not 1 <= len(sections) <= _native.MAX_AXES or min(sections) < 0 or sum(sections) != _HALF:
        raise ValueError(f"sections must be 1 to {_native.MAX_AXES} counts of pairs that add up to {_HALF}, "
                         f"got {sections}")
    return (ctypes.c_int32 * len(sections))(*sections), len(sections)


def _axes(positions: torch.Tensor, sections: Optional[Sequence[int]], tokens: int, index: int):
    """Sections array, axes and position stride; positions checked against them."""
    _check(positions, "positions", torch.int64, index)
    if sections is None:
        array, axes = _sections((_HALF,))
        _vector(positions, "positions", tokens)
        return array, axes, 0
    array, axes = _sections(tuple(sections))
    if positions.shape != (axes, tokens) or (tokens > 1 and positions.stride(1) != 1):
        raise ValueError(f"positions must have shape [{axes}, {tokens}] (axes, tokens) and contiguous rows, got "
                         f"{tuple(positions.shape)} with strides {positions.stride()}")
    return array, axes, positions.stride(0)


def _cos_sin(cache: torch.Tensor, index: int) -> int:
    _check(cache, "cos_sin_cache", torch.float32, index)
    if cache.dim() != 2 or cache.shape[1] != ROPE_DIM or not cache.is_contiguous() or cache.data_ptr() & 15:
        raise ValueError(f"cos_sin_cache must be a contiguous, 16-byte aligned [max_position, {ROPE_DIM}] float32 "
                         "tensor")
    return cache.shape[0]


def _cache(cache: torch.Tensor, name: str, index: int) -> ctypes.Array:
    """Strides of a [num_blocks, block_size, heads, 256] cache."""
    _check(cache, name, torch.bfloat16, index)
    if cache.dim() != 4 or cache.shape[3] != HEAD_DIM:
        raise ValueError(f"{name} must have shape [num_blocks, block_size, heads, {HEAD_DIM}], got "
                         f"{tuple(cache.shape)}")
    strides = cache.stride()
    if strides[3] != 1 or (strides[0] | strides[1] | strides[2]) & 7 or cache.data_ptr() & 15:
        raise ValueError(f"{name} must have lane stride 1, other strides that are multiples of 8, and a 16-byte "
                         "aligned start")
    return (ctypes.c_int64 * 3)(*strides[:3])


def _status(status: Optional[torch.Tensor], index: int) -> Optional[int]:
    if status is None:
        return None
    _check(status, "status", torch.int32, index)
    if status.numel() < 1:
        raise ValueError("status must hold at least one int32")
    return status.data_ptr()


def _launch(name: str, index: int, *args) -> None:
    """Calls a library entry on the current stream of device ``index``, made current for the call."""
    fn = getattr(_native.load(), name)
    stream = torch._C._cuda_getCurrentRawStream(index)
    if torch._C._cuda_getDevice() == index:
        rc = fn(*args, stream)
    else:
        with torch.cuda.device(index):
            rc = fn(*args, stream)
    if rc:
        _native.check(name, rc)


def _no_grad(name: str, *tensors: Optional[torch.Tensor]) -> None:
    """Refuses tensors whose gradient the call would lose."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise ValueError(f"{name} has no backward pass: call it under torch.no_grad() or on detached tensors")


def _written(*tensors: Optional[torch.Tensor]) -> None:
    """Tells autograd that tensors were written in place."""
    if torch.is_grad_enabled():
        torch.autograd.graph.increment_version([t for t in tensors if t is not None])


# ---------------------------------------------------------------------------
# Rotary embedding with several axes.
# ---------------------------------------------------------------------------
def _rotate(q, q_out, k, k_out, positions, cos_sin_cache, sections, interleaved, inverse, status, index) -> None:
    """welm_rope_multi_axis; q or k (with its output) may be None."""
    tokens = None
    rows: list[int] = []
    heads: list[int] = []
    for src, dst, name in ((q, q_out, "query"), (k, k_out, "key")):
        if src is None:
            heads.append(0)
            rows += (0, 0, 0, 0)
            continue
        _check(src, name, torch.bfloat16, index)
        n, count, token, head = _rows(src, name)
        if tokens is not None and n != tokens:
            raise ValueError("query and key need the same number of tokens")
        tokens = n
        heads.append(count)
        rows += (token, head) + ((token, head) if dst is src else dst.stride()[:2])
    array, axes, position_stride = _axes(positions, sections, tokens, index)
    max_position = _cos_sin(cos_sin_cache, index)
    ptr = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    _launch("welm_rope_multi_axis", index, ptr(q), ptr(q_out), ptr(k), ptr(k_out), positions.data_ptr(),
            cos_sin_cache.data_ptr(), array, axes, int(bool(interleaved)), int(inverse), tokens, heads[0], heads[1],
            *rows, position_stride, max_position, _status(status, index))


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
    and flagged.  For tensors that require gradients use
    :func:`rope_multi_axis`.
    """
    index = _index(q)
    _no_grad("rope_multi_axis_inplace", q, k)
    _rotate(q, q, k, k, positions, cos_sin_cache, sections, interleaved, inverse, status, index)
    _written(q, k)


def _readable(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    """``t`` in a layout that the kernel reads: lanes next to one another, 16-byte steps."""
    if t is None or t.dim() != 3:
        return t
    token, head, lane = t.stride()
    if lane == 1 and not (token | head) & 7 and not t.data_ptr() & 15:
        return t
    return t.clone(memory_format=torch.contiguous_format)


class _MultiAxis(torch.autograd.Function):
    """Rotated copies; the gradient of a rotation is the inverse rotation."""

    @staticmethod
    def forward(ctx, q, k, positions, cos_sin_cache, sections, interleaved, inverse, status):
        q, k = _readable(q), _readable(k)
        first = k if q is None else q
        index = _index(first)
        new = lambda t: None if t is None else torch.empty(t.shape, dtype=t.dtype, device=t.device)  # noqa: E731
        q_out, k_out = new(q), new(k)
        _rotate(q, q_out, k, k_out, positions, cos_sin_cache, sections, interleaved, inverse, status, index)
        ctx.save_for_backward(positions, cos_sin_cache)
        ctx.args = (sections, interleaved, inverse)
        ctx.set_materialize_grads(False)
        return q_out, k_out

    @staticmethod
    def backward(ctx, dq, dk):
        positions, cos_sin_cache = ctx.saved_tensors
        sections, interleaved, inverse = ctx.args
        dq = dq if ctx.needs_input_grad[0] else None
        dk = dk if ctx.needs_input_grad[1] else None
        if dq is not None or dk is not None:
            dq, dk = _MultiAxis.apply(dq, dk, positions, cos_sin_cache, sections, interleaved, not inverse, None)
        return dq, dk, None, None, None, None, None, None


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
    """Rotated copies of Q and K, differentiable in both (any number of times).

    Arguments as for :func:`rope_multi_axis_inplace`; q and k keep their values
    and may have any strides, the results are contiguous.  A token with a
    position outside the cache is copied as it is, its gradient too.
    """
    _index(q)
    return _MultiAxis.apply(q, k, positions, cos_sin_cache, tuple(sections), interleaved, inverse, status)


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
    The slots of one call must differ.
    """
    index = _index(k)
    _no_grad("rope_kv_append", q, k, v)
    _check(k, "key", torch.bfloat16, index)
    _check(v, "v", torch.bfloat16, index)
    tokens, k_heads, k_token, k_head = _rows(k, "key")
    v_tokens, v_heads, v_token, v_head = _rows(v, "v")
    if (v_tokens, v_heads) != (tokens, k_heads):
        raise ValueError("key and v need the same tokens and heads")
    q_ptr, q_heads, q_token, q_head = None, 0, 0, 0
    if q is not None:
        _check(q, "query", torch.bfloat16, index)
        q_tokens, q_heads, q_token, q_head = _rows(q, "query")
        if q_tokens != tokens:
            raise ValueError("query and key need the same number of tokens")
        q_ptr = q.data_ptr()
    array, axes, position_stride = _axes(positions, sections, tokens, index)
    max_position = _cos_sin(cos_sin_cache, index)
    _check(slot_mapping, "slot_mapping", torch.int64, index)
    _vector(slot_mapping, "slot_mapping", tokens)
    key_strides = _cache(key_cache, "key_cache", index)
    value_strides = _cache(value_cache, "value_cache", index)
    shape = key_cache.shape
    if value_cache.shape != shape or shape[2] != k_heads:
        raise ValueError("key_cache and value_cache need the same shape, with the heads of key and v")
    _launch("welm_rope_kv_append", index, q_ptr, k.data_ptr(), v.data_ptr(), positions.data_ptr(),
            cos_sin_cache.data_ptr(), array, axes, int(bool(interleaved)), slot_mapping.data_ptr(),
            key_cache.data_ptr(), value_cache.data_ptr(), tokens, q_heads, k_heads, q_token, q_head, k_token, k_head,
            v_token, v_head, shape[0], shape[1], key_strides, value_strides, position_stride, max_position,
            _status(status, index))
    _written(q, key_cache, value_cache)


# ---------------------------------------------------------------------------
# Attention with a shared prefix.
# ---------------------------------------------------------------------------
@lru_cache(maxsize=1024)
def _workspace_bytes(tokens: int, batch: int, q_heads: int, k_heads: int, prefix_len: int, index: int) -> int:
    out = ctypes.c_int64(0)
    with torch.cuda.device(index):
        rc = _native.load().welm_rope_attend_workspace(tokens, batch, q_heads, k_heads, prefix_len, ctypes.byref(out))
    _native.check("welm_rope_attend_workspace", rc)
    return out.value


def attend_workspace_bytes(tokens: int, batch: int, q_heads: int, k_heads: int, prefix_len: int,
                           device: torch.device | str = "cuda") -> int:
    """Bytes of the workspace that :func:`attend_shared_prefix` needs for these sizes."""
    device = torch.device(device)
    index = torch.cuda.current_device() if device.index is None else device.index
    return _workspace_bytes(int(tokens), int(batch), int(q_heads), int(k_heads), int(prefix_len), index)


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
    is zeros, its logarithm minus infinity; so are rows of no request in an
    ``out`` that the call allocates, while a given ``out`` keeps them.

    ``workspace``: device memory of :func:`attend_workspace_bytes`, 32-byte
    aligned, for one call at a time; by default the call takes it from torch's
    allocator.  Lengths, starts and tables are read on the device, so a captured
    call follows them; ``prefix_len`` is part of the capture.  There is no
    backward pass.
    """
    index = _index(q)
    _no_grad("attend_shared_prefix", q)
    _check(q, "query", torch.bfloat16, index)
    tokens, q_heads, q_token, q_head = _rows(q, "query")
    key_strides = _cache(key_cache, "key_cache", index)
    value_strides = _cache(value_cache, "value_cache", index)
    blocks, block_size, k_heads, _ = shape = key_cache.shape
    if value_cache.shape != shape:
        raise ValueError("key_cache and value_cache need the same shape")
    if k_heads < 1 or q_heads < 1 or q_heads % k_heads:
        raise ValueError(f"query heads ({q_heads}) must be a multiple of the cache's heads ({k_heads})")
    if block_size < 1 or block_size % 8:
        raise ValueError(f"block_size must be a multiple of 8, got {block_size}")
    _check(block_table, "block_table", torch.int32, index)
    if block_table.dim() != 2 or (block_table.shape[1] > 1 and block_table.stride(1) != 1):
        raise ValueError("block_table must be a [batch, blocks] int32 tensor with contiguous rows")
    batch, width = block_table.shape
    _check(seq_lens, "seq_lens", torch.int64, index)
    _vector(seq_lens, "seq_lens", batch)
    starts_ptr = None
    if query_starts is not None:
        _check(query_starts, "query_starts", torch.int64, index)
        _vector(query_starts, "query_starts", batch + 1)
        starts_ptr = query_starts.data_ptr()
    elif tokens != batch:
        raise ValueError("without query_starts every request has one query token: q rows must equal block_table rows")
    prefix_len = int(prefix_len)
    prefix_ptr = None
    if prefix_len < 0:
        raise ValueError("prefix_len must not be negative")
    if prefix_len:
        _check(prefix_table, "prefix_table", torch.int32, index)
        if prefix_table.dim() != 1 or prefix_table.shape[0] * block_size < prefix_len or (
                prefix_table.shape[0] > 1 and prefix_table.stride(0) != 1):
            raise ValueError("prefix_table must be a contiguous 1-D int32 tensor with a block for every prefix key")
        prefix_ptr = prefix_table.data_ptr()
    scale = HEAD_DIM ** -0.5 if scale is None else float(scale)
    if not 0.0 < scale < 3.0e38:
        raise ValueError(f"scale must be positive and finite, got {scale}")
    fill = 0
    if out is None:
        out = torch.empty((tokens, q_heads, HEAD_DIM), dtype=torch.bfloat16, device=q.device)
        fill = 1
    else:
        _check(out, "out", torch.bfloat16, index)
        if out.shape != q.shape:
            raise ValueError(f"out must have the shape of q, got {tuple(out.shape)}")
        _no_grad("attend_shared_prefix", out)
    _, _, out_token, out_head = _rows(out, "out")
    lse = torch.empty((tokens, q_heads), dtype=torch.float32, device=q.device) if return_lse else None
    if tokens and batch and blocks:
        need = _workspace_bytes(tokens, batch, q_heads, k_heads, prefix_len, index)
        if workspace is None:
            workspace = torch.empty(need, dtype=torch.uint8, device=q.device)
        elif not isinstance(workspace, torch.Tensor) or workspace.get_device() != index:
            raise ValueError("workspace must be a tensor on the device of q")
        size = workspace.numel() * workspace.element_size()
        if size < need or not workspace.is_contiguous() or workspace.data_ptr() & 31:
            raise ValueError(f"workspace must be contiguous, 32-byte aligned and hold {need} bytes")
        _launch("welm_rope_attend", index, q.data_ptr(), out.data_ptr(), None if lse is None else lse.data_ptr(),
                key_cache.data_ptr(), value_cache.data_ptr(), block_table.data_ptr(), seq_lens.data_ptr(), starts_ptr,
                prefix_ptr, prefix_len, tokens, batch, q_heads, k_heads, q_token, q_head, out_token, out_head, width,
                block_table.stride(0), blocks, block_size, key_strides, value_strides, scale, fill,
                workspace.data_ptr(), size, _status(status, index))
    else:  # no request, or no block to hold a key
        if blocks == 0 and tokens and batch:
            raise ValueError("the cache has no blocks")
        if fill:
            out.zero_()
        if lse is not None:
            lse.fill_(float("-inf"))
    _written(out)
    return (out, lse) if return_lse else out

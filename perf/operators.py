"""Measurement cases of the multi-axis rotary embedding, the rotating KV-cache
append and the paged attention with a shared prefix, with their plain forms.

``run`` computes an operator in elementary torch operations where ``own`` is
false, and through ``testfiles_b200`` where it is true; ``exact`` computes the
same outputs from the definitions in 64 bits.  Heads are the package's: 256
lanes, of which the last 64 are rotated (lanes 192..223 against 224..255).
"""

from __future__ import annotations

import math
import random

import torch

own = False

HEAD_DIM = 256
ROPE_DIM = 64
HALF = 32
LANE0 = HEAD_DIM - ROPE_DIM
MAX_POSITION = 32768
ROPE_BASE = 10000.0


def listed() -> list[dict]:
    return [
        # one decode step of a small multimodal batch: launch latency
        dict(name="axes_decode_16", op="axes", tokens=16, q_heads=6, k_heads=1, sections="16,8,8",
             interleaved=False, fused=False, train=False),
        # prefill of an image's tokens, in place on the fused projection output, pairs dealt out in turn
        dict(name="axes_image_4099", op="axes", tokens=4099, q_heads=6, k_heads=1, sections="12,10,10",
             interleaved=True, fused=True, train=False),
        # a training step over video tokens: rotated copies and the gradients of both inputs
        dict(name="axes_train_16384", op="axes", tokens=16384, q_heads=6, k_heads=1, sections="16,8,8",
             interleaved=False, fused=False, train=True),
        # one decode step of 32 requests, padded to the captured batch size: launch latency
        dict(name="append_decode_32", op="append", tokens=32, pad=5, q_heads=6, k_heads=1, block_size=64,
             sections="", fused=True),
        # prefill of a ragged batch with several KV heads, small pages
        dict(name="append_prefill_5001", op="append", tokens=5001, pad=0, q_heads=8, k_heads=2, block_size=16,
             sections="", fused=True),
        # the longest prefill chunk, multi-axis positions
        dict(name="append_prefill_16384", op="append", tokens=16384, pad=0, q_heads=6, k_heads=1, block_size=64,
             sections="16,8,8", fused=True),
        # a single request's decode step: latency
        dict(name="attend_decode_1", op="attend", batch=1, q_len=1, prefix=0, length=300, spread=False, q_heads=6,
             k_heads=1, block_size=64, lse=False),
        # decode of unrelated requests, no prefix in common: the own keys' bandwidth
        dict(name="attend_decode_48", op="attend", batch=48, q_len=1, prefix=0, length=4000, spread=True, q_heads=6,
             k_heads=1, block_size=64, lse=False),
        # many continuations of one long document
        dict(name="attend_shared_128", op="attend", batch=128, q_len=1, prefix=16384, length=512, spread=True,
             q_heads=6, k_heads=1, block_size=64, lse=False),
        # verification of a few drafted tokens a request, several KV heads, odd prefix, small pages
        dict(name="attend_verify_24", op="attend", batch=24, q_len=5, prefix=4097, length=700, spread=True,
             q_heads=8, k_heads=2, block_size=16, lse=True),
        # several prompts' chunks read against one shared system prompt
        dict(name="attend_chunk_4", op="attend", batch=4, q_len=640, prefix=8192, length=900, spread=False, q_heads=6,
             k_heads=1, block_size=64, lse=False),
        # the largest serving batch over the longest prefix
        dict(name="attend_shared_256", op="attend", batch=256, q_len=1, prefix=32768, length=1500, spread=True,
             q_heads=6, k_heads=1, block_size=64, lse=False),
    ]


def _log_int(rng: random.Random, low: int, high: int) -> int:
    """An integer of [low, high], its logarithm uniform."""
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


_SECTIONS = ("16,8,8", "12,10,10", "32", "8,12,12", "10,22", "8,8,8,8")


def draw(rng: random.Random) -> dict:
    kind = rng.choice(("axes", "append", "attend", "attend"))
    q_heads, k_heads = rng.choice(((6, 1), (6, 1), (8, 2), (4, 4), (12, 2)))
    if kind == "axes":
        train = rng.random() < 0.5
        return dict(op="axes", tokens=_log_int(rng, 1, 16384 if q_heads == 6 else 8000), q_heads=q_heads,
                    k_heads=k_heads, sections=rng.choice(_SECTIONS), interleaved=rng.random() < 0.5,
                    fused=rng.random() < 0.5, train=train)
    if kind == "append":
        tokens = _log_int(rng, 1, 16384 if q_heads == 6 else 8000)
        return dict(op="append", tokens=tokens, pad=rng.randint(0, tokens // 4), q_heads=q_heads, k_heads=k_heads,
                    block_size=rng.choice((16, 32, 64, 128)), sections=rng.choice(("",) + _SECTIONS),
                    fused=rng.random() < 0.5)
    form = rng.choice(("decode", "shared", "verify", "chunk"))
    block_size = rng.choice((16, 32, 64, 128))
    if form == "decode":
        case = dict(batch=_log_int(rng, 1, 48), q_len=1, prefix=0, length=_log_int(rng, 1, 3500))
    elif form == "shared":
        case = dict(batch=_log_int(rng, 2, 200), q_len=1, prefix=_log_int(rng, 64, 24000),
                    length=_log_int(rng, 1, 800))
    elif form == "verify":
        case = dict(batch=_log_int(rng, 1, 48), q_len=rng.randint(2, 12), prefix=_log_int(rng, 1, 12000),
                    length=_log_int(rng, 16, 1500))
    else:
        case = dict(batch=rng.randint(1, 4), q_len=_log_int(rng, 32, 640), prefix=_log_int(rng, 1, 8000),
                    length=_log_int(rng, 700, 1000))
    if k_heads > 1:  # more rows, and pages of its own for every KV head
        case["batch"], case["prefix"] = -(-case["batch"] // k_heads), -(-case["prefix"] // k_heads)
    return dict(op="attend", **case, spread=rng.random() < 0.75, q_heads=q_heads, k_heads=k_heads,
                block_size=block_size, lse=rng.random() < 0.3)


# ---------------------------------------------------------------------------
# Shapes that follow from a case alone.
# ---------------------------------------------------------------------------
def _sections(case: dict) -> tuple[int, ...]:
    return tuple(int(x) for x in case["sections"].split(",")) if case["sections"] else ()


def _pair_axes(sections: tuple[int, ...], interleaved: bool) -> list[int]:
    """The axis of each of the 32 rotated pairs."""
    if not interleaved:
        return [a for a, n in enumerate(sections) for _ in range(n)]
    left, axes = list(sections), []
    while len(axes) < HALF:
        for a in range(len(left)):
            if left[a]:
                left[a] -= 1
                axes.append(a)
    return axes


def _lens(case: dict) -> tuple[list[int], list[int]]:
    """Each request's own cached length and its query tokens."""
    rng = random.Random("%d %d %d %d" % (case["batch"], case["q_len"], case["length"], case["prefix"]))
    lens, q_lens = [], []
    for _ in range(case["batch"]):
        n = rng.randint(1, case["q_len"]) if case["spread"] and case["q_len"] > 1 else case["q_len"]
        length = rng.randint(1, case["length"]) if case["spread"] else case["length"]
        q_lens.append(n)
        lens.append(max(length, n))
    return lens, q_lens


def work(case: dict) -> dict:
    if case["op"] == "axes":
        heads, tokens = case["q_heads"] + case["k_heads"], case["tokens"]
        gather = tokens * (8 * len(_sections(case)) + 4 * ROPE_DIM)
        if case["train"]:  # rotated copies of whole heads, and gradients of whole heads
            return {"bytes": 2 * (2 * heads * tokens * HEAD_DIM * 2) + gather, "flops": 2 * 6 * HALF * heads * tokens}
        return {"bytes": 2 * heads * tokens * ROPE_DIM * 2 + gather, "flops": 6 * HALF * heads * tokens}
    if case["op"] == "append":
        tokens = case["tokens"] - case["pad"]
        axes = max(1, len(_sections(case)))
        row = 2 * case["q_heads"] * ROPE_DIM * 2 + 4 * case["k_heads"] * HEAD_DIM * 2 + 8 * axes + 4 * ROPE_DIM
        return {"bytes": tokens * row + 8 * case["tokens"],
                "flops": 6 * HALF * (case["q_heads"] + case["k_heads"]) * tokens}
    lens, q_lens = _lens(case)
    tokens = sum(q_lens)
    pairs = sum(n * case["prefix"] + sum(length - n + i + 1 for i in range(n)) for length, n in zip(lens, q_lens))
    kv = (case["prefix"] + sum(lens)) * case["k_heads"] * HEAD_DIM * 2 * 2
    io = tokens * case["q_heads"] * (2 * HEAD_DIM * 2 + (4 if case["lse"] else 0))
    return {"bytes": kv + io, "flops": 4 * HEAD_DIM * case["q_heads"] * pairs}


# ---------------------------------------------------------------------------
# Inputs.
# ---------------------------------------------------------------------------
def _cos_sin(device: torch.device) -> torch.Tensor:
    inv = 1.0 / (ROPE_BASE ** (torch.arange(0, ROPE_DIM, 2, dtype=torch.float64, device=device) / ROPE_DIM))
    angle = torch.arange(MAX_POSITION, dtype=torch.float64, device=device)[:, None] * inv
    return torch.cat((angle.cos(), angle.sin()), dim=1).to(torch.float32)


def _heads(tokens: int, counts: tuple[int, ...], fused: bool, gen: torch.Generator) -> list[torch.Tensor]:
    """[tokens, n, 256] tensors for each count: views of one projection output, or tensors of their own."""
    if fused:
        whole = torch.randn((tokens, sum(counts), HEAD_DIM), dtype=torch.bfloat16, device="cuda", generator=gen)
        return list(whole.split(counts, dim=1))
    return [torch.randn((tokens, n, HEAD_DIM), dtype=torch.bfloat16, device="cuda", generator=gen) for n in counts]


def _axis_positions(tokens: int, axes: int, gen: torch.Generator) -> torch.Tensor:
    """Positions of a frame of image tokens that starts at a random place: time, height, width, ..."""
    start = torch.randint(0, MAX_POSITION - tokens, (1,), device="cuda", generator=gen)
    index = torch.arange(tokens, device="cuda")
    rows = [index] if axes == 1 else [index // 1024, index // 32 % 32, index % 32, index % 7][:axes]
    return start + torch.stack(rows)


def prepare(case: dict, seed: int) -> dict:
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    state = dict(case=case)
    if case["op"] == "axes":
        counts = (case["q_heads"], case["k_heads"])
        state["q"], state["k"] = _heads(case["tokens"], counts, case["fused"], gen)
        state["sections"] = _sections(case)
        state["positions"] = _axis_positions(case["tokens"], len(state["sections"]), gen)
        state["cos_sin"] = _cos_sin(state["q"].device)
        if case["train"]:
            state["grads"] = _heads(case["tokens"], counts, False, gen)
            state["q"].requires_grad_(True)
            state["k"].requires_grad_(True)
        return state
    if case["op"] == "append":
        tokens, live = case["tokens"], case["tokens"] - case["pad"]
        state["q"], state["k"], state["v"] = _heads(tokens, (case["q_heads"], case["k_heads"], case["k_heads"]),
                                                    case["fused"], gen)
        blocks = -(-(live + live // 4 + 1) // case["block_size"])
        shape = (blocks, case["block_size"], case["k_heads"], HEAD_DIM)
        state["key_cache"] = torch.randn(shape, dtype=torch.bfloat16, device="cuda", generator=gen)
        state["value_cache"] = torch.randn(shape, dtype=torch.bfloat16, device="cuda", generator=gen)
        slots = torch.full((tokens,), -1, dtype=torch.int64, device="cuda")
        index = torch.arange(live, device="cuda")  # whole pages in a random order
        pages = torch.randperm(blocks, device="cuda", generator=gen)
        slots[:live] = pages[index // case["block_size"]] * case["block_size"] + index % case["block_size"]
        state["slots"] = slots
        state["sections"] = _sections(case)
        positions = _axis_positions(tokens, max(1, len(state["sections"])), gen)
        state["positions"] = positions if state["sections"] else positions[0]
        state["cos_sin"] = _cos_sin(slots.device)
        return state
    lens, q_lens = _lens(case)
    size, k_heads = case["block_size"], case["k_heads"]
    state["q"] = torch.randn((sum(q_lens), case["q_heads"], HEAD_DIM), dtype=torch.bfloat16, device="cuda",
                             generator=gen)
    prefix_blocks = -(-case["prefix"] // size)
    own_blocks = [-(-n // size) for n in lens]
    blocks = prefix_blocks + sum(own_blocks) + 1
    shape = (blocks, size, k_heads, HEAD_DIM)
    state["key_cache"] = torch.randn(shape, dtype=torch.bfloat16, device="cuda", generator=gen)
    state["value_cache"] = torch.randn(shape, dtype=torch.bfloat16, device="cuda", generator=gen)
    pages = torch.randperm(blocks, generator=gen, device="cuda").to(torch.int32).cpu()
    table = torch.zeros((len(lens), max(own_blocks)), dtype=torch.int32)
    at = prefix_blocks
    for b, n in enumerate(own_blocks):
        table[b, :n] = pages[at:at + n]
        at += n
    starts = torch.zeros(len(lens) + 1, dtype=torch.int64)
    starts[1:] = torch.tensor(q_lens).cumsum(0)
    state["block_table"] = table.cuda()
    state["prefix_table"] = pages[:prefix_blocks].cuda()
    state["seq_lens"] = torch.tensor(lens, dtype=torch.int64).cuda()
    state["query_starts"] = starts.cuda() if case["q_len"] > 1 else None
    state["most"] = (max(lens), max(q_lens))
    return state


# ---------------------------------------------------------------------------
# One pass.
# ---------------------------------------------------------------------------
def run(state: dict):
    if own:
        return _run_own(state)
    return {"axes": _plain_axes, "append": _plain_append, "attend": _plain_attend}[state["case"]["op"]](state)


def _run_own(state: dict):
    import testfiles_b200 as welm

    case = state["case"]
    if case["op"] == "axes":
        if not case["train"]:
            welm.rope_multi_axis_inplace(state["q"], state["k"], state["positions"], state["cos_sin"],
                                         state["sections"], case["interleaved"])
            return state["q"], state["k"]
        q, k = welm.rope_multi_axis(state["q"], state["k"], state["positions"], state["cos_sin"], state["sections"],
                                    case["interleaved"])
        dq, dk = torch.autograd.grad((q, k), (state["q"], state["k"]), state["grads"])
        return q, k, dq, dk
    if case["op"] == "append":
        welm.rope_kv_append(state["q"], state["k"], state["v"], state["positions"], state["cos_sin"], state["slots"],
                            state["key_cache"], state["value_cache"], sections=state["sections"] or None)
        return state["q"], state["key_cache"], state["value_cache"]
    return welm.attend_shared_prefix(state["q"], state["key_cache"], state["value_cache"], state["block_table"],
                                     state["seq_lens"], query_starts=state["query_starts"],
                                     prefix_table=state["prefix_table"], prefix_len=case["prefix"],
                                     return_lse=case["lse"])


def _plain_cos_sin(state: dict, interleaved: bool) -> tuple[torch.Tensor, torch.Tensor]:
    """cos and sin of each (token, pair), [tokens, 1, 32] in 32 bits."""
    positions = state["positions"]
    if positions.dim() == 1:
        rows = state["cos_sin"][positions]
        return rows[:, None, :HALF], rows[:, None, HALF:]
    axes = torch.tensor(_pair_axes(state["sections"], interleaved), device=positions.device)
    at = positions[axes].t()  # [tokens, 32]
    pair = torch.arange(HALF, device=positions.device)
    return state["cos_sin"][at, pair][:, None], state["cos_sin"][at, pair + HALF][:, None]


def _plain_rotate(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    x1, x2 = x[..., LANE0:LANE0 + HALF].float(), x[..., LANE0 + HALF:].float()
    return torch.cat((x1 * cos - x2 * sin, x1 * sin + x2 * cos), dim=-1).to(x.dtype)


def _plain_whole(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    return torch.cat((x[..., :LANE0], _plain_rotate(x, cos, sin)), dim=-1)


def _plain_axes(state: dict):
    q, k = state["q"].detach(), state["k"].detach()
    cos, sin = _plain_cos_sin(state, state["case"]["interleaved"])
    if not state["case"]["train"]:
        q[..., LANE0:] = _plain_rotate(q, cos, sin)
        k[..., LANE0:] = _plain_rotate(k, cos, sin)
        return q, k
    dq, dk = state["grads"]
    return (_plain_whole(q, cos, sin), _plain_whole(k, cos, sin), _plain_whole(dq, cos, -sin),
            _plain_whole(dk, cos, -sin))


def _plain_append(state: dict):
    q, k, v, slots = state["q"], state["k"], state["v"], state["slots"]
    live = (slots >= 0).nonzero()[:, 0]
    cos, sin = _plain_cos_sin(state, False)
    q[live, :, LANE0:] = _plain_rotate(q[live], cos[live], sin[live])
    k_heads = k.shape[1]
    state["key_cache"].view(-1, k_heads, HEAD_DIM)[slots[live]] = _plain_whole(k[live], cos[live], sin[live])
    state["value_cache"].view(-1, k_heads, HEAD_DIM)[slots[live]] = v[live]
    return q, state["key_cache"], state["value_cache"]


def _plain_attend(state: dict):
    case, q = state["case"], state["q"]
    k_heads, group, prefix = case["k_heads"], case["q_heads"] // case["k_heads"], case["prefix"]
    tokens, batch = q.shape[0], case["batch"]
    most_len, most_q = state["most"]
    scale = HEAD_DIM ** -0.5
    starts = state["query_starts"]
    if starts is None:
        starts = torch.arange(batch + 1, device=q.device)
    count = starts[1:] - starts[:-1]
    step = torch.arange(most_q, device=q.device)
    there = step < count[:, None]  # [batch, most_q]
    token = torch.where(there, starts[:-1, None] + step, 0)
    qf = q.float() * scale
    # each request against its own pages, padded to the longest
    rows = qf.view(tokens, k_heads, group, HEAD_DIM)[token]  # [batch, most_q, k_heads, group, 256]
    rows = rows.permute(0, 2, 1, 3, 4).reshape(batch, k_heads, most_q * group, HEAD_DIM)
    keys = state["key_cache"][state["block_table"].long()].flatten(1, 2)[:, :most_len].float().transpose(1, 2)
    values = state["value_cache"][state["block_table"].long()].flatten(1, 2)[:, :most_len].float().transpose(1, 2)
    score = rows @ keys.transpose(2, 3)
    last = (state["seq_lens"] - count)[:, None] + step  # the last position that a query token sees
    seen = torch.arange(most_len, device=q.device) <= last[:, :, None]
    seen = seen.repeat_interleave(group, dim=1)[:, None]
    score = score.masked_fill(~seen, -math.inf)
    top = score.amax(dim=3)
    if prefix:
        flat = qf.view(tokens, k_heads, group, HEAD_DIM).transpose(0, 1).reshape(k_heads, tokens * group, HEAD_DIM)
        table = state["prefix_table"].long()
        p_keys = state["key_cache"][table].flatten(0, 1)[:prefix].float().transpose(0, 1)
        p_values = state["value_cache"][table].flatten(0, 1)[:prefix].float().transpose(0, 1)
        p_score = flat @ p_keys.transpose(1, 2)  # [k_heads, tokens * group, prefix]
        place = (token[:, :, None] * group + torch.arange(group, device=q.device)).flatten(1)
        top = torch.maximum(top, p_score.amax(dim=2)[:, place].transpose(0, 1))
    shift = torch.where(top == -math.inf, 0, top)
    weight = torch.exp(score - shift[..., None])
    total = weight.sum(dim=3)
    mixed = weight @ values
    # back to one row for each token and head: [k_heads, tokens, group, ...]
    whole = lambda x: x.unflatten(2, (most_q, group)).transpose(1, 2)[there].transpose(0, 1)  # noqa: E731
    total, mixed, shift = whole(total), whole(mixed), whole(shift)
    if prefix:
        weight = torch.exp(p_score - shift.reshape(k_heads, tokens * group)[..., None])
        total = total + weight.sum(dim=2).view_as(total)
        mixed = mixed + (weight @ p_values).view_as(mixed)
    out = torch.where(total[..., None] > 0, mixed / total[..., None], 0)
    out = out.transpose(0, 1).reshape(tokens, k_heads * group, HEAD_DIM).to(q.dtype)
    if not case["lse"]:
        return out
    return out, (shift + total.log()).transpose(0, 1).reshape(tokens, k_heads * group)


# ---------------------------------------------------------------------------
# The definitions in 64 bits.
# ---------------------------------------------------------------------------
def _exact_rotated(x: torch.Tensor, state: dict, interleaved: bool, sign: float) -> torch.Tensor:
    """Each pair (x1, x2) as the complex number x1 + i x2, times cos + i sin."""
    positions = state["positions"] if state["positions"].dim() == 2 else state["positions"][None]
    sections = state["sections"] or (HALF,)
    out = x.double().clone()
    for pair, axis in enumerate(_pair_axes(sections, interleaved)):
        row = state["cos_sin"].double()[positions[axis]]
        turn = torch.complex(row[:, pair], sign * row[:, HALF + pair])[:, None]
        turned = torch.complex(out[..., LANE0 + pair], out[..., LANE0 + HALF + pair]) * turn
        out[..., LANE0 + pair], out[..., LANE0 + HALF + pair] = turned.real, turned.imag
    return out


def exact(case: dict, seed: int):
    state = prepare(case, seed)
    if case["op"] == "axes":
        q, k = state["q"].detach(), state["k"].detach()
        rotated = [_exact_rotated(x, state, case["interleaved"], 1.0) for x in (q, k)]
        if not case["train"]:
            return tuple(rotated)
        return (*rotated, *(_exact_rotated(x, state, case["interleaved"], -1.0) for x in state["grads"]))
    if case["op"] == "append":
        live = case["tokens"] - case["pad"]
        q = _exact_rotated(state["q"], state, False, 1.0)
        q[live:] = state["q"][live:].double()
        keys, values = state["key_cache"].double(), state["value_cache"].double()
        block, place = state["slots"][:live] // case["block_size"], state["slots"][:live] % case["block_size"]
        keys[block, place] = _exact_rotated(state["k"], state, False, 1.0)[:live]
        values[block, place] = state["v"][:live].double()
        return q, keys, values
    lens, q_lens = _lens(case)
    group = case["q_heads"] // case["k_heads"]
    outs, sums = [], []
    table = state["prefix_table"].long()
    p_keys = state["key_cache"][table].flatten(0, 1)[:case["prefix"]].double()
    p_values = state["value_cache"][table].flatten(0, 1)[:case["prefix"]].double()
    at = 0
    for b, (length, n) in enumerate(zip(lens, q_lens)):
        pages = state["block_table"][b].long()
        keys = torch.cat((p_keys, state["key_cache"][pages].flatten(0, 1)[:length].double()))
        values = torch.cat((p_values, state["value_cache"][pages].flatten(0, 1)[:length].double()))
        mask = torch.ones((n, keys.shape[0]), dtype=torch.bool, device=keys.device).tril(keys.shape[0] - n)
        o = torch.empty((n, case["q_heads"], HEAD_DIM), dtype=torch.float64, device=keys.device)
        s = torch.empty((n, case["q_heads"]), dtype=torch.float64, device=keys.device)
        for h in range(case["q_heads"]):
            logit = state["q"][at:at + n, h].double() @ keys[:, h // group].t() / math.sqrt(HEAD_DIM)
            logit[~mask] = -math.inf
            s[:, h] = logit.logsumexp(dim=1)
            o[:, h] = logit.softmax(dim=1) @ values[:, h // group]
        outs.append(o)
        sums.append(s)
        at += n
    if not case["lse"]:
        return torch.cat(outs)
    return torch.cat(outs), torch.cat(sums)

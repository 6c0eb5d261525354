"""GPU tests of the multi-axis rotary embedding, in place and differentiable,
against the 64-bit oracle, finite differences and the ordinary entry."""

from __future__ import annotations

import pytest
import torch

import paged_oracle
import testfiles_b200 as welm
from testfiles_b200 import _native, workloads

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
ROWS = 4096


def make(tokens, axes, heads=(6, 1), seed=0):
    g = torch.Generator().manual_seed(seed + tokens)
    qkv = torch.randn((tokens, sum(heads) + heads[1], 256), generator=g).to(torch.bfloat16)
    positions = torch.randint(0, ROWS, (axes, tokens), generator=g)
    return qkv, qkv[:, :heads[0]], qkv[:, heads[0]:sum(heads)], positions, workloads.make_cos_sin_cache(ROWS, 10000.0)


def close(got, x, positions, cos_sin, sections, interleaved, inverse=False):
    exact = paged_oracle.rotate(x.cpu(), positions, cos_sin, sections, interleaved, inverse)
    off = (got.cpu().double() - exact).abs()
    assert (off <= paged_oracle.rotate_bound(x.cpu(), exact)).all()
    assert torch.equal(got.cpu()[..., :192], x.cpu()[..., :192])


@pytest.mark.parametrize("sections", [(16, 8, 8), (12, 10, 10), (32,), (0, 32), (1, 30, 1), (8, 8, 8, 8), (0, 5, 0, 27)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,heads", [(1, (6, 1)), (77, (6, 1)), (300, (8, 2)), (33, (1, 3))])
def test_in_place_and_copies(tokens, heads, sections, interleaved):
    qkv, q, k, positions, cos_sin = make(tokens, len(sections), heads)
    for inverse in (False, True):
        d = qkv.to(DEV)
        dq, dk = d[:, :heads[0]], d[:, heads[0]:sum(heads)]
        status = torch.zeros(1, dtype=torch.int32, device=DEV)
        args = (positions.to(DEV), cos_sin.to(DEV), sections, interleaved, inverse, status)
        q_out, k_out = welm.rope_multi_axis(dq, dk, *args)
        assert torch.equal(d.cpu(), qkv)
        welm.rope_multi_axis_inplace(dq, dk, *args)
        assert torch.equal(dq, q_out) and torch.equal(dk, k_out)
        assert torch.equal(d[:, sum(heads):].cpu(), qkv[:, sum(heads):])
        close(dq, q, positions, cos_sin, sections, interleaved, inverse)
        close(dk, k, positions, cos_sin, sections, interleaved, inverse)
        assert status.item() == 0


def test_one_axis_equals_the_ordinary_entry():
    qkv, q, k, positions, cos_sin = make(5000, 1)
    a, b = qkv.to(DEV), qkv.to(DEV)
    welm.rope_multi_axis_inplace(a[:, :6], a[:, 6:7], positions.to(DEV), cos_sin.to(DEV), (32,))
    welm.welmv4_inplace_rope_npu(b[:, :6], b[:, 6:7], positions[0].to(DEV), cos_sin.to(DEV))
    assert torch.equal(a, b)


def test_axis_rows_may_be_views():
    qkv, q, k, positions, cos_sin = make(90, 3)
    wide = torch.full((3, 200), -1, dtype=torch.int64, device=DEV)
    wide[:, 50:140] = positions.to(DEV)
    d = qkv.to(DEV)
    welm.rope_multi_axis_inplace(d[:, :6], d[:, 6:7], wide[:, 50:140], cos_sin.to(DEV), (16, 8, 8))
    close(d[:, :6], q, positions, cos_sin, (16, 8, 8), False)
    same = positions[:1].expand(3, 90)  # one position for every axis
    e = qkv.to(DEV)
    welm.rope_multi_axis_inplace(e[:, :6], e[:, 6:7], same.to(DEV)[:1].expand(3, 90), cos_sin.to(DEV), (16, 8, 8))
    close(e[:, :6], q, same, cos_sin, (16, 8, 8), False)


def test_bad_positions_leave_the_token():
    qkv, q, k, positions, cos_sin = make(64, 3)
    positions[0, 3], positions[1, 9], positions[2, 20] = -1, ROWS, 2 ** 40
    for sections, skipped in (((16, 16, 0), (3, 9)), ((16, 8, 8), (3, 9, 20))):  # an axis of no pairs is not read
        d = qkv.to(DEV)
        status = torch.zeros(1, dtype=torch.int32, device=DEV)
        args = (positions.to(DEV), cos_sin.to(DEV), sections, False, False, status)
        q_out, k_out = welm.rope_multi_axis(d[:, :6], d[:, 6:7], *args)
        assert status.item() == _native.DEV_BAD_POSITION
        status.zero_()
        welm.rope_multi_axis_inplace(d[:, :6], d[:, 6:7], *args)
        assert status.item() == _native.DEV_BAD_POSITION
        assert torch.equal(d[:, :6], q_out) and torch.equal(d[:, 6:7], k_out)
        for t in skipped:
            assert torch.equal(d[t].cpu(), qkv[t])
        close(d[:, :6], q, positions, cos_sin, sections, False)


def test_not_a_number_stays_in_its_pair():
    qkv, q, k, positions, cos_sin = make(10, 3)
    qkv[4, 2, 200] = float("nan")
    qkv[5, 6, 230] = float("inf")
    d = qkv.to(DEV)
    welm.rope_multi_axis_inplace(d[:, :6], d[:, 6:7], positions.to(DEV), cos_sin.to(DEV), (16, 8, 8))
    bad = (~torch.isfinite(d.cpu())).nonzero().tolist()
    assert set(map(tuple, bad)) <= {(4, 2, 200), (4, 2, 232), (5, 6, 198), (5, 6, 230)}
    assert [4, 2, 200] in bad and [4, 2, 232] in bad and [5, 6, 230] in bad


def test_head_major_and_odd_layouts():
    qkv, q, k, positions, cos_sin = make(50, 3, (4, 2))
    args = (positions.to(DEV), cos_sin.to(DEV), (16, 8, 8))
    turned = q.to(DEV).transpose(0, 1).contiguous().transpose(0, 1)
    want_q, want_k = welm.rope_multi_axis(q.to(DEV), k.to(DEV), *args)
    got = welm.rope_multi_axis(turned, k.to(DEV), *args)
    assert torch.equal(got[0], want_q)
    kk = k.to(DEV).contiguous()
    welm.rope_multi_axis_inplace(turned, kk, *args)
    assert torch.equal(turned, want_q) and torch.equal(kk, want_k)
    # the function takes any layout: lanes apart, a start off 16 bytes, one row for all
    lanes = torch.empty((50, 4, 512), dtype=torch.bfloat16, device=DEV)[..., ::2]
    lanes.copy_(q)
    odd = torch.empty(50 * 4 * 256 + 1, dtype=torch.bfloat16, device=DEV)[1:].view(50, 4, 256)
    odd.copy_(q)
    for x in (lanes, odd):
        assert torch.equal(welm.rope_multi_axis(x, k.to(DEV), *args)[0], want_q)
    one = q[:1].to(DEV).expand(50, 4, 256)
    assert torch.equal(welm.rope_multi_axis(one, k.to(DEV), *args)[0],
                       welm.rope_multi_axis(one.contiguous(), k.to(DEV), *args)[0])


def test_gradients():
    """The gradients against the formula: the inverse rotation of what comes back."""
    qkv, q, k, positions, cos_sin = make(200, 3, (8, 2))
    args = (positions.to(DEV), cos_sin.to(DEV), (12, 10, 10), True)
    a, b = q.to(DEV).contiguous().requires_grad_(), k.to(DEV).contiguous().requires_grad_()
    out = welm.rope_multi_axis(a, b, *args)
    grads = [torch.randn_like(x) for x in out]
    for got, grad in zip(torch.autograd.grad(out, (a, b), grads, retain_graph=True), grads):
        close(got, grad, positions, cos_sin, (12, 10, 10), True, inverse=True)
    # one output alone, a broadcast gradient, one input that needs none
    only_q, only_k = torch.autograd.grad(out[0], (a, b), grads[0], allow_unused=True, retain_graph=True)
    assert only_k is None
    close(only_q, grads[0], positions, cos_sin, (12, 10, 10), True, inverse=True)
    ones = torch.ones((), dtype=torch.bfloat16, device=DEV).expand(out[1].shape)
    from_sum = torch.autograd.grad(out[1].sum(), b, retain_graph=True)[0]
    close(from_sum, ones, positions, cos_sin, (12, 10, 10), True, inverse=True)
    frozen = welm.rope_multi_axis(a, b.detach(), *args)
    assert not torch.autograd.grad(frozen[0].float().sum(), a)[0].isnan().any()


def test_gradients_of_shared_and_expanded_inputs():
    qkv, q, k, positions, cos_sin = make(64, 3)
    args = (positions.to(DEV), cos_sin.to(DEV), (16, 8, 8))
    row = q[:1, :1].to(DEV).contiguous().requires_grad_()
    out, _ = welm.rope_multi_axis(row.expand(64, 6, 256), k.to(DEV), *args)
    grad = torch.randn_like(out)
    got = torch.autograd.grad(out, row, grad)[0]
    each = paged_oracle.rotate(grad.cpu(), positions, cos_sin, (16, 8, 8), inverse=True)
    bound = paged_oracle.rotate_bound(grad.cpu(), each)
    # the sum over 384 rows in FP32 and its rounding
    want = each.sum((0, 1))
    allowed = bound.sum((0, 1)) + 384 * 2.0 ** -24 * each.abs().sum((0, 1)) + want.abs() * 2.0 ** -8
    assert ((got.cpu().double()[0, 0] - want).abs() <= allowed).all()
    both = q[:, :1].to(DEV).contiguous().requires_grad_()  # the same tensor as Q and K
    a, b = welm.rope_multi_axis(both, both, *args)
    assert torch.equal(a, b)
    g = torch.randn_like(a)
    one = torch.autograd.grad(a, both, g, retain_graph=True)[0]
    two = torch.autograd.grad((a, b), both, (g, g))[0]
    assert torch.equal(two, one * 2)


def test_gradient_against_differences():
    """The rotation is linear: with a step that BF16 holds exactly, the difference quotient of sum(w * out) in the
    kernel's own outputs is the gradient up to the outputs' roundings."""
    qkv, q, k, positions, cos_sin = make(8, 3)
    args = (positions.to(DEV), cos_sin.to(DEV), (16, 8, 8))
    a = q.to(DEV).contiguous().requires_grad_()
    b = k.to(DEV).contiguous()
    out, _ = welm.rope_multi_axis(a, b, *args)
    w = torch.randn_like(out)
    grad = torch.autograd.grad(out, a, w)[0]
    step = 64.0
    for t, h, lane in ((0, 0, 192), (3, 5, 255), (7, 2, 223), (5, 1, 100)):
        ends = []
        for sign in (1, -1):
            x = torch.zeros_like(a)
            x[t, h, lane] = sign * step
            ends.append((welm.rope_multi_axis(x, b, *args)[0].double() * w.double()).sum().item())
        weight = w[t, h].double().abs()
        pair = {lane} if lane < 192 else {192 + lane % 32, 224 + lane % 32}
        allowed = (2.0 ** -8 + 2.0 ** -22) * sum(weight[i].item() for i in pair) * 2  # outputs, and the gradient
        assert abs((ends[0] - ends[1]) / (2 * step) - grad[t, h, lane].item()) <= allowed


def test_second_derivative():
    qkv, q, k, positions, cos_sin = make(16, 3)
    args = (positions.to(DEV), cos_sin.to(DEV), (16, 8, 8))
    a, b = q.to(DEV).contiguous().requires_grad_(), k.to(DEV).contiguous()
    out, _ = welm.rope_multi_axis(a, b, *args)
    w = torch.randn_like(out).requires_grad_()
    grad, = torch.autograd.grad(out, a, w, create_graph=True)
    v = torch.randn_like(a)
    back, = torch.autograd.grad(grad, w, v)  # the rotation of v
    assert torch.equal(back, welm.rope_multi_axis(v, b, *args)[0])


def test_captured_step_and_other_stream():
    qkv, q, k, positions, cos_sin = make(700, 3)
    d, pos, cache = qkv.to(DEV), positions.to(DEV), cos_sin.to(DEV)
    source = d.clone()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        a = d[:, :6].contiguous().requires_grad_()
        b = d[:, 6:7].contiguous().requires_grad_()
        w = torch.ones_like(a)
        torch.autograd.grad(welm.rope_multi_axis(a, b, pos, cache, (16, 8, 8))[0], a, w)  # warm up
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            d.copy_(source)
            welm.rope_multi_axis_inplace(d[:, :6], d[:, 6:7], pos, cache, (16, 8, 8))
            out = welm.rope_multi_axis(a, b, pos, cache, (16, 8, 8))
            grad, = torch.autograd.grad(out[0], a, w)
    torch.cuda.synchronize()
    for seed in (1, 2):
        new = torch.randint(0, ROWS, positions.shape, generator=torch.Generator().manual_seed(seed))
        pos.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        close(d[:, :6], q, new, cos_sin, (16, 8, 8), False)
        assert torch.equal(out[0], d[:, :6]) and torch.equal(out[1], d[:, 6:7])
        close(grad, torch.ones_like(q), new, cos_sin, (16, 8, 8), False, inverse=True)


def test_no_tokens():
    cos_sin = workloads.make_cos_sin_cache(64, 10000.0).to(DEV)
    q = torch.zeros((0, 6, 256), dtype=torch.bfloat16, device=DEV).requires_grad_()
    k = torch.zeros((0, 1, 256), dtype=torch.bfloat16, device=DEV)
    pos = torch.zeros((3, 0), dtype=torch.int64, device=DEV)
    a, b = welm.rope_multi_axis(q, k, pos, cos_sin, (16, 8, 8))
    assert a.shape == q.shape and b.shape == k.shape
    assert torch.autograd.grad(a.float().sum(), q)[0].shape == q.shape


def test_in_place_write_is_seen_by_autograd():
    """A tensor saved for a backward pass and then rotated in place must not go unnoticed."""
    qkv, q, k, positions, cos_sin = make(4, 3)
    a, b = q.to(DEV).contiguous(), k.to(DEV).contiguous()
    w = torch.ones_like(a).requires_grad_()
    y = (a * w).sum()
    welm.rope_multi_axis_inplace(a, b, positions.to(DEV), cos_sin.to(DEV), (16, 8, 8))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_gradients_of_one_input_and_of_one_output():
    """Inputs and outputs that no gradient is wanted of or comes from; a second pass through a freed graph is refused."""
    qkv, q, k, positions, cos_sin = make(33, 3)
    pos, cache = positions.to(DEV), cos_sin.to(DEV)
    for wants in ((True, False), (False, True), (True, True)):
        a, b = (t.to(DEV).contiguous().requires_grad_(w) for t, w in zip((q, k), wants))
        outs = welm.rope_multi_axis(a, b, pos, cache, (16, 8, 8))
        for which in (0, 1):
            w = torch.ones_like(outs[which])
            got = torch.autograd.grad(outs[which], [t for t in (a, b) if t.requires_grad], w, retain_graph=True,
                                      allow_unused=True)
            whole = iter(got)
            for i, t in enumerate((a, b)):
                if not t.requires_grad:
                    continue
                g = next(whole)
                if i != which:
                    assert g is None or (g == 0).all()
                else:
                    close(g, torch.ones_like((q, k)[i]), positions, cos_sin, (16, 8, 8), False, inverse=True)
        outs[0].sum().backward()
        with pytest.raises(RuntimeError, match="second time"):
            outs[0].sum().backward()


def test_positions_changed_before_the_backward_pass_are_noticed():
    qkv, q, k, positions, cos_sin = make(5, 3)
    a, b, pos = q.to(DEV).contiguous().requires_grad_(), k.to(DEV).contiguous(), positions.to(DEV)
    out = welm.rope_multi_axis(a, b, pos, cos_sin.to(DEV), (16, 8, 8))[0]
    pos.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()


def test_forward_mode_is_refused():
    import torch.autograd.forward_ad as fwad
    qkv, q, k, positions, cos_sin = make(5, 3)
    a, b = q.to(DEV).contiguous(), k.to(DEV).contiguous()
    with fwad.dual_level(), pytest.raises(NotImplementedError):
        welm.rope_multi_axis(fwad.make_dual(a, torch.ones_like(a)), b, positions.to(DEV), cos_sin.to(DEV), (16, 8, 8))

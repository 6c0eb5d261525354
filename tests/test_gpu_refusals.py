"""GPU tests: what the paged operators refuse beside types, shapes and devices,
before anything is launched."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

import testfiles_b200 as welm
from test_paged_refusals import DEV, tensors

pytestmark = pytest.mark.gpu


def axes_args(**change):
    t = tensors()
    args = dict(q=t["q"], k=t["k"], positions=torch.zeros((3, 4), dtype=torch.int64, device=DEV),
                cos_sin_cache=t["cos_sin_cache"], sections=(16, 8, 8))
    return {**args, **change}


def test_q_and_k_that_overlap():
    whole = torch.zeros((4, 8, 256), dtype=torch.bfloat16, device=DEV)
    for q, k in ((whole, whole), (whole[:, :6], whole[:, 5:6]), (whole[:, :6], whole[:, 2:4])):
        with pytest.raises(ValueError, match="overlap"):
            welm.rope_multi_axis_inplace(**axes_args(q=q, k=k))
    q_out, _ = welm.rope_multi_axis(**axes_args(q=whole, k=whole))  # copies may come from the same rows
    assert q_out.shape == whole.shape
    welm.rope_multi_axis_inplace(**axes_args(q=whole[:, :6], k=whole[:, 6:7]))


def test_append_with_tensors_that_overlap():
    def append(**change):
        args = {**tensors(), **change}
        welm.rope_kv_append(**args)
        return args

    t = tensors()
    whole = torch.zeros((4, 8, 256), dtype=torch.bfloat16, device=DEV)
    pages = torch.zeros((2, 2, 16, 1, 256), dtype=torch.bfloat16, device=DEV)
    flat = pages.view(-1, 1, 256)
    for bad in (dict(value_cache=t["key_cache"], key_cache=t["key_cache"]), dict(q=whole, k=whole[:, 7:]),
                dict(q=whole, v=whole[:, :1]), dict(q=flat[:4], key_cache=pages[:, 0], value_cache=pages[:, 1]),
                dict(q=flat[16:20], key_cache=pages[:, 0], value_cache=pages[:, 1])):
        with pytest.raises(ValueError, match="overlap"):
            append(**bad)
    # interleaved caches, views of one projection, and keys that are rotated where they lie
    append(q=whole[:, :6], k=whole[:, 6:7], v=whole[:, 7:], key_cache=pages[:, 0], value_cache=pages[:, 1])
    keys = torch.randn((32, 1, 256), device=DEV).to(torch.bfloat16)
    cos_sin = torch.randn((8, 64), device=DEV)
    want = append(k=keys[:4].clone(), cos_sin_cache=cos_sin)["key_cache"].view(32, 1, 256)[:4]
    append(q=None, k=keys[:4], key_cache=keys.view(2, 16, 1, 256), cos_sin_cache=cos_sin)
    assert torch.equal(keys[:4], want)


def attend_args(**change):
    t = tensors()
    args = dict(q=t["q"], key_cache=t["key_cache"], value_cache=t["value_cache"],
                block_table=torch.zeros((4, 1), dtype=torch.int32, device=DEV),
                seq_lens=torch.ones(4, dtype=torch.int64, device=DEV))
    return {**args, **change}


def test_an_out_that_overlaps_what_attention_reads():
    q = torch.zeros((4, 12, 256), dtype=torch.bfloat16, device=DEV)
    pages = torch.zeros((2, 16, 1, 256), dtype=torch.bfloat16, device=DEV)
    for bad in (dict(q=q[:, :6], out=q[:, :6]), dict(q=q[:, :6], out=q[:, 5:11]),
                dict(key_cache=pages, out=pages.view(-1)[:6144].view(4, 6, 256)),
                dict(value_cache=pages, out=pages.view(-1)[:6144].view(4, 6, 256))):
        with pytest.raises(ValueError, match="overlap"):
            welm.attend_shared_prefix(**attend_args(**bad))
    args = attend_args(q=q[:, :6], out=q[:, 6:])
    assert welm.attend_shared_prefix(**args) is args["out"]  # heads of one tensor, apart


@pytest.mark.parametrize("entry,args,names", [
    (welm.rope_multi_axis_inplace, axes_args, ("q", "k")),
    (welm.rope_kv_append, lambda **c: {**tensors(), **c}, ("q", "k", "v", "key_cache", "value_cache")),
    (welm.attend_shared_prefix, attend_args, ("q", "key_cache", "value_cache", "out")),
])
def test_forward_mode_tensors(entry, args, names):
    """Their tangents would be lost, or stay as they were beside a tensor that has changed."""
    for name in names:
        given = args()
        plain = given.get(name, torch.zeros((4, 6, 256), dtype=torch.bfloat16, device=DEV))
        with forward_ad.dual_level():
            dual = forward_ad.make_dual(plain, torch.ones_like(plain))
            for ctx in (torch.enable_grad, torch.no_grad):
                with ctx(), pytest.raises(NotImplementedError, match="forward-mode"):
                    entry(**args(**{name: dual}))
        assert (plain == 0).all()


@pytest.mark.parametrize("entry,args", [
    (welm.rope_multi_axis_inplace, axes_args), (welm.rope_multi_axis, axes_args),
    (welm.rope_kv_append, lambda **c: {**tensors(), **c}),
])
def test_a_cos_sin_cache_whose_gradient_would_be_lost(entry, args):
    table = torch.zeros((8, 64), device=DEV, requires_grad=True)
    with pytest.raises(ValueError, match="no backward pass"):
        entry(**args(cos_sin_cache=table))
    with torch.no_grad():
        entry(**args(cos_sin_cache=table))
    entry(**args(cos_sin_cache=table.detach()))
    with forward_ad.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
        entry(**args(cos_sin_cache=forward_ad.make_dual(table.detach(), torch.ones((8, 64), device=DEV))))


@pytest.mark.parametrize("scale", [1e-60, 2.9e38, 1e60, float("inf"), float("nan"), -1.0])
def test_scales_that_fp32_does_not_hold(scale):
    with pytest.raises(ValueError, match="scale"):
        welm.attend_shared_prefix(**attend_args(scale=scale))

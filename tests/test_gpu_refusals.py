"""GPU tests: what the paged operators refuse beside types, shapes and devices,
before anything is launched."""

from __future__ import annotations

import pytest
import torch

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

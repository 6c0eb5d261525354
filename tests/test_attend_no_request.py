"""The C entry of attention with no request at all: every row is one of none."""

from __future__ import annotations

import math

import pytest
import torch

from testfiles_b200 import _native
from test_paged_refusals import FAKE, attend


def test_refusals():
    none = dict(b=0, starts=FAKE, fill=1)
    assert attend(**none, out=None) == _native.ERR_NULL_POINTER
    assert attend(**none, oh=4) == attend(**none, oh=0) == attend(**none, out=FAKE + 2) == _native.ERR_BAD_STRIDE
    assert attend(b=0, starts=FAKE, out=None) == _native.OK  # nothing to do


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,heads", [(1, 1), (5, 6), (700, 7)])
@pytest.mark.parametrize("fill", [0, 1])
@pytest.mark.parametrize("with_lse", [False, True])
def test_rows_become_zeros_or_stay_and_their_lse_is_minus_infinity(tokens, heads, fill, with_lse):
    whole = torch.full((tokens + 1, heads + 1, 256), 7.0, dtype=torch.bfloat16, device="cuda:0")
    lse = torch.full((tokens + 1, heads), 7.0, device="cuda:0")
    args = dict(n=tokens, b=0, hq=heads, hk=1, starts=FAKE, out=whole.data_ptr(), ot=whole.stride(0), oh=256, fill=fill,
                lse=lse.data_ptr() if with_lse else None)
    assert attend(**args) == _native.OK
    out = whole[:tokens, :heads]
    assert (out == (0.0 if fill else 7.0)).all()
    out.fill_(7.0)
    assert (whole == 7.0).all()
    assert (lse[:tokens] == (-math.inf if with_lse else 7.0)).all() and (lse[tokens] == 7.0).all()

"""GPU tests of attention where a wait inside the kernel gives up, and without
programmatic dependent launches.  Both switches are read once a process, so
children run them."""

from __future__ import annotations

import os
import subprocess
import sys
import textwrap

import pytest

from conftest import REPO

pytestmark = pytest.mark.gpu

SHAPES = textwrap.dedent("""
    import math, sys, torch
    sys.path[:0] = [".", "tests"]
    from testfiles_b200 import _native
    from test_gpu_attend import Batch, agree
    shapes = [dict(lens=[300]), dict(lens=[0, 1, 700], prefix=1000), dict(lens=[30] * 40, prefix=130),
              dict(lens=[1 + 37 * b % 150 for b in range(400)], prefix=70), dict(lens=[900], counts=[700], prefix=1500),
              dict(lens=[70, 20], counts=[2, 1], prefix=100, spare=4), dict(lens=[0, 0], prefix=0)]
""")


def child(code, **env):
    out = subprocess.run([sys.executable, "-c", SHAPES + textwrap.dedent(code)], cwd=REPO, env={**os.environ, **env},
                         capture_output=True, text=True, timeout=240)
    assert out.returncode == 0 and out.stdout.strip().endswith("ok"), out.stdout[-1000:] + out.stderr[-2000:]


def test_rows_of_a_call_that_gave_up_are_no_numbers():
    """The first wait that is not over ends the call.  Its status says so, no row keeps what memory held
    before, rows of no request are as ever, and the next call of the process can be made."""
    child("""
        for shape in shapes:
            batch = Batch(**shape)
            n = batch.tokens
            for out in (None, torch.full_like(batch.q, 7.0)):
                got, lse = batch.run(out=out)
                torch.cuda.synchronize()
                assert batch.status.item() == _native.DEV_WAIT_TIMEOUT, shape
                assert torch.isnan(got[:n]).all() and torch.isnan(lse[:n]).all(), shape
                assert (got[n:] == (0.0 if out is None else 7.0)).all() and (lse[n:] == -math.inf).all(), shape
                batch.status.zero_()
        assert (torch.ones(5, device="cuda:0") * 2).sum().item() == 10.0
        print("ok")
    """, WELM_ROPE_GIVE_UP="1")


@pytest.mark.parametrize("env", [dict(WELM_ROPE_PDL="0"), dict(WELM_ROPE_GIVE_UP="0")])
def test_results_with_other_settings(env):
    child("""
        for shape in shapes:
            batch = Batch(**shape)
            agree(batch, [x[:batch.tokens] for x in batch.run()])
            assert batch.status.item() == 0
        print("ok")
    """, **env)

"""CPU checks of the bench's result check: the recorded digests hold for the
recorded inputs, and a host whose cos/sin table differs in a last bit is not
told that the results are wrong."""

from __future__ import annotations

import pytest
import torch

from oracle import rope_oracle
from test_bench_contract import load_bench
from testfiles_b200 import workloads

CASE = "b_prefill_m577"


def outputs(inp):
    return rope_oracle.reference_outputs(inp.query, inp.key, inp.positions, inp.last_index, inp.cache)


def record(bench, q, k):
    return bench.parity_record(None, 0, q, k, [q.shape[0]], [k.shape[0]], CASE)


@pytest.mark.parametrize("table", ["recorded", "other"])
def test_results_are_compared_with_those_of_the_same_inputs(monkeypatch, table):
    bench = load_bench()
    if table == "other":  # every sine and cosine off by one step in FP32, enough to turn some BF16 roundings
        cache = workloads.cache_for("baseline")
        off = (cache.view(torch.int32) + (cache != 0)).view(torch.float32)
        monkeypatch.setattr(workloads, "cache_for", lambda flavour: off)
    inp = workloads.make_inputs(workloads.find_case(CASE), "cpu")
    recorded = bench.sha256_rows(inp.cache) == bench.golden_case(CASE)["cache"]
    assert table == "recorded" or not recorded
    q, k = outputs(inp)
    right = record(bench, q, k)
    assert right["bit_exact"] is True and right["max_ulp"] == 0
    assert ("reference's own" in right["compared_with"]) == recorded
    q[3, 2, 200] += 1
    assert record(bench, q, k)["bit_exact"] is False

"""CPU tests: tensors whose rows share memory where the call would write one
while another is read or written are refused, and views that merely interleave
are not taken for such."""

from __future__ import annotations

import ctypes
import random
import subprocess

import pytest

from testfiles_b200 import _native, build
from test_paged_refusals import AXES, FAKE, append, attend, i64, multi_axis

SOURCE = r"""
#include "rope_rows.h"
extern "C" int meet(int64_t a, const int64_t* an, const int64_t* as, int64_t b, const int64_t* bn, const int64_t* bs) {
  RowSet x{uintptr_t(a), {an[0], an[1], an[2]}, {as[0], as[1], as[2]}};
  RowSet y{uintptr_t(b), {bn[0], bn[1], bn[2]}, {bs[0], bs[1], bs[2]}};
  return rows_meet(x, y);
}
"""


@pytest.fixture(scope="module")
def meet(tmp_path_factory):
    """rows_meet of csrc/rope_rows.h: addresses in bytes, strides in elements of two bytes."""
    where = tmp_path_factory.mktemp("rows")
    (where / "meet.cpp").write_text(SOURCE)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", "-I", str(build.CSRC), "-I",
                    str(build.REPO_ROOT / "include"), str(where / "meet.cpp"), "-o", str(where / "meet.so")],
                   check=True)
    f = ctypes.CDLL(str(where / "meet.so")).meet
    arr = lambda v: (ctypes.c_int64 * 3)(*v)  # noqa: E731
    return lambda a, an, as_, b, bn, bs: bool(f(ctypes.c_int64(a), arr(an), arr(as_), ctypes.c_int64(b), arr(bn),
                                               arr(bs)))


def brute(a, an, as_, b, bn, bs):
    def starts(at, n, s):
        return {at // 2 + i * s[0] + j * s[1] + k * s[2]
                for i in range(n[0]) for j in range(n[1]) for k in range(n[2])}

    right = sorted(starts(b, bn, bs))
    return any(abs(x - y) < 256 for x in starts(a, an, as_) for y in right)


def test_against_every_pair_of_rows(meet):
    rng = random.Random(7)
    seen = {False: 0, True: 0}
    for _ in range(4000):
        step = rng.choice([8, 64, 256])
        a, b = (2 * step * rng.randint(0, 60) for _ in range(2))
        an, bn = ([rng.choice([0, 1, 1, 2, 3, 5, 9]) for _ in range(3)] for _ in range(2))
        pool = [step * rng.randint(0, 40) for _ in range(4)]
        as_, bs = ([rng.choice(pool) for _ in range(3)] for _ in range(2))
        want = brute(a, an, as_, b, bn, bs)
        assert meet(a, an, as_, b, bn, bs) == want, (a, an, as_, b, bn, bs)
        assert meet(b, bn, bs, a, an, as_) == want
        seen[want] += 1
    assert min(seen.values()) > 500


def test_usual_views(meet):
    n, one = 16384, [1, 1, 1]
    fused = [2048, 256, 0]  # [tokens, 8 heads, 256]
    assert not meet(0, [n, 6, 1], fused, 2 * 1536, [n, 1, 1], fused)
    assert not meet(0, [n, 6, 1], fused, 2 * 1792, [n, 1, 1], fused)
    assert meet(0, [n, 6, 1], fused, 2 * 1280, [n, 1, 1], fused)
    assert meet(0, [n, 6, 1], fused, 0, [n, 6, 1], fused)
    major = [256, n * 256, 0]  # [heads, tokens, 256], turned
    assert not meet(0, [n, 6, 1], major, 2 * 6 * n * 256, [n, 1, 1], major)
    assert meet(0, [n, 6, 1], major, 2 * 5 * n * 256, [n, 2, 1], major)
    mixed = [5 * 768, 768, 0]  # [tokens, 5 heads, (q, k, v), 256]
    for i in range(3):
        for j in range(3):
            assert meet(512 * i, [n, 5, 1], mixed, 512 * j, [n, 5, 1], mixed) == (i == j)
    pages = [2 * 64 * 256, 256, 256]  # [blocks, (K, V), 64, 1, 256]
    assert not meet(0, [9999, 64, 1], pages, 2 * 64 * 256, [9999, 64, 1], pages)
    assert meet(0, [9999, 64, 1], pages, 2 * 63 * 256, [9999, 64, 1], pages)
    row = [4096, 256, 0]
    assert not meet(0, one, row, 512, one, row) and meet(0, one, row, 510, one, row)
    assert not meet(0, [n, 0, 1], fused, 0, [n, 6, 1], fused)  # no rows
    big = 2 ** 60
    assert not meet(0, [2 ** 30, 6, 1], [big, 256, 0], 2 * 1536, [2 ** 30, 1, 1], [big, 256, 0])


def test_multi_axis_refuses_q_and_k_that_share_rows():
    """In place both are rotated, so a shared row would be rotated once or twice, as it happens."""
    other = FAKE + 2 * 1536 * 4
    assert multi_axis() == _native.ERR_BAD_STRIDE  # the same memory as Q and K
    assert multi_axis(k=FAKE + 2 * 1280, ko=FAKE + 2 * 1280, kt=1536, kot=1536) == _native.ERR_BAD_STRIDE
    # copies: outputs apart from one another, and from inputs that another thread may still read
    far = 1 << 30
    assert multi_axis(qo=far, ko=far) == _native.ERR_BAD_STRIDE
    assert multi_axis(k=other, ko=far, qo=FAKE + 512) == _native.ERR_BAD_STRIDE
    assert multi_axis(k=other, qo=other, ko=far) == _native.ERR_BAD_STRIDE
    assert multi_axis(k=other, qo=far, ko=FAKE) == _native.ERR_BAD_STRIDE
    assert set(AXES) >= {"q", "qo", "k", "ko"}


def test_append_refuses_what_it_writes_to_overlap():
    """Q, keys and values are written: none may share a row with another, nor Q with what is read."""
    qkv = dict(q=FAKE, k=FAKE + 2 * 1536, v=FAKE + 2 * 1792)
    far, page = 1 << 30, 2 * 4096
    for bad in (dict(q=None, hq=0, kc=far, vc=far),  # one cache for both
                dict(qkv, kc=far, vc=far + 3 * page), dict(qkv, kc=FAKE, vc=far), dict(qkv, kc=far, vc=FAKE + 2 * 2048),
                dict(qkv, k=FAKE + 2 * 1280, kc=far, vc=2 * far), dict(qkv, v=FAKE, kc=far, vc=2 * far),
                dict(qkv, kc=far, vc=far + 2 * 256, ks=i64(8192, 512, 256), vs=i64(8192, 256, 256))):
        assert append(**bad) == _native.ERR_BAD_STRIDE, bad


def test_attend_refuses_an_out_that_overlaps_what_it_reads():
    far, page = 1 << 30, 2 * 4096
    for bad in (dict(kc=far, vc=far), dict(q=FAKE + 2 * 256, kc=far, vc=far), dict(out=far, vc=2 * far),
                dict(out=far, kc=2 * far), dict(out=far + 3 * page, kc=far, vc=2 * far),
                dict(q=2 * far, out=far - 2 * 5376, kc=3 * far, vc=far)):  # its last rows in the first page
        assert attend(**{**dict(kc=far, vc=far), **bad}) == _native.ERR_BAD_STRIDE, bad

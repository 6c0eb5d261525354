"""CPU tests: what the multi-axis rotary embedding, the cache append and the
paged attention refuse, at the C entries (before any CUDA call) and in Python."""

from __future__ import annotations

import ctypes

import pytest
import torch

import testfiles_b200 as welm
from testfiles_b200 import _native, build

FAKE = 0x1000  # a non-NULL address; every call below is rejected before it is used


def i32(*v):
    return (ctypes.c_int32 * len(v))(*v)


def i64(*v):
    return (ctypes.c_int64 * len(v))(*v)


AXES = dict(q=FAKE, qo=FAKE, k=FAKE, ko=FAKE, pos=FAKE, cache=FAKE, sec=i32(16, 8, 8), axes=3, inter=0, inv=0, n=4,
            hq=6, hk=1, qt=1536, qh=256, qot=1536, qoh=256, kt=256, kh=256, kot=256, koh=256, ps=4, mp=16)


def multi_axis(**kw):
    return _native.load().welm_rope_multi_axis(*{**AXES, **kw}.values(), None, None)


def test_multi_axis_entry():
    assert multi_axis(axes=0) == multi_axis(axes=5) == multi_axis(inter=2) == multi_axis(inv=-1) == _native.ERR_BAD_MODE
    assert multi_axis(sec=i32(16, 8, 7)) == multi_axis(sec=i32(16, 17, -1)) == _native.ERR_BAD_MODE
    assert multi_axis(sec=i32(2 ** 31 - 1, 2 ** 31 - 1, 34)) == _native.ERR_BAD_MODE
    assert multi_axis(n=-1) == multi_axis(hq=-1) == multi_axis(mp=-1) == _native.ERR_BAD_SIZE
    assert multi_axis(n=2 ** 40) == multi_axis(hq=2 ** 62) == _native.ERR_BAD_SIZE
    for name in ("q", "qo", "k", "ko", "pos", "cache", "sec"):
        assert multi_axis(**{name: None}) == _native.ERR_NULL_POINTER, name
    assert multi_axis(qt=1535, qot=1535) == multi_axis(koh=4, kh=4, hk=2) == _native.ERR_BAD_STRIDE
    assert multi_axis(qot=255, qt=255) == multi_axis(kot=0, kt=0) == _native.ERR_BAD_STRIDE  # outputs overlap
    assert multi_axis(qt=2048) == _native.ERR_BAD_STRIDE  # in place with other strides
    assert multi_axis(q=FAKE + 2, qo=FAKE + 2) == multi_axis(cache=FAKE + 4) == _native.ERR_BAD_STRIDE
    assert multi_axis(ps=-4) == multi_axis(qo=FAKE + 16, qt=-8) == _native.ERR_BAD_STRIDE
    assert multi_axis(n=0) == multi_axis(hq=0, hk=0) == _native.OK


APPEND = dict(q=FAKE, k=FAKE, v=FAKE, pos=FAKE, cache=FAKE, sec=i32(32), axes=1, inter=0, slots=FAKE, kc=FAKE, vc=FAKE,
              n=4, hq=6, hk=1, qt=2048, qh=256, kt=2048, kh=256, vt=2048, vh=256, nb=4, bs=16, ks=i64(4096, 256, 256),
              vs=i64(4096, 256, 256), ps=0, mp=16)


def append(**kw):
    return _native.load().welm_rope_kv_append(*{**APPEND, **kw}.values(), None, None)


def test_append_entry():
    assert append(axes=0) == append(sec=i32(31)) == append(inter=7) == _native.ERR_BAD_MODE
    assert append(n=-1) == append(hk=0) == append(bs=0) == append(nb=-1) == append(mp=-1) == _native.ERR_BAD_SIZE
    assert append(n=2 ** 40) == append(nb=2 ** 62, bs=4) == append(hk=2 ** 62) == _native.ERR_BAD_SIZE
    for name in ("q", "k", "v", "pos", "cache", "sec", "slots", "kc", "vc", "ks", "vs"):
        assert append(**{name: None}) == _native.ERR_NULL_POINTER, name
    assert append(qt=1528) == append(kt=2047) == append(vh=-8) == _native.ERR_BAD_STRIDE
    assert append(ks=i64(4088, 256, 256)) == append(vs=i64(4096, 0, 256)) == _native.ERR_BAD_STRIDE  # slots overlap
    assert append(ks=i64(4096, 260, 256)) == append(k=FAKE + 8) == append(vc=FAKE + 2) == _native.ERR_BAD_STRIDE
    assert append(n=0) == _native.OK


ATTEND = dict(q=FAKE, out=FAKE, lse=None, kc=FAKE, vc=FAKE, table=FAKE, lens=FAKE, starts=None, pt=FAKE, p=10, n=4, b=4,
              hq=6, hk=1, qt=1536, qh=256, ot=1536, oh=256, width=2, ts=2, nb=4, bs=16, ks=i64(4096, 256, 256),
              vs=i64(4096, 256, 256), scale=0.0625, fill=0, ws=FAKE, wb=2 ** 40)


def attend(**kw):
    return _native.load().welm_rope_attend(*{**ATTEND, **kw}.values(), None, None)


def test_attend_entry():
    assert attend(n=-1) == attend(b=-1) == attend(hk=0) == attend(hq=0) == attend(p=-1) == _native.ERR_BAD_SIZE
    assert attend(hq=7, hk=2) == attend(n=2 ** 40, b=2 ** 40) == attend(p=2 ** 40) == _native.ERR_BAD_SIZE
    assert attend(b=3) == _native.ERR_BAD_SIZE  # one token a request, but 4 tokens for 3
    assert attend(bs=12) == attend(bs=0) == attend(nb=0) == attend(nb=2 ** 40) == _native.ERR_BAD_SIZE
    assert attend(width=-1) == attend(width=2 ** 30) == _native.ERR_BAD_SIZE
    nan, inf = float("nan"), float("inf")
    assert attend(scale=0.0) == attend(scale=-1.0) == attend(scale=nan) == attend(scale=inf) == _native.ERR_BAD_MODE
    assert attend(fill=2) == _native.ERR_BAD_MODE
    for name in ("q", "out", "kc", "vc", "table", "lens", "pt", "ks", "vs", "ws"):
        assert attend(**{name: None}) == _native.ERR_NULL_POINTER, name
    assert attend(ot=1528) == attend(oh=0) == attend(qt=-8) == attend(ts=-1) == _native.ERR_BAD_STRIDE
    assert attend(qh=260) == attend(q=FAKE + 2) == attend(kc=FAKE + 8) == attend(ws=FAKE + 8) == _native.ERR_BAD_STRIDE
    assert attend(ks=i64(4096, 128, 256)) == attend(vs=i64(2 ** 40, 256, 256)) == _native.ERR_BAD_STRIDE
    assert attend(n=0, b=0) == attend(n=0, b=3, starts=FAKE) == attend(b=0, starts=FAKE) == _native.OK


def test_workspace_entry():
    size = ctypes.c_int64(-1)
    f = _native.load().welm_rope_attend_workspace
    assert f(4, 4, 6, 1, 10, None) == _native.ERR_NULL_POINTER
    assert f(4, 4, 6, 4, 10, ctypes.byref(size)) == _native.ERR_BAD_SIZE
    assert f(-1, 4, 6, 1, 10, ctypes.byref(size)) == _native.ERR_BAD_SIZE
    assert size.value == -1


def test_python_refuses_cpu_tensors():
    q, k = torch.zeros((4, 6, 256), dtype=torch.bfloat16), torch.zeros((4, 1, 256), dtype=torch.bfloat16)
    pos, cache = torch.zeros((3, 4), dtype=torch.int64), torch.zeros((8, 64))
    for call in (welm.rope_multi_axis, welm.rope_multi_axis_inplace):
        with pytest.raises(ValueError, match="CUDA"):
            call(q, k, pos, cache, (16, 8, 8))
    with pytest.raises(ValueError, match="CUDA"):
        welm.rope_kv_append(q, k, k, pos[0], cache, pos[0], k[None], k[None])
    with pytest.raises(ValueError, match="CUDA"):
        welm.attend_shared_prefix(q, k[None], k[None], pos.int(), pos[0])


def test_binding_is_built_and_of_the_librarys_version():
    assert build.BINDING.exists(), "run python -m testfiles_b200.build"
    from testfiles_b200 import _welm_torch

    with pytest.raises(TypeError, match="13 arguments"):
        _welm_torch.attend()


DEV = "cuda:0"


def tensors():
    bf = dict(dtype=torch.bfloat16, device=DEV)
    return dict(q=torch.zeros((4, 6, 256), **bf), k=torch.zeros((4, 1, 256), **bf), v=torch.zeros((4, 1, 256), **bf),
                positions=torch.zeros(4, dtype=torch.int64, device=DEV), cos_sin_cache=torch.zeros((8, 64), device=DEV),
                slot_mapping=torch.arange(4, device=DEV), key_cache=torch.zeros((2, 16, 1, 256), **bf),
                value_cache=torch.zeros((2, 16, 1, 256), **bf))


@pytest.mark.gpu
@pytest.mark.parametrize("change,error", [
    (dict(q=lambda t: t.float()), TypeError), (dict(k=lambda t: t.cpu()), ValueError),
    (dict(v=lambda t: t.cpu()), ValueError), (dict(q=lambda t: t[:3]), ValueError),
    (dict(v=lambda t: t.expand(4, 2, 256)), ValueError), (dict(q=lambda t: t[..., :128]), ValueError),
    (dict(q=lambda t: t[:1].expand(4, 6, 256)), RuntimeError), (dict(positions=lambda t: t.int()), TypeError),
    (dict(positions=lambda t: t[:3]), ValueError), (dict(positions=lambda t: t[None]), ValueError),
    (dict(slot_mapping=lambda t: t[::2]), ValueError), (dict(cos_sin_cache=lambda t: t[:, :32]), ValueError),
    (dict(key_cache=lambda t: t[0]), ValueError), (dict(key_cache=lambda t: t[:1]), ValueError),
    (dict(key_cache=lambda t: t.expand(2, 16, 2, 256), value_cache=lambda t: t.expand(2, 16, 2, 256)), ValueError),
    (dict(key_cache=lambda t: t[:, :1].expand(2, 16, 1, 256)), RuntimeError),
    (dict(k=lambda t: t.requires_grad_()), ValueError), (dict(status=torch.zeros(1)), TypeError),
    (dict(key_cache=lambda t: t.requires_grad_()), ValueError),
    (dict(value_cache=lambda t: t.requires_grad_()), ValueError),
    (dict(sections=(16, 16)), ValueError),
])
def test_append_refuses(change, error):
    args = tensors()
    for name, how in change.items():
        args[name] = how(args[name]) if callable(how) else how
    with pytest.raises(error):
        welm.rope_kv_append(**args)


@pytest.mark.gpu
@pytest.mark.parametrize("change,error", [
    (dict(positions=lambda t: t[:2]), ValueError), (dict(positions=lambda t: t.t().contiguous().t()), ValueError),
    (dict(sections=(16, 8)), ValueError), (dict(sections=()), ValueError), (dict(sections=(8,) * 5), ValueError),
    (dict(sections=(40, -8, 0)), ValueError), (dict(sections="abc"), TypeError), (dict(sections=3), TypeError),
    (dict(sections=(16.0, 8, 8)), TypeError), (dict(q=None), ValueError), (dict(k=None), ValueError),
    (dict(positions=[0]), TypeError), (dict(q=lambda t: t[:3]), ValueError), (dict(k=lambda t: t.half()), TypeError),
    (dict(q=lambda t: t.requires_grad_()), ValueError), (dict(cos_sin_cache=lambda t: t.double()), TypeError),
    (dict(q=lambda t: torch.zeros(4 * 6 * 256 + 1, dtype=t.dtype, device=DEV)[1:].view(4, 6, 256)), ValueError),
    (dict(q=lambda t: t[:1].expand(4, 6, 256)), RuntimeError),
])
def test_multi_axis_inplace_refuses(change, error):
    t = tensors()
    args = dict(q=t["q"], k=t["k"], positions=torch.zeros((3, 4), dtype=torch.int64, device=DEV),
                cos_sin_cache=t["cos_sin_cache"], sections=(16, 8, 8))
    for name, how in change.items():
        args[name] = how(args[name]) if callable(how) else how
    with pytest.raises(error):
        welm.rope_multi_axis_inplace(**args)


@pytest.mark.gpu
@pytest.mark.parametrize("change,error", [
    (dict(q=lambda t: t[:3]), ValueError), (dict(q=lambda t: t.half()), TypeError),
    (dict(q=lambda t: t.requires_grad_()), ValueError), (dict(block_table=lambda t: t.long()), TypeError),
    (dict(key_cache=lambda t: t.requires_grad_()), ValueError),
    (dict(value_cache=lambda t: t.requires_grad_()), ValueError),
    (dict(block_table=lambda t: t[0]), ValueError), (dict(seq_lens=lambda t: t.int()), TypeError),
    (dict(seq_lens=lambda t: t[:2]), ValueError), (dict(query_starts=torch.zeros(3, dtype=torch.int64)), ValueError),
    (dict(prefix_len=17), ValueError), (dict(prefix_len=-1), ValueError), (dict(prefix_table=None), ValueError),
    (dict(scale=0.0), ValueError), (dict(scale=float("nan")), ValueError),
    (dict(value_cache=lambda t: t[:1]), ValueError),
    (dict(key_cache=lambda t: t[:, :12], value_cache=lambda t: t[:, :12]), ValueError),
    (dict(key_cache=lambda t: t.expand(2, 16, 4, 256), value_cache=lambda t: t.expand(2, 16, 4, 256)), ValueError),
    (dict(key_cache=lambda t: t[:0], value_cache=lambda t: t[:0]), ValueError),
    (dict(out=lambda t: torch.zeros((4, 6, 255), dtype=torch.bfloat16, device=DEV)), ValueError),
    (dict(out=lambda t: torch.zeros((4, 1, 256), dtype=torch.bfloat16, device=DEV).expand(4, 6, 256)), RuntimeError),
    (dict(workspace=lambda t: torch.zeros(64, dtype=torch.uint8, device=DEV)), ValueError),
    (dict(workspace=lambda t: torch.zeros(2 ** 26, dtype=torch.uint8)), ValueError),
])
def test_attend_refuses(change, error):
    t = tensors()
    args = dict(q=t["q"], key_cache=t["key_cache"], value_cache=t["value_cache"],
                block_table=torch.zeros((4, 1), dtype=torch.int32, device=DEV),
                seq_lens=torch.ones(4, dtype=torch.int64, device=DEV),
                prefix_table=torch.zeros(1, dtype=torch.int32, device=DEV), prefix_len=16)
    for name, how in change.items():
        args[name] = how(args.get(name)) if callable(how) else how
    with pytest.raises(error):
        welm.attend_shared_prefix(**args)

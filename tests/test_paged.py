"""CPU checks of the paged cache's host side: axis maps, argument checks that need no GPU."""
import ctypes
import struct

import pytest
import torch

from scope_b200 import _lib, paged

# ws_paged_kv and ws_rope (include/scope_b200.h)
paged_kv_pack = struct.Struct("@QQQQq12q6i").pack
rope_pack = struct.Struct("@QQqq6i32s").pack


def axes_of(packed, n):
    words = [int.from_bytes(packed[4 * i:4 * i + 4], "little") for i in range(8)]
    return [(words[i >> 4] >> (2 * (i & 15))) & 3 for i in range(n)]


@pytest.mark.parametrize("rot", [16, 48, 64, 128, 256])
def test_axis_map_of_one_axis_is_zero(rot):
    assert axes_of(paged.rope_axis_map(rot, None, False), rot // 2) == [0] * (rot // 2)


@pytest.mark.parametrize("rot,sections", [(128, (16, 24, 24)), (16, (4, 2, 2)), (256, (32, 32, 32, 32)), (64, (32, 0))])
def test_axis_map_blocks(rot, sections):
    want = [a for a, s in enumerate(sections) for _ in range(s)]
    assert axes_of(paged.rope_axis_map(rot, sections, False), rot // 2) == want


def test_axis_map_cyclic():
    got = axes_of(paged.rope_axis_map(128, (24, 20, 20), True), 64)
    assert [got.count(a) for a in range(3)] == [24, 20, 20]
    assert got[:6] == [0, 1, 2, 0, 1, 2] and got[60:] == [0, 0, 0, 0]


@pytest.mark.parametrize("rot,sections,cyclic", [
    (128, (16, 24, 23), False), (128, (), False), (64, (8, 8, 8, 4, 4), False), (16, (10, -2), False),
    (64, (4, 28), True)])
def test_axis_map_refuses(rot, sections, cyclic):
    with pytest.raises(RuntimeError, match="rope"):
        paged.rope_axis_map(rot, sections, cyclic)


def test_cpu_tensors_are_refused():
    i32 = torch.zeros(2, dtype=torch.int32)
    h = torch.zeros(2, 4, 32, dtype=torch.bfloat16)
    pool = torch.zeros(3, 8, 2, 32, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="CUDA"):
        paged.paged_slots(i32, i32, i32.view(1, 2), i32, i32, 16, 2)
    with pytest.raises(RuntimeError, match="CUDA"):
        paged.paged_release(i32, i32.bool(), i32.view(1, 2), i32, i32, 16)
    with pytest.raises(RuntimeError, match="CUDA"):
        paged.rope(h, i32, torch.zeros(8, 32))
    with pytest.raises(RuntimeError, match="CUDA"):
        paged.rope_append(None, h[:, :2], h[:, :2], None, None, torch.zeros(2, dtype=torch.int64), pool, pool)
    with pytest.raises(RuntimeError, match="CUDA"):
        paged.paged_decode(h, pool, pool, i32.view(2, 1), i32, 1.0)


def test_entries_check_their_arguments_before_any_launch():
    """Each of these is turned down on the host (there is no GPU here to launch on)."""
    L = _lib.lib()
    buf = ctypes.create_string_buffer(1 << 12)
    p = (ctypes.addressof(buf) + 255) // 256 * 256

    def kv(**change):
        f = dict(k=p, v=p, ks=0, vs=0, n=4, kp=2048, kt=128, kh=32, vp=2048, vt=128, vh=32, P=16, Hkv=4, Dk=32, Dv=32,
                 dt=_lib.WS_DTYPE_BF16)
        f.update(change)
        return paged_kv_pack(f["k"], f["v"], f["ks"], f["vs"], f["n"], f["kp"], f["kt"], f["kh"], f["vp"], f["vt"],
                                  f["vh"], 0, 0, 0, 0, 0, 0, f["P"], f["Hkv"], f["Dk"], f["Dv"], f["dt"], 0)

    def decode(pool, q=p, B=2, G=2, q_dtype=_lib.WS_DTYPE_BF16, stride=128, window=0, ws=p, nbytes=1 << 30, out=p):
        return L.ws_paged_decode(q, stride * G, stride, q_dtype, B, G, pool, p, 1, 1, p, window, 1.0, out, None, ws,
                                 nbytes, None)

    bad, unsupported, space = _lib.WS_ERR_INVALID_ARG, _lib.WS_ERR_UNSUPPORTED, _lib.WS_ERR_WORKSPACE
    for pool, want in ((kv(Dk=40), unsupported), (kv(Dv=272), unsupported), (kv(dt=_lib.WS_DTYPE_F32), bad),
                       (kv(kt=129), bad), (kv(k=p + 2), bad), (kv(P=0), bad), (kv(Hkv=0), bad), (kv(k=0), bad),
                       (kv(dt=_lib.WS_DTYPE_I8), bad), (kv(dt=_lib.WS_DTYPE_F16), bad)):
        assert decode(pool) == want
        assert L.ws_last_error().startswith(b"paged_decode")
    assert decode(kv(), G=0) == bad and decode(kv(), window=-1) == bad and decode(kv(), q=p + 2) == bad
    assert decode(kv(), stride=36) == bad and decode(kv(), q_dtype=_lib.WS_DTYPE_F32) == bad
    assert decode(kv(), out=None) == bad and decode(kv(), ws=None) == space and decode(kv(), nbytes=16) == space
    assert decode(kv(), B=0) == _lib.WS_OK

    def slots(B=2, width=4, stride=4, ring=8, P=16, n=2, ws=p, nbytes=1 << 30, lens=p):
        return L.ws_paged_slots(lens, p, B, p, stride, width, p, ring, p, P, n, p, p, p, p, p, ws, nbytes, None)

    assert slots(B=8193) == unsupported and slots(P=0) == bad and slots(width=0) == bad and slots(stride=3) == bad
    assert slots(ring=0) == bad and slots(n=-1) == bad and slots(lens=None) == bad
    assert slots(ws=None) == space and slots(nbytes=64) == space

    def append(rope, pool=kv(), H=2, D=32, dtype=_lib.WS_DTYPE_BF16, k=p):
        return L.ws_rope_append(rope, p, 64, 32, H, D, p, 64, 32, k, 128, 32, p, 128, 32, dtype, 3, p, pool, None)

    def rope(rot=32, axes=1, top=4, positions=p, amap=b""):
        return rope_pack(positions, p, 0, top, 0, axes, rot, 0, 0, 0, amap)

    assert append(rope(rot=8)) == bad and append(rope(rot=48)) == bad and append(rope(rot=24)) == bad
    assert append(rope(axes=5)) == bad and append(rope(top=0)) == bad and append(rope(positions=0)) == bad
    assert append(rope(axes=2, amap=b"\x02")) == bad   # a pair of axis 2 where two axes have positions
    assert append(rope(), D=48) == bad and append(rope(), k=None) == bad and append(rope(), pool=kv(n=0)) == bad
    assert append(rope(), dtype=_lib.WS_DTYPE_F32) == bad and append(rope(), dtype=_lib.WS_DTYPE_F16) == bad
    assert append(None, pool=None, D=20) == unsupported

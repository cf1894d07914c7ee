"""CPU checks of the 8-bit pages' and differential attention's host side: arguments that are turned down before any launch."""
import ctypes

import pytest
import torch

from scope_b200 import PagedKVCache, _lib, paged
from test_paged import paged_kv_pack

BAD, UNSUPPORTED, SPACE, OK = _lib.WS_ERR_INVALID_ARG, _lib.WS_ERR_UNSUPPORTED, _lib.WS_ERR_WORKSPACE, _lib.WS_OK
I8, E4, BF = _lib.WS_DTYPE_I8, _lib.WS_DTYPE_E4M3, _lib.WS_DTYPE_BF16


@pytest.fixture(scope="module")
def p():
    buf = ctypes.create_string_buffer(1 << 12)
    test = (ctypes.addressof(buf) + 255) // 256 * 256
    yield test
    del buf


def pool(p, **change):
    f = dict(k=p, v=p, ks=p, vs=p, n=4, kp=2048, kt=128, kh=32, P=16, Hkv=4, Dk=32, Dv=32, dt=I8, block=16)
    f.update(change)
    return paged_kv_pack(f["k"], f["v"], f["ks"], f["vs"], f["n"], f["kp"], f["kt"], f["kh"], f["kp"], f["kt"], f["kh"], 4, 4, 1,
                         4, 4, 1, f["P"], f["Hkv"], f["Dk"], f["Dv"], f["dt"], f["block"])


BAD_POOLS = [dict(block=3), dict(block=-1), dict(block=32), dict(P=24, dt=E4), dict(ks=0), dict(vs=0, dt=E4), dict(dt=5), dict(kt=120),
             dict(k=0), dict(Hkv=0)]


@pytest.mark.parametrize("change", range(len(BAD_POOLS)))
def test_pools_that_are_turned_down(p, change):
    L, kv = _lib.lib(), pool(p, **BAD_POOLS[change])
    assert L.ws_paged_decode(p, 256, 32, BF, 2, 2, kv, p, 1, 1, p, 0, 1.0, p, None, p, 1 << 30, None) == BAD
    assert L.ws_last_error().startswith(b"paged_decode: ")
    assert L.ws_paged_diff_decode(p, 256, 32, BF, 2, 2, kv, p, 1, 1, p, 0, 1.0, p, 1, None, 0.0, p, None, p, 1 << 30, None) == BAD
    assert L.ws_last_error().startswith(b"paged_diff_decode: ")
    assert L.ws_paged_read(kv, p, 1, 1, 2, p, None, 3, BF, p, p, None) == BAD
    assert L.ws_last_error().startswith(b"paged_read: ")
    assert L.ws_rope_append(None, None, 0, 0, 0, 32, None, 0, 0, p, 128, 32, p, 128, 32, BF, 3, p, kv, None) == BAD


def test_differential_decode(p):
    L = _lib.lib()

    def call(kv=pool(p), q=p, B=2, G=2, dt=BF, stride=32, lam=p, out=p, ws=p, nbytes=1 << 30, window=0):
        return L.ws_paged_diff_decode(q, 8 * stride, stride, dt, B, G, kv, p, 1, 1, p, window, 1.0, lam, 1, None, 1e-5, out, None,
                                      ws, nbytes, None)

    assert call(pool(p, Hkv=3)) == BAD and b"pairs" in L.ws_last_error()
    assert call(pool(p, Dk=144)) == UNSUPPORTED and call(pool(p, Dv=256)) == UNSUPPORTED and call(pool(p, Dk=24)) == UNSUPPORTED
    assert call(G=0) == BAD and call(G=1 << 20) == UNSUPPORTED and call(B=-1) == BAD and call(lam=None) == BAD
    assert call(q=p + 2) == BAD and call(stride=36) == BAD and call(out=p + 8) == BAD and call(dt=_lib.WS_DTYPE_F32) == BAD
    assert call(pool(p, dt=_lib.WS_DTYPE_F16)) == BAD and call(window=-1) == BAD
    assert call(ws=None) == SPACE and call(nbytes=64) == SPACE and call(B=0) == OK


def test_read(p):
    L = _lib.lib()

    def call(kv=pool(p), B=2, cu=p, n=3, dt=BF, k=p, v=p, pages=1, table=p):
        return L.ws_paged_read(kv, table, 1, pages, B, cu, None, n, dt, k, v, None)

    assert call(None) == BAD and call(B=-1) == BAD and call(n=-1) == BAD and call(pages=-1) == BAD
    assert call(dt=_lib.WS_DTYPE_F32) == BAD and call(pool(p, dt=_lib.WS_DTYPE_F16)) == BAD
    assert call(cu=None) == BAD and call(k=None) == BAD and call(v=p + 4) == BAD and call(table=None) == BAD
    assert call(pool(p, Dk=40)) == UNSUPPORTED
    assert call(B=0) == OK and call(n=0) == OK


def test_cpu_tensors_are_refused():
    i32, pages = torch.zeros(2, dtype=torch.int32), torch.zeros(3, 8, 2, 32, dtype=torch.int8)
    q, scales = torch.zeros(2, 4, 32, dtype=torch.bfloat16), torch.zeros(3, 1, 2)
    with pytest.raises(RuntimeError, match="CUDA"):
        paged.paged_diff_decode(q, pages, pages, i32.view(2, 1), i32, 1.0, torch.zeros(2), k_scales=scales, v_scales=scales)
    with pytest.raises(RuntimeError, match="CUDA"):
        paged.paged_read(pages, pages, i32.view(2, 1), torch.zeros(3, dtype=torch.int32), 4, k_scales=scales, v_scales=scales)


@pytest.mark.parametrize("kw", [dict(scale_block=3, dtype=torch.int8), dict(scale_block=0, dtype=torch.int8), dict(scale_block=16),
                                dict(scale_block=32, dtype=torch.float8_e4m3fn)])
def test_a_cache_of_blocks_that_do_not_fit(kw):
    with pytest.raises(RuntimeError, match="scale_block"):
        PagedKVCache(1, 4, 16, 1, 32, 1, 32, device="cpu", **kw)

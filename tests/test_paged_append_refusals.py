"""CPU checks that an append into blocks is turned down whole: before its queries, which may lie in place, are launched."""
import ctypes

import pytest

from scope_b200 import _lib
from test_paged import rope_pack
from test_paged_blocks import E4, I8, pool


@pytest.mark.parametrize("dt", [I8, E4])
@pytest.mark.parametrize("N,stride,why", [(3, 1 << 33, b"stride"), (1 << 20, 1 << 33, b"stride"), (1 << 20, -32, b"stride"),
                                          ((1 << 31) - 1000, 128, b"tokens")])
def test_an_append_is_turned_down_before_any_launch(dt, N, stride, why):
    """Long calls turn their queries in a launch of their own: without a device that one would fail as WS_ERR_CUDA."""
    L = _lib.lib()
    buf = ctypes.create_string_buffer(1 << 12)
    p = (ctypes.addressof(buf) + 255) // 256 * 256
    for rope in (None, rope_pack(p, p, 0, 4, 0, 1, 32, 0, 0, 0, b"")):
        rc = L.ws_rope_append(rope, p, 128, 32, 4, 32, p, 128, 32, p, stride, 32, p, 128, 32, _lib.WS_DTYPE_BF16, N, p, pool(p, dt=dt),
                              None)
        assert rc == _lib.WS_ERR_UNSUPPORTED and why in L.ws_last_error()

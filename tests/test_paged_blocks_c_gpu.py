"""GPU checks of the block append through the C ABI, where it takes what the Python call has no argument for.

Rotations and codes are whole formulas of fp32 operations: compared bit for bit.
"""
import ctypes

import pytest
import torch

import scope_b200
from scope_b200 import _lib, paged
from test_paged import paged_kv_pack, rope_pack
from test_paged_blocks_gpu import E4, I8, append_reference, make_pool, raw
from test_paged_gpu import BF, DEV, HF, gen, table_of, turned

pytestmark = pytest.mark.gpu
DTYPE = {BF: _lib.WS_DTYPE_BF16, HF: _lib.WS_DTYPE_F16, I8: _lib.WS_DTYPE_I8, E4: _lib.WS_DTYPE_E4M3}


def kv_of(k, v, ks, vs):
    """ws_paged_kv of a pool's tensors."""
    block = k.shape[1] // ks.shape[1] if ks is not None else 0
    at = [x.data_ptr() if x is not None else 0 for x in (k, v, ks, vs)]
    floats = [x.stride(i) if x is not None else 0 for x in (ks, vs) for i in range(3)]
    return paged_kv_pack(*at, k.shape[0], *k.stride()[:3], *v.stride()[:3], *floats, k.shape[1], k.shape[2], k.shape[3], v.shape[3],
                         DTYPE[k.dtype], block)


def append(rope, q, q_out, k, v, slots, kv):
    s = torch.cuda.current_stream().cuda_stream
    return _lib.lib().ws_rope_append(rope, q.data_ptr(), q.stride(0), q.stride(1), q.shape[1], q.shape[2], q_out.data_ptr(),
                                     q_out.stride(0), q_out.stride(1), k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(),
                                     v.stride(0), v.stride(1), DTYPE[q.dtype], q.shape[0], slots.data_ptr(), kv, ctypes.c_void_p(s))


# few tokens and many: the queries go with the keys, or ahead of them
@pytest.mark.parametrize("pool,block,N", [(I8, 16, 20), (I8, 16, 700), (E4, 16, 700), (E4, 128, 20), (E4, 128, 700), (E4, 1, 60)])
@pytest.mark.parametrize("aligned", [True, False])
@pytest.mark.parametrize("adjacent,axes", [(0, 1), (1, 1), (0, 2)])
def test_append_turned_back(pool, block, N, aligned, adjacent, axes):
    """`inverse` turns queries and keys back, wherever the rows go and however the turns lie."""
    g, H, Hkv, D, rot, P = gen(N + block), 4, 2, 80, 64, 128
    table = table_of(200, rot)
    if not aligned:   # 4 bytes past a boundary
        table = torch.cat([table.new_zeros(1), table.flatten()])[1:].view(200, rot)
    pos = torch.randint(0, 200, (axes, N), generator=g, device=DEV, dtype=torch.int32)
    of = [i * axes // (rot // 2) for i in range(rot // 2)]
    words = [sum(a << (2 * i) for i, a in enumerate(of[w:w + 16])) for w in range(0, rot // 2, 16)]
    q, k, v = (torch.randn(N, h, D, generator=g, device=DEV).to(BF) for h in (H, Hkv, Hkv))
    n_pages = -(-N // P) + 2
    (kp, ks), (vp, vs) = (make_pool(g, n_pages, P, block, Hkv, D, pool) for _ in range(2))
    slots = torch.arange(N, device=DEV) + 5
    pairs = "adjacent" if adjacent else "half"
    wk, wks = append_reference(turned(k, pos, table, of, pairs, True), slots, kp, ks, block)
    wv, wvs = append_reference(v.float(), slots, vp, vs, block)
    out = torch.empty_like(q)
    rope = rope_pack(pos.data_ptr(), table.data_ptr(), pos.stride(0), 200, 0, axes, rot, adjacent, 1, 0,
                     b"".join(w.to_bytes(4, "little") for w in words))
    assert append(rope, q, out, k, v, slots, kv_of(kp, vp, ks, vs)) == _lib.WS_OK
    assert torch.equal(out, turned(q, pos, table, of, pairs, True).to(BF))
    assert torch.equal(ks, wks) and torch.equal(vs, wvs)
    assert torch.equal(raw(kp), raw(wk)) and torch.equal(raw(vp), raw(wv))
    assert scope_b200.status_take() == 0


@pytest.mark.parametrize("N", [20, 3000])
def test_a_refused_append_leaves_the_queries(N):
    """In place, so a caller who falls back after the refusal does not turn them twice."""
    g, H, Hkv, D = gen(N), 4, 2, 64
    q, k, v = (torch.randn(N, h, D, generator=g, device=DEV).to(BF) for h in (H, Hkv, Hkv))
    (kp, ks), (vp, vs) = (make_pool(g, 200, 16, 16, Hkv, D, I8) for _ in range(2))
    table, pos = table_of(100, D), torch.randint(1, 100, (N,), generator=g, device=DEV, dtype=torch.int32)
    rope = rope_pack(pos.data_ptr(), table.data_ptr(), 0, 100, 0, 1, D, 0, 0, 0, b"")
    was, pages = q.clone(), kp.clone()
    kv = kv_of(kp, vp, ks, vs)
    L, s = _lib.lib(), ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    slots = torch.arange(N, device=DEV)
    rc = L.ws_rope_append(rope, q.data_ptr(), q.stride(0), q.stride(1), H, D, q.data_ptr(), q.stride(0), q.stride(1), k.data_ptr(),
                          1 << 33, D, v.data_ptr(), v.stride(0), v.stride(1), DTYPE[BF], N, slots.data_ptr(), kv, s)
    assert rc == _lib.WS_ERR_UNSUPPORTED
    torch.cuda.synchronize()
    assert torch.equal(q, was) and torch.equal(raw(kp), raw(pages))


def test_append_where_heads_lie_past_32_bits():
    """A pool with its heads outermost, each of more than 2^32 codes: its last pages."""
    n_pages, P, Hkv, D, block = 270000, 128, 2, 128, 16
    kp = torch.zeros(Hkv, n_pages, P, D, dtype=I8, device=DEV).permute(1, 2, 0, 3)
    vp = torch.zeros(n_pages, P, Hkv, 16, dtype=I8, device=DEV)
    ks, vs = (torch.zeros(n_pages, P // block, Hkv, device=DEV) for _ in range(2))
    assert kp.stride(2) > 1 << 32
    for N in (3, 1000):
        k = torch.randn(N, Hkv, D, generator=gen(N), device=DEV).to(BF)
        near = torch.arange(N, device=DEV) + 5     # in the last nine pages
        want = append_reference(k.float(), near, kp[-9:], ks[-9:], block)
        paged.rope_append(None, k, k[..., :16], None, None, near + (n_pages - 9) * P, kp, vp, k_scales=ks, v_scales=vs)
        assert torch.equal(raw(kp[-9:]), raw(want[0])) and torch.equal(ks[-9:], want[1])
    assert scope_b200.status_take() == 0

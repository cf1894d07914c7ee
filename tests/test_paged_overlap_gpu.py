"""GPU checks that an output given to a paged operator shares no memory with the pages, scales or tables it is made from."""
import pytest
import torch

from scope_b200 import paged
from test_paged_gpu import BF, DEV, table_of

pytestmark = pytest.mark.gpu
SHARED = "overlap|memory location"


@pytest.mark.parametrize("diff", [False, True])
def test_decode(diff):
    B, H, Hkv, D, P = 2, 4, 2, 32, 16
    flat = torch.zeros(3, 4 * P * Hkv * D, dtype=BF, device=DEV)
    k, v = (x.view(4, P, Hkv, D) for x in flat[:2])
    q, lens = torch.zeros(B, H, D, dtype=BF, device=DEV), torch.ones(B, dtype=torch.int32, device=DEV)
    table = torch.zeros(B, 1, dtype=torch.int32, device=DEV)
    shape = (B, H // 2, 2 * D) if diff else (B, H, D)

    def call(k, v, ks=None, vs=None, **kw):
        if diff:
            return paged.paged_diff_decode(q, k, v, table, lens, 1.0, torch.zeros(H // 2, device=DEV), k_scales=ks, v_scales=vs, **kw)
        return paged.paged_decode(q, k, v, table, lens, 1.0, k_scales=ks, v_scales=vs, **kw)

    for x in flat[:2]:
        with pytest.raises(RuntimeError, match=SHARED):
            call(k, v, out=x[-B * H * D:].view(shape))
        with pytest.raises(RuntimeError, match=SHARED):
            call(k, v, lse=x[:2 * B * H].view(torch.float32).view(B, H))
    with pytest.raises(RuntimeError, match=SHARED):   # the two outputs
        call(k, v, out=flat[2, :B * H * D].view(shape), lse=flat[2, :2 * B * H].view(torch.float32).view(B, H))
    codes, scales = (torch.zeros(4, P, Hkv, D, dtype=torch.int8, device=DEV) for _ in range(2)), torch.zeros(2, 4, P, Hkv, device=DEV)
    kc, vc = codes
    for s in scales:
        with pytest.raises(RuntimeError, match=SHARED):
            call(kc, vc, *scales, lse=s.view(-1)[:B * H].view(B, H))
        with pytest.raises(RuntimeError, match=SHARED):
            call(kc, vc, *scales, out=s.view(-1).view(BF)[:B * H * D].view(shape))
    got = call(k, v, out=flat[2, :B * H * D].view(shape))
    assert got[0].data_ptr() == flat[2].data_ptr()


def test_rope_and_append():
    N, H, Hkv, D, P, pages = 8, 2, 2, 32, 16, 16
    k, q = (torch.ones(N, Hkv, D, dtype=BF, device=DEV) for _ in range(2))
    pool, scales = torch.zeros(2, pages, P, Hkv, D, dtype=torch.int8, device=DEV), torch.zeros(2, pages, P, Hkv, device=DEV)
    slots, pos, turns = torch.arange(256, device=DEV), torch.zeros(512, dtype=torch.int32, device=DEV), table_of(32, D)

    def over(x):   # an output for q in x's memory
        return x.view(-1).view(BF)[:N * H * D].view(N, H, D)

    for x in (*pool, *scales, slots, pos, turns):
        with pytest.raises(RuntimeError, match=SHARED):
            paged.rope_append(q, k, k, pos[:N], turns, slots[:N], *pool, k_scales=scales[0], v_scales=scales[1], q_out=over(x))
    for x in (pos, turns):
        with pytest.raises(RuntimeError, match=SHARED):
            paged.rope(q, pos[:N], turns, out=over(x))
    assert paged.rope(q, pos[:N], turns, out=q) is q
    assert paged.rope_append(q, k, k, pos[:N], turns, slots[:N], *pool, k_scales=scales[0], v_scales=scales[1], q_out=q) is q

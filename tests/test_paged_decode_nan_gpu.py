"""GPU checks of what is not finite in a paged cache: it reaches what the formula says, and nothing else."""
import pytest
import torch

import scope_b200
from test_paged_blocks_gpu import E4, decode, make_decode, raw, widened
from test_paged_gpu import BF, DEV, HF

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("Dk,Dv", [(16, 16), (48, 48), (80, 80), (112, 112), (144, 144), (176, 64), (208, 208), (240, 240), (80, 128),
                                   (128, 80), (64, 64)])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("P,block", [(16, 16), (24, 8), (32, 1)])
def test_a_nan_value_in_e4m3_reaches_its_dim_only(Dk, Dv, dtype, P, block):
    """A NaN code in every row of a subtile and every group of dims, a request each: the other dims, the other heads and the
    lse are bit for bit what a finite code in its place gives."""
    B, Hkv, G = 131, 2, 3
    s = make_decode([70] * B, Hkv * G, Hkv, Dk, Dv, P, block, dtype, E4, seed=Dk + Dv)
    b = torch.arange(B, device=DEV)
    t, dim = b % 67, 5 * b % Dv
    page, off = s["table"].long()[b, t // P], t % P
    want, want_lse = decode(s)
    assert want.isfinite().all() and want_lse.isfinite().all()
    raw(s["v"])[page, off, 1, dim] = 0x7f + 0x80 * (b % 2).to(torch.uint8)
    nan = torch.zeros(B, Hkv * G, Dv, dtype=torch.bool, device=DEV)
    nan[b, G:, dim] = True
    for x in (s, widened(s, 600 // P)):
        out, lse = decode(x)
        assert torch.equal(out.isnan(), nan) and torch.equal(lse, want_lse)
        assert torch.equal(out[~nan], want[~nan])
    assert scope_b200.status_take() == 0

"""GPU checks of what is not finite in a paged cache: it reaches what the formula says, and nothing else."""
import pytest
import torch

import scope_b200
from test_paged_blocks_gpu import E4, I8, decode, make_decode, raw, widened
from test_paged_diff_gpu import diff, make
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


def far(s, n=600):
    """The same requests behind a table of more than n tokens: rows by TMA, where they can come so."""
    return dict(s, table=torch.cat([s["table"], s["table"].new_full((s["table"].shape[0], n // s["k"].shape[1] + 1), 1 << 20)], 1))


@pytest.mark.parametrize("Dk,Dv", [(16, 16), (32, 32), (48, 48), (64, 64), (80, 80), (96, 96), (112, 16), (128, 128)])
@pytest.mark.parametrize("dtype,pool,block", [(BF, BF, 1), (HF, HF, 1), (BF, E4, 16), (HF, E4, 64), (BF, E4, 8)])
@pytest.mark.parametrize("heads", [4, 12])
@pytest.mark.parametrize("m", [0, 1])
def test_a_key_of_one_map_does_not_reach_the_other(Dk, Dv, dtype, pool, block, heads, m):
    """A NaN key of one head of a pair, in every row of a subtile and every group of dims, a request each: that map's heads
    have a NaN lse and outputs; the other map's lse, and the other pair, are bit for bit what they were."""
    B, pairs = 131, 2
    G = heads // pairs
    s = make([70] * B, heads, pairs, Dk, Dv, 64, dtype, pool, block, seed=Dk + heads)
    b = torch.arange(B, device=DEV)
    t, dim = b % 67, 5 * b % Dk
    page, off = s["table"].long()[b, t // 64], t % 64
    want, want_lse = diff(s)
    assert want.isfinite().all() and want_lse.isfinite().all()
    if pool == E4:
        raw(s["k"])[page, off, 2 + m, dim] = 0xff
    else:
        s["k"][page, off, 2 + m, dim] = float("nan")
    for x in (s, far(s)):
        out, lse = diff(x)
        assert lse[:, 2 * G + m::2].isnan().all() and out[:, G:].isnan().all()
        assert torch.equal(lse[:, :2 * G], want_lse[:, :2 * G]) and torch.equal(out[:, :G], want[:, :G])
        assert torch.equal(lse[:, 2 * G + 1 - m::2], want_lse[:, 2 * G + 1 - m::2])
    assert scope_b200.status_take() == 0


@pytest.mark.parametrize("Dk", [32, 48, 64, 96, 128])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("m", [0, 1])
def test_a_score_of_minus_infinity_leaves_a_token_out_of_its_map(Dk, dtype, m):
    """Keys of -inf against positive queries weigh nothing in their map, as ones do whose score is finite and far below."""
    s = make([70, 700, 33], 4, 2, Dk, Dk, 64, dtype, dtype, seed=Dk)
    s["q"][:, :, 7] = 32.0
    got = []
    for x in (torch.finfo(dtype).min, float("-inf")):   # times 32 and the scale: far below any other score
        for b, t in ((0, 3), (0, 69), (1, 0), (1, 511), (2, 32)):
            s["k"][s["table"][b, t // 64].long(), t % 64, 2 + m, 7] = x
        got += [diff(s), diff(far(s))]
    for out, lse in got:
        assert out.isfinite().all() and lse.isfinite().all()
        assert torch.equal(out, got[0][0]) and torch.equal(lse, got[0][1])


@pytest.mark.parametrize("D", [32, 48, 64, 96, 128])
@pytest.mark.parametrize("dtype,pool,block", [(BF, I8, 1), (HF, I8, 16), (BF, I8, 64), (HF, E4, 1), (BF, E4, 16), (BF, E4, 64)])
@pytest.mark.parametrize("m", [0, 1])
def test_a_scale_that_is_not_finite_stays_with_its_head(D, dtype, pool, block, m):
    """A block (or row) of one head of a pair that reads back as NaN: of a key its map's lse, of a value its half of the dims.

    The other map's scores are the same, but the reference of its softmax moves with the pair's: two sums over n tokens of the
    same terms, each off by (n + 64) 2^-24 and 2^-22 |lse|."""
    s = make([70, 333, 200], 4, 2, D, D, 64, dtype, pool, block, seed=D + block)
    b, t = torch.tensor([0, 1, 2], device=DEV), torch.tensor([5, 200, 199], device=DEV)
    page, j = s["table"].long()[b, t // 64], t % 64 // block
    bad = torch.tensor([float("nan"), float("inf"), float("nan")], device=DEV)
    for form in (lambda z: z, far):
        want, want_lse = diff(form(s), False)
        for x in "kv":
            codes, scales = s[x].clone(), s[x + "s"].clone()
            for p, i in zip(page.tolist(), j.tolist()):
                raw(codes)[p, i * block:(i + 1) * block, 2 + m] = 0    # as an append leaves it
            scales[page, j, 2 + m] = bad
            out, lse = diff(form(dict(s, **{x: codes, x + "s": scales})), False)
            assert torch.equal(out[:, :2], want[:, :2]) and torch.equal(lse[:, :4], want_lse[:, :4])   # the other pair
            if x == "k":
                other, want_other = lse[:, 5 - m::2], want_lse[:, 5 - m::2]
                assert lse[:, 4 + m::2].isnan().all() and out[:, 2:].isnan().all()
                assert ((other - want_other).abs() <= 2 * ((333 + 64) * 2.0 ** -24 + 2.0 ** -22 * want_other.abs()) + 2e-6).all()
            else:
                mine, others = (slice(h * D, (h + 1) * D) for h in (m, 1 - m))
                assert out[:, 2:, mine].isnan().all() and torch.equal(out[:, 2:, others], want[:, 2:, others])
                assert torch.equal(lse, want_lse)
    assert scope_b200.status_take() == 0

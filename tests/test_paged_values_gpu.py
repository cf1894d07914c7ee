"""GPU checks of the paged operators on values that are no numbers, or no finite ones, and of how exactly values come
through."""
import pytest
import torch

from scope_b200 import paged
from test_paged_gpu import BF, DEV, HF, U, codes, decode, gen, make_decode, reference, table_of, turned

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ append into int8 pools


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("H,Hkv,D,Dv,rot", [(4, 2, 128, 128, 128), (6, 3, 80, 48, 64), (2, 1, 16, 256, 16), (0, 2, 192, 16, 64)])
@pytest.mark.parametrize("pairs", ["half", "adjacent"])
def test_append_into_int8_keeps_what_is_no_number(dtype, H, Hkv, D, Dv, rot, pairs):
    """A row with a NaN or an infinity anywhere reads back as NaN; every other row has its own codes and scale."""
    g = gen(D + Dv)
    bad = [float("nan"), float("inf"), float("-inf")]
    N = 3 * (D + Dv) + 5   # one token for every place and value, and a few sound ones
    k = torch.randn(N, Hkv, D, generator=g, device=DEV).to(dtype)
    v = torch.randn(N, Hkv, Dv, generator=g, device=DEV).to(dtype)
    at = 0
    for x, width in ((k, D), (v, Dv)):
        for d in range(width):
            for value in bad:
                x[at, (at // 7) % Hkv, d] = value
                at += 1
    table, pos = table_of(300, rot), torch.randint(0, 300, (N,), generator=g, device=DEV, dtype=torch.int32)
    q = torch.randn(N, H, D, generator=g, device=DEV).to(dtype) if H else None
    P = 16
    n_pages = -(-N // P)
    kp, vp = (torch.full((n_pages, P, Hkv, w), 99, dtype=torch.int8, device=DEV) for w in (D, Dv))
    ks, vs = (torch.zeros(n_pages, P, Hkv, device=DEV) for _ in range(2))
    slots = torch.randperm(n_pages * P, generator=g, device=DEV)[:N].contiguous()
    paged.rope_append(q, k, v, pos, table, slots, kp, vp, k_scales=ks, v_scales=vs, pairs=pairs)
    rows = ((kp, ks, turned(k, pos[None], table, [0] * (rot // 2), pairs)), (vp, vs, v.float()))
    for pool, scales, x in rows:
        got, scale = pool.view(-1, Hkv, x.shape[-1])[slots], scales.view(-1, Hkv)[slots]
        want, most = codes(x)
        sound = torch.isfinite(x).all(-1)
        assert torch.equal(torch.isfinite(scale), sound) and torch.equal(scale.isnan(), x.isnan().any(-1))
        assert torch.equal(got[sound], want[sound]) and torch.equal(scale[sound], most[sound])
        assert (got[~sound] == 0).all() and (got.float() * scale[..., None])[~sound].isnan().all()
        assert 0 < int((~sound).sum()) < sound.numel()


def test_a_nan_key_appended_into_int8_reaches_the_output():
    g = gen(2)
    Hkv, D, P = 2, 64, 16
    kp, vp = (torch.zeros(4, P, Hkv, D, dtype=torch.int8, device=DEV) for _ in range(2))
    ks, vs = (torch.zeros(4, P, Hkv, device=DEV) for _ in range(2))
    k, v = (torch.randn(40, Hkv, D, generator=g, device=DEV).to(BF) for _ in range(2))
    k[7, 1, 30] = float("nan")
    paged.rope_append(None, k, v, None, None, torch.arange(40, device=DEV), kp, vp, k_scales=ks, v_scales=vs)
    q = torch.randn(1, 4, D, generator=g, device=DEV).to(BF)
    out, lse = paged.paged_decode(q, kp, vp, torch.arange(4, dtype=torch.int32, device=DEV)[None],
                                  torch.tensor([40], dtype=torch.int32, device=DEV), 0.1, k_scales=ks, v_scales=vs)
    assert torch.isfinite(out[0, :2]).all() and torch.isfinite(lse[0, :2]).all()
    assert out[0, 2:].isnan().all() and lse[0, 2:].isnan().all()


# ------------------------------------------------------------------ how exactly the decode adds up


@pytest.mark.parametrize("pool", [HF, torch.int8])
def test_decode_long_sums_are_rounded_to_nearest(pool):
    """Rows of values 1 and then -1: a sum that rises to half of the weights and falls back to about nothing.

    Adding in fp32 rounds up to m = 8192 / 16 partial sums of at most l / 2 (l: the weights' sum) to nearest, each by at
    most 2^-25 l, either way: six standard deviations of a row's are below 6 sqrt(m / 3) 2^-25 l = 2.4e-6 l, and what is
    left at other places (scores, products, the subtiles' own sums) has no side that it prefers: 0.6e-6 for its mean.
    Sums that are cut off at every step lose half a unit each time, always the same way: 1024 / 2 2^-24 / 4 = 7.6e-6.
    """
    g = gen(71)
    n, D, P, B = 8192, 64, 16, 2960
    k = torch.randn(n // P, P, 1, D, generator=g, device=DEV).to(HF)
    v = torch.ones(n // P, P, 1, D, dtype=HF, device=DEV)
    v[n // P // 2:] = -1
    q = torch.randn(B, 1, D, generator=g, device=DEV).to(HF)
    table = torch.arange(n // P, dtype=torch.int32, device=DEV).expand(B, -1).contiguous()   # all read the same pages
    lens = torch.full((B,), n, dtype=torch.int32, device=DEV)
    scale, kw, kd = D ** -0.5, {}, k.double().view(n, D)
    if pool == torch.int8:
        one = torch.full((n // P, P, 1), 0.03, device=DEV)
        k, kw = (k.float() * 32).round().clamp(-127, 127).to(torch.int8), dict(k_scales=one, v_scales=torch.ones_like(one))
        v, kd = v.to(torch.int8), k.double().view(n, D) * one.double().view(n, 1)
    out, _ = paged.paged_decode(q, k, v, table, lens, scale, **kw)
    p = torch.softmax(q.double().view(B, D) @ kd.t() * scale, 1)
    exact = p[:, :n // 2].sum(1) - p[:, n // 2:].sum(1)
    off = out.double().view(B, D) - exact[:, None]
    assert off.mean().abs() <= 3e-6


VARIANTS = [  # D, page size, query heads a kv head, width of the table: every compiled head dim, by TMA and by cp.async
    (64, 16, 4, 200), (128, 16, 4, 200), (128, 24, 4, 100), (128, 16, 12, 200), (192, 32, 4, 100), (256, 16, 2, 200),
    (80, 16, 4, 200), (112, 7, 9, 300)]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("D,P,G,width", VARIANTS)
@pytest.mark.parametrize("spread", [0.0, 1.0, 4.0])
def test_decode_passes_infinite_values_on(dtype, D, P, G, width, spread):
    """One infinite value gives every head of its request and kv head that infinity in its dim, both signs in a dim give
    NaN, and every other output is what it was."""
    lens = [1, 2, 40, 300, 1300]
    s = make_decode(lens, 2 * G, 2, D, D, P, dtype, width=width, seed=81, spread=spread)
    want, want_lse = (x.clone() for x in decode(s))
    inf = float("inf")
    # with P = 16 the places are in a request's first, second and last subtile
    for b, n in enumerate(lens):
        for t, h, d, value in ((0, 0, 0, inf), (min(17, n - 1), 0, 3, -inf), (n - 1, 1, D - 1, inf), (n // 2, 0, 9, inf),
                               (0, 1, 16, inf), (n - 1, 1, 16, -inf if n > 1 else inf)):
            page, off = s["rows"][b]
            s["v"][page[t], off[t], h, d] = value
            want[b, h * G:(h + 1) * G, d] = value if (h, d) != (1, 16) or n == 1 else float("nan")
    out, lse = decode(s)
    assert torch.equal(lse, want_lse)
    odd = ~torch.isfinite(want)
    assert torch.equal(out[~odd], want[~odd])
    assert torch.equal(out[odd].nan_to_num(nan=7.0), want[odd].nan_to_num(nan=7.0))


def test_decode_of_one_token_gives_its_value_row():
    """Probability 1, nothing to round: whatever the row holds comes out, infinities too."""
    for dtype in (BF, HF):
        v = torch.cat([torch.linspace(-8, 8, 61, device=DEV), torch.tensor([float("inf"), float("-inf"), 0.0], device=DEV)]).to(dtype)
        k = torch.randn(1, 16, 1, 64, device=DEV).to(dtype)
        pages = torch.full((1, 16, 1, 64), float("nan"), dtype=dtype, device=DEV)
        pages[0, 0, 0] = v
        one = torch.ones(1, dtype=torch.int32, device=DEV)
        out, _ = paged.paged_decode(torch.randn(1, 3, 64, device=DEV).to(dtype), k, pages, one.view(1, 1) * 0, one, 1.0)
        assert torch.equal(out, v.expand(1, 3, 64))


@pytest.mark.parametrize("dtype,pool", [(BF, BF), (HF, HF), (BF, torch.int8), (HF, torch.int8)])
@pytest.mark.parametrize("D,P,G,width", VARIANTS)
def test_decode_keeps_all_bits_of_a_probability(dtype, pool, D, P, G, width):
    """Values that cancel: tokens of probability 1 (times l) and value 1, and as many of just below 1 and value -1, which
    a probability rounded once would make equal.

    Probabilities enter exactly or to 2^-22, so what is left is a score's error (exact here: one product), exp2's 2^-22,
    the sums' (n + 64) 2^-24 and the result's rounding."""
    n, step = 96, 2.0 ** (-10 if dtype == BF else -13)
    s = make_decode([n, 5 * n], 2 * G, 2, D, D, P, dtype, pool, width=width, seed=82)
    s["q"].zero_()
    s["q"][..., 0] = 1
    s["scale"] = 1.0
    for page, off in s["rows"]:
        low = (torch.arange(len(page), device=DEV) % 2).bool()
        for name in ("k", "v"):
            s[name][page, off] = 0
        if pool == torch.int8:
            s["k"][page[low], off[low], :, 0], s["ks"][page, off] = -1, step
            s["v"][page, off], s["vs"][page, off] = 64, 1 / 64
            s["v"][page[low], off[low]] = -64
        else:
            s["k"][page[low], off[low], :, 0] = -step
            s["v"][page, off] = 1
            s["v"][page[low], off[low]] = -1
    out, lse = decode(s)
    exact, exact_lse, _, _ = reference(s)
    total = (2.0 ** -22 + 2.0 ** -22 + (5 * n + 64) * 2.0 ** -24)
    assert (1 - U[dtype]) * exact.min() > total   # of the inputs: a probability rounded once would be seen
    assert ((out.double() - exact).abs() <= U[dtype] * exact.abs() + total).all()
    assert ((lse.double() - exact_lse).abs() <= 1e-5).all()


@pytest.mark.parametrize("dtype", [BF, HF])
def test_decode_int8_scales_of_every_size(dtype):
    """Scales from 1e-30 to 1e30 within a request, and the largest on a token that does not count or counts for nothing."""
    s = make_decode([600, 64, 33], 8, 2, 128, 128, 16, dtype, torch.int8, seed=83)
    g = gen(84)
    for (page, off), low, high in zip(s["rows"], (-3.0, -30.0, 20.0), (0.0, -27.0, 24.0)):
        s["vs"][page, off] = 10 ** (torch.rand(len(page), 2, generator=g, device=DEV) * (high - low) + low)
    out, lse = decode(s)
    exact, exact_lse, room, lse_room = reference(s)
    exact = exact.clamp(-torch.finfo(dtype).max, torch.finfo(dtype).max) if dtype == HF else exact
    ok = exact.abs() < torch.finfo(dtype).max
    least = 2.0 ** -133 if dtype == BF else 2.0 ** -25   # half of the type's least step
    assert ((out.double() - exact).abs() <= room + least)[ok].all()
    assert ((lse.double() - exact_lse).abs() <= lse_room).all()

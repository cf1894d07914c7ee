"""GPU checks of the paged cache's operators against plain implementations: whole numbers exactly, values in 64 bits.

Tolerances.  u(bf16) = 2^-8, u(fp16) = 2^-11 (rounding to nearest of one value).  A score is a sum of Dk products, exact
in fp32, accumulated in fp32: |ds| <= (Dk + 4) 2^-24 scale sum|q k|.  An output rounds each probability once to the
type the second product takes (u sum p|v|), accumulates in fp32 (n 2^-24) and rounds the result once, so
    |do| <= (2 u + 2 ds + (n + 64) 2^-24) sum p|v| + 1e-7,    |dlse| <= ds + (min(n, 4096) + 64) 2^-24 + 2^-22 |lse|.
Rotations round every product and sum by itself, so they are compared bit for bit with the same formula in torch fp32.
"""
import numpy as np
import pytest
import torch

import scope_b200
from scope_b200 import PagedKVCache, paged

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
BF, HF = torch.bfloat16, torch.float16


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


# ------------------------------------------------------------------ decode


def make_pool(g, n_pages, P, Hkv, Dk, Dv, pool, heads_major):
    """(k_pages, v_pages, k_scales, v_scales), every entry NaN or infinite (codes and scales for int8: NaN scales)."""
    def one(D):
        shape = (n_pages, Hkv, P, D) if heads_major else (n_pages, P, Hkv, D)
        if pool == torch.int8:
            x = torch.full(shape, 127, dtype=torch.int8, device=DEV)
            s = torch.full(shape[:3], float("nan"), device=DEV)
        else:
            x = torch.full(shape, float("nan"), dtype=pool, device=DEV)
            x.view(-1)[::3] = float("inf")
            s = None
        return (x.transpose(1, 2), None if s is None else s.transpose(1, 2)) if heads_major else (x, s)

    (k, ks), (v, vs) = one(Dk), one(Dv)
    return k, v, ks, vs


def make_decode(lens, H, Hkv, Dk, Dv, P, dtype, pool=None, heads_major=False, width=None, seed=0, spread=1.0):
    """Requests whose pages hold values up to their lengths and NaN or infinity everywhere else."""
    g, pool = gen(seed), dtype if pool is None else pool
    B = len(lens)
    held = [-(-n // P) for n in lens]
    n_pages = sum(held) + 3
    width = max(held + [1]) if width is None else width
    ids = torch.randperm(n_pages, generator=g, device=DEV).int()
    table = torch.full((B, width), n_pages + 7, dtype=torch.int32, device=DEV)   # entries past a length: no page
    k, v, ks, vs = make_pool(g, n_pages, P, Hkv, Dk, Dv, pool, heads_major)
    at, rows = 0, []
    for b, n in enumerate(lens):
        table[b, :held[b]] = ids[at:at + held[b]]
        at += held[b]
        t = torch.arange(n, device=DEV)
        page, off = table[b].long()[t // P], t % P
        for x, s, D in ((k, ks, Dk), (v, vs, Dv)):
            val = torch.randn(n, Hkv, D, generator=g, device=DEV)
            if pool == torch.int8:
                x[page, off] = (val * 32).round().clamp(-127, 127).to(torch.int8)
                s[page, off] = torch.rand(n, Hkv, generator=g, device=DEV) * 0.04 + 0.01
            else:
                x[page, off] = val.to(pool)
        rows.append((page, off))
    q = (torch.randn(B, H, Dk, generator=g, device=DEV) * spread).to(dtype)
    return dict(q=q, k=k, v=v, ks=ks, vs=vs, table=table, lens=torch.tensor(lens, dtype=torch.int32, device=DEV),
                rows=rows, scale=Dk ** -0.5)


def reference(s, window=0, leave_out=None):
    """Per request in float64: (out, lse, bound of out, bound of lse)."""
    q, Hkv = s["q"], s["k"].shape[2]
    B, H, Dk = q.shape
    G, Dv = H // Hkv, s["v"].shape[3]
    u = U[q.dtype]
    out = torch.zeros(B, H, Dv, dtype=torch.float64, device=DEV)
    lse = torch.full((B, H), float("-inf"), dtype=torch.float64, device=DEV)
    bo, bl = torch.full_like(out, 1e-7), torch.full_like(lse, 1e-6)
    for b, (page, off) in enumerate(s["rows"]):
        if window:
            page, off = page[-window:], off[-window:]
        if leave_out is not None:
            keep = leave_out(page)
            page, off = page[keep], off[keep]
        n = len(page)
        if n == 0:
            continue
        for h in range(Hkv):
            k, v = s["k"][page, off, h].double(), s["v"][page, off, h].double()
            if s["ks"] is not None:
                k, v = k * s["ks"][page, off, h].double()[:, None], v * s["vs"][page, off, h].double()[:, None]
            qs = q[b, h * G:(h + 1) * G].double()
            z = qs @ k.t() * s["scale"]
            ds = (Dk + 4) * 2.0 ** -24 * s["scale"] * (qs.abs() @ k.abs().t()).amax(1)
            L = torch.logsumexp(z, 1)
            p = torch.exp(z - L[:, None])
            sl = slice(h * G, (h + 1) * G)
            out[b, sl], lse[b, sl] = p @ v, L
            bo[b, sl] += (2 * u + 2 * ds[:, None] + (n + 64) * 2.0 ** -24) * (p @ v.abs())
            bl[b, sl] = ds + (min(n, 4096) + 64) * 2.0 ** -24 + 2.0 ** -22 * L.abs()
    return out, lse, bo, bl


def decode(s, window=0, **kw):
    return paged.paged_decode(s["q"], s["k"], s["v"], s["table"], s["lens"], s["scale"], window=window,
                              k_scales=s["ks"], v_scales=s["vs"], **kw)


def agrees(s, out, lse, window=0, leave_out=None):
    ro, rl, bo, bl = reference(s, window, leave_out)
    assert out.dtype == s["q"].dtype and lse.dtype == torch.float32
    assert torch.isfinite(out.float()).all()
    empty = torch.isneginf(rl)
    assert torch.equal(torch.isneginf(lse), empty) and (out[empty] == 0).all()
    assert ((out.double() - ro).abs() <= bo).all(), ((out.double() - ro).abs() / bo).max().item()
    d = (lse.double() - rl).abs()[~empty]
    assert (d <= bl[~empty]).all(), (d / bl[~empty]).max().item()


LENS = [0, 1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 200]


@pytest.mark.parametrize("P", [1, 7, 16, 24, 64, 256])
@pytest.mark.parametrize("dtype,pool", [(BF, BF), (HF, HF), (BF, torch.int8), (HF, torch.int8)])
def test_decode_lengths_and_page_sizes(P, dtype, pool):
    s = make_decode(LENS, 8, 2, 128, 128, P, dtype, pool, seed=P)
    agrees(s, *decode(s))
    assert scope_b200.status_take() == 0


@pytest.mark.parametrize("Dk,Dv", [(16, 16), (32, 64), (64, 64), (80, 80), (96, 96), (112, 48), (128, 128), (192, 128),
                                   (64, 256), (256, 256), (240, 16)])
@pytest.mark.parametrize("dtype,pool", [(BF, BF), (HF, torch.int8)])
def test_decode_head_dims(Dk, Dv, dtype, pool):
    s = make_decode([300, 0, 45, 16], 6, 3, Dk, Dv, 16, dtype, pool, seed=Dk + Dv)
    agrees(s, *decode(s))


@pytest.mark.parametrize("G", [1, 2, 3, 5, 8, 9, 12, 16, 17, 24, 32, 48, 64])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_decode_groups(G, D):
    s = make_decode([257, 1, 0, 90], 2 * G, 2, D, D, 32, BF, seed=G)
    agrees(s, *decode(s))


@pytest.mark.parametrize("heads_major", [False, True])
@pytest.mark.parametrize("pool", [BF, torch.int8])
def test_decode_layouts_and_strided_queries(heads_major, pool):
    s = make_decode([500, 3, 0, 129], 16, 4, 128, 128, 16, BF, pool, heads_major, width=77, seed=5)
    packed = torch.full((4, 16, 3 * 128 + 8), float("nan"), dtype=BF, device=DEV)
    packed[..., 8:136] = s["q"]
    want = decode(s)
    agrees(s, *want)
    s["q"] = packed[..., 8:136]
    wide = torch.full((4, 200), 1 << 30, dtype=torch.int32, device=DEV)
    wide[:, 50:127] = s["table"]
    s["table"] = wide[:, 50:127]
    got = decode(s)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert scope_b200.status_take() == 0


@pytest.mark.parametrize("window", [1, 2, 16, 17, 100, 129, 4000])
def test_decode_window(window):
    s = make_decode([0, 1, 16, 100, 129, 1000, 2500], 8, 2, 128, 128, 24, BF, seed=window)
    agrees(s, *decode(s, window), window=window)


@pytest.mark.parametrize("B,lens", [
    (1, [1]), (1, [4096]), (1, [50001]), (3, [40000, 17, 9000]), (40, None), (300, None), (1100, None)])
@pytest.mark.parametrize("pool", [BF, torch.int8])
def test_decode_splits(B, lens, pool):
    """From one long request, whose length is split over the device, to more requests than it has SMs."""
    if lens is None:
        lens = np.random.RandomState(B).randint(0, 300, B).tolist()
    s = make_decode(lens, 8, 2, 64, 64, 16, BF, pool, seed=B)
    got = decode(s)
    agrees(s, *got)
    again = decode(s)   # the split does not depend on which block ran first
    assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])


def test_decode_large_and_small_scores():
    """Scores of hundreds either way: the running maximum has to move both ways without overflow."""
    for spread in (60.0, 1e-3):
        s = make_decode([1000, 5, 77], 8, 2, 128, 128, 16, BF, seed=11, spread=spread)
        agrees(s, *decode(s))
    s = make_decode([1000, 40], 4, 1, 64, 64, 16, HF, seed=12)
    s["k"][:] = 0   # every score 0: the plain mean
    agrees(s, *decode(s))
    s = make_decode([1000, 40], 4, 1, 64, 64, 16, BF, seed=13)
    page, off = s["rows"][0]
    s["k"][page, off] = (-3.0e38 * torch.sign(s["q"][0].float().sum(0))).to(BF)[None, None]   # near the type's lowest
    s["q"][0] = s["q"][0, :1]
    s["q"][0, :, 1:] = 0
    agrees(s, *decode(s))


def test_decode_extremely_low_scores_keep_their_differences():
    """Scores around -1e30, equal ones: weights are even, lse is the score itself."""
    s = make_decode([64, 7], 2, 1, 16, 16, 16, BF, seed=14)
    s["q"][:] = 0
    s["q"][..., 0] = 1
    for page, off in s["rows"]:
        s["k"][page, off, 0, 0] = -1e30
    out, lse = decode(s)
    for b, (page, off) in enumerate(s["rows"]):
        mean = s["v"][page, off, 0].double().mean(0)
        assert (out[b].double() - mean).abs().max() <= 3 * U[BF] * s["v"][page, off, 0].double().abs().mean(0).max()
        assert (lse[b].double() / (-1e30 * s["scale"]) - 1).abs().max() < 2 * U[BF]


def test_decode_leaves_out_pages_that_are_none():
    s = make_decode([100, 64, 10], 8, 2, 128, 128, 16, BF, seed=15)
    n_pages = s["k"].shape[0]
    gone = [int(s["table"][0, 2]), int(s["table"][2, 0])]
    t = s["table"].clone()
    t[0, 2], t[2, 0] = -1, n_pages
    s["table"] = t
    out, lse = decode(s)
    agrees(s, out, lse, leave_out=lambda page: ~torch.isin(page, torch.tensor(gone, device=DEV, dtype=page.dtype)))
    assert scope_b200.status_take() == 5 and scope_b200.status_take() == 0


def test_decode_length_past_the_table_and_negative():
    s = make_decode([40, 5, 0], 8, 2, 128, 128, 16, BF, seed=16)
    want = decode(s)
    lens = torch.tensor([48, 5, -3], dtype=torch.int32, device=DEV)   # the table is three pages wide
    page, off = torch.tensor([int(s["table"][0, 2])] * 8, device=DEV), torch.arange(8, 16, device=DEV)
    s["k"][page, off], s["v"][page, off] = 0, 0
    s["rows"][0] = (torch.cat([s["rows"][0][0], page.to(s["rows"][0][0].dtype)]), torch.cat([s["rows"][0][1], off]))
    for L0 in (48, 1000000):
        lens[0] = L0
        s["lens"] = lens
        out, lse = decode(s)
        agrees(s, out, lse)
        assert torch.equal(out[1:], want[0][1:])


def test_decode_offsets_past_32_bits():
    """Pages whose elements lie more than 2^31 (and 2^32 bytes) from the pool's start."""
    P, Hkv, D = 64, 8, 128
    n_pages = (1 << 31) // (P * Hkv * D) + 40
    k = torch.empty(n_pages, P, Hkv, D, dtype=BF, device=DEV)
    v = torch.empty(n_pages, P, Hkv, D, dtype=BF, device=DEV)
    g = gen(17)
    pages = torch.tensor([n_pages - 1, 0, n_pages - 20, n_pages // 2], device=DEV)
    for p in pages.tolist():
        k[p], v[p] = torch.randn(P, Hkv, D, generator=g, device=DEV).to(BF), torch.randn(P, Hkv, D, generator=g, device=DEV).to(BF)
    n = 3 * P + 11
    t = torch.arange(n, device=DEV)
    s = dict(q=torch.randn(1, 32, D, generator=g, device=DEV).to(BF), k=k, v=v, ks=None, vs=None,
             table=pages.int()[None].contiguous(), lens=torch.tensor([n], dtype=torch.int32, device=DEV),
             rows=[(pages[t // P], t % P)], scale=D ** -0.5)
    agrees(s, *decode(s))
    # and the append writes there
    kk, vv = torch.randn(2, Hkv, D, generator=g, device=DEV).to(BF), torch.randn(2, Hkv, D, generator=g, device=DEV).to(BF)
    slots = torch.tensor([(n_pages - 3) * P + 5, 9 * P], device=DEV)
    paged.rope_append(None, kk, vv, None, None, slots, k, v)
    assert torch.equal(k[n_pages - 3, 5], kk[0]) and torch.equal(v[9, 0], vv[1])


def test_decode_on_another_stream_and_outputs_given():
    s = make_decode([700, 30], 8, 2, 128, 128, 16, BF, seed=18)
    out = torch.full((2, 8, 128), float("nan"), dtype=BF, device=DEV)
    lse = torch.full((2, 8), float("nan"), device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = decode(s, out=out, lse=lse)
    side.synchronize()
    assert got[0] is out and got[1] is lse
    agrees(s, out, lse)


def test_decode_of_no_requests_and_no_pages():
    k = torch.empty(0, 16, 2, 64, dtype=BF, device=DEV)
    lens = torch.zeros(0, dtype=torch.int32, device=DEV)
    out, lse = paged.paged_decode(torch.empty(0, 4, 64, dtype=BF, device=DEV), k, k, lens.view(0, 1)[:, :1], lens, 1.0)
    assert out.shape == (0, 4, 64) and lse.shape == (0, 4)
    q = torch.randn(3, 4, 64, device=DEV).to(BF)
    zero = torch.zeros(3, dtype=torch.int32, device=DEV)
    out, lse = paged.paged_decode(q, k, k, torch.zeros(3, 2, dtype=torch.int32, device=DEV), zero, 1.0)
    assert (out == 0).all() and torch.isneginf(lse).all()


def test_decode_refusals():
    s = make_decode([20], 4, 2, 64, 64, 16, BF, seed=19)
    q, k, v, t, n = s["q"], s["k"], s["v"], s["table"], s["lens"]

    def no(match, *a, **kw):
        with pytest.raises(RuntimeError, match=match):
            paged.paged_decode(*a, **kw)

    no("bf16 or fp16", q.float(), k, v, t, n, 1.0)
    no("type or int8", q.half(), k, v, t, n, 1.0)
    no("Hkv \\* G", q[:, :3], k, v, t, n, 1.0)
    no("page_table", q, k, v, t.long(), n, 1.0)
    no("page_table", q, k, v, t[0], n, 1.0)
    no("seq_lens", q, k, v, t, n.long(), 1.0)
    no("scales", q, k, v, t, n, 1.0, k_scales=torch.ones(k.shape[:3], device=DEV))
    no("int8 pool needs", q, k.to(torch.int8), v.to(torch.int8), t, n, 1.0)
    no("k_pages", q, k, v[:-1], t, n, 1.0)
    no("out must", q, k, v, t, n, 1.0, out=torch.empty(1, 4, 64, device=DEV))
    no("lse must", q, k, v, t, n, 1.0, lse=torch.empty(1, 5, device=DEV))
    no("window|bad shape", q, k, v, t, n, 1.0, window=-1)
    no("cpu|on cuda", q, k, v, t.cpu(), n, 1.0)
    odd = torch.zeros(2, 16, 2, 72, dtype=BF, device=DEV)
    no("multiples of 16", torch.zeros(1, 4, 72, dtype=BF, device=DEV), odd, odd, t, n, 1.0)


# ------------------------------------------------------------------ pages and slots


def slots_reference(lens, new, table, free, ring, P, n):
    table, head, count = table.copy(), int(ring[0]), int(ring[1])
    slots, pos = np.full(n, -1, np.int64), np.zeros(n, np.int32)
    out, start, took, wanted, refused = lens.copy(), 0, 0, 0, 0
    cu = np.concatenate([[0], np.cumsum(np.maximum(new, 0))]).astype(np.int32)
    for b in range(len(lens)):
        L, m = max(int(lens[b]), 0), max(int(new[b]), 0)
        held, want = -(-L // P), -(-(L + m) // P)
        fits = want <= table.shape[1] and cu[b + 1] <= n
        need = want - held if fits else 0
        wanted += need
        if not fits or (need and wanted > count):
            refused += 1
            continue
        for i in range(need):
            table[b, held + i] = free[(head + took + i) % len(free)]
        took += need
        for j in range(m):
            p = L + j
            slots[cu[b] + j] = int(table[b, p // P]) * P + p % P
            pos[cu[b] + j] = p
        out[b] = L + m
    return slots, pos, cu, out, np.array([(head + took) % len(free), count - took, refused], np.int32), table


def run_slots(lens, new, table, free, ring, P, n, in_place=False):
    d = [torch.from_numpy(np.ascontiguousarray(x)).to(DEV) for x in (lens, new, table, free, ring)]
    kw = dict(seq_lens_out=d[0], ring_out=d[4]) if in_place else {}
    r = paged.paged_slots(*d, P, n, **kw)
    if in_place:
        assert r.seq_lens is d[0] and r.ring is d[4]
    return [x.cpu().numpy() for x in (r.slots, r.positions, r.cu_new, r.seq_lens, r.ring, d[2])], d


def slots_case(seed, B, P, most, prompt, width, n_ring, spare=0):
    r = np.random.RandomState(seed)
    lens = r.randint(0, most + 1, B).astype(np.int32)
    new = np.where(r.rand(B) < 0.5, 1, r.randint(0, prompt + 1, B)).astype(np.int32)
    held = -(-lens // P)
    ids = r.permutation(int(held.sum()) + n_ring).astype(np.int32)
    table = np.full((B, width), -1, np.int32)
    at = 0
    for b in range(B):
        w = min(held[b], width)
        table[b, :w] = ids[at:at + w]
        at += w
    free = ids[len(ids) - n_ring:].copy()
    ring = np.array([r.randint(n_ring), r.randint(n_ring // 2, n_ring + 1), 0], np.int32)
    return lens, new, table, free, ring, P, int(new.sum()) + spare


@pytest.mark.parametrize("seed,B,P,most,prompt,width,n_ring,spare", [
    (1, 1, 16, 40, 1, 8, 4, 0), (2, 5, 1, 9, 3, 20, 40, 3), (3, 64, 16, 500, 1, 40, 100, 0),
    (4, 200, 24, 700, 300, 50, 900, 17), (5, 200, 24, 700, 300, 30, 300, 0),     # a narrow table and few pages: refusals
    (6, 1025, 8, 100, 40, 30, 4000, 0), (7, 3000, 16, 60, 20, 8, 2000, 5), (8, 31, 7, 30, 2000, 400, 6000, 1)])
@pytest.mark.parametrize("in_place", [False, True])
def test_slots_match_the_definition(seed, B, P, most, prompt, width, n_ring, spare, in_place):
    case = slots_case(seed, B, P, most, prompt, width, n_ring, spare)
    got, _ = run_slots(*case, in_place=in_place)
    for x, y, name in zip(got, slots_reference(*case), ("slots", "positions", "cu_new", "seq_lens", "ring", "table")):
        assert np.array_equal(x, y), name


def test_slots_refuse_tokens_past_the_step_and_odd_counts():
    lens, new, table, free, ring, P, n = slots_case(9, 40, 16, 100, 30, 20, 300)
    new[3], new[7] = -5, 0
    for room in (0, 1, n // 2, n - 1):
        got, _ = run_slots(lens, new, table, free, ring, P, room)
        for x, y in zip(got, slots_reference(lens, new, table, free, ring, P, room)):
            assert np.array_equal(x, y)
    zero = np.zeros(0, np.int32)
    got, _ = run_slots(zero, zero, np.zeros((0, 4), np.int32), free, ring, P, 3)
    assert (got[0] == -1).all() and got[2].tolist() == [0] and got[4].tolist() == [ring[0], ring[1], 0]


def test_slots_of_many_requests_at_the_limit_and_past_it():
    case = slots_case(10, 8192, 16, 40, 3, 8, 9000)
    got, _ = run_slots(*case)
    for x, y in zip(got, slots_reference(*case)):
        assert np.array_equal(x, y)
    z = torch.zeros(8193, dtype=torch.int32, device=DEV)
    with pytest.raises(RuntimeError, match="8192"):
        paged.paged_slots(z, z, z.view(-1, 1), z, torch.zeros(3, dtype=torch.int32, device=DEV), 16, 1)


@pytest.mark.parametrize("B,width,P", [(1, 4, 16), (70, 30, 8), (2000, 60, 4)])
def test_release_and_take_again(B, width, P):
    """Pages go out and come back over many steps: never one page twice, the ring's order is the definition's."""
    r = np.random.RandomState(B)
    n_pages = max(4, B * width // 3)
    lens = torch.zeros(B, dtype=torch.int32, device=DEV)
    table = torch.full((B, width), -1, dtype=torch.int32, device=DEV)
    free = torch.randperm(n_pages, generator=gen(B), device=DEV).int()
    ring = torch.tensor([n_pages - 1, n_pages, 0], dtype=torch.int32, device=DEV)
    for step in range(6):
        new = r.randint(0, width * P // 2, B).astype(np.int32)
        before = [x.cpu().numpy() for x in (lens, table, free, ring)]
        step_out = paged.paged_slots(lens, torch.from_numpy(new).to(DEV), table, free, ring, P, int(new.sum()),
                                     seq_lens_out=lens, ring_out=ring)
        want = slots_reference(before[0], new, before[1], before[2], before[3], P, int(new.sum()))
        assert np.array_equal(step_out.slots.cpu().numpy(), want[0])
        assert np.array_equal(lens.cpu().numpy(), want[3]) and np.array_equal(ring.cpu().numpy(), want[4])
        held = -(-want[3] // P)
        owned = np.concatenate([want[5][b, :held[b]] for b in range(B)])
        h, c = want[4][0], want[4][1]
        loose = free.cpu().numpy()[(h + np.arange(c)) % n_pages]
        assert sorted(np.concatenate([owned, loose]).tolist()) == list(range(n_pages))
        done = r.rand(B) < 0.5
        paged.paged_release(lens, torch.from_numpy(done).to(DEV), table, free, ring, P, seq_lens_out=lens, ring_out=ring)
        back = np.concatenate([want[5][b, :held[b]] for b in range(B) if done[b]] + [np.zeros(0, np.int32)])
        assert ring.cpu().numpy().tolist() == [h, c + len(back), 0]
        f = free.cpu().numpy()
        assert np.array_equal(f[(h + c + np.arange(len(back))) % n_pages], back)
        assert np.array_equal(lens.cpu().numpy(), np.where(done, 0, want[3]))
    assert scope_b200.status_take() == 0


def test_release_twice_is_reported():
    lens = torch.tensor([32, 16], dtype=torch.int32, device=DEV)
    table = torch.tensor([[0, 1], [2, -1]], dtype=torch.int32, device=DEV)
    free = torch.tensor([3, 9, 9, 9], dtype=torch.int32, device=DEV)
    ring = torch.tensor([0, 1, 0], dtype=torch.int32, device=DEV)
    done = torch.ones(2, dtype=torch.bool, device=DEV)
    lens2, ring2 = paged.paged_release(lens, done, table, free, ring, 16)
    assert ring2.tolist() == [0, 4, 0] and free.tolist() == [3, 0, 1, 2] and lens2.tolist() == [0, 0]
    assert scope_b200.status_take() == 0
    paged.paged_release(lens, done, table, free, ring2, 16)   # the same pages again: the ring is full
    assert scope_b200.status_take() == 5
    assert free.tolist() == [3, 0, 1, 2]


def test_slots_refusals():
    i = torch.zeros(4, dtype=torch.int32, device=DEV)
    t, ring = i.view(2, 2), i[:3].contiguous()
    with pytest.raises(RuntimeError, match="new_lens"):
        paged.paged_slots(i[:2], i[:3], t, i, ring, 16, 1)
    with pytest.raises(RuntimeError, match="page_table"):
        paged.paged_slots(i[:2], i[:2], i.view(4, 1), i, ring, 16, 1)
    with pytest.raises(RuntimeError, match="ring"):
        paged.paged_slots(i[:2], i[:2], t, i, i, 16, 1)
    with pytest.raises(RuntimeError, match="seq_lens"):
        paged.paged_slots(i[::2], i[:2], t, i, ring, 16, 1)
    with pytest.raises(RuntimeError, match="bad shape"):
        paged.paged_slots(i[:2], i[:2], t, i, ring, 0, 1)
    with pytest.raises(RuntimeError, match="done"):
        paged.paged_release(i[:2], i[:2], t, i, ring, 16)


# ------------------------------------------------------------------ rotary positions


def table_of(top, rot):
    a = torch.arange(top, dtype=torch.float64, device=DEV)[:, None] * 1e4 ** (
        -torch.arange(0, rot, 2, dtype=torch.float64, device=DEV) / rot)
    return torch.cat([a.cos(), a.sin()], 1).float()


def turned(x, pos, table, axes, pairs, inverse=False, dt=torch.float32):
    """The formula, elementwise in ``dt``; axes: the axis of each pair; pos [A, N]."""
    n = table.shape[1] // 2
    a = torch.tensor(axes, device=DEV)
    at = pos.long()[a]                                     # [n, N]
    i = torch.arange(n, device=DEV)[:, None]
    c, s = table[at, i].t()[:, None].to(dt), table[at, n + i].t()[:, None].to(dt)
    s = -s if inverse else s
    x = x.to(dt)
    x1, x2 = (x[..., 0:2 * n:2], x[..., 1:2 * n:2]) if pairs == "adjacent" else (x[..., :n], x[..., n:2 * n])
    y1, y2 = x1 * c - x2 * s, x2 * c + x1 * s
    y = torch.stack([y1, y2], -1).flatten(-2) if pairs == "adjacent" else torch.cat([y1, y2], -1)
    return torch.cat([y, x[..., 2 * n:]], -1)


ROPE = [  # N, H, D, rot, sections, cyclic
    (1, 1, 16, 16, None, False), (3, 5, 128, 128, None, False), (1000, 32, 128, 128, (16, 24, 24), False),
    (77, 7, 80, 64, (12, 10, 10), True), (300, 12, 96, 96, (24, 8, 8, 8), False), (5, 40, 256, 256, (64, 64), True),
    (513, 3, 64, 32, None, False), (9, 2, 240, 144, None, False), (4097, 1, 112, 112, (20, 18, 18), True)]


@pytest.mark.parametrize("N,H,D,rot,sections,cyclic", ROPE)
@pytest.mark.parametrize("pairs", ["half", "adjacent"])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("inverse", [False, True])
def test_rope_is_the_formula(N, H, D, rot, sections, cyclic, pairs, dtype, inverse):
    g = gen(N + D)
    A = 1 if sections is None else len(sections)
    table = table_of(999, rot)
    pos = torch.randint(0, 999, (A, N), generator=g, device=DEV, dtype=torch.int32 if N % 2 else torch.int64)
    x = torch.randn(N, H, D, generator=g, device=DEV).to(dtype)
    words = paged.rope_axis_map(rot, sections, cyclic)
    axes = [(int.from_bytes(words[4 * (i >> 4):4 * (i >> 4) + 4], "little") >> (2 * (i & 15))) & 3 for i in range(rot // 2)]
    kw = dict(sections=sections, cyclic=cyclic, pairs=pairs, inverse=inverse)
    want = turned(x, pos, table, axes, pairs, inverse)
    got = paged.rope(x, pos[0] if A == 1 else pos, table, **kw)
    assert torch.equal(got, want.to(dtype))
    exact = turned(x, pos, table, axes, pairs, inverse, torch.float64)
    size = x.double().abs().amax() * 2
    assert ((got.double() - exact).abs() <= U[dtype] * exact.abs() + 4 * 2.0 ** -24 * size + 2.0 ** -25).all()
    # views, an odd start and in place
    wide = torch.zeros(N, H + 2, D + 24, dtype=dtype, device=DEV)
    for d in (8, 5):
        view = wide[:, 1:H + 1, d:d + D]
        view.copy_(x)
        assert torch.equal(paged.rope(view, pos[0] if A == 1 else pos, table, **kw), got)
        paged.rope(view, pos[0] if A == 1 else pos, table, out=view, **kw)
        assert torch.equal(view, got)
        assert (wide[:, 0] == 0).all() and (wide[:, :, :d] == 0).all() and (wide[:, :, d + D:] == 0).all()
        wide.zero_()


@pytest.mark.parametrize("pairs", ["half", "adjacent"])
def test_rope_inverse_is_the_gradient(pairs):
    """<g, d rope(x)> for the formula's gradient (autograd of it) and for differences of the forward (it is linear)."""
    g = gen(3)
    N, H, D, rot, sections = 40, 4, 64, 48, (10, 8, 6)
    table, pos = table_of(500, rot), torch.randint(0, 500, (3, N), generator=g, device=DEV, dtype=torch.int32)
    axes = [a for a, s in enumerate(sections) for _ in range(s)]
    x = torch.randn(N, H, D, generator=g, device=DEV, dtype=torch.float64, requires_grad=True)
    gy = torch.randn(N, H, D, generator=g, device=DEV).to(BF)
    turned(x, pos, table, axes, pairs, dt=torch.float64).backward(gy.double())
    got = paged.rope(gy, pos, table, sections=sections, pairs=pairs, inverse=True)
    assert ((got.double() - x.grad).abs() <= U[BF] * x.grad.abs() + 1e-5).all()
    # differences: rope(x + d) - rope(x) of the kernel, against the kernel's gradient
    x0 = torch.randn(N, H, D, generator=g, device=DEV).to(HF)
    d = torch.randn(N, H, D, generator=g, device=DEV).to(HF)
    x1 = (x0.float() + d.float()).to(HF)
    d = x1.double() - x0.double()
    y0, y1 = (paged.rope(t, pos, table, sections=sections, pairs=pairs).double() for t in (x0, x1))
    left, right = (gy.double() * (y1 - y0)).sum(), (got.double() * d).sum()
    # each of the forward's values is rounded once to fp16, each gradient once to bf16
    room = (gy.double().abs() * (y0.abs() + y1.abs())).sum() * U[HF] + (got.double().abs() * d.abs()).sum() * U[BF]
    assert (left - right).abs() <= room


def test_rope_positions_outside_the_table_are_clamped_and_reported():
    table = table_of(100, 32)
    x = torch.randn(4, 2, 32, device=DEV).to(BF)
    bad = torch.tensor([-1, 100, 1 << 30, 7], dtype=torch.int32, device=DEV)
    got = paged.rope(x, bad, table)
    assert scope_b200.status_take() == 5
    assert torch.equal(got, paged.rope(x, torch.tensor([0, 99, 99, 7], dtype=torch.int32, device=DEV), table))
    assert scope_b200.status_take() == 0


def test_rope_of_no_tokens_and_refusals():
    table = table_of(100, 32)
    x = torch.randn(4, 2, 32, device=DEV).to(BF)
    pos = torch.zeros(4, dtype=torch.int32, device=DEV)
    assert paged.rope(x[:0], pos[:0], table).shape == (0, 2, 32)
    for match, a, kw in [
            ("bf16 or fp16", (x.float(), pos, table), {}), ("cos_sin", (x, pos, table.half()), {}),
            ("positions", (x, pos[:3], table), {}), ("positions", (x, pos.float(), table), {}),
            ("positions", (x, pos, table), dict(sections=(8, 4, 4))), ("sections", (x, pos.expand(3, 4), table), dict(sections=(8, 4, 5))),
            ("pairs", (x, pos, table), dict(pairs="both")), ("rope_dim", (x, pos, table_of(10, 48)), {}),
            ("rope_dim", (x, pos, table_of(10, 24)), {}), ("multiples of 16", (x[..., :24], pos, table_of(10, 16)), {}),
            ("out", (x, pos, table), dict(out=torch.empty(4, 3, 32, dtype=BF, device=DEV)))]:
        with pytest.raises(RuntimeError, match=match):
            paged.rope(*a, **kw)


# ------------------------------------------------------------------ append


def codes(x):
    """fp32 rows -> (int8 codes, scales), the rule of the framework's row quantiser."""
    most = x.abs().amax(-1).clamp(min=1e-6)
    inv = torch.full_like(most, 127.0) / most   # one division (127.0 / most is a reciprocal and a product)
    return torch.round(x * inv[..., None]).clamp(-128, 127).to(torch.int8), most * (1.0 / 127.0)


@pytest.mark.parametrize("N,H,Hkv,D,Dv,rot,sections,P,heads_major", [
    (1, 8, 2, 128, 128, 128, None, 16, False), (64, 32, 8, 128, 128, 128, None, 16, False),
    (513, 12, 3, 80, 80, 64, None, 24, True), (1000, 4, 4, 64, 64, 64, (12, 10, 10), 1, False),
    (200, 6, 2, 192, 128, 64, None, 64, True), (37, 5, 1, 256, 256, 128, (32, 32), 256, False),
    (90, 3, 3, 16, 240, 16, None, 7, False)])
@pytest.mark.parametrize("dtype,pool", [(BF, BF), (HF, HF), (BF, torch.int8), (HF, torch.int8)])
@pytest.mark.parametrize("pairs", ["half", "adjacent"])
def test_append_writes_exactly_the_rows(N, H, Hkv, D, Dv, rot, sections, P, heads_major, dtype, pool, pairs):
    g = gen(N)
    A = 1 if sections is None else len(sections)
    table, pos = table_of(400, rot), torch.randint(0, 400, (A, N), generator=g, device=DEV, dtype=torch.int32)
    axes = [0] * (rot // 2) if A == 1 else [a for a, s in enumerate(sections) for _ in range(s)]
    qkv = torch.randn(N, H * D + Hkv * (D + Dv), generator=g, device=DEV).to(dtype)
    q, k, v = (x.view(N, h, d) for x, h, d in zip(qkv.split([H * D, Hkv * D, Hkv * Dv], 1), (H, Hkv, Hkv), (D, D, Dv)))
    if N > 2:
        k[2] = 0   # a row of zeros: scale of the least maximum, codes 0
    n_pages = -(-N // P) + 5
    kp, vp, ks, vs = make_pool(g, n_pages, P, Hkv, D, Dv, pool, heads_major)
    slots = torch.randperm(n_pages * P, generator=g, device=DEV)[:N].contiguous()
    slots[torch.rand(N, generator=g, device=DEV) < 0.1] = -1
    wk, wv = kp.clone(), vp.clone()
    wks, wvs = (None, None) if ks is None else (ks.clone(), vs.clone())
    at = torch.nonzero(slots >= 0)[:, 0]
    page, off = slots[at] // P, slots[at] % P
    rk, rv = turned(k, pos, table, axes, pairs), v.float()
    if pool == torch.int8:
        (ck, sk), (cv, sv) = codes(rk), codes(rv)
        wk[page, off], wv[page, off], wks[page, off], wvs[page, off] = ck[at], cv[at], sk[at], sv[at]
    else:
        wk[page, off], wv[page, off] = rk[at].to(pool), rv[at].to(pool)
    got = paged.rope_append(q, k, v, pos[0] if A == 1 else pos, table, slots, kp, vp, k_scales=ks, v_scales=vs,
                            sections=sections, pairs=pairs)
    assert torch.equal(got, turned(q, pos, table, axes, pairs).to(dtype))

    def same(a, b):
        return torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))

    assert same(kp, wk) and same(vp, wv)
    if ks is not None:
        assert same(ks, wks) and same(vs, wvs)
    assert scope_b200.status_take() == 0


def test_append_without_rotation_in_place_and_unaligned():
    g = gen(7)
    N, H, Hkv, D, P = 33, 6, 2, 64, 16
    pool = torch.zeros(2, 4, P, Hkv, D, dtype=BF, device=DEV)
    slots = torch.randperm(4 * P, generator=g, device=DEV)[:N].contiguous()
    flat = torch.randn(N * (H + 2 * Hkv) * D + 3, generator=g, device=DEV).to(BF)[3:]   # 6 bytes past a boundary
    q, k, v = (x.view(N, h, D) for x, h in zip(flat.view(N, -1).split([H * D, Hkv * D, Hkv * D], 1), (H, Hkv, Hkv)))
    assert paged.rope_append(None, k, v, None, None, slots, pool[0], pool[1]) is None
    for p, x in ((pool[0], k), (pool[1], v)):
        assert torch.equal(p.view(-1, Hkv, D)[slots], x)
    same = q.clone()
    assert torch.equal(paged.rope_append(q, k, v, None, None, slots, pool[0], pool[1]), same)
    table, pos = table_of(50, D), torch.randint(0, 50, (N,), generator=g, device=DEV)
    want = paged.rope(q.contiguous(), pos, table)
    assert paged.rope_append(q, k, v, pos, table, slots, pool[0], pool[1], q_out=q) is q
    assert torch.equal(q, want) and torch.equal(pool[0].view(-1, Hkv, D)[slots], paged.rope(k.contiguous(), pos, table))


def test_append_slot_past_the_pool_is_dropped_and_reported():
    pool = torch.zeros(2, 2, 16, 1, 32, dtype=BF, device=DEV)
    k = torch.ones(3, 1, 32, dtype=BF, device=DEV)
    paged.rope_append(None, k, k, None, None, torch.tensor([32, 5, 1 << 40], device=DEV), pool[0], pool[1])
    assert scope_b200.status_take() == 5
    assert pool[0].view(32, 32).sum(1).tolist() == [32.0 if i == 5 else 0.0 for i in range(32)]


def test_append_refusals():
    pool = torch.zeros(2, 2, 16, 2, 32, dtype=BF, device=DEV)
    k, slots = torch.ones(3, 2, 32, dtype=BF, device=DEV), torch.zeros(3, dtype=torch.int64, device=DEV)
    pos, table = slots.int(), table_of(10, 32)
    for match, a, kw in [
            ("as the pool", (None, k[:, :1], k, None, None, slots, pool[0], pool[1]), {}),
            ("slots", (None, k, k, None, None, slots.int(), pool[0], pool[1]), {}),
            ("slots", (None, k, k, None, None, slots[:2], pool[0], pool[1]), {}),
            ("both or neither", (None, k, k, pos, None, slots, pool[0], pool[1]), {}),
            ("inputs' type", (None, k.half(), k.half(), None, None, slots, pool[0], pool[1]), {}),
            ("q must be", (torch.ones(3, 2, 48, dtype=BF, device=DEV), k, k, pos, table, slots, pool[0], pool[1]), {}),
            ("q_out without q", (None, k, k, pos, table, slots, pool[0], pool[1]), dict(q_out=k)),
            ("v must be", (None, k, k.half(), None, None, slots, pool[0], pool[1]), {}),
            ("unit stride", (None, k, k, None, None, slots, pool[0].transpose(2, 3).contiguous().transpose(2, 3), pool[1]), {})]:
        with pytest.raises(RuntimeError, match=match):
            paged.rope_append(*a, **kw)


# ------------------------------------------------------------------ together


def serve(cache, steps, H, Hkv, D, sections, capture):
    """Drive a cache through ``steps`` (new_lens, done) and check every decode against tokens kept apart."""
    g, R, P = gen(21), cache.max_requests, cache.page_size
    scale, top = D ** -0.5, 4096
    table = table_of(top, D)
    int8 = cache.k_pages[0].dtype == torch.int8
    kept = [[[], []] for _ in range(R)]
    N = max(sum(n) for n, _ in steps)
    new = torch.zeros(R, dtype=torch.int32, device=DEV)
    qkv = torch.zeros(N, (H + 2 * Hkv) * D, dtype=BF, device=DEV)
    last = torch.zeros(R, dtype=torch.int64, device=DEV)
    held = {}

    def body():
        step = cache.begin_step(new, N)
        q, k, v = qkv.split([H * D, Hkv * D, Hkv * D], 1)
        pos = step.positions.expand(3, N).contiguous() if sections else None
        q = cache.append(1, q.view(N, H, D), k.view(N, Hkv, D), v.view(N, Hkv, D), step, table, positions=pos,
                         sections=sections)
        held.update(step=step, q=q, out=cache.decode(1, q[last], scale))

    graph = None
    for n, done in steps:
        new.copy_(torch.tensor(n, dtype=torch.int32))
        qkv.copy_(torch.randn(qkv.shape, generator=g, device=DEV).to(BF))
        ends = np.cumsum(n)
        last.copy_(torch.tensor([max(int(e) - 1, 0) for e in ends]))
        if not capture:
            body()
        else:
            if graph is None:   # the first step outside, so that the workspace is there, then the same step again in a graph
                before = cache.seq_lens.clone(), cache._ring.clone()
                side = torch.cuda.Stream()
                side.wait_stream(torch.cuda.current_stream())
                with torch.cuda.stream(side):
                    body()
                    side.synchronize()
                    cache.seq_lens.copy_(before[0]), cache._ring.copy_(before[1])
                    graph = torch.cuda.CUDAGraph()
                    with torch.cuda.graph(graph, stream=side):
                        body()
            graph.replay()
        torch.cuda.synchronize()
        assert cache.refused() == 0
        q, k, v = qkv.split([H * D, Hkv * D, Hkv * D], 1)
        at = 0
        for b in range(R):
            L = sum(x.shape[0] for x in kept[b][0])
            p = torch.arange(L, L + n[b], device=DEV)
            kk = turned(k[at:at + n[b]].view(-1, Hkv, D), p[None], table, [0] * (D // 2), "half")
            vv = v[at:at + n[b]].view(-1, Hkv, D).float()
            if int8:
                (ck, sk), (cv, sv) = codes(kk), codes(vv)
                kk, vv = ck.double() * sk.double()[..., None], cv.double() * sv.double()[..., None]
            else:
                kk, vv = kk.to(BF).double(), vv.double()
            kept[b][0].append(kk), kept[b][1].append(vv)
            at += n[b]
        out, lse = held["out"]
        for b in range(R):
            kk, vv = torch.cat(kept[b][0]), torch.cat(kept[b][1])
            assert int(cache.seq_lens[b]) == kk.shape[0]
            if kk.shape[0] == 0:
                assert (out[b] == 0).all() and torch.isneginf(lse[b]).all()
                continue
            qb = held["q"][last[b]].double().view(Hkv, H // Hkv, D)
            z = torch.einsum("hgd,thd->hgt", qb, kk) * scale
            want = torch.einsum("hgt,thd->hgd", torch.softmax(z, -1), vv).reshape(H, D)
            room = torch.einsum("hgt,thd->hgd", torch.softmax(z, -1), vv.abs()).reshape(H, D)
            assert ((out[b].double() - want).abs() <= (2 * U[BF] + 1e-4) * room + 1e-7).all()
            assert (lse[b].double() - torch.logsumexp(z, -1).view(H)).abs().max() < 1e-4
        cache.release(torch.tensor(done, device=DEV))
        for b in range(R):
            if done[b]:
                kept[b] = [[], []]
    pages = sum(-(-sum(x.shape[0] for x in kept[b][0]) // P) for b in range(R))
    assert cache.free_pages() == cache.num_pages - pages
    assert scope_b200.status_take() == 0


@pytest.mark.parametrize("dtype", [BF, torch.int8])
@pytest.mark.parametrize("sections", [None, (16, 8, 8)])
@pytest.mark.parametrize("capture", [False, True])
def test_requests_come_and_go(dtype, sections, capture):
    H, Hkv, D = 8, 2, 64
    cache = PagedKVCache(2, 60, 16, Hkv, D, 5, 400, dtype=dtype, device=DEV)
    F, T = False, True
    steps = [([33, 0, 1, 16, 100], [F] * 5), ([1, 1, 1, 1, 1], [F, F, T, F, F]), ([1, 50, 17, 1, 1], [T, F, F, F, T]),
             ([200, 1, 1, 1, 90], [F] * 5), ([1, 1, 1, 1, 1], [F] * 5), ([1, 1, 1, 1, 1], [T] * 5), ([7, 0, 0, 9, 1], [F] * 5)]
    serve(cache, steps, H, Hkv, D, sections, capture)


def test_cache_refuses_what_does_not_fit_and_goes_on():
    cache = PagedKVCache(1, 4, 16, 1, 32, 3, 64, device=DEV)
    new = torch.tensor([40, 20, 16], dtype=torch.int32, device=DEV)
    step = cache.begin_step(new, 76)
    assert cache.refused() == 2 and cache.free_pages() == 1 and cache.seq_lens.tolist() == [40, 0, 0]
    assert (step.slots[40:] == -1).all() and (step.slots[:40] >= 0).all()
    cache.release(torch.tensor([True, False, False], device=DEV))
    cache.begin_step(torch.tensor([0, 20, 16], dtype=torch.int32, device=DEV), 36)
    assert cache.refused() == 0 and cache.free_pages() == 1 and cache.seq_lens.tolist() == [0, 20, 16]
    cache.reset()
    assert cache.free_pages() == 4 and cache.seq_lens.tolist() == [0, 0, 0]


def test_decode_more_requests_than_one_launch_counts():
    """A table so wide that its rows, were they full, pass the kernel's 32-bit count: several launches, one result."""
    g = gen(30)
    P, D, B = 1 << 20, 16, 20
    k, v = (torch.empty(1, P, 1, D, dtype=BF, device=DEV) for _ in range(2))
    k[0, :100], v[0, :100] = (torch.randn(100, 1, D, generator=g, device=DEV).to(BF) for _ in range(2))
    lens = [(7 * b) % 101 for b in range(B)]
    t = torch.zeros(B, 1024, dtype=torch.int32, device=DEV)
    s = dict(q=torch.randn(B, 2, D, generator=g, device=DEV).to(BF), k=k, v=v, ks=None, vs=None, table=t,
             lens=torch.tensor(lens, dtype=torch.int32, device=DEV), scale=D ** -0.5,
             rows=[(torch.zeros(n, dtype=torch.long, device=DEV), torch.arange(n, device=DEV)) for n in lens])
    agrees(s, *decode(s))
    wide = torch.zeros(1, 1 << 11, dtype=torch.int32, device=DEV)
    pool = torch.empty(1, P, 17, D, dtype=BF, device=DEV)
    with pytest.raises(RuntimeError, match="too many tokens"):
        paged.paged_decode(torch.zeros(1, 17, D, dtype=BF, device=DEV), pool, pool, wide, s["lens"][:1].contiguous(), 1.0)


@pytest.mark.parametrize("dtype,pool", [(BF, BF), (HF, HF), (BF, torch.int8), (HF, torch.int8)])
@pytest.mark.parametrize("D,Dv", [(64, 64), (128, 128), (256, 256), (192, 128), (80, 80)])
def test_decode_variants_with_whole_and_split_pages(dtype, pool, D, Dv):
    """Each compiled variant over lengths that end in every part of a subtile, pages of whole tiles and not."""
    lens = list(range(1, 34)) + [47, 48, 49, 63, 64, 65, 96, 97, 700]
    for P in (16, 32, 48, 20):
        s = make_decode(lens, 12, 2, D, Dv, P, dtype, pool, heads_major=P == 32, seed=D + P)
        agrees(s, *decode(s))
        agrees(s, *decode(s, 33), window=33)
    assert scope_b200.status_take() == 0


def test_decode_int8_values_are_exact():
    """One token: the output is its value row, code * scale, for every code."""
    codes_ = torch.arange(-128, 128, dtype=torch.int16, device=DEV).to(torch.int8).view(1, 1, 1, 256)
    for dtype in (BF, HF):
        scale = torch.tensor([0.0371], device=DEV).view(1, 1, 1)
        q = torch.randn(1, 1, 256, device=DEV).to(dtype)
        one = torch.ones(1, dtype=torch.int32, device=DEV)
        out, lse = paged.paged_decode(q, codes_, codes_, one.view(1, 1) * 0, one, 0.01, k_scales=scale, v_scales=scale)
        want = codes_.view(-1).double() * scale.double().view(-1)
        # the probability is 1: its product with the scale as two 16-bit values (2^-16), then one rounding of the result
        assert ((out.view(-1).double() - want).abs() <= (U[dtype] + 2.0 ** -15) * want.abs()).all()
        z = 0.01 * 0.0371 * (q.double().view(-1) @ codes_.view(-1).double())
        assert (lse.double().view(()) - z).abs() <= 260 * 2.0 ** -24 * 0.01 * 0.0371 * (q.double().abs().view(-1) @ codes_.view(-1).double().abs()) + 1e-6


@pytest.mark.parametrize("pool", [BF, torch.int8])
def test_decode_passes_a_nan_on_to_its_rows_alone(pool):
    """A NaN key gives its request and kv head NaN, in the output and in lse; every other row stays as it was."""
    s = make_decode([700, 40, 300], 8, 2, 64, 64, 16, BF, pool=pool, seed=53)
    out, lse = (x.clone() for x in decode(s))
    page, at = int(s["table"][0, 5]), 3
    if pool == torch.int8:
        s["ks"][page, at, 1] = float("nan")
    else:
        s["k"][page, at, 1, 0] = float("nan")
    bad, bad_lse = decode(s)
    assert bad[0, 4:].isnan().all() and bad_lse[0, 4:].isnan().all()
    out[0, 4:], lse[0, 4:], bad[0, 4:], bad_lse[0, 4:] = 0, 0, 0, 0
    assert torch.equal(out, bad) and torch.equal(lse, bad_lse)


def test_decode_refuses_more_heads_than_it_counts():
    k = torch.zeros(1, 16, 1, 16, dtype=BF, device=DEV).expand(1, 16, 40000, 16)
    table, lens = torch.zeros(1, 1, dtype=torch.int32, device=DEV), torch.ones(1, dtype=torch.int32, device=DEV)
    with pytest.raises(RuntimeError, match="too many heads"):
        paged.paged_decode(torch.zeros(1, 40000, 16, dtype=BF, device=DEV), k, k, table, lens, 1.0)
    k = torch.zeros(1, 16, 1, 16, dtype=BF, device=DEV)
    with pytest.raises(RuntimeError, match="too many heads"):
        paged.paged_decode(torch.zeros(1, (1 << 18) + 8, 16, dtype=BF, device=DEV), k, k, table, lens, 1.0)


def test_slots_take_a_negative_head_as_the_rings_start():
    """The ring's words are the caller's memory: whatever they hold, a page comes from within the ring."""
    free = np.arange(100, 108, dtype=np.int32)
    lens, new, table = np.zeros(1, np.int32), np.full(1, 20, np.int32), np.full((1, 4), -1, np.int32)
    for count in (8, 1 << 30):
        got, d = run_slots(lens, new, table, free, np.array([-5, count, 0], np.int32), 16, 20)
        assert got[0].tolist() == [1600 + i for i in range(20)] and got[4].tolist() == [2, 6, 0]
    d[4].copy_(torch.tensor([-5, 6, 0]))
    lens_out, ring = paged.paged_release(torch.full((1,), 20, dtype=torch.int32, device=DEV),
                                         torch.ones(1, dtype=torch.bool, device=DEV), d[2], d[3], d[4], 16)
    assert ring.tolist() == [0, 8, 0] and d[3].tolist() == [100, 101, 102, 103, 104, 105, 100, 101]


LONG = [0, 1, 15, 16, 17, 31, 33, 64, 65, 200, 511, 601, 1300, 2000]


@pytest.mark.parametrize("heads_major", [False, True])
@pytest.mark.parametrize("dtype,pool", [(BF, BF), (HF, HF), (BF, torch.int8), (HF, torch.int8)])
@pytest.mark.parametrize("D", [64, 128, 192, 256])
@pytest.mark.parametrize("P,Hkv,G,window", [(16, 2, 4, 0), (64, 1, 12, 600), (48, 3, 1, 0)])
def test_decode_wide_tables_of_whole_tiles(heads_major, dtype, pool, D, P, Hkv, G, window):
    """Long rows and short ones in pages of whole 16-token tiles: what lies past a length in a tile is NaN."""
    s = make_decode(LONG, Hkv * G, Hkv, D, D, P, dtype, pool=pool, heads_major=heads_major, seed=61)
    agrees(s, *decode(s, window=window), window=window)
    out, lse = decode(s, window=window)
    again, lse2 = decode(s, window=window)
    assert torch.equal(out, again) and torch.equal(lse, lse2)
    assert scope_b200.status_take() == 0


@pytest.mark.parametrize("pool", [BF, torch.int8])
def test_decode_wide_tables_leave_out_pages_that_are_none(pool):
    s = make_decode([900, 40, 17, 3000], 8, 2, 128, 128, 16, BF, pool=pool, seed=62)
    bad = torch.zeros(s["k"].shape[0] + 1, dtype=torch.bool, device=DEV)
    for b, col, put in ((0, 3, -1), (0, 4, s["k"].shape[0]), (0, 56, 1 << 30), (1, 0, -5), (2, 1, -1), (3, 100, -1)):
        bad[int(s["table"][b, col])] = True
        s["table"][b, col] = put
    agrees(s, *decode(s), leave_out=lambda page: ~bad[page])
    assert scope_b200.status_take() != 0 and scope_b200.status_take() == 0


@pytest.mark.parametrize("head,tok", [(136, 272), (136, 280), (128, 256), (144, 456)])
def test_decode_wide_tables_of_a_pool_with_gaps(head, tok):
    """Rows and tokens further apart than they are long, pages that are every other one of a larger buffer."""
    s = make_decode(LONG, 8, 2, 128, 128, 16, BF, seed=63)
    n = s["k"].shape[0]
    for name in ("k", "v"):
        wide = torch.full((n * 2 * 16 * tok,), float("nan"), dtype=BF, device=DEV)
        wide = wide.as_strided(s[name].shape, (2 * 16 * tok, tok, head, 1), 16 * tok)
        wide.copy_(s[name])
        s[name] = wide
    agrees(s, *decode(s))


@pytest.mark.parametrize("heads_major", [False, True])
@pytest.mark.parametrize("dtype,pool", [(BF, BF), (HF, HF), (BF, torch.int8), (HF, torch.int8)])
@pytest.mark.parametrize("Dk,Dv", [(16, 16), (32, 32), (48, 48), (80, 80), (96, 96), (112, 112), (64, 16), (128, 64), (80, 128),
                                   (96, 192), (192, 128), (160, 160), (224, 64), (256, 80), (144, 240)])
def test_decode_wide_tables_of_any_head_dims(heads_major, dtype, pool, Dk, Dv):
    s = make_decode(LONG, 12, 2, Dk, Dv, 32, dtype, pool=pool, heads_major=heads_major, seed=64)
    agrees(s, *decode(s))
    assert scope_b200.status_take() == 0

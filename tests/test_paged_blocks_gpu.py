"""GPU checks of pages held in 8 bits with one scale for each block of tokens and head: the append that quantises, the way
back to rows, the decode.

Codes, scales and rows read back are whole formulas of fp32 operations, so they are compared bit for bit with the same
formulas in torch; how far a written value is from the one it stands for is bounded in 64 bits: half a step, s / 2 (int8) or
2^-4 |x| and 2^-10 s (e4m3, normal and subnormal), each widened by 2^-20 for the fp32 product and the scale's own rounding.

Decode.  A score is a sum of Dk products, exact in fp32, added in fp32: ds = (Dk + 4) 2^-24 scale sum |q k| (queries that
went to fp16 under a power of two are exact to 2^-38 of the head's largest).  A probability enters its product to 2^-21
(two fp16 parts; its scale's product), sums over n tokens are fp32, the result is rounded once, by u / 2 steps:
    |do| <= (u + 2 ds + (n + 64) 2^-24 + 2^-20) sum p|v| + 2^-24,    |dlse| <= ds + (min(n, 4096) + 64) 2^-24 + 2^-22 |lse|
with u = 2^-8 for bf16 and 2^-11 for fp16 (half a step, relative).
"""
import pytest
import torch

import scope_b200
from scope_b200 import PagedKVCache, paged
from test_paged_gpu import BF, DEV, HF, U, gen, table_of, turned

pytestmark = pytest.mark.gpu
E4, I8 = torch.float8_e4m3fn, torch.int8


def raw(x):
    return x.view(torch.uint8)


def to_codes(x, inv, pool):
    if pool == I8:
        return torch.round(x * inv).clamp(-127, 127).to(I8)
    return (x * inv).clamp(-448, 448).to(E4)


def scale_for(most, pool):
    """The scale that a block's largest value asks for."""
    if not bool(torch.isfinite(most)):
        return most
    most = most.clamp(min=1e-6)
    if pool == I8:
        return most * (1.0 / 127.0)
    part, up = torch.frexp(most)
    return torch.exp2((up - 9 + (part > 0.875).int()).float())


def append_reference(x, slots, pages, scales, block):
    """The rule, block by block and head by head, on copies of (pages, scales); x fp32 [N, heads, D]."""
    pages, scales = pages.clone(), scales.clone()
    P, pool = pages.shape[1], pages.dtype
    by_block = {}
    for t, s in enumerate(slots.tolist()):
        if 0 <= s < pages.shape[0] * P:
            by_block.setdefault(s // block, []).append((t, s % block))
    one = torch.ones((), device=DEV)
    for key, tokens in by_block.items():
        page, j = key * block // P, key * block % P // block
        first = min(o for _, o in tokens)
        for h in range(x.shape[1]):
            rows = x[[t for t, _ in tokens], h]
            most = rows.abs().amax() if not rows.isnan().any() else rows.new_tensor(float("nan"))
            need, held = scale_for(most, pool), scales[page, j, h].clone()
            s = torch.maximum(held, need) if first else need      # maximum keeps a NaN
            fine = bool(torch.isfinite(s))
            inv = one / s if fine else one * 0
            block_rows = raw(pages[page, j * block:(j + 1) * block, h])
            new = to_codes(rows, inv, pool) if fine else torch.zeros_like(rows, dtype=torch.uint8)
            if first and not bool(s == held):
                old = pages[page, j * block:j * block + first, h].float()
                block_rows[:first] = raw(to_codes(old, held * inv, pool)) if fine else 0
            block_rows[[o for _, o in tokens]] = raw(new)
            scales[page, j, h] = s
    return pages, scales


def make_pool(g, n_pages, P, block, Hkv, D, pool, heads_major=False, lo=0.01):
    shape, blocks = ((n_pages, Hkv, P), (n_pages, Hkv, P // block)) if heads_major else ((n_pages, P, Hkv), (n_pages, P // block, Hkv))
    x = torch.randn(*shape, D, generator=g, device=DEV)
    x = (x * 32).round().clamp(-127, 127).to(I8) if pool == I8 else (x * 100).clamp(-448, 448).to(E4)
    s = torch.rand(*blocks, generator=g, device=DEV) * 0.02 + lo
    if pool == E4:
        s = torch.exp2(torch.floor(torch.log2(s)))
    return (x.transpose(1, 2), s.transpose(1, 2)) if heads_major else (x, s)


def chunk_slots(g, starts, news, P, n_pages):
    """Slots of requests that hold starts[b] tokens and add news[b], each with pages of its own."""
    ids, at, out = torch.randperm(n_pages, generator=g, device=DEV), 0, []
    for L, n in zip(starts, news):
        held = -(-(L + n) // P)
        t = torch.arange(L, L + n, device=DEV)
        out.append(ids[at + t // P] * P + t % P)
        at += held
    assert at <= n_pages
    return torch.cat(out)


APPENDS = [  # starts, news, H, Hkv, D, Dv, rot, P, block
    ([5], [1], 8, 2, 128, 128, 128, 16, 16),
    ([0, 3, 15, 16, 31, 17], [1, 1, 1, 1, 1, 1], 8, 8, 128, 128, 128, 16, 16),
    ([0, 7, 64, 100], [130, 3, 64, 29], 4, 2, 64, 64, 64, 64, 32),
    ([0, 23, 11], [50, 70, 1], 5, 5, 80, 80, 64, 24, 8),
    ([2, 0], [300, 9], 2, 1, 256, 64, 128, 256, 256),
    ([1, 90], [700, 40], 3, 3, 16, 240, 16, 128, 128),
    ([0, 511], [1030, 600], 2, 1, 192, 128, 64, 512, 512),
    ([4, 9, 0], [9, 2, 31], 2, 2, 96, 96, 96, 10, 5),
    ([3, 0, 1], [4, 6, 1], 2, 2, 32, 32, 32, 7, 1),
]


@pytest.mark.parametrize("case", range(len(APPENDS)))
@pytest.mark.parametrize("dtype,pool", [(BF, I8), (HF, E4), (BF, E4), (HF, I8)])
@pytest.mark.parametrize("heads_major,pairs", [(False, "half"), (True, "adjacent")])
def test_append_quantises_blocks(case, dtype, pool, heads_major, pairs):
    starts, news, H, Hkv, D, Dv, rot, P, block = APPENDS[case]
    if block == 1 and pool == I8:
        pytest.skip("a scale per row: tests of the plain append")
    g = gen(case)
    N, n_pages = sum(news), sum(-(-(a + b) // P) for a, b in zip(starts, news)) + 2
    table, pos = table_of(1200, rot), torch.cat([torch.arange(a, a + b, device=DEV) for a, b in zip(starts, news)]).int() % 1200
    qkv = torch.randn(N, H * D + Hkv * (D + Dv), generator=g, device=DEV).to(dtype)
    q, k, v = (x.view(N, h, d) for x, h, d in zip(qkv.split([H * D, Hkv * D, Hkv * Dv], 1), (H, Hkv, Hkv), (D, D, Dv)))
    k.mul_(torch.rand(N, 1, 1, generator=g, device=DEV).to(dtype) * 3)
    v[::3] *= 0.01
    kp, ks = make_pool(g, n_pages, P, block, Hkv, D, pool, heads_major)
    vp, vs = make_pool(g, n_pages, P, block, Hkv, Dv, pool, heads_major, lo=1e-4)
    slots = chunk_slots(g, starts, news, P, n_pages)
    rk = turned(k, pos[None], table, [0] * (rot // 2), pairs)
    wk, wks = append_reference(rk, slots, kp, ks, block)
    wv, wvs = append_reference(v.float(), slots, vp, vs, block)
    got = paged.rope_append(q, k, v, pos, table, slots, kp, vp, k_scales=ks, v_scales=vs, pairs=pairs)
    assert torch.equal(got, turned(q, pos[None], table, [0] * (rot // 2), pairs).to(dtype))
    assert torch.equal(ks, wks) and torch.equal(vs, wvs)
    assert torch.equal(raw(kp), raw(wk)) and torch.equal(raw(vp), raw(wv))
    for x, pages, scales in ((rk, kp, ks), (v.float(), vp, vs)):
        page, off = slots // P, slots % P
        s = scales[page, off // block].double()[..., None]
        err = (pages.view(torch.uint8)[page, off].view(pool).double() * s - x.double()).abs()
        bound = s / 2 if pool == I8 else torch.maximum(x.double().abs() * 2.0 ** -4, s * 2.0 ** -10)
        assert (err <= bound * (1 + 2.0 ** -20) + s * 127 * 2.0 ** -22).all()
    assert scope_b200.status_take() == 0


@pytest.mark.parametrize("pool", [I8, E4])
def test_append_token_by_token_is_the_rule_each_time(pool):
    """A decode's appends, a block's scale growing now and then; what is kept is within the sum of half steps."""
    g, P, block, Hkv, D = gen(3), 32, 16, 2, 64
    kp, ks = make_pool(g, 2, P, block, Hkv, D, pool)
    vp, vs = make_pool(g, 2, P, block, Hkv, D, pool)
    ks.fill_(float("nan"))   # of earlier owners of the page
    x = torch.randn(40, Hkv, D, generator=g, device=DEV) * torch.exp2(torch.arange(40, device=DEV) % 16 / 4.0)[:, None, None]
    x = x.to(BF)
    slots = torch.arange(40, device=DEV) + 8 * 0
    wk, wks = kp, ks
    for t in range(40):
        wk, wks = append_reference(x[t:t + 1].float(), slots[t:t + 1], wk, wks, block)
    for t in range(40):
        paged.rope_append(None, x[t:t + 1], x[t:t + 1], None, None, slots[t:t + 1], kp, vp, k_scales=ks, v_scales=vs)
    assert torch.equal(raw(kp)[:1], raw(wk)[:1]) and torch.equal(ks[:1], wks[:1])
    s = ks.view(-1, Hkv)[slots // block].double()[..., None]
    err = (kp.view(2 * P, Hkv, D)[slots].double() * s - x.double()).abs()
    # at most 16 roundings, each to half a step of a scale that is not above the last
    assert (err <= (8 * s if pool == I8 else x.double().abs() * 2.0 ** -4 + s * 2.0 ** -9 * 16)).all()


@pytest.mark.parametrize("pool", [I8, E4])
def test_append_dropped_tokens_between_and_around(pool):
    g, P, block = gen(4), 64, 32
    kp, ks = make_pool(g, 9, P, block, 3, 48, pool)
    vp, vs = make_pool(g, 9, P, block, 3, 48, pool)
    slots = chunk_slots(g, [10, 0, 40], [100, 200, 60], P, 9)
    drop = torch.rand(len(slots), generator=g, device=DEV) < 0.3
    slots[drop] = -1
    slots = torch.cat([torch.full((40,), -1, device=DEV), slots[:90], torch.full((31,), -5, device=DEV), slots[90:],
                       torch.full((70,), -1, device=DEV)])
    k, v = (torch.randn(len(slots), 3, 48, generator=g, device=DEV).to(BF) for _ in range(2))
    wk, wks = append_reference(k.float(), slots, kp, ks, block)
    wv, wvs = append_reference(v.float(), slots, vp, vs, block)
    paged.rope_append(None, k, v, None, None, slots, kp, vp, k_scales=ks, v_scales=vs)
    # rows between the first and the last of a block that were dropped are nobody's, and left as they were
    assert torch.equal(ks, wks) and torch.equal(vs, wvs)
    assert torch.equal(raw(kp), raw(wk)) and torch.equal(raw(vp), raw(wv))
    assert scope_b200.status_take() == 0


@pytest.mark.parametrize("pool", [I8, E4])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_append_what_is_not_finite_makes_the_block_nan(pool, bad):
    g, P, block = gen(5), 16, 8
    kp, ks = make_pool(g, 2, P, block, 2, 32, pool)
    vp, vs = make_pool(g, 2, P, block, 2, 32, pool)
    k = torch.randn(6, 2, 32, generator=g, device=DEV).to(BF)
    k[4, 1, 7] = bad
    slots = torch.arange(3, 9, device=DEV)      # offsets 3..7 of block 0, 0 of block 1
    wk, wks = append_reference(k.float(), slots, kp, ks, block)
    paged.rope_append(None, k, k, None, None, slots, kp, vp, k_scales=ks, v_scales=vs)
    assert torch.equal(raw(kp), raw(wk)) and torch.equal(ks.nan_to_num(nan=-7.0), wks.nan_to_num(nan=-7.0))
    table, cu = torch.zeros(1, 1, dtype=torch.int32, device=DEV), torch.tensor([0, 9], dtype=torch.int32, device=DEV)
    rows, _ = paged.paged_read(kp, vp, table, cu, 9, k_scales=ks, v_scales=vs)
    assert rows[:8, 1].isnan().all() and rows[8, 1].isfinite().all() and rows[:, 0].isfinite().all()
    # the block stays so, and the next one is its own
    k2 = torch.ones(2, 2, 32, dtype=BF, device=DEV)
    paged.rope_append(None, k2, k2, None, None, torch.tensor([7, 9], device=DEV), kp, vp, k_scales=ks, v_scales=vs)
    assert not ks[0, 0, 1].isfinite() and ks[0, 1].isfinite().all()


def test_append_scale_limits():
    """Rows of zeros, the least and the largest bf16 values; e4m3's border between two powers."""
    for pool in (I8, E4):
        x = torch.zeros(6, 1, 16, device=DEV)
        x[1, 0, 0], x[2, 0, 0], x[3, 0, 0], x[4, 0, 0], x[5, 0, 0] = 3.3e38, 448.0, 450.0, 1e-30, 2.0 ** -28 * 448
        x = x.to(BF)
        kp, ks = make_pool(gen(6), 6, 4, 4, 1, 16, pool)
        vp, vs = make_pool(gen(7), 6, 4, 4, 1, 16, pool)
        slots = torch.arange(6, device=DEV) * 4
        wk, wks = append_reference(x.float(), slots, kp, ks, 4)
        paged.rope_append(None, x, x, None, None, slots, kp, vp, k_scales=ks, v_scales=vs)
        assert torch.equal(raw(kp), raw(wk)) and torch.equal(ks, wks)
        if pool == E4:
            assert ks[2, 0, 0] == 1 and ks[3, 0, 0] == 2 and ks[0, 0, 0] == 2.0 ** -28


@pytest.mark.parametrize("sections,cyclic", [((12, 10, 10), False), ((12, 10, 10), True), (None, False)])
@pytest.mark.parametrize("i64,odd", [(False, False), (True, True)])
@pytest.mark.parametrize("N", [30, 3000])
def test_append_turns_by_axes_positions_out_of_range_and_unaligned_turns(sections, cyclic, i64, odd, N):
    g, Hkv, D, P, block = gen(8), 2, 80, 32, 16
    A = 1 if sections is None else 3
    table = table_of(50, 64)
    if odd:   # 4 bytes past a boundary
        table = torch.cat([table.new_zeros(1), table.flatten()])[1:].view(50, 64)
    pos = torch.randint(0, 50, (A, N), generator=g, device=DEV, dtype=torch.int64 if i64 else torch.int32)
    given = pos.clone()
    given[:, 3], pos[:, 3] = -7, 0
    given[:, 9], pos[:, 9] = (1 << 40) if i64 else (1 << 30), 49
    axes = [0] * 32
    if sections and cyclic:
        axes = [i % 3 if i // 3 < sections[i % 3] else 0 for i in range(32)]
    elif sections:
        axes = [a for a, n in enumerate(sections) for _ in range(n)]
    q, k, v = (torch.randn(N, h, D, generator=g, device=DEV).to(HF) for h in (4, Hkv, Hkv))
    kp, ks = make_pool(g, 100, P, block, Hkv, D, E4)
    vp, vs = make_pool(g, 100, P, block, Hkv, D, E4)
    slots = torch.arange(N, device=DEV) + 5
    rk = turned(k, pos, table, axes, "half")
    wk, wks = append_reference(rk, slots, kp, ks, block)
    got = paged.rope_append(q, k, v, given[0] if A == 1 else given, table, slots, kp, vp, k_scales=ks, v_scales=vs, sections=sections,
                            cyclic=cyclic)
    assert torch.equal(got, turned(q, pos, table, axes, "half").to(HF))
    assert torch.equal(ks, wks) and torch.equal(raw(kp), raw(wk))
    assert scope_b200.status_take() == 5


@pytest.mark.parametrize("N,H,Hkv,D,Dv,rot,P", [(1, 8, 2, 128, 128, 128, 16), (513, 12, 3, 80, 80, 64, 24), (3000, 8, 4, 64, 192, 64, 1)])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("pairs", ["half", "adjacent"])
def test_append_e4m3_rows_in_any_order(N, H, Hkv, D, Dv, rot, P, dtype, pairs):
    """A scale a row: rows of zeros, of one NaN and of one infinity among them, slots in any order."""
    g = gen(N)
    table, pos = table_of(400, rot), torch.randint(0, 400, (1, N), generator=g, device=DEV)
    q, k, v = (torch.randn(N, h, d, generator=g, device=DEV).to(dtype) for h, d in ((H, D), (Hkv, D), (Hkv, Dv)))
    if N > 5:
        k[2], v[3, 0, 5], v[4, 1, 0] = 0, float("nan"), float("-inf")
    n_pages = -(-N // P) + 5
    (kp, ks), (vp, vs) = (make_pool(g, n_pages, P, 1, Hkv, d, E4, heads_major=D == 80) for d in (D, Dv))
    slots = torch.randperm(n_pages * P, generator=g, device=DEV)[:N].contiguous()
    slots[torch.rand(N, generator=g, device=DEV) < 0.1] = -1
    wk, wks, wv, wvs = kp.clone(), ks.clone(), vp.clone(), vs.clone()
    rk = turned(k, pos, table, [0] * (rot // 2), pairs)
    at = torch.nonzero(slots >= 0)[:, 0]
    page, off = slots[at] // P, slots[at] % P
    for x, pages, scales in ((rk, wk, wks), (v.float(), wv, wvs)):
        most = x.abs().amax(-1).clamp(min=1e-6)      # clamp keeps a NaN
        part, up = torch.frexp(most)
        s = torch.where(most.isfinite(), torch.exp2((up - 9 + (part > 0.875).int()).float()), most)
        codes = torch.where(most.isfinite()[..., None], (x * (torch.ones_like(s) / s)[..., None]).clamp(-448, 448), 0.0).to(E4)
        raw(pages)[page, off], scales[page, off] = raw(codes)[at], s[at]
    got = paged.rope_append(q, k, v, pos, table, slots, kp, vp, k_scales=ks, v_scales=vs, pairs=pairs)
    assert torch.equal(got, turned(q, pos, table, [0] * (rot // 2), pairs).to(dtype))
    assert torch.equal(raw(kp), raw(wk)) and torch.equal(raw(vp), raw(wv))
    assert torch.equal(ks, wks) and torch.equal(vs.nan_to_num(nan=-3.0), wvs.nan_to_num(nan=-3.0))
    assert scope_b200.status_take() == 0


def test_append_of_a_slot_beside_others_and_in_place():
    """Queries turned in place in the packed projection that keys and values are read from; a call without a token."""
    g, N, H, Hkv, D = gen(12), 70, 4, 2, 64
    for n in (N, 4000):
        qkv = torch.randn(n, (H + 2 * Hkv) * D, generator=g, device=DEV).to(BF)
        q, k, v = (x.view(n, h, D) for x, h in zip(qkv.split([H * D, Hkv * D, Hkv * D], 1), (H, Hkv, Hkv)))
        table, pos = table_of(100, D), torch.randint(0, 100, (n,), generator=g, device=DEV)
        kp, ks = make_pool(g, 260, 16, 16, Hkv, D, I8)
        vp, vs = make_pool(g, 260, 16, 16, Hkv, D, I8)
        slots = torch.arange(n, device=DEV)
        want = turned(q, pos[None], table, [0] * 32, "half").to(BF)
        wk, wks = append_reference(turned(k, pos[None], table, [0] * 32, "half"), slots, kp, ks, 16)
        wv, wvs = append_reference(v.float(), slots, vp, vs, 16)
        assert paged.rope_append(q, k, v, pos, table, slots, kp, vp, k_scales=ks, v_scales=vs, q_out=q) is q
        assert torch.equal(q, want)
        assert torch.equal(raw(kp), raw(wk)) and torch.equal(raw(vp), raw(wv)) and torch.equal(ks, wks) and torch.equal(vs, wvs)
    none = torch.empty(0, Hkv, D, dtype=BF, device=DEV)
    paged.rope_append(None, none, none, None, None, slots[:0], kp, vp, k_scales=ks, v_scales=vs)
    assert torch.equal(raw(kp), raw(wk))


def test_append_behind_many_dropped_tokens():
    """A block that goes on behind thousands of dropped tokens, in a call that ends in as many."""
    g, P, block = gen(13), 64, 64
    kp, ks = make_pool(g, 3, P, block, 1, 32, I8)
    vp, vs = make_pool(g, 3, P, block, 1, 32, I8)
    slots = torch.full((9000,), -1, dtype=torch.int64, device=DEV)
    slots[10], slots[4000], slots[4100], slots[4101] = 70, 72, 71 + 5, 128
    k, v = (torch.randn(9000, 1, 32, generator=g, device=DEV).to(BF) for _ in range(2))
    wk, wks = append_reference(k.float(), slots, kp, ks, block)
    wv, wvs = append_reference(v.float(), slots, vp, vs, block)
    paged.rope_append(None, k, v, None, None, slots, kp, vp, k_scales=ks, v_scales=vs)
    assert torch.equal(ks, wks) and torch.equal(vs, wvs) and torch.equal(raw(kp), raw(wk)) and torch.equal(raw(vp), raw(wv))


def test_append_slots_past_the_pool_and_unaligned_rows():
    pool, scales = torch.zeros(2, 2, 16, 1, 32, dtype=I8, device=DEV), torch.zeros(2, 2, 2, 1, device=DEV)
    flat = torch.ones(4 * 32 + 3, device=DEV).to(BF)
    k = flat[3:].view(4, 1, 32)
    paged.rope_append(None, k, k, None, None, torch.tensor([32, 5, 1 << 40, 6], device=DEV), pool[0], pool[1], k_scales=scales[0],
                      v_scales=scales[1])
    assert scope_b200.status_take() == 5
    assert pool[0].view(32, 32).float().sum(1).tolist() == [127.0 * 32 if i in (5, 6) else 0.0 for i in range(32)]


# ------------------------------------------------------------------ read


@pytest.mark.parametrize("P,block,heads_major", [(16, 16, False), (24, 8, True), (7, 7, False), (64, 1, False), (256, 128, True)])
@pytest.mark.parametrize("Hkv,Dk,Dv", [(2, 128, 128), (5, 80, 48), (1, 16, 256), (11, 192, 128)])
@pytest.mark.parametrize("pool,dtype", [(I8, BF), (I8, HF), (E4, BF), (E4, HF), (BF, BF), (HF, HF)])
def test_read_back(P, block, heads_major, Hkv, Dk, Dv, pool, dtype):
    g = gen(P + Dk)
    lens, starts = [0, 1, 300, 64, 0, 17], [0, 5, 11, 0, 9, 30]
    held = [-(-(a + n) // P) for a, n in zip(starts, lens)]
    n_pages = sum(held) + 1
    ids = torch.randperm(n_pages, generator=g, device=DEV).int()
    table = torch.full((6, max(held) + 2), -1, dtype=torch.int32, device=DEV)
    at = 0
    for b, h in enumerate(held):
        table[b, :h] = ids[at:at + h]
        at += h
    if pool in (I8, E4):
        (kp, ks), (vp, vs) = (make_pool(g, n_pages, P, block, Hkv, D, pool, heads_major) for D in (Dk, Dv))
    else:
        kp, vp = (torch.randn(n_pages, P, Hkv, D, generator=g, device=DEV).to(pool) for D in (Dk, Dv))
        ks = vs = None
    n = sum(lens)
    cu = torch.tensor([0] + lens, device=DEV).cumsum(0).int()
    outs = [torch.full((n + 5, Hkv, D), 7.0, dtype=dtype, device=DEV) for D in (Dk, Dv)]
    k, v = paged.paged_read(kp, vp, table, cu, n + 5, starts=torch.tensor(starts, dtype=torch.int32, device=DEV), k_scales=ks,
                            v_scales=vs, dtype=dtype, k_out=outs[0], v_out=outs[1])
    assert k is outs[0] and v is outs[1]
    for got, pages, scales in ((k, kp, ks), (v, vp, vs)):
        want = []
        for b in range(6):
            t = torch.arange(starts[b], starts[b] + lens[b], device=DEV)
            page, off = table[b].long()[t // P], t % P
            if scales is None:
                want.append(pages[page, off])
            else:
                want.append((pages.view(torch.uint8)[page, off].view(pool).float() * scales[page, off // block][..., None]).to(dtype))
        assert torch.equal(got[:n], torch.cat(want))
        assert (got[n:] == 7).all()   # rows behind the last sequence
    assert scope_b200.status_take() == 0


def test_read_of_tokens_without_a_place():
    kp, ks = make_pool(gen(1), 3, 16, 16, 2, 32, I8)
    table = torch.tensor([[0, 9], [1, -1]], dtype=torch.int32, device=DEV)
    cu, starts = torch.tensor([0, 40, 60], dtype=torch.int32, device=DEV), torch.tensor([0, -4], dtype=torch.int32, device=DEV)
    k, v = paged.paged_read(kp, kp, table, cu, 60, starts=starts, k_scales=ks, v_scales=ks)
    assert scope_b200.status_take() == 5
    assert torch.equal(k, v) and (k[16:44] == 0).all() and (k[:16] != 0).any() and (k[44:60] != 0).any()
    assert paged.paged_read(kp, kp, table[:0], cu[:1], 0, k_scales=ks, v_scales=ks)[0].shape == (0, 2, 32)
    full = torch.full((4, 2, 32), 3.0, dtype=BF, device=DEV)   # no request has a row here
    paged.paged_read(kp, kp, table, torch.tensor([2, 2, 3], dtype=torch.int32, device=DEV), 4, k_scales=ks, v_scales=ks, k_out=full)
    assert (full[:2] == 3).all() and (full[3] == 3).all() and (full[2] != 3).any()
    assert scope_b200.status_take() == 0


def test_read_past_32_bits():
    """A pool of more than 2^31 bytes, and of codes, its last page."""
    n_pages, P, Hkv, D = 33000, 64, 8, 128
    kp = torch.zeros(n_pages, P, Hkv, D, dtype=I8, device=DEV)
    ks = torch.full((n_pages, 1, Hkv), 0.5, device=DEV)
    vp = kp[:, :, :, :16]
    kp[n_pages - 1, 63, 7] = torch.arange(128, device=DEV).to(I8)
    table = torch.tensor([[3, n_pages - 1]], dtype=torch.int32, device=DEV)
    cu = torch.tensor([0, 128], dtype=torch.int32, device=DEV)
    k, v = paged.paged_read(kp, vp, table, cu, 128, k_scales=ks, v_scales=ks)
    assert torch.equal(k[127, 7], (torch.arange(128, device=DEV) * 0.5).to(BF)) and (k[:127] == 0).all() and v.shape == (128, 8, 16)
    x = torch.full((1, Hkv, D), 2.0, dtype=BF, device=DEV)
    paged.rope_append(None, x, x[:, :, :16], None, None, torch.tensor([n_pages * P - 2], device=DEV), kp, vp, k_scales=ks,
                      v_scales=ks.clone())
    assert (kp[n_pages - 1, 62, :, 16:] == 4).all()   # under the block's scale of 0.5


# ------------------------------------------------------------------ decode


def make_decode(lens, H, Hkv, Dk, Dv, P, block, dtype, pool, heads_major=False, seed=0):
    """Pages of requests; past a length codes are what they may be (e4m3: NaN), and scales of blocks past it NaN."""
    g, B = gen(seed), len(lens)
    held = [-(-n // P) for n in lens]
    n_pages = sum(held) + 2
    ids = torch.randperm(n_pages, generator=g, device=DEV).int()
    table = torch.full((B, max(held + [1])), n_pages + 7, dtype=torch.int32, device=DEV)
    (k, ks), (v, vs) = (make_pool(g, n_pages, P, block, Hkv, D, pool, heads_major) for D in (Dk, Dv))
    keep, keep_s = torch.zeros(n_pages, P, dtype=torch.bool, device=DEV), torch.zeros(n_pages, P // block, dtype=torch.bool, device=DEV)
    rows, at = [], 0
    for b, n in enumerate(lens):
        table[b, :held[b]] = ids[at:at + held[b]]
        at += held[b]
        t = torch.arange(n, device=DEV)
        page, off = table[b].long()[t // P], t % P
        keep[page, off] = True
        keep_s[page, off // block] = True
        rows.append((page, off))
    for x, s in ((k, ks), (v, vs)):
        raw(x)[~keep] = 0x7f
        s[~keep_s] = float("nan")
    q = torch.randn(B, H, Dk, generator=g, device=DEV).to(dtype)
    return dict(q=q, k=k, v=v, ks=ks, vs=vs, table=table, lens=torch.tensor(lens, dtype=torch.int32, device=DEV), rows=rows,
                scale=Dk ** -0.5, block=block)


def values(pages, scales, page, off, h, block):
    x = raw(pages)[page, off, h].view(pages.dtype) if pages.element_size() == 1 else pages[page, off, h]
    return x.double() if scales is None else x.double() * scales[page, off // block, h].double()[:, None]


def agrees(s, out, lse, window=0):
    q, Hkv = s["q"], s["k"].shape[2]
    B, H, Dk = q.shape
    G, u = H // Hkv, U[q.dtype]
    assert out.dtype == q.dtype and lse.dtype == torch.float32
    for b, (page, off) in enumerate(s["rows"]):
        if window:
            page, off = page[-window:], off[-window:]
        n = len(page)
        if n == 0:
            assert (out[b] == 0).all() and torch.isneginf(lse[b]).all()
            continue
        for h in range(Hkv):
            k, v = (values(s[x], s[x + "s"], page, off, h, s["block"]) for x in "kv")
            sl = slice(h * G, (h + 1) * G)
            qs = q[b, sl].double()
            z = qs @ k.t() * s["scale"]
            ds = (Dk + 4) * 2.0 ** -24 * abs(s["scale"]) * (qs.abs() @ k.abs().t()).amax(1)
            L = torch.logsumexp(z, 1)
            p = torch.exp(z - L[:, None])
            bound = (u + 2 * ds[:, None] + (n + 64) * 2.0 ** -24 + 2.0 ** -20) * (p @ v.abs()) + 2.0 ** -24
            d = (out[b, sl].double() - p @ v).abs()
            assert (d <= bound).all(), (b, h, (d / bound).max().item())
            dl = (lse[b, sl].double() - L).abs()
            assert (dl <= ds + (min(n, 4096) + 64) * 2.0 ** -24 + 2.0 ** -22 * L.abs() + 1e-6).all(), (b, h, dl.max().item())


def decode(s, **kw):
    return paged.paged_decode(s["q"], s["k"], s["v"], s["table"], s["lens"], s["scale"], k_scales=s["ks"], v_scales=s["vs"], **kw)


LENS = [0, 1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 200]


@pytest.mark.parametrize("P,block", [(1, 1), (7, 7), (16, 16), (16, 2), (24, 8), (64, 64), (64, 16), (96, 48), (256, 32)])
@pytest.mark.parametrize("dtype,pool", [(BF, I8), (HF, I8), (BF, E4), (HF, E4)])
def test_decode_blocks_and_page_sizes(P, block, dtype, pool):
    s = make_decode(LENS, 8, 2, 128, 128, P, block, dtype, pool, seed=P + block)
    agrees(s, *decode(s))
    agrees(s, *decode(s, window=40), window=40)
    assert scope_b200.status_take() == 0


@pytest.mark.parametrize("Dk,Dv", [(16, 16), (32, 64), (64, 64), (80, 80), (112, 48), (128, 128), (192, 128), (192, 192), (64, 256),
                                   (256, 256)])
@pytest.mark.parametrize("dtype,pool", [(BF, E4), (HF, I8), (HF, E4)])
def test_decode_head_dims(Dk, Dv, dtype, pool):
    s = make_decode([300, 0, 45, 16, 700], 6, 3, Dk, Dv, 32, 16, dtype, pool, heads_major=Dk % 32 == 0, seed=Dk + Dv)
    agrees(s, *decode(s))
    wide = dict(s, table=torch.cat([s["table"], torch.full((5, 40), 1 << 20, dtype=torch.int32, device=DEV)], 1))
    agrees(s, *decode(wide))
    assert scope_b200.status_take() == 0


def widened(s, n=60):
    """The same requests behind a table too wide for the form that short tables take."""
    B = s["table"].shape[0]
    return dict(s, table=torch.cat([s["table"], torch.full((B, n), 1 << 20, dtype=torch.int32, device=DEV)], 1))


@pytest.mark.parametrize("P,block", [(32, 32), (64, 32), (64, 64), (96, 96), (96, 32), (16, 16), (48, 48), (256, 128), (64, 8)])
@pytest.mark.parametrize("D", [64, 128, 192, 256])
@pytest.mark.parametrize("dtype,pool", [(BF, I8), (HF, E4), (BF, E4)])
def test_decode_where_a_subtile_has_one_scale_and_where_not(P, block, D, dtype, pool):
    """Lengths at every border of pages, blocks and subtiles, rows by TMA; e4m3 codes behind a length are NaN."""
    lens = [0, 1, 15, 16, 17, 31, 32, 33, 47, 63, 64, 65, 95, 96, 97, 700, 1500]
    s = widened(make_decode(lens, 6, 2, D, D, P, block, dtype, pool, heads_major=P == 64, seed=P + block + D))
    agrees(s, *decode(s))
    agrees(s, *decode(s, window=601), window=601)
    assert scope_b200.status_take() == 0


def test_decode_leaves_bad_pages_out():
    for pool, P, block in ((I8, 64, 64), (E4, 64, 64), (E4, 16, 16)):
        s = widened(make_decode([700, 90], 4, 2, 128, 128, P, block, BF, pool, seed=9))
        s["table"][0, 1], s["table"][0, 3] = -1, s["k"].shape[0]
        page, off = s["rows"][0]
        t = torch.arange(700, device=DEV) // P
        keep = (t != 1) & (t != 3)
        s["rows"][0] = (page[keep], off[keep])
        agrees(s, *decode(s))
        assert scope_b200.status_take() == 5


@pytest.mark.parametrize("G", [1, 3, 8, 9, 16, 20])
@pytest.mark.parametrize("dtype,pool", [(BF, E4), (HF, E4), (BF, I8)])
def test_decode_query_heads_and_long_rows(G, dtype, pool):
    s = make_decode([3000, 1, 9000], 2 * G, 2, 64 if G == 3 else 128, 128, 64, 64, dtype, pool, seed=G)
    agrees(s, *decode(s))
    agrees(s, *decode(s, window=2500), window=2500)


def test_decode_many_requests_and_empty_slots():
    g = torch.Generator().manual_seed(5)
    lens = [int(x) for x in torch.randint(0, 300, (157,), generator=g)]
    lens[3] = lens[80] = 0
    s = make_decode(lens, 4, 1, 64, 64, 16, 8, BF, E4, seed=11)
    agrees(s, *decode(s))


@pytest.mark.parametrize("size", [1e-30, 1e30, 3e38])
def test_decode_queries_of_any_size_over_e4m3(size):
    """bf16 queries pass through fp16 under a power of two: none too large or too small for it."""
    s = make_decode([100, 700], 4, 2, 64, 64, 16, 16, BF, E4, seed=2)
    s["q"] = (s["q"].float() / s["q"].float().abs().max() * size).to(BF)
    s["scale"] = 1.0 / size if size < 1e38 else 2.0 ** -126
    agrees(s, *decode(s))


@pytest.mark.parametrize("pool,block", [(I8, 64), (E4, 64), (I8, 16)])
def test_decode_past_32_bits(pool, block):
    """A pool of more than 2^32 bytes, its first and last pages, as one cache and as pairs of heads."""
    n_pages, P, Hkv, D = 70000, 64, 8, 128
    codes = torch.zeros(n_pages, P, Hkv, D, dtype=I8, device=DEV)
    scales = torch.full((n_pages, P // block, Hkv), float("nan"), device=DEV)
    g, at = gen(21), torch.tensor([n_pages - 1, 3, n_pages - 2], device=DEV)
    x, sc = make_pool(g, 3, P, block, Hkv, D, pool)
    raw(codes)[at], scales[at] = raw(x), sc
    pages = codes.view(pool)
    s = dict(q=torch.randn(2, 32, D, generator=g, device=DEV).to(BF), k=pages, v=pages, ks=scales, vs=scales, block=block,
             table=torch.full((2, 20), -1, dtype=torch.int32, device=DEV), scale=D ** -0.5,
             lens=torch.tensor([180, 64], dtype=torch.int32, device=DEV))
    s["table"][0, :3], s["table"][1, :1] = at.int(), at[:1].int()
    t = torch.arange(180, device=DEV)
    s["rows"] = [(at[t // P], t % P), (at[:1].expand(64), t[:64])]
    agrees(s, *decode(s))
    lam = torch.full((1,), 0.3, device=DEV)
    out, lse = paged.paged_diff_decode(s["q"], pages, pages, s["table"], s["lens"], s["scale"], lam, k_scales=scales, v_scales=scales)
    small = torch.tensor([[0, 1, 2], [0, 0, 0]], dtype=torch.int32, device=DEV)   # the same pages in a pool of three
    table = torch.cat([small, torch.full((2, 17), -1, dtype=torch.int32, device=DEV)], 1)
    out2, lse2 = paged.paged_diff_decode(s["q"], x, x, table, s["lens"], s["scale"], lam, k_scales=sc, v_scales=sc)
    assert torch.equal(out, out2) and torch.equal(lse, lse2) and scope_b200.status_take() == 0


def test_decode_queries_in_a_packed_projection_and_lengths_past_the_table():
    s = make_decode([100, 64], 8, 2, 64, 64, 16, 16, BF, E4, seed=14)
    wide = torch.randn(2, 8, 96, device=DEV).to(BF)
    wide[:, :, 16:80] = s["q"]
    more = s["lens"].clone()
    more[0] += 1000     # the table ends at 112 tokens: what lies there counts
    raw(s["k"])[s["table"][0, 6].long(), 4:], raw(s["v"])[s["table"][0, 6].long(), 4:] = 0, 0
    t = torch.arange(112, device=DEV)
    s["rows"][0] = (s["table"][0].long()[t // 16], t % 16)
    out, lse = paged.paged_decode(wide[:, :, 16:80], s["k"], s["v"], s["table"], more, s["scale"], k_scales=s["ks"], v_scales=s["vs"])
    agrees(s, out, lse)


def test_decode_values_that_are_nan():
    """A NaN code of a token that counts reaches its dim only; one past the length, nobody."""
    s = make_decode([50, 700], 4, 2, 128, 128, 16, 16, HF, E4, seed=3)
    page, off = s["rows"][1]
    raw(s["v"])[page[5], off[5], 1, 9] = 0x7f
    wide = torch.cat([s["table"], torch.full((2, 40), 1 << 20, dtype=torch.int32, device=DEV)], 1)
    for table in (s["table"], wide):
        out, lse = paged.paged_decode(s["q"], s["k"], s["v"], table, s["lens"], s["scale"], k_scales=s["ks"], v_scales=s["vs"])
        assert out[1, 2:, 9].isnan().all() and int(out.isnan().sum()) == 2 and lse.isfinite().all()


def test_scale_per_row_and_per_block_of_one_agree():
    """int8: the same codes with a scale per row, and blocks whose rows share it, give the same bits."""
    s = make_decode([33, 700, 5], 8, 2, 128, 128, 32, 8, BF, I8, seed=4)
    rows = {x: s[x].repeat_interleave(8, 1).contiguous() for x in ("ks", "vs")}
    a = decode(s)
    b = paged.paged_decode(s["q"], s["k"], s["v"], s["table"], s["lens"], s["scale"], k_scales=rows["ks"], v_scales=rows["vs"])
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


# ------------------------------------------------------------------ together


@pytest.mark.parametrize("pool,block,page", [(I8, 16, 16), (E4, 32, 32), (I8, 6, 24), (E4, 1, 16)])
@pytest.mark.parametrize("graph", [False, True])
def test_a_cache_served(pool, block, page, graph):
    """Prompts and then single tokens through begin_step, append, decode, read, release: each decode against 64 bits over the
    rows read back, and those against the tokens that went in."""
    B, H, Hkv, D, g = 5, 8, 2, 64, gen(6)
    cache = PagedKVCache(1, 60, page, Hkv, D, B, 300, dtype=pool, device=DEV, scale_block=block)
    turns = table_of(300, D)
    kept = [([], []) for _ in range(B)]

    def step(new, n):
        q, k, v = (torch.randn(n, h, D, generator=g, device=DEV).to(BF) for h in (H, Hkv, Hkv))
        return q, k, v, torch.tensor(new, dtype=torch.int32, device=DEV)

    def launch(q, k, v, new, last):
        st = cache.begin_step(new, q.shape[0])
        q = cache.append(0, q, k, v, st, turns)
        return cache.decode(0, q[last], D ** -0.5), st, q

    captured = None
    news = [[40, 0, 7, 100, 1], [1, 33, 1, 1, 1]] + [[1] * B] * 20 + [[0, 50, 0, 0, 0]] + [[1] * B] * 3
    for i, new in enumerate(news):
        n = sum(new)
        q, k, v, nt = step(new, n)
        last = (torch.tensor(new, device=DEV).cumsum(0) - 1).clamp(min=0)
        before = cache.seq_lens.clone()
        if graph and new == [1] * B:
            if captured is None:
                buf = [x.clone() for x in (q, k, v, nt, last)]
                side = torch.cuda.Stream()
                side.wait_stream(torch.cuda.current_stream())
                with torch.cuda.stream(side):
                    captured = torch.cuda.CUDAGraph()
                    with torch.cuda.graph(captured, stream=side):
                        result = launch(*buf)
                torch.cuda.current_stream().wait_stream(side)
            for x, y in zip(buf, (q, k, v, nt, last)):
                x.copy_(y)
            captured.replay()
            (out, lse), st, rq = result
        else:
            (out, lse), st, rq = launch(q, k, v, nt, last)
        assert cache.refused() == 0
        rk = paged.rope(k, st.positions, turns).float()
        at = 0
        for b in range(B):
            kept[b][0].append(rk[at:at + new[b]])
            kept[b][1].append(v[at:at + new[b]].float())
            at += new[b]
        lens = cache.seq_lens.tolist()
        assert lens == [x + y for x, y in zip(before.tolist(), new)]
        cu = torch.tensor([0] + lens, device=DEV).cumsum(0).int()
        rows = cache.read(0, cu, sum(lens), dtype=HF)
        for b in range(B):
            r = [x[cu[b]:cu[b + 1]].double() for x in rows]
            for x, y in zip(r, kept[b]):
                y = torch.cat(y).double()
                # at most `block` roundings of half a step of the block's largest |x| <= 6, and that of the read
                step_of = 6 / 127 if pool == I8 else 6 * 2.0 ** -3
                assert ((x - y).abs() <= block * step_of / 2 + 6 * 2.0 ** -8).all()
            if lens[b] == 0 or new[b] == 0:
                continue
            t = torch.arange(lens[b], device=DEV)
            page_, off = cache.page_table[b].long()[t // page], t % page
            for h in range(Hkv):
                kk, vv = (values(p[0], s[0], page_, off, h, block) for p, s in ((cache.k_pages, cache.k_scales), (cache.v_pages, cache.v_scales)))
                z = rq[last[b], h * 4:h * 4 + 4].double() @ kk.t() * D ** -0.5
                p = torch.softmax(z, 1)
                assert ((out[b, h * 4:h * 4 + 4].double() - p @ vv).abs() <= 2.0 ** -8 * (p @ vv.abs()) * 1.01 + 1e-6).all()
    cache.release(torch.ones(B, dtype=torch.bool, device=DEV))
    assert cache.free_pages() == 60 and scope_b200.status_take() == 0


def test_on_another_stream():
    s = make_decode([700, 30], 8, 2, 128, 128, 16, 16, BF, E4, seed=18)
    cu = torch.tensor([0, 700, 730], dtype=torch.int32, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out, lse = decode(s)
        k, v = paged.paged_read(s["k"], s["v"], s["table"], cu, 730, k_scales=s["ks"], v_scales=s["vs"])
        slots = s["table"][0, :1].long() * 16
        paged.rope_append(None, k[:1], v[:1], None, None, slots, s["k"], s["v"], k_scales=s["ks"], v_scales=s["vs"])
    side.synchronize()
    agrees(make_decode([700, 30], 8, 2, 128, 128, 16, 16, BF, E4, seed=18), out, lse)


def test_refusals():
    kp, ks = make_pool(gen(1), 3, 16, 16, 2, 32, I8)
    k, slots = torch.ones(3, 2, 32, dtype=BF, device=DEV), torch.arange(3, device=DEV)
    for scales in (ks.new_ones(3, 3, 2), ks.new_ones(3, 0, 2), ks.new_ones(3, 32, 2), ks.new_ones(3, 1, 1), ks.new_ones(2, 1, 2), ks.half(),
                   ks[:, :, :, None]):
        with pytest.raises(RuntimeError, match="scales must be"):
            paged.rope_append(None, k, k, None, None, slots, kp, kp, k_scales=scales, v_scales=scales)
    with pytest.raises(RuntimeError, match="scales must be"):   # one block size for both
        paged.rope_append(None, k, k, None, None, slots, kp, kp, k_scales=ks, v_scales=ks.new_ones(3, 2, 2))
    with pytest.raises(RuntimeError, match="e4m3fn pool needs"):
        paged.rope_append(None, k, k, None, None, slots, kp.float().to(E4), kp.float().to(E4))
    with pytest.raises(RuntimeError, match="the pool must be"):
        paged.rope_append(None, k, k, None, None, slots, kp.float().to(torch.float8_e5m2), kp.float().to(torch.float8_e5m2))
    with pytest.raises(RuntimeError, match="overlap|memory location"):   # blocks of a page that share their scale
        paged.rope_append(None, k, k, None, None, slots, kp, kp, k_scales=ks.expand(3, 1, 2)[:1].expand(3, 1, 2), v_scales=ks)
    table, cu = torch.zeros(2, 1, dtype=torch.int32, device=DEV), torch.tensor([0, 2, 4], dtype=torch.int32, device=DEV)
    sc = dict(k_scales=ks, v_scales=ks)

    def no(match, *a, **kw):
        with pytest.raises(RuntimeError, match=match):
            paged.paged_read(*a, **{**sc, **kw})

    no("bf16 or fp16", kp, kp, table, cu, 4, dtype=torch.float32)
    no("torch.dtype", kp, kp, table, cu, 4, dtype="bf16")
    no("cu_seqlens", kp, kp, table, cu.long(), 4)
    no("page_table", kp, kp, table, cu[:2], 4)
    no("cu_seqlens|n_tokens", kp, kp, table, cu, -1)
    no("cu_seqlens", kp, kp, table, cu[:0], 4)
    no("starts", kp, kp, table, cu, 4, starts=cu)
    no("starts", kp, kp, table, cu, 4, starts=cu[:2].long())
    no("k_out", kp, kp, table, cu, 4, k_out=torch.empty(4, 2, 32, dtype=HF, device=DEV))
    no("v_out", kp, kp, table, cu, 4, v_out=torch.empty(5, 2, 32, dtype=BF, device=DEV))
    both = torch.empty(4, 2, 32, dtype=BF, device=DEV)
    no("overlap|memory location", kp, kp, table, cu, 4, k_out=both, v_out=both)
    no("overlap|memory location", kp, kp, table, cu, 3, k_out=raw(kp).view(-1)[:384].view(BF).view(3, 2, 32))
    no("own type", kp.to(HF), kp.to(HF), table, cu, 4, dtype=BF, k_scales=None, v_scales=None)
    no("belong to", kp.to(HF), kp.to(HF), table, cu, 4)
    for kw in (dict(scale_block=3, dtype=I8), dict(scale_block=0, dtype=I8), dict(scale_block=16), dict(scale_block=32, dtype=E4)):
        with pytest.raises(RuntimeError, match="scale_block"):
            PagedKVCache(1, 4, 16, 1, 32, 1, 32, device=DEV, **kw)

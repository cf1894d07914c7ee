"""GPU checks of how near a decode over 8-bit pages comes to 64 bits, and of what a cache holds, each as tight as its arithmetic.

Decode.  With ds = (Dk + 4) 2^-24 scale sum |q k| for a score's error, a sum's error over n tokens added one after the other
and the probabilities' 2^-20, a head's sum is off by
    e = (2 ds + (n + 64) 2^-24 + 2^-20) sum p|v|
and is rounded once: |do| <= e + u (|o| + e) + 2^-25, with u = 2^-8 for bf16 and 2^-11 for fp16 (2^-25: half a step of fp16's
least values).  At the few hundred tokens here e is far below u |o| of most dims in bf16, so a probability rounded once to
bf16 passes no longer: its sum alone is off by some u sqrt(sum p^2 v^2) / 2, more than u |o| for the dims near the mean.
"""
import pytest
import torch

import scope_b200
from scope_b200 import PagedKVCache, paged
from test_paged_blocks_gpu import E4, I8, append_reference, decode, make_decode, raw, values, widened
from test_paged_gpu import BF, DEV, HF, U, gen, table_of

pytestmark = pytest.mark.gpu


def exact_and_room(s, window=0):
    """Per request: (exact out, its room before the rounding, lse, its room) of all heads, fp64."""
    q, Hkv = s["q"], s["k"].shape[2]
    B, H, Dk = q.shape
    G = H // Hkv
    for b, (page, off) in enumerate(s["rows"]):
        if window:
            page, off = page[-window:], off[-window:]
        n = len(page)
        if n == 0:
            continue
        for h in range(Hkv):
            k, v = (values(s[x], s[x + "s"], page, off, h, s["block"]) for x in "kv")
            qs = q[b, h * G:(h + 1) * G].double()
            z = qs @ k.t() * s["scale"]
            ds = (Dk + 4) * 2.0 ** -24 * abs(s["scale"]) * (qs.abs() @ k.abs().t()).amax(1)
            L = torch.logsumexp(z, 1)
            p = torch.exp(z - L[:, None])
            e = (2 * ds[:, None] + (n + 64) * 2.0 ** -24 + 2.0 ** -20) * (p @ v.abs())
            yield b, slice(h * G, (h + 1) * G), p, v, e, L, ds + (n + 64) * 2.0 ** -24 + 2.0 ** -22 * L.abs() + 1e-6


@pytest.mark.parametrize("P,block", [(16, 16), (64, 64), (32, 32), (64, 32), (24, 8), (16, 1)])
@pytest.mark.parametrize("Dk,Dv", [(64, 64), (80, 80), (128, 128), (192, 128), (256, 256)])
@pytest.mark.parametrize("dtype,pool", [(BF, I8), (HF, I8), (BF, E4), (HF, E4)])
def test_decode_is_rounded_once(P, block, Dk, Dv, dtype, pool):
    s = make_decode([300, 0, 1, 33, 177, 256], 8, 2, Dk, Dv, P, block, dtype, pool, heads_major=P == 64, seed=P + block + Dk)
    u, caught = U[dtype], 0
    outs = [decode(x) for x in (s, widened(s, 600 // P))]
    for b, sl, p, v, e, L, room in exact_and_room(s):
        o = p @ v
        bound = e + u * (o.abs() + e) + 2.0 ** -25
        for out, lse in outs:
            d = (out[b, sl].double() - o).abs()
            assert (d <= bound).all(), (b, (d / bound).max().item())
            assert ((lse[b, sl].double() - L).abs() <= room).all()
        if len(v) > 100:   # the mistake that the bound is for, made here: probabilities rounded once
            wrong = ((p.float().to(dtype).double() @ v).to(dtype).double() - o).abs()
            caught += int((wrong > bound).sum())
    assert caught > 0 or dtype == HF   # one dim out of its bound is enough; in fp16 e comes near the mistake
    assert scope_b200.status_take() == 0


@pytest.mark.parametrize("pool,block,page", [(I8, 16, 16), (E4, 32, 32), (I8, 6, 24), (E4, 64, 64)])
def test_a_cache_holds_what_went_in(pool, block, page):
    """Prompts and single tokens, a prompt that joins later: pages, scales and rows read back are the rule's, bit for bit."""
    B, H, Hkv, D, g = 4, 4, 2, 48, gen(block)
    cache = PagedKVCache(1, 30, page, Hkv, D, B, 200, dtype=pool, device=DEV, scale_block=block)
    turns = table_of(200, D)
    held = [x[0] for x in (cache.k_pages, cache.k_scales, cache.v_pages, cache.v_scales)]
    for x in held:
        raw(x).zero_() if x.element_size() == 1 else x.zero_()
    want = [x.clone() for x in held]
    for new in [[40, 0, 7, 100], [1, 33, 1, 1]] + [[1] * B] * 18 + [[0, 50, 0, 0]] + [[1, 0, 1, 1]] * 3:
        n = sum(new)
        q, k, v = (torch.randn(n, h, D, generator=g, device=DEV).to(BF) for h in (H, Hkv, Hkv))
        k *= torch.exp2(torch.randint(-2, 3, (n, 1, 1), generator=g, device=DEV).float()).to(BF)
        step = cache.begin_step(torch.tensor(new, dtype=torch.int32, device=DEV), n)
        cache.append(0, q, k, v, step, turns)
        t = turns[step.positions.long()][:, None]
        x1, x2, c, s = k[..., :D // 2].float(), k[..., D // 2:].float(), t[..., :D // 2], t[..., D // 2:]
        rk = torch.cat([x1 * c - x2 * s, x2 * c + x1 * s], -1)
        want = [*append_reference(rk, step.slots, *want[:2], block), *append_reference(v.float(), step.slots, *want[2:], block)]
        assert all(torch.equal(raw(x.contiguous()), raw(y.contiguous())) for x, y in zip(held, want))
    lens = cache.seq_lens.tolist()
    cu = torch.tensor([0] + lens, device=DEV).cumsum(0).int()
    rows = cache.read(0, cu, sum(lens), dtype=HF)
    for x, pages, scales in zip(rows, want[::2], want[1::2]):
        for b in range(B):
            t = torch.arange(lens[b], device=DEV)
            p, off = cache.page_table[b].long()[t // page], t % page
            y = raw(pages)[p, off].view(pool).float() * scales[p, off // block][..., None]
            assert torch.equal(x[cu[b]:cu[b + 1]], y.to(HF))
    assert cache.refused() == 0 and scope_b200.status_take() == 0

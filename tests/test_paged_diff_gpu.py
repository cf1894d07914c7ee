"""GPU checks of differential attention over pages, against 64 bits.

With (e1, e2) the bounds of the two maps' outputs before rounding (tests of the block-scaled decode: 2 ds + (n + 64) 2^-24 +
2^-20 of sum p|v|), the difference x = o1 - lam o2 is off by
    dx <= e1 + |lam| e2 + 2^-22 (|o1| + |lam o2|),
the normalised y = x r w, r = (mean x^2 + eps)^-1/2, to first order by |w| r (dx + |x| r^2 mean(|x| dx)) + 2^-20 |y|, and
the result is rounded once, by u |y|.  Of second order are, with d = max dx r and m = mean(x dx) r^2 <= d: 1.5 m^2 and, of the
other sign, mean(dx^2) r^2 / 2 <= d^2 / 2 from the root, and dx r m: together at most 1.5 d of the first order, which is
below a tenth of it while d < 0.066 (the cases keep to it; the factor 1.1 below).
"""
import pytest
import torch

import scope_b200
from scope_b200 import PagedKVCache, paged
from test_paged_blocks_gpu import E4, I8, make_pool, raw, values
from test_paged_gpu import BF, DEV, HF, U, gen, table_of

pytestmark = pytest.mark.gpu


def make(lens, H, pairs, Dk, Dv, P, dtype, pool, block=1, heads_major=False, seed=0):
    g, B, hs = gen(seed), len(lens), 2 * pairs
    held = [-(-n // P) for n in lens]
    n_pages = sum(held) + 2
    ids = torch.randperm(n_pages, generator=g, device=DEV).int()
    table = torch.full((B, max(held + [1])), n_pages + 7, dtype=torch.int32, device=DEV)
    if pool in (I8, E4):
        (k, ks), (v, vs) = (make_pool(g, n_pages, P, block, hs, D, pool, heads_major) for D in (Dk, Dv))
    else:
        k, v = (torch.randn(n_pages, *((hs, P) if heads_major else (P, hs)), D, generator=g, device=DEV).to(pool) for D in (Dk, Dv))
        if heads_major:
            k, v = k.transpose(1, 2), v.transpose(1, 2)
        ks = vs = None
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
        if s is None:
            x[~keep] = float("nan")
        else:
            raw(x)[~keep] = 0x7f
            s[~keep_s] = float("nan")
    return dict(q=torch.randn(B, 2 * H, Dk, generator=g, device=DEV).to(dtype), k=k, v=v, ks=ks, vs=vs, table=table,
                lens=torch.tensor(lens, dtype=torch.int32, device=DEV), rows=rows, scale=Dk ** -0.5, block=block,
                lam=torch.rand(H, generator=g, device=DEV) * 0.7 + 0.1, w=1 + 0.2 * torch.randn(2 * Dv, generator=g, device=DEV))


def diff(s, norm=True, **kw):
    return paged.paged_diff_decode(s["q"], s["k"], s["v"], s["table"], s["lens"], s["scale"], s["lam"],
                                   norm_weight=s["w"] if norm else None, norm_eps=1e-5, k_scales=s["ks"], v_scales=s["vs"], **kw)


def agrees(s, out, lse, norm=True, window=0, chain=None):
    """chain: how many additions one after the other a sum over tokens takes (None: as many as tokens)."""
    q, pairs = s["q"], s["k"].shape[2] // 2
    B, H2, Dk = q.shape
    G, u, H = H2 // 2 // pairs, U[q.dtype], H2 // 2
    assert out.shape == (B, H, 2 * s["v"].shape[3]) and out.dtype == q.dtype and lse.shape == (B, H2)
    for b, (page, off) in enumerate(s["rows"]):
        if window:
            page, off = page[-window:], off[-window:]
        n = len(page)
        if n == 0:
            assert (out[b] == 0).all() and torch.isneginf(lse[b]).all()
            continue
        for p_ in range(pairs):
            v = torch.cat([values(s["v"], s["vs"], page, off, 2 * p_ + m, s["block"]) for m in (0, 1)], 1)
            o, e = [], []
            for m in (0, 1):
                k = values(s["k"], s["ks"], page, off, 2 * p_ + m, s["block"])
                heads = [2 * (p_ * G + i) + m for i in range(G)]
                qs = q[b, heads].double()
                z = qs @ k.t() * s["scale"]
                ds = (Dk + 4) * 2.0 ** -24 * s["scale"] * (qs.abs() @ k.abs().t()).amax(1)
                L = torch.logsumexp(z, 1)
                p = torch.exp(z - L[:, None])
                o.append(p @ v)
                e.append((2 * ds[:, None] + ((chain or n) + 64) * 2.0 ** -24 + 2.0 ** -20) * (p @ v.abs()))
                dl = (lse[b, heads].double() - L).abs()
                assert (dl <= ds + (min(n, 4096) + 64) * 2.0 ** -24 + 2.0 ** -22 * L.abs() + 1e-6).all(), dl.max().item()
            lam = s["lam"].expand(H)[p_ * G:(p_ + 1) * G].double()[:, None]
            x = o[0] - lam * o[1]
            dx = e[0] + lam.abs() * e[1] + 2.0 ** -22 * (o[0].abs() + (lam * o[1]).abs())
            if norm:
                r = ((x * x).mean(1, keepdim=True) + 1e-5) ** -0.5
                assert (dx * r).max() < 0.066
                w = s["w"].double()
                y = x * r * w
                dy = 1.1 * w.abs() * r * (dx + x.abs() * r ** 2 * (x.abs() * dx).mean(1, keepdim=True)) + 2.0 ** -20 * y.abs()
            else:
                y, dy = x, dx
            d = (out[b, p_ * G:(p_ + 1) * G].double() - y).abs()
            bound = dy + u * (y.abs() + dy) + 2.0 ** -24
            assert (d <= bound).all(), (b, p_, (d / bound).max().item())


TYPES = [(BF, BF, 1), (HF, HF, 1), (BF, I8, 1), (HF, I8, 8), (BF, E4, 8), (HF, E4, 4)]
LENS = [0, 1, 2, 15, 16, 17, 31, 33, 64, 65, 127, 129, 200]


@pytest.mark.parametrize("P,heads_major", [(8, False), (16, True), (24, False), (64, False)])
@pytest.mark.parametrize("dtype,pool,block", TYPES)
def test_lengths_and_pages(P, heads_major, dtype, pool, block):
    s = make(LENS, 6, 2, 64, 64, P, dtype, pool, block, heads_major, seed=P)
    agrees(s, *diff(s))
    agrees(s, *diff(s, False), norm=False)
    agrees(s, *diff(s, window=40), window=40)
    assert scope_b200.status_take() == 0


@pytest.mark.parametrize("Dk,Dv", [(16, 16), (32, 32), (48, 48), (64, 32), (80, 80), (96, 96), (112, 16), (128, 128), (64, 128)])
@pytest.mark.parametrize("dtype,pool,block", TYPES)
def test_head_dims(Dk, Dv, dtype, pool, block):
    s = make([300, 0, 45, 16, 640], 3, 3, Dk, Dv, 16, dtype, pool, block, heads_major=Dk % 32 == 0, seed=Dk + Dv)
    agrees(s, *diff(s))
    wide = dict(s, table=torch.cat([s["table"], torch.full((5, 40), 1 << 20, dtype=torch.int32, device=DEV)], 1))
    agrees(s, *diff(wide))    # rows by TMA, where they can come so
    agrees(s, *diff(wide, False), norm=False)


@pytest.mark.parametrize("P,block", [(16, 16), (32, 32), (64, 64), (64, 32), (96, 48), (64, 8)])
@pytest.mark.parametrize("D", [32, 64, 96, 128])
@pytest.mark.parametrize("dtype,pool", [(BF, I8), (HF, E4)])
def test_where_a_subtile_has_one_scale_and_where_not(P, block, D, dtype, pool):
    lens = [0, 1, 15, 16, 17, 31, 32, 33, 63, 64, 65, 700, 1500]
    s = make(lens, 4, 2, D, D, P, dtype, pool, block, heads_major=P == 64, seed=P + block + D)
    s["table"] = torch.cat([s["table"], torch.full((len(lens), 60), 1 << 20, dtype=torch.int32, device=DEV)], 1)
    agrees(s, *diff(s))
    agrees(s, *diff(s, False, window=601), norm=False, window=601)
    assert scope_b200.status_take() == 0


@pytest.mark.parametrize("G", [1, 2, 4, 5, 8, 9])
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("dtype,pool,block", [(BF, BF, 1), (HF, I8, 16)])
def test_query_heads_and_long_rows(G, D, dtype, pool, block):
    s = make([3000, 1, 7000, 1500], 2 * G, 2, D, D, 64, dtype, pool, block, seed=G)
    agrees(s, *diff(s))
    agrees(s, *diff(s, window=2500), window=2500)


@pytest.mark.parametrize("dtype,pool,block", [(BF, BF, 1), (BF, E4, 16)])
def test_one_long_request_is_joined_from_every_cta(dtype, pool, block):
    # 148 CTAs of 8 warps and more share the tokens: 96 of them at most a warp (three subtiles of 32), then 16 warps' and 148
    # CTAs' parts, one after the other
    s = make([60000], 4, 1, 64, 64, 64, dtype, pool, block, seed=3)
    a = diff(s)
    agrees(s, *a, chain=96 + 16 + 148)
    b = diff(s)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_many_short_requests():
    g = torch.Generator().manual_seed(5)
    lens = [int(x) for x in torch.randint(0, 300, (157,), generator=g)]
    s = make(lens, 4, 2, 64, 64, 16, BF, BF, seed=11)
    agrees(s, *diff(s))


def test_lam_of_one_value_and_strided():
    s = make([100, 700], 4, 2, 64, 64, 16, BF, BF, seed=4)
    for lam in (torch.tensor(0.35, device=DEV), torch.tensor([0.35], device=DEV), torch.full((8,), 0.35, device=DEV)[::2],
                torch.tensor(0.35, device=DEV).expand(4)):
        one = dict(s, lam=lam)
        agrees(one, *diff(one))


def test_the_difference_of_equal_maps_is_nothing_and_of_lam_zero_the_first_map():
    s = make([100, 900], 4, 2, 64, 64, 16, HF, HF, seed=6)
    twin = dict(s, q=s["q"].view(2, 4, 2, 64)[:, :, :1].expand(2, 4, 2, 64).reshape(2, 8, 64), lam=torch.ones(4, device=DEV))
    twin["k"] = s["k"].unflatten(2, (2, 2))[:, :, :, :1].expand(-1, -1, -1, 2, -1).flatten(2, 3).contiguous()
    out, lse = diff(twin, False)
    assert (out.float().abs() <= 2.0 ** -18).all() and torch.equal(lse[:, ::2], lse[:, 1::2])
    first = dict(s, lam=torch.zeros(1, device=DEV))
    out, lse = diff(first, False)
    half = [paged.paged_decode(s["q"][:, ::2].contiguous(), s["k"][:, :, ::2], s["v"][:, :, m::2], s["table"], s["lens"], s["scale"])
            for m in (0, 1)]
    assert torch.allclose(out.float(), torch.cat([h[0] for h in half], 2).float(), rtol=2.0 ** -9, atol=2.0 ** -16)
    assert torch.allclose(lse[:, ::2], half[0][1], rtol=2.0 ** -20)


def test_through_a_cache_and_a_graph():
    """The same cache as any other: keys [N, 2 pairs, D], values viewed as such; the step captured and replayed."""
    B, H, pairs, D, g = 3, 4, 2, 64, gen(9)
    cache = PagedKVCache(1, 40, 16, 2 * pairs, D, B, 200, device=DEV)
    turns, lam, w = table_of(200, D), torch.rand(H, generator=g, device=DEV), torch.ones(2 * D, device=DEV)
    kept_k, kept_v = [[] for _ in range(B)], [[] for _ in range(B)]

    def launch(q, k, v, new, last):
        st = cache.begin_step(new, q.shape[0])
        q = cache.append(0, q, k, v.view(-1, 2 * pairs, D), st, turns)
        return cache.diff_decode(0, q[last], D ** -0.5, lam, w), st, q

    captured = None
    for i, new in enumerate([[30, 1, 90], [1, 1, 1], [1, 1, 1], [1, 1, 1], [1, 1, 1]]):
        n = sum(new)
        q, k, v = (torch.randn(n, h, d, generator=g, device=DEV).to(BF) for h, d in ((2 * H, D), (2 * pairs, D), (pairs, 2 * D)))
        nt, last = torch.tensor(new, dtype=torch.int32, device=DEV), torch.tensor(new, device=DEV).cumsum(0) - 1
        if i == 0:
            result = launch(q, k, v, nt, last)
        else:
            if captured is None:
                buf = [x.clone() for x in (q, k, v, nt, last)]
                side = torch.cuda.Stream()
                side.wait_stream(torch.cuda.current_stream())
                with torch.cuda.stream(side):
                    captured = torch.cuda.CUDAGraph()
                    with torch.cuda.graph(captured, stream=side):
                        held = launch(*buf)
                torch.cuda.current_stream().wait_stream(side)
            for x, y in zip(buf, (q, k, v, nt, last)):
                x.copy_(y)
            captured.replay()
            result = held
        (out, lse), st, rq = result
        rk, at = paged.rope(k, st.positions, turns), 0
        for b in range(B):
            kept_k[b].append(rk[at:at + new[b]])
            kept_v[b].append(v[at:at + new[b]])
            at += new[b]
        # the same through rows kept apart, one page a request
        n_max = max(sum(len(x) for x in kk) for kk in kept_k)
        kp, vp = (torch.zeros(B, n_max, 2 * pairs, D, dtype=BF, device=DEV) for _ in range(2))
        for b in range(B):
            kk, vv = torch.cat(kept_k[b]), torch.cat(kept_v[b])
            kp[b, :len(kk)], vp[b, :len(vv)] = kk, vv.view(-1, 2 * pairs, D)
        lens = cache.seq_lens.tolist()
        rows = [(torch.full((L,), b, device=DEV), torch.arange(L, device=DEV)) for b, L in enumerate(lens)]
        agrees(dict(q=rq[last], k=kp, v=vp, ks=None, vs=None, rows=rows, scale=D ** -0.5, block=1, lam=lam, w=w), out, lse)
    assert scope_b200.status_take() == 0


def test_queries_in_a_packed_projection_and_another_stream():
    s = make([100, 700], 4, 2, 64, 64, 16, BF, I8, 16, seed=15)
    wide = torch.randn(2, 8, 96, device=DEV).to(BF)
    wide[:, :, 16:80] = s["q"]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = diff(dict(s, q=wide[:, :, 16:80]))
    side.synchronize()
    agrees(s, *got)


def test_two_captured_graphs_replayed_in_turn():
    """Graphs of one stream share its workspace; replayed one after the other each gives what it gave alone."""
    a, b = make([3000, 40], 4, 2, 64, 64, 16, BF, BF, seed=16), make([10, 5000], 8, 2, 64, 64, 64, BF, E4, 64, seed=17)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs, held = [], []
    with torch.cuda.stream(side):
        for s in (a, b):
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[-1], stream=side):
                held.append(diff(s))
        for _ in range(3):
            for graph in graphs:
                graph.replay()
    side.synchronize()
    agrees(a, *held[0])
    agrees(b, *held[1])


def test_outputs_given_and_refusals():
    s = make([100, 30], 4, 2, 64, 64, 16, BF, BF, seed=7)
    out, lse = torch.empty(2, 4, 128, dtype=BF, device=DEV), torch.empty(2, 8, device=DEV)
    got = diff(s, out=out, lse=lse)
    assert got[0] is out and got[1] is lse
    agrees(s, out, lse)

    def no(match, **kw):
        a = dict(q=s["q"], k_pages=s["k"], v_pages=s["v"], page_table=s["table"], seq_lens=s["lens"], scale=0.1, lam=s["lam"])
        a.update(kw)
        with pytest.raises(RuntimeError, match=match):
            paged.paged_diff_decode(**a)

    no("bf16 or fp16", q=s["q"].float())
    no("type or int8", q=s["q"].half())
    no("pairs", k_pages=s["k"][:, :, :3], v_pages=s["v"][:, :, :3])
    no("2 \\* H", q=s["q"][:, :6])
    no("2 \\* H", q=s["q"][:, :, :32])
    no("lam must", lam=s["lam"].half())
    no("lam must", lam=s["lam"][:3])
    no("lam must", lam=s["lam"].cpu())
    no("lam must", lam=s["lam"].view(2, 2))
    no("norm_weight", norm_weight=s["w"][:64])
    no("norm_weight", norm_weight=s["w"].half())
    no("norm_eps", norm_eps=-1.0)
    no("out must", out=torch.empty(2, 8, 64, dtype=BF, device=DEV))
    no("lse must", lse=torch.empty(2, 4, device=DEV))
    no("overlap|memory location", out=s["q"].view(2, 4, 128))
    no("window", window=-1)
    wide = torch.zeros(2, 16, 2, 144, dtype=BF, device=DEV)
    no("at most 128", q=torch.zeros(2, 4, 144, dtype=BF, device=DEV), k_pages=wide, v_pages=wide, lam=s["lam"][:2])
    no("torch|tensor", lam=0.5)

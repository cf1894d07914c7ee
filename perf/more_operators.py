"""Cases of a paged key-value cache held in 8 bits with one scale for each block of tokens and head -- written as it is
quantised, read back, attended by a decode step -- and of differential attention over a paged cache.  Each case has a
plain form (elementary torch operations in 32 bits) and, with ``own`` set, the framework's calls.
"""
import numpy as np
import torch

own = False

HALF = {"bf16": torch.bfloat16, "fp16": torch.float16}
LARGEST = 4.2e9   # bytes that a drawn case may move when every request is as long as the longest


def listed():
    return [
        # one decode step of 64 requests, 32 query and 8 kv heads: each new row lands inside an open block
        dict(name="append-decode", op="append", B=64, least=1, most=4096, new_least=1, new_most=1, refused=False, H=32, Hkv=8,
             D=128, Dv=128, rot=128, adjacent=False, dtype="bf16", pool="int8", page=16, block=16, heads_major=False,
             packed=True, lens_seed=1),
        # prompts of 16 thousand tokens in all, some of them going on where an earlier chunk ended
        dict(name="append-prompts", op="append", B=6, least=0, most=3000, new_least=1500, new_most=4000, refused=False, H=32,
             Hkv=4, D=128, Dv=128, rot=128, adjacent=False, dtype="bf16", pool="e4m3", page=64, block=64, heads_major=False,
             packed=True, lens_seed=5),
        # ragged chunks, heads of 80, small blocks in odd pages, head-major, one request refused
        dict(name="append-ragged", op="append", B=23, least=0, most=700, new_least=1, new_most=400, refused=True, H=20, Hkv=5,
             D=80, Dv=80, rot=64, adjacent=True, dtype="fp16", pool="int8", page=24, block=8, heads_major=True, packed=False,
             lens_seed=3),
        # one chat's context for the attention of its next chunk: latency
        dict(name="read-1x1000", op="read", B=1, least=1000, most=1000, empty=False, Hkv=4, D=128, Dv=128, dtype="bf16",
             pool="int8", page=16, block=16, heads_major=False, lens_seed=4),
        # a ragged batch of documents, the part behind a shared beginning
        dict(name="read-16-ragged", op="read", B=16, least=1024, most=32768, empty=True, Hkv=8, D=128, Dv=128, dtype="bf16",
             pool="e4m3", page=64, block=32, heads_major=False, lens_seed=5),
        # one user, 4096 tokens: latency
        dict(name="decode-1x4096", op="decode", B=1, H=32, Hkv=4, D=128, Dv=128, dtype="bf16", pool="e4m3", page=16, block=16,
             heads_major=False, least=4096, most=4096, empty=False, window=0, lens_seed=3),
        # many short chats, one slot of the batch empty, a window that cuts the longer ones, odd pages and heads
        dict(name="decode-128-short", op="decode", B=128, H=20, Hkv=4, D=80, Dv=80, dtype="fp16", pool="int8", page=24, block=12,
             heads_major=True, least=1, most=1024, empty=True, window=700, lens_seed=4),
        # long documents
        dict(name="decode-8-long", op="decode", B=8, H=32, Hkv=4, D=128, Dv=128, dtype="bf16", pool="int8", page=64, block=64,
             heads_major=False, least=16384, most=65536, empty=False, window=0, lens_seed=6),
        # the largest: 32 requests of 65536 tokens, 8 kv heads
        dict(name="decode-32x65536", op="decode", B=32, H=64, Hkv=8, D=128, Dv=128, dtype="bf16", pool="e4m3", page=64, block=64,
             heads_major=False, least=65536, most=65536, empty=False, window=0, lens_seed=7),
        # differential attention, one user: 16 heads of two 64-dim maps, values of 128: latency
        dict(name="diff-1x2000", op="diff", B=1, H=16, Hkv=4, D=64, Dv=64, dtype="bf16", pool="bf16", page=16, block=1,
             heads_major=False, least=2000, most=2000, empty=False, window=0, norm=True, lens_seed=8),
        # a ragged batch in 16 bits
        dict(name="diff-16-ragged", op="diff", B=16, H=16, Hkv=8, D=64, Dv=64, dtype="bf16", pool="bf16", page=64, block=1,
             heads_major=False, least=1024, most=32768, empty=True, window=0, norm=True, lens_seed=5),
        # maps of 128 dims over an 8-bit cache, a window, no norm
        dict(name="diff-24-blocks", op="diff", B=24, H=32, Hkv=8, D=128, Dv=128, dtype="fp16", pool="int8", page=32, block=32,
             heads_major=True, least=100, most=16384, empty=False, window=8000, norm=False, lens_seed=10),
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], even over the logarithm."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["append", "append", "append", "read", "read", "decode", "decode", "decode", "diff", "diff", "diff"])
    page = rng.choice([8, 16, 16, 24, 32, 48, 64, 64, 128, 256])
    block = rng.choice([b for b in range(2, page + 1) if page % b == 0])
    dtype = rng.choice(["bf16", "fp16"])
    Hkv = rng.randint(1, 8)
    c = dict(op=op, dtype=dtype, page=page, block=block, pool=rng.choice(["int8", "e4m3"]), heads_major=rng.random() < 0.4,
             lens_seed=rng.randrange(1 << 30), Hkv=Hkv)
    D = rng.choice([32, 64, 80, 96, 112, 128, 128, 192, 256])
    Dv = rng.choice([D, D, D, 128 if D == 192 else D, 64])
    if op == "append":
        new_most = _spread(rng, 1, 4096)
        B = _spread(rng, 1, max(1, min(256, 16384 // new_most)))
        return dict(c, B=B, least=0, most=_spread(rng, 1, 8192), new_least=_spread(rng, 1, new_most), new_most=new_most,
                    refused=B > 2 and rng.random() < 0.2, H=Hkv * rng.randint(1, 8), D=D, Dv=Dv,
                    rot=rng.choice([D, 16 * rng.randint(1, D // 16)]), adjacent=rng.random() < 0.4, packed=rng.random() < 0.5)
    B = _spread(rng, 1, 256)
    if op == "diff":
        D = rng.choice([32, 48, 64, 64, 80, 96, 128, 128])
        Dv = rng.choice([D, D, 64])
        if rng.random() < 0.5:
            c.update(pool=dtype, block=1)
    per = 3 if op == "read" else 2 if c["pool"] in HALF else 1   # bytes a value
    most = _spread(rng, 1, int(min(131072, LARGEST / (B * _heads(c) * ((D + Dv) * per + 8)))))
    c.update(B=B, D=D, Dv=Dv, least=_spread(rng, 1, most), most=most, empty=B > 1 and rng.random() < 0.3)
    if op == "read":
        return c
    c.update(H=Hkv * rng.choice([1, 2, 3, 4, 5, 6, 8] + ([12, 16] if op == "decode" else [])),
             window=rng.choice([0, 0, 0, _spread(rng, 1, most)]))
    return dict(c, norm=rng.random() < 0.7) if op == "diff" else c


# ------------------------------------------------------------------ what the cases hold


def _rng(c):
    return np.random.RandomState(c["lens_seed"] % (1 << 32))


def _lens(c):
    """The requests' lengths."""
    r = _rng(c)
    lens = r.randint(c["least"], c["most"] + 1, c["B"])
    if c.get("empty"):
        lens[r.randint(c["B"])] = 0
    return lens


def _chunks(c):
    """An append's (lengths before the step, new tokens, which requests are served)."""
    r = _rng(c)
    lens = r.randint(c["least"], c["most"] + 1, c["B"])
    new = r.randint(c["new_least"], c["new_most"] + 1, c["B"])
    if c["new_most"] > 1:   # half of the prompts begin
        lens[r.rand(c["B"]) < 0.5] = 0
    served = np.ones(c["B"], dtype=bool)
    if c["refused"]:
        served[c["B"] // 2] = False
    return lens, new, served


def _parts(c):
    """A read's (first token, tokens) of each request: an append's touched blocks; else most of what is held."""
    if c["op"] == "append":
        lens, new, served = _chunks(c)
        first = lens // c["block"] * c["block"]
        return first, np.where(served, lens + new - first, 0)
    lens = _lens(c)
    first = lens // 16
    return first, lens - first


def _heads(c):
    """The pool's heads."""
    return c["Hkv"] * (2 if c["op"] == "diff" else 1)


def _pool(n_pages, c, Dx, g, dev):
    """A pool of pages [n_pages, page, heads, Dx] filled with values, and its scales [n_pages, blocks, heads]."""
    hs, P, nb = _heads(c), c["page"], c["page"] // c["block"]
    shape = (n_pages, hs, P) if c["heads_major"] else (n_pages, P, hs)
    blocks = (n_pages, hs, nb) if c["heads_major"] else (n_pages, nb, hs)
    if c["pool"] in HALF:
        x, s = torch.randn(*shape, Dx, generator=g, device=dev, dtype=HALF[c["pool"]]), None
    else:
        x = torch.randn(*shape, Dx, generator=g, device=dev, dtype=torch.bfloat16)
        if c["pool"] == "int8":
            x = (x * 32).round_().clamp_(-127, 127).to(torch.int8)
            s = torch.rand(*blocks, generator=g, device=dev) * 0.02 + 0.015
        else:   # scales of powers of two
            x = (x * 100).clamp_(-448, 448).to(torch.float8_e4m3fn)
            s = torch.exp2(torch.randint(-8, -5, blocks, generator=g, device=dev).float())
    if c["heads_major"]:
        x, s = x.transpose(1, 2), None if s is None else s.transpose(1, 2)
    return x, s


def prepare(case, seed):
    c, dev = case, torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=dev, dtype=HALF[c["dtype"]])

    def i32(x):
        return torch.from_numpy(np.ascontiguousarray(x)).to(dev).int()

    P = c["page"]
    lens = sum(_chunks(c)[:2]) if c["op"] == "append" else _lens(c)   # what the pages have to hold
    held = -(-lens // P)
    n_pages = int(held.sum()) + 1 + int(held.sum()) // 64
    ids = torch.randperm(n_pages, generator=g, device=dev).int()
    width = max(1, int(held.max()))
    table = torch.full((c["B"], width), -1, dtype=torch.int32, device=dev)
    table[torch.arange(width, device=dev)[None] < i32(held)[:, None]] = ids[: int(held.sum())]
    s = {"case": c, "table": table}
    s["k_pages"], s["k_scales"] = _pool(n_pages, c, c["D"], g, dev)
    s["v_pages"], s["v_scales"] = _pool(n_pages, c, c["Dv"], g, dev)
    if c["op"] in ("append", "read"):
        first, n = _parts(c)
        s.update(starts=i32(first), cu=i32(np.concatenate([[0], np.cumsum(n)])), n=int(n.sum()))
    if c["op"] == "append":
        old, new, served = _chunks(c)
        N, H, Hkv, D, Dv = int(new.sum()), c["H"], c["Hkv"], c["D"], c["Dv"]
        if c["packed"]:   # views of the projection's one output
            q, k, v = randn(N, H * D + Hkv * (D + Dv)).split([H * D, Hkv * D, Hkv * Dv], 1)
        else:
            q, k, v = randn(N, H * D), randn(N, Hkv * D), randn(N, Hkv * Dv)
        # some tokens' keys and values are larger, as they are in earnest: blocks' scales differ, and open ones grow
        loud = torch.exp2(torch.randint(-1, 3, (N, 1, 1), generator=g, device=dev).float()).to(k.dtype)
        s.update(q=q.view(N, H, D), k=k.view(N, Hkv, D).mul_(loud), v=v.view(N, Hkv, Dv).mul_(loud))
        b = np.repeat(np.arange(c["B"]), new)
        pos = np.arange(N) - np.repeat(np.cumsum(new) - new, new) + old[b]
        page = table.long()[torch.from_numpy(b).to(dev), torch.from_numpy(pos // P).to(dev)]
        at = torch.from_numpy(pos).to(dev)
        s["slots"] = torch.where(torch.from_numpy(served[b]).to(dev), page * P + at % P, -1)
        s["pos"] = at.int()
        inv = 1e6 ** (-torch.arange(0, c["rot"], 2, dtype=torch.float64, device=dev) / c["rot"])
        a = torch.arange(int(lens.max()) + 1, dtype=torch.float64, device=dev)[:, None] * inv
        s["turns"] = torch.cat([a.cos(), a.sin()], 1).float()
    if c["op"] in ("decode", "diff"):
        s.update(lens=i32(lens), scale=c["D"] ** -0.5, q=randn(c["B"], c["H"] * (2 if c["op"] == "diff" else 1), c["D"]))
    if c["op"] == "diff":
        s["lam"] = torch.rand(c["H"], generator=g, device=dev) * 0.6 + 0.2
        s["weight"] = 1 + 0.1 * torch.randn(2 * c["Dv"], generator=g, device=dev) if c["norm"] else None
    return s


# ------------------------------------------------------------------ the plain forms


def _turned(x, s):
    """x in 32 bits with its first ``rot`` dims rotated."""
    c, x = s["case"], x.float()
    n = c["rot"] // 2
    turns = s["turns"][s["pos"].long()]
    cos, sin = turns[:, None, :n], turns[:, None, n:]
    if c["adjacent"]:
        x1, x2 = x[..., 0:2 * n:2], x[..., 1:2 * n:2]
    else:
        x1, x2 = x[..., :n], x[..., n:2 * n]
    y1, y2 = x1 * cos - x2 * sin, x2 * cos + x1 * sin
    y = torch.stack([y1, y2], -1).flatten(-2) if c["adjacent"] else torch.cat([y1, y2], -1)
    return torch.cat([y, x[..., 2 * n:]], -1)


def _codes(x, inv, pool):
    if pool == "int8":
        return torch.round(x * inv).clamp(-127, 127).to(torch.int8)
    return (x * inv).clamp(-448, 448).to(torch.float8_e4m3fn)


def _at(pages, *at):
    """pages[at], whatever 8-bit type they hold."""
    return pages.view(torch.int8)[at].view(pages.dtype) if pages.element_size() == 1 else pages[at]


def _own_scale(most, pool):
    """The scale that values of up to ``most`` ask for."""
    most = most.clamp(min=1e-6)
    if pool == "int8":
        return most * (1.0 / 127.0)
    part, up = torch.frexp(most)   # most = part * 2^up, part of [0.5, 1); 448 = 0.875 * 2^9
    return torch.exp2((up - 9 + (part > 0.875).int()).float())


def _write(x, pages, scales, s):
    """Rows x [N, heads, D] in 32 bits into their blocks: the pool's codes and scales in place."""
    c, slots = s["case"], s["slots"]
    P, blk, nb = c["page"], c["block"], c["page"] // c["block"]
    at = torch.nonzero(slots >= 0)[:, 0]
    x, slot = x[at], slots[at]
    page, off = slot // P, slot % P
    place, n_blocks = page * nb + off // blk, pages.shape[0] * nb
    most = x.new_zeros(n_blocks, x.shape[1]).index_reduce_(0, place, x.abs().amax(-1), "amax")
    front = torch.full((n_blocks,), blk, device=x.device).index_reduce_(0, place, off % blk, "amin")
    # the rows before the first new one stay: those of each request's open block
    had = s["starts"].long()
    held = had // P
    b_page = s["table"].long()[torch.arange(had.numel(), device=x.device), held]
    b_off = (had - held * P)[:, None] + torch.arange(blk, device=x.device)
    b_place = b_page * nb + b_off[:, 0] // blk
    before = torch.where((front[b_place] > 0) & (front[b_place] < blk), 1.0, 0.0)[:, None]
    old = scales[b_page, b_off[:, 0] // blk] * before
    new = _own_scale(most, c["pool"])
    full = new.index_reduce(0, b_place, old, "amax")
    ratio = old * (torch.ones_like(old) / full[b_place])
    keep = (torch.arange(blk, device=x.device)[None] < front[b_place][:, None]) & (before > 0)
    rows, raw = _at(pages, b_page[:, None], b_off), pages.view(torch.int8)
    again = _codes(rows.float(), ratio[:, None, :, None], c["pool"])
    grows = keep[..., None, None] & (ratio < 1)[:, None, :, None]
    raw[b_page[:, None], b_off] = torch.where(grows, again.view(torch.int8), rows.view(torch.int8))
    raw[page, off] = _codes(x, (torch.ones_like(full) / full)[place][..., None], c["pool"]).view(torch.int8)
    scales[page, off // blk] = full[place]


def _read(s):
    c = s["case"]
    P, blk = c["page"], c["block"]
    n = (s["cu"][1:] - s["cu"][:-1]).long()
    b = torch.repeat_interleave(torch.arange(c["B"], device=n.device), n, output_size=s["n"])
    t = torch.arange(s["n"], device=n.device) - s["cu"].long()[b] + s["starts"].long()[b]
    page, off = s["table"].long()[b, t // P], t % P

    def rows(pages, scales):
        return (_at(pages, page, off).float() * scales[page, off // blk][..., None]).to(HALF[c["dtype"]])

    return rows(s["k_pages"], s["k_scales"]), rows(s["v_pages"], s["v_scales"])


def _plain_append(s):
    q = _turned(s["q"], s).to(s["q"].dtype)
    _write(_turned(s["k"], s), s["k_pages"], s["k_scales"], s)
    _write(s["v"].float(), s["v_pages"], s["v_scales"], s)
    k, v = _read(s)
    return {"q": q, "k": k, "v": v}


def _rows(pages, scales, s):
    """[B, heads, tokens, D] in 32 bits: every request's rows, padded to the table's width."""
    table = s["table"].long().clamp(min=0)
    x = _at(pages, table).float()
    if scales is not None:
        x = x * torch.repeat_interleave(scales[table], s["case"]["block"], 2)[..., None]
    return x.flatten(1, 2).transpose(1, 2)


def _softmax(score, s):
    """score [B, heads, queries, tokens] -> (exp(score - max), their sums, lse), 0 and -inf where nothing is seen."""
    c, lens = s["case"], s["lens"].long()
    t = torch.arange(score.shape[3], device=lens.device)[None]
    seen = t < lens[:, None]
    if c["window"]:
        seen &= t >= lens[:, None] - c["window"]
    score = (score * s["scale"]).masked_fill(~seen[:, None, None], float("-inf"))
    most = score.amax(3, keepdim=True)
    p = torch.exp(score - most.clamp(min=-1e30))
    total = p.sum(3)
    return p, total, most[..., 0] + total.log()


def _plain_decode(s):
    c = s["case"]
    B, H, Hkv = c["B"], c["H"], c["Hkv"]
    q = s["q"].float().view(B, Hkv, H // Hkv, -1)
    p, total, lse = _softmax(q @ _rows(s["k_pages"], s["k_scales"], s).transpose(2, 3), s)
    o = p @ _rows(s["v_pages"], s["v_scales"], s) / total.clamp(min=1e-30)[..., None]
    return {"out": o.reshape(B, H, -1).to(s["q"].dtype), "lse": lse.reshape(B, H)}


def _plain_diff(s):
    c = s["case"]
    B, H, Hkv, Dv = c["B"], c["H"], c["Hkv"], c["Dv"]
    q = s["q"].float().view(B, Hkv, H // Hkv, 2, -1).transpose(2, 3).flatten(1, 2)   # heads of a map together
    p, total, lse = _softmax(q @ _rows(s["k_pages"], s["k_scales"], s).transpose(2, 3), s)
    v = _rows(s["v_pages"], s["v_scales"], s).unflatten(1, (Hkv, 2))
    p = p.view(B, Hkv, 2 * (H // Hkv), -1)
    o = torch.cat([p @ v[:, :, 0], p @ v[:, :, 1]], -1).view(B, Hkv, 2, H // Hkv, 2 * Dv)
    o = o / total.clamp(min=1e-30).view(B, Hkv, 2, H // Hkv, 1)
    o = o[:, :, 0] - s["lam"].view(Hkv, H // Hkv, 1) * o[:, :, 1]
    if s["weight"] is not None:
        o = o * torch.rsqrt((o * o).mean(-1, keepdim=True) + 1e-5) * s["weight"]
    return {"out": o.reshape(B, H, -1).to(s["q"].dtype),
            "lse": lse.view(B, Hkv, 2, H // Hkv).transpose(2, 3).reshape(B, 2 * H)}


def run(state):
    s, c = state, state["case"]
    if not own:
        if c["op"] == "read":
            k, v = _read(s)
            return {"k": k, "v": v}
        return {"append": _plain_append, "decode": _plain_decode, "diff": _plain_diff}[c["op"]](s)
    from scope_b200 import paged
    pool, scales = (s["k_pages"], s["v_pages"]), dict(k_scales=s["k_scales"], v_scales=s["v_scales"])
    if c["op"] == "decode":
        out, lse = paged.paged_decode(s["q"], *pool, s["table"], s["lens"], s["scale"], window=c["window"], **scales)
        return {"out": out, "lse": lse}
    if c["op"] == "diff":
        out, lse = paged.paged_diff_decode(s["q"], *pool, s["table"], s["lens"], s["scale"], s["lam"], norm_weight=s["weight"],
                                           norm_eps=1e-5, window=c["window"], **scales)
        return {"out": out, "lse": lse}
    outs = {}
    if c["op"] == "append":
        outs["q"] = paged.rope_append(s["q"], s["k"], s["v"], s["pos"], s["turns"], s["slots"], *pool,
                                      pairs="adjacent" if c["adjacent"] else "half", **scales)
    # what an append touched is read back by the other operator
    outs["k"], outs["v"] = paged.paged_read(*pool, s["table"], s["cu"], s["n"], starts=s["starts"], dtype=HALF[c["dtype"]],
                                            **scales)
    return outs


# ------------------------------------------------------------------ what a pass cannot do without


def work(case):
    c = case
    D, Dv, P, blk, hs = c["D"], c["Dv"], c["page"], c["block"], _heads(c)
    if c["op"] in ("append", "read"):
        first, n = _parts(c)
        n = int(n.sum())
        scales = 8 * hs * int((-(-(first + _parts(c)[1]) // blk) - first // blk).sum())
        nbytes = n * hs * (D + Dv) * 2 + scales + 4 * int((-(-(first + _parts(c)[1]) // P) - first // P).sum())
        if c["op"] == "read":
            return {"bytes": nbytes + n * hs * (D + Dv), "flops": n * hs * (D + Dv)}
        N = int(_chunks(c)[1].sum())
        # the tokens' rows and turns in; queries, codes and scales out; the read's codes are those, and a few older ones
        return {"bytes": nbytes + scales + N * (4 * c["H"] * D + 2 * hs * (D + Dv) + 4 * c["rot"] + 12) + n * hs * (D + Dv),
                "flops": 3 * N * (c["H"] + hs) * c["rot"] + 2 * N * hs * (D + Dv)}
    lens = _lens(c)
    if c["window"]:
        lens = np.minimum(lens, c["window"])
    n = int(lens.sum())
    eight = c["pool"] not in HALF
    nbytes = n * hs * (D + Dv) * (1 if eight else 2) + 4 * int((-(-lens // P)).sum()) + 4 * c["B"]
    if eight:
        nbytes += 8 * hs * int((-(-lens // blk)).sum())
    maps = hs // c["Hkv"]
    nbytes += c["B"] * c["H"] * maps * (2 * D + 2 * Dv + 4)
    return {"bytes": nbytes, "flops": 2 * n * c["H"] * maps * (D + maps * Dv)}


# ------------------------------------------------------------------ in 64 bits


def _exact_turn(x, s):
    c, n = s["case"], s["case"]["rot"] // 2
    z, pos = x.double().clone(), s["pos"].long()
    for i in range(n):
        cos, sin = s["turns"][pos, i].double()[:, None], s["turns"][pos, n + i].double()[:, None]
        d1, d2 = (2 * i, 2 * i + 1) if c["adjacent"] else (i, n + i)
        x1, x2 = x[..., d1].double(), x[..., d2].double()
        z[..., d1], z[..., d2] = x1 * cos - x2 * sin, x2 * cos + x1 * sin
    return z


def _near(x, pool):
    """The nearest code's value, ties to even."""
    if pool == "int8":
        return torch.round(x).clamp(-127, 127)
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return (torch.round(x / step) * step).clamp(-448, 448)


def _exact_write(x, pages, scales, s):
    """The pool's codes and scales in 64 bits after the rows x went in, request by request and block by block."""
    c, P, blk = s["case"], s["case"]["page"], s["case"]["block"]
    codes, scales, slots = pages.double(), scales.double(), s["slots"].cpu().numpy()
    keys = np.where(slots >= 0, slots // blk, -1)   # blocks are counted through: a page holds a whole number of them
    cuts = np.concatenate([[0], np.nonzero(np.diff(keys))[0] + 1, [len(keys)]])
    runs = [(a, b) for a, b in zip(cuts[:-1], cuts[1:]) if keys[a] >= 0]
    page = torch.tensor([slots[a] // P for a, _ in runs], device=x.device)
    off = torch.tensor([slots[a] % P for a, _ in runs], device=x.device)
    start = torch.tensor([a for a, _ in runs], device=x.device)
    size = torch.tensor([b - a for a, b in runs], device=x.device)
    for i in range(0, len(runs), 2048):   # the blocks side by side
        pg, of, st, sz = (t[i:i + 2048] for t in (page, off, start, size))
        j, o = of // blk, of % blk
        row = torch.arange(blk, device=x.device)[None]
        new = (row >= o[:, None]) & (row < (o + sz)[:, None])
        src = x[(st[:, None] + row - o[:, None]).clamp(0, len(x) - 1)] * new[..., None, None]
        old = scales[pg, j] * (o > 0)[:, None]
        most = src.abs().amax((1, 3)).clamp(min=1e-6)
        need = most / 127 if c["pool"] == "int8" else torch.exp2(torch.ceil(torch.log2(most / 448)))
        now = torch.maximum(old, need)
        at = (pg[:, None], (j * blk)[:, None] + row)
        was = codes[at]
        kept = torch.where((now > old)[:, None, :, None], _near(was * (old / now)[:, None, :, None], c["pool"]), was)
        is_old = (row < o[:, None])[..., None, None]
        codes[at] = torch.where(is_old, kept, torch.where(new[..., None, None], _near(src / now[:, None, :, None], c["pool"]), was))
        scales[pg, j] = now
    return codes, scales


def exact(case, seed):
    c = case
    s = prepare(case, seed)
    P, blk, hs = c["page"], c["block"], _heads(c)
    if c["op"] in ("append", "read"):
        outs, pools = {}, []
        for name, x in (("k", s.get("k")), ("v", s.get("v"))):
            pages, scales = s[name + "_pages"], s[name + "_scales"]
            if c["op"] == "append":
                pages, scales = _exact_write(_exact_turn(x, s) if name == "k" else x.double(), pages, scales, s)
            pools.append((name, pages, scales))
        if c["op"] == "append":
            outs["q"] = _exact_turn(s["q"], s)
        first, n = _parts(c)
        for name, pages, scales in pools:
            rows = []
            for b in range(c["B"]):
                t = torch.arange(first[b], first[b] + n[b], device="cuda")
                page, off = s["table"][b].long()[t // P], t % P
                rows.append(_at(pages, page, off).double() * scales[page, off // blk].double()[..., None])
            outs[name] = torch.cat(rows)
        return outs
    outs, lses = [], []
    maps = hs // c["Hkv"]
    G, wide = c["H"] // c["Hkv"], maps * c["Dv"]
    for b, L in enumerate(_lens(c).tolist()):
        lo = max(0, L - c["window"]) if c["window"] else 0
        if L == 0:
            outs.append(torch.zeros(c["H"], wide, dtype=torch.float64, device="cuda"))
            lses.append(torch.full((c["H"] * maps,), float("-inf"), dtype=torch.float64, device="cuda"))
            continue
        t = torch.arange(lo, L, device="cuda")
        page, off = s["table"][b].long()[t // P], t % P

        def head(pages, scales, h):
            x = _at(pages, page, off, h).double()
            return x if scales is None else x * scales[page, off // blk, h].double()[:, None]

        heads_o, heads_l = [], []
        for kvh in range(c["Hkv"]):
            v = torch.cat([head(s["v_pages"], s["v_scales"], kvh * maps + m) for m in range(maps)], 1)
            q = s["q"][b].view(c["Hkv"], G, maps, -1)[kvh].double()
            got, ls = [], []
            for m in range(maps):
                z = q[:, m] @ head(s["k_pages"], s["k_scales"], kvh * maps + m).t() * s["scale"]
                ls.append(torch.logsumexp(z, 1))
                got.append(torch.exp(z - ls[-1][:, None]) @ v)
            o = got[0]
            if maps == 2:
                o = o - s["lam"].double()[kvh * G:(kvh + 1) * G, None] * got[1]
                if s["weight"] is not None:
                    o = o / torch.sqrt((o * o).mean(1, keepdim=True) + 1e-5) * s["weight"].double()
            heads_o.append(o)
            heads_l.append(torch.stack(ls, 1).flatten())
        outs.append(torch.cat(heads_o))
        lses.append(torch.cat(heads_l))
    return {"out": torch.stack(outs), "lse": torch.stack(lses)}

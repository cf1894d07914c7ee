"""Cases of the paged key-value cache's operators: page tables and slot maps from request lengths, rotary
positions with several axes, the append of rotated keys and values into pages, and the decode attention that
reads them.  Each case has a plain form (elementary torch operations in 32 bits) and, with ``own`` set, the
framework's call.
"""
import numpy as np
import torch

own = False

HALF = {"bf16": torch.bfloat16, "fp16": torch.float16}
LARGEST = 8.7e9   # bytes of keys and values that a drawn decode may span when every request is padded to the longest


def listed():
    return [
        # one decode step's bookkeeping of a running batch: every request gets one token
        dict(name="slots-decode", op="slots", B=64, page=16, most=4096, prompts=0.0, prompt=1, short=False, lens_seed=1),
        # a large server's step that admits prompts beside decodes, with fewer free pages than it would take
        dict(name="slots-mixed", op="slots", B=512, page=32, most=32768, prompts=0.5, prompt=1024, short=True,
             lens_seed=2),
        # queries of a decode step: 20 heads of 96, the first 64 dims rotated in adjacent pairs, backwards
        dict(name="rope-decode", op="rope", N=8, H=20, D=96, rot=64, axes=1, cyclic=False, adjacent=True, inverse=True,
             dtype="fp16", top=32768),
        # queries of a long prompt of images and text: time, height and width share the 64 pairs
        dict(name="rope-3axes-prompt", op="rope", N=16384, H=32, D=128, rot=128, axes=3, cyclic=False, adjacent=False,
             inverse=False, dtype="bf16", top=32768),
        # one decode step of 64 requests, 32 query and 8 kv heads
        dict(name="append-decode", op="append", N=64, H=32, Hkv=8, D=128, Dv=128, rot=128, axes=1, cyclic=False,
             adjacent=False, dtype="bf16", pool="bf16", page=16, heads_major=False, packed=True, top=131072),
        # a long prompt of images and text, read from the packed projection
        dict(name="append-prompt", op="append", N=16384, H=32, Hkv=4, D=128, Dv=128, rot=128, axes=3, cyclic=True,
             adjacent=False, dtype="bf16", pool="bf16", page=64, heads_major=False, packed=True, top=32768),
        # a ragged chunk into an int8 pool, heads of 80 (an odd number of 16-byte pieces), head-major pages
        dict(name="append-int8", op="append", N=4097, H=20, Hkv=5, D=80, Dv=80, rot=64, axes=1, cyclic=False,
             adjacent=False, dtype="fp16", pool="int8", page=24, heads_major=True, packed=False, top=8192),
        # one user, 4096 tokens: latency
        dict(name="decode-1x4096", op="decode", B=1, H=32, Hkv=4, D=128, Dv=128, dtype="bf16", pool="bf16", page=16,
             heads_major=False, least=4096, most=4096, empty=False, window=0, lens_seed=3),
        # many short chats, one slot of the batch empty, a window that cuts the longer ones, odd pages and heads
        dict(name="decode-128-short", op="decode", B=128, H=20, Hkv=4, D=80, Dv=80, dtype="fp16", pool="fp16", page=24,
             heads_major=True, least=1, most=1024, empty=True, window=700, lens_seed=4),
        # a ragged batch of documents
        dict(name="decode-16-ragged", op="decode", B=16, H=32, Hkv=8, D=128, Dv=128, dtype="bf16", pool="bf16", page=64,
             heads_major=False, least=1024, most=32768, empty=False, window=0, lens_seed=5),
        # long documents in an int8 pool
        dict(name="decode-8-int8", op="decode", B=8, H=32, Hkv=4, D=128, Dv=128, dtype="bf16", pool="int8", page=32,
             heads_major=False, least=16384, most=65536, empty=False, window=0, lens_seed=6),
        # the largest: 32 requests of 131072 tokens
        dict(name="decode-32x131072", op="decode", B=32, H=32, Hkv=4, D=128, Dv=128, dtype="bf16", pool="bf16", page=64,
             heads_major=False, least=131072, most=131072, empty=False, window=0, lens_seed=7),
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], even over the logarithm."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["slots", "rope", "append", "append", "decode", "decode", "decode", "decode"])
    page = rng.choice([8, 16, 16, 24, 32, 48, 64, 128, 256])
    if op == "slots":
        return dict(op=op, B=_spread(rng, 1, 1024), page=page, most=_spread(rng, 64, 65536),
                    prompts=rng.choice([0.0, 0.1, 0.5]), prompt=_spread(rng, 8, 1024), short=rng.random() < 0.3,
                    lens_seed=rng.randrange(1 << 30))
    axes = rng.choice([1, 1, 2, 3, 4])
    turn = dict(axes=axes, cyclic=axes > 1 and rng.random() < 0.5, adjacent=rng.random() < 0.4,
                dtype=rng.choice(["bf16", "fp16"]), top=_spread(rng, 1024, 131072))
    D = rng.choice([32, 64, 80, 96, 112, 128, 128, 192, 256])
    if op == "rope":
        return dict(op=op, N=_spread(rng, 1, 16384), H=rng.randint(1, 40), D=D, rot=rng.choice([D, 16 * rng.randint(1, D // 16)]),
                    inverse=rng.random() < 0.3, **turn)
    Hkv = rng.randint(1, 8)
    G = rng.choice([1, 2, 3, 4, 5, 6, 7, 8, 8, 12, 16])
    Dv = rng.choice([D, D, D, 128 if D == 192 else D, 64])
    if op == "append":
        return dict(op=op, N=_spread(rng, 1, 16384), H=Hkv * min(G, 8), Hkv=Hkv, D=D, Dv=Dv,
                    rot=rng.choice([D, 16 * rng.randint(1, D // 16)]), pool=rng.choice([turn["dtype"], turn["dtype"], "int8"]),
                    page=page, heads_major=rng.random() < 0.5, packed=rng.random() < 0.5, **turn)
    pool = rng.choice([turn["dtype"], turn["dtype"], "int8"])
    B = _spread(rng, 1, 256)
    room = LARGEST / (B * Hkv * (D + Dv) * (1 if pool == "int8" else 2))
    most = _spread(rng, 1, int(min(131072, room)))
    return dict(op=op, B=B, H=Hkv * G, Hkv=Hkv, D=D, Dv=Dv, dtype=turn["dtype"], pool=pool, page=page,
                heads_major=rng.random() < 0.5, least=_spread(rng, 1, most), most=most, empty=B > 1 and rng.random() < 0.3,
                window=rng.choice([0, 0, 0, _spread(rng, 1, most)]), lens_seed=rng.randrange(1 << 30))


# ------------------------------------------------------------------ what the cases hold


def _lens(c):
    """A decode case's request lengths."""
    r = np.random.RandomState(c["lens_seed"] % (1 << 32))
    lens = r.randint(c["least"], c["most"] + 1, c["B"])
    if c["empty"]:
        lens[r.randint(c["B"])] = 0
    return lens


def _requests(c):
    """A bookkeeping case's (lengths before the step, new tokens): decodes take one, prompts start from nothing
    or go on in a chunk, and a few requests wait."""
    r = np.random.RandomState(c["lens_seed"] % (1 << 32))
    lens = r.randint(1, c["most"] + 1, c["B"])
    new = np.ones(c["B"], dtype=np.int64)
    prompt = r.rand(c["B"]) < c["prompts"]
    new[prompt] = r.randint(1, c["prompt"] + 1, int(prompt.sum()))
    fresh = prompt & (r.rand(c["B"]) < 0.7)
    lens[fresh] = 0
    if c["prompts"]:
        new[r.rand(c["B"]) < 0.05] = 0
    return lens, new


def _sections(c):
    """How many pairs each axis takes: the first the most, the others the same number."""
    if c["axes"] == 1:
        return None
    each = (c["rot"] // 2) // (c["axes"] + 1 if c["axes"] < 4 else 4)
    return (c["rot"] // 2 - each * (c["axes"] - 1),) + (each,) * (c["axes"] - 1)


def _axis_of_pair(c):
    """The axis that each pair turns by."""
    n, sections = c["rot"] // 2, _sections(c)
    if sections is None:
        return [0] * n
    if c["cyclic"]:
        return [i % c["axes"] if i // c["axes"] < sections[i % c["axes"]] else 0 for i in range(n)]
    return [a for a, s in enumerate(sections) for _ in range(s)]


def _turns(c, dev):
    """cos | sin of every position, fp32 [top, rot]."""
    inv = 1e6 ** (-torch.arange(0, c["rot"], 2, dtype=torch.float64, device=dev) / c["rot"])
    a = torch.arange(c["top"], dtype=torch.float64, device=dev)[:, None] * inv
    return torch.cat([a.cos(), a.sin()], 1).float()


def _positions(c, g, dev):
    if c["axes"] == 1:
        first = torch.randint(0, max(1, c["top"] - c["N"]), (1,), generator=g, device=dev)
        return ((first + torch.arange(c["N"], device=dev)) % c["top"]).int()
    return torch.randint(0, c["top"], (c["axes"], c["N"]), generator=g, device=dev, dtype=torch.int32)


def _pool(n_pages, c, Dx, g, dev):
    """A pool of pages [n_pages, page, Hkv, Dx] and its scales, filled with values (pages of an earlier request)."""
    shape = (n_pages, c["Hkv"], c["page"]) if c["heads_major"] else (n_pages, c["page"], c["Hkv"])
    if c["pool"] == "int8":
        x = (torch.randn(*shape, Dx, generator=g, device=dev, dtype=torch.bfloat16) * 32).round_().clamp_(-127, 127).to(torch.int8)
        s = torch.rand(*shape, generator=g, device=dev) * 0.04 + 0.01
    else:
        x = torch.randn(*shape, Dx, generator=g, device=dev, dtype=HALF[c["pool"]])
        s = None
    if c["heads_major"]:
        x, s = x.transpose(1, 2), None if s is None else s.transpose(1, 2)
    return x, s


def prepare(case, seed):
    c, dev = case, torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    s = {"case": c}

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=dev, dtype=HALF[c["dtype"]])

    if c["op"] == "slots":
        lens, new = _requests(c)
        P = c["page"]
        held, need = -(-lens // P), -(-(lens + new) // P) - -(-lens // P)
        n_free = int(need.sum() * (0.8 if c["short"] else 1.2)) + (0 if c["short"] else 4)
        n_pages = int(held.sum()) + n_free
        ids = torch.randperm(n_pages, generator=g, device=dev).int()
        width = -(-(c["most"] + c["prompt"]) // P)
        table = torch.full((c["B"], width), -1, dtype=torch.int32, device=dev)
        h = torch.from_numpy(held).to(dev)
        has = torch.arange(width, device=dev)[None] < h[:, None]
        table[has] = ids[: int(held.sum())]
        ring = torch.full((n_pages,), -1, dtype=torch.int32, device=dev)
        head = int(torch.randint(0, n_pages, (1,), generator=g, device=dev))
        ring[(head + torch.arange(n_free, device=dev)) % n_pages] = ids[int(held.sum()):]
        s.update(lens=torch.from_numpy(lens).to(dev).int(), new=torch.from_numpy(new).to(dev).int(), table=table,
                 free=ring, ring=torch.tensor([head, n_free, 0], dtype=torch.int32, device=dev), n=int(new.sum()))
        return s
    if c["op"] in ("rope", "append"):
        s.update(turns=_turns(c, dev), pos=_positions(c, g, dev))
        if c["op"] == "rope":
            s["x"] = randn(c["N"], c["H"], c["D"])
            return s
        N, H, Hkv, D, Dv = c["N"], c["H"], c["Hkv"], c["D"], c["Dv"]
        if c["packed"]:   # views of the projection's one output
            qkv = randn(N, H * D + Hkv * (D + Dv))
            q, k, v = qkv.split([H * D, Hkv * D, Hkv * Dv], 1)
        else:
            q, k, v = randn(N, H * D), randn(N, Hkv * D), randn(N, Hkv * Dv)
        s.update(q=q.view(N, H, D), k=k.view(N, Hkv, D), v=v.view(N, Hkv, Dv))
        n_pages = -(-N // c["page"]) + 2
        s["k_pages"], s["k_scales"] = _pool(n_pages, c, D, g, dev)
        s["v_pages"], s["v_scales"] = _pool(n_pages, c, Dv, g, dev)
        # tokens lie in whole pages, the pages anywhere; a few tokens of refused requests have no slot
        page = torch.randperm(n_pages, generator=g, device=dev)
        t = torch.arange(N, device=dev)
        slots = page[t // c["page"]] * c["page"] + t % c["page"]
        slots[torch.rand(N, generator=g, device=dev) < 0.01] = -1
        s["slots"] = slots
        return s
    lens = _lens(c)
    held = -(-lens // c["page"])
    n_pages = int(held.sum()) + 1 + int(held.sum()) // 64
    ids = torch.randperm(n_pages, generator=g, device=dev).int()
    width = max(1, int(held.max()))
    table = torch.full((c["B"], width), -1, dtype=torch.int32, device=dev)
    table[torch.arange(width, device=dev)[None] < torch.from_numpy(held).to(dev)[:, None]] = ids[: int(held.sum())]
    s["q"] = randn(c["B"], c["H"], c["D"])
    s["k_pages"], s["k_scales"] = _pool(n_pages, c, c["D"], g, dev)
    s["v_pages"], s["v_scales"] = _pool(n_pages, c, c["Dv"], g, dev)
    s.update(table=table, lens=torch.from_numpy(lens).to(dev).int(), scale=c["D"] ** -0.5)
    return s


# ------------------------------------------------------------------ the plain forms


def _plain_slots(s):
    P, B, n = s["case"]["page"], s["lens"].numel(), s["n"]
    lens, new, table, ring = s["lens"].long(), s["new"].long(), s["table"], s["ring"].long()
    end = new.cumsum(0)
    held, want = -(-lens // P), -(-(lens + new) // P)
    fits = (want <= table.shape[1]) & (end <= n)
    need = torch.where(fits, want - held, 0)
    upto = need.cumsum(0)
    served = fits & ((need == 0) | (upto <= ring[1]))
    b = torch.repeat_interleave(torch.arange(B, device=lens.device), new, output_size=n)
    p = lens[b] + torch.arange(n, device=lens.device) - (end - new)[b]
    fresh = served[b] & (p // P >= held[b])
    taken = s["free"][(ring[0] + (upto - need)[b] + p // P - held[b]) % s["free"].numel()]
    col = (p // P).clamp(max=table.shape[1] - 1)
    page = torch.where(fresh, taken, table[b, col])
    # every token of a fresh page writes the same entry, the others write back what is there
    table[b, col] = page
    slots = torch.where(served[b], page.long() * P + p % P, -1)
    took = (need * served).sum()
    ring_out = torch.stack([(ring[0] + took) % s["free"].numel(), ring[1] - took, (~served).sum()]).int()
    return {"slots": slots, "positions": torch.where(served[b], p, 0).int(),
            "cu_new": torch.cat([end.new_zeros(1), end]).int(), "seq_lens": (lens + new * served).int(),
            "ring": ring_out, "table": table}


def _turned(x, s, inverse=False):
    """x in 32 bits with its first ``rot`` dims rotated."""
    c, x = s["case"], x.float()
    n = c["rot"] // 2
    if c["axes"] == 1:
        turns = s["turns"][s["pos"].long()]
    else:
        axis = torch.tensor(_axis_of_pair(c) * 2, device=x.device)
        turns = s["turns"][s["pos"].long()[axis].t(), torch.arange(2 * n, device=x.device)]
    cos, sin = turns[:, None, :n], turns[:, None, n:]
    if inverse:
        sin = -sin
    if c["adjacent"]:
        x1, x2 = x[..., 0:2 * n:2], x[..., 1:2 * n:2]
    else:
        x1, x2 = x[..., :n], x[..., n:2 * n]
    y1, y2 = x1 * cos - x2 * sin, x2 * cos + x1 * sin
    y = torch.stack([y1, y2], -1).flatten(-2) if c["adjacent"] else torch.cat([y1, y2], -1)
    return torch.cat([y, x[..., 2 * n:]], -1)


def _codes(x):
    most = x.abs().amax(-1).clamp(min=1e-6)
    inv = torch.full_like(most, 127.0) / most   # one division (127.0 / most is a reciprocal and a product)
    return torch.round(x * inv[..., None]).clamp(-128, 127).to(torch.int8), most * (1.0 / 127.0)


def _values(s):
    """The pools as the values that they stand for."""
    if s["case"]["pool"] != "int8":
        return s["k_pages"], s["v_pages"]
    dt = HALF[s["case"]["dtype"]]
    return (s["k_pages"] * s["k_scales"][..., None]).to(dt), (s["v_pages"] * s["v_scales"][..., None]).to(dt)


def _plain_append(s):
    c = s["case"]
    k, v = _turned(s["k"], s), s["v"].float()
    at = torch.nonzero(s["slots"] >= 0)[:, 0]
    page, off = s["slots"][at] // c["page"], s["slots"][at] % c["page"]
    if c["pool"] == "int8":
        (k, ks), (v, vs) = _codes(k), _codes(v)
        s["k_scales"][page, off], s["v_scales"][page, off] = ks[at], vs[at]
    s["k_pages"][page, off] = k[at].to(s["k_pages"].dtype)
    s["v_pages"][page, off] = v[at].to(s["v_pages"].dtype)
    kp, vp = _values(s)
    return {"q": _turned(s["q"], s).to(s["q"].dtype), "k": kp, "v": vp}


def _plain_decode(s):
    c, lens = s["case"], s["lens"].long()
    B, H, Hkv = c["B"], c["H"], c["Hkv"]
    table = s["table"].long().clamp(min=0)

    def rows(pages, scales):   # [B, Hkv, tokens, D] in 32 bits
        x = pages[table].float()
        if scales is not None:
            x = x * scales[table][..., None]
        return x.flatten(1, 2).transpose(1, 2)

    score = rows(s["k_pages"], s["k_scales"]) @ s["q"].float().view(B, Hkv, H // Hkv, -1).transpose(2, 3)
    t = torch.arange(score.shape[2], device=lens.device)[None]
    seen = t < lens[:, None]
    if c["window"]:
        seen &= t >= lens[:, None] - c["window"]
    score = (score * s["scale"]).masked_fill(~seen[:, None, :, None], float("-inf"))
    most = score.amax(2, keepdim=True)
    p = torch.exp(score - most.clamp(min=-1e30))
    total = p.sum(2)
    o = p.transpose(2, 3) @ rows(s["v_pages"], s["v_scales"])
    o = o / total.clamp(min=1e-30)[..., None]
    return {"out": o.reshape(B, H, -1).to(s["q"].dtype), "lse": (most[:, :, 0] + total.log()).reshape(B, H)}


def run(state):
    s, c = state, state["case"]
    if not own:
        return {"slots": _plain_slots, "append": _plain_append, "decode": _plain_decode,
                "rope": lambda s: _turned(s["x"], s, c["inverse"]).to(s["x"].dtype)}[c["op"]](s)
    from scope_b200 import paged
    if c["op"] == "slots":
        r = paged.paged_slots(s["lens"], s["new"], s["table"], s["free"], s["ring"], c["page"], s["n"])
        return {"slots": r.slots, "positions": r.positions, "cu_new": r.cu_new, "seq_lens": r.seq_lens, "ring": r.ring,
                "table": s["table"]}
    if c["op"] == "decode":
        out, lse = paged.paged_decode(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lens"], s["scale"],
                                      window=c["window"], k_scales=s["k_scales"], v_scales=s["v_scales"])
        return {"out": out, "lse": lse}
    turn = dict(sections=_sections(c), cyclic=c["cyclic"], pairs="adjacent" if c["adjacent"] else "half")
    if c["op"] == "rope":
        return paged.rope(s["x"], s["pos"], s["turns"], inverse=c["inverse"], **turn)
    q = paged.rope_append(s["q"], s["k"], s["v"], s["pos"], s["turns"], s["slots"], s["k_pages"], s["v_pages"],
                          k_scales=s["k_scales"], v_scales=s["v_scales"], **turn)
    k, v = _values(s)
    return {"q": q, "k": k, "v": v}


# ------------------------------------------------------------------ what a pass cannot do without


def work(case):
    c = case
    if c["op"] == "slots":
        lens, new = _requests(c)
        P = c["page"]
        need = int((-(-(lens + new) // P) - -(-lens // P)).sum())
        # lengths in and out, offsets; a slot and a position for each token; a free page read and a table entry written
        # for each page, and the last page's entry of each request
        return {"bytes": 20 * c["B"] + 12 * int(new.sum()) + 8 * need, "flops": 0}
    if c["op"] in ("rope", "append"):
        turns = c["N"] * c["rot"] * 4 + c["N"] * c["axes"] * 4
        if c["op"] == "rope":
            return {"bytes": 4 * c["N"] * c["H"] * c["D"] + turns, "flops": 3 * c["N"] * c["H"] * c["rot"]}
        rows = c["Hkv"] * (c["D"] + c["Dv"])
        kept = rows + 8 * c["Hkv"] if c["pool"] == "int8" else 2 * rows
        return {"bytes": c["N"] * (4 * c["H"] * c["D"] + 2 * rows + kept + 8) + turns,
                "flops": 3 * c["N"] * (c["H"] + c["Hkv"]) * c["rot"]}
    lens = _lens(c)
    if c["window"]:
        lens = np.minimum(lens, c["window"])
    n = int(lens.sum())
    row = (c["D"] + c["Dv"]) * (1 if c["pool"] == "int8" else 2) + (8 if c["pool"] == "int8" else 0)
    return {"bytes": n * c["Hkv"] * row + 4 * int((-(-lens // c["page"])).sum()) + 4 * c["B"]
            + c["B"] * c["H"] * (2 * c["D"] + 2 * c["Dv"] + 4), "flops": 2 * n * c["H"] * (c["D"] + c["Dv"])}


# ------------------------------------------------------------------ in 64 bits


def _exact_turn(x, s, inverse=False):
    c, n = s["case"], s["case"]["rot"] // 2
    pos = s["pos"].long().view(c["axes"], c["N"])
    z = x.double().clone()
    for i, a in enumerate(_axis_of_pair(c)):
        cos, sin = s["turns"][pos[a], i].double()[:, None], s["turns"][pos[a], n + i].double()[:, None]
        if inverse:
            sin = -sin
        d1, d2 = (2 * i, 2 * i + 1) if c["adjacent"] else (i, n + i)
        x1, x2 = x[..., d1].double(), x[..., d2].double()
        z[..., d1], z[..., d2] = x1 * cos - x2 * sin, x2 * cos + x1 * sin
    return z


def exact(case, seed):
    c = case
    if c["op"] == "slots":
        return None
    s = prepare(case, seed)
    if c["op"] == "rope":
        return _exact_turn(s["x"], s, c["inverse"])
    if c["op"] == "append":
        k, v = _exact_turn(s["k"], s), s["v"].double()
        kp, vp = s["k_pages"].double(), s["v_pages"].double()
        if c["pool"] == "int8":
            kp, vp = kp * s["k_scales"].double()[..., None], vp * s["v_scales"].double()[..., None]

            def near(x):   # the nearest of the 255 values that the row's largest spans
                most = x.abs().amax(-1, keepdim=True).clamp(min=1e-6)
                return torch.round(x * 127 / most) * (most / 127)

            k, v = near(k), near(v)
        for t, slot in enumerate(s["slots"].tolist()):
            if slot >= 0:
                kp[slot // c["page"], slot % c["page"]] = k[t]
                vp[slot // c["page"], slot % c["page"]] = v[t]
        return {"q": _exact_turn(s["q"], s), "k": kp, "v": vp}
    outs, lses = [], []
    G = c["H"] // c["Hkv"]
    for b, L in enumerate(_lens(c).tolist()):
        lo = max(0, L - c["window"]) if c["window"] else 0
        if L == 0:
            outs.append(torch.zeros(c["H"], c["Dv"], dtype=torch.float64, device="cuda"))
            lses.append(torch.full((c["H"],), float("-inf"), dtype=torch.float64, device="cuda"))
            continue
        t = torch.arange(lo, L, device="cuda")
        page, off = s["table"][b].long()[t // c["page"]], t % c["page"]
        heads_o, heads_l = [], []
        for h in range(c["Hkv"]):
            k, v = s["k_pages"][page, off, h].double(), s["v_pages"][page, off, h].double()
            if c["pool"] == "int8":
                k = k * s["k_scales"][page, off, h].double()[:, None]
                v = v * s["v_scales"][page, off, h].double()[:, None]
            z = s["q"][b, h * G:(h + 1) * G].double() @ k.t() * s["scale"]
            lse = torch.logsumexp(z, 1)
            heads_o.append(torch.exp(z - lse[:, None]) @ v)
            heads_l.append(lse)
        outs.append(torch.cat(heads_o))
        lses.append(torch.cat(heads_l))
    return {"out": torch.stack(outs), "lse": torch.stack(lses)}

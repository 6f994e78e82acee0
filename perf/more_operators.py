"""Operators next to the 8-bit paged key / value cache: what is done to a step's queries and keys before it, and attention for
sequences that begin alike; in plain torch and by this library.

Rows [rows, heads, D] in bfloat16, each row a token at a position. Channels [first, first + rot) of a head are rotated in pairs
by the angle position * freq[pair]: channels 2i and 2i + 1 of the part (interleaved) or i and i + rot / 2 (halves); with a
factor `mscale` on the rotated part, and frequencies that are scaled for contexts longer than the trained one.

- rope: the rotation of heads, or (inverse) its transpose.
- norm_rope: queries and keys divided by the root mean square of their head, times a weight for each channel, then rotated.
- append: the same for the rows of a serving step, whose keys, rounded to bfloat16, go into the paged cache with the values:
  e4m3 codes [page, D] of the keys and [D, page] of the values, a power-of-two scale (e8m0) for each page and head. Position t
  of sequence b lies in slot t % page of page table[b][t // page]; sequence b brings rows cu[b] .. cu[b + 1], and lens[b]
  counts its tokens, the new ones included. A block's scale is the smallest power of two that fits its tokens and never shrinks.
- shared: causal softmax attention of the step's rows over their sequences' cached tokens, in groups of sequences whose tables
  begin with the same pages.
"""
import math

import torch

own = False

EPS = 1e-6


def listed():
    gqa = {"Hq": 32, "Hkv": 8, "D": 128, "page": 64}
    full = {"first": 0, "rot": 128, "interleaved": False, "base": 500000.0, "factor": 1.0, "orig": 0}
    return [
        # A few draft tokens through the layers of a model whose heads of 80 channels are rotated in part; latency.
        {"name": "rope_draft_7", "op": "rope", "rows": 7, "heads": 40, "D": 80, "first": 0, "rot": 32, "interleaved": False,
         "base": 10000.0, "factor": 1.0, "orig": 0, "inverse": False, "far": 2000, "layers": 16, "graph": True},
        # A prompt's wide heads, of which the last 64 channels are rotated, far past the trained length.
        {"name": "rope_prompt_4099", "op": "rope", "rows": 4099, "heads": 64, "D": 192, "first": 128, "rot": 64,
         "interleaved": True, "base": 10000.0, "factor": 16.0, "orig": 4096, "inverse": False, "far": 60000, "layers": 1,
         "graph": False},
        # One token of each sequence of a batch through the layers.
        {"name": "norm_rope_decode_32", "op": "norm_rope", "rows": 32, "Hq": 32, "Hkv": 8, "D": 128, **full, "far": 8000,
         "layers": 16, "graph": True},
        # A long prompt of a model with many query heads.
        {"name": "norm_rope_prompt_8191", "op": "norm_rope", "rows": 8191, "Hq": 64, "Hkv": 8, "D": 128, **full, "far": 0,
         "layers": 1, "graph": False},
        # One token of each sequence of a batch into its layers' caches.
        {"name": "append_decode_64", "op": "append", "B": 64, "n": 1, "chunk": 0, "ctx_lo": 1, "ctx_hi": 5000, **gqa, **full,
         "layers": 8, "graph": True},
        # Three prompts of different lengths, half of each head rotated.
        {"name": "append_prompt_3", "op": "append", "B": 3, "n": 2001, "chunk": 8000, "ctx_lo": 0, "ctx_hi": 90, **gqa,
         "first": 0, "rot": 64, "interleaved": False, "base": 10000.0, "factor": 8.0, "orig": 8192, "layers": 1,
         "graph": False},
        # Four answers to one short question, a token at a time, through the layers; latency and launches.
        {"name": "shared_decode_4", "op": "shared", "groups": 1, "each": 4, "n": 1, "pre_lo": 700, "pre_hi": 700, "own_lo": 3,
         "own_hi": 60, **gqa, "layers": 16, "graph": True, "told": False},
        # A service whose requests all begin with the same instructions.
        {"name": "shared_decode_64", "op": "shared", "groups": 1, "each": 64, "n": 1, "pre_lo": 8003, "pre_hi": 8003,
         "own_lo": 1, "own_hi": 500, **gqa, "layers": 4, "graph": True, "told": False},
        # Parallel sampling: eight answers to each of eight prompts; small heads and small pages.
        {"name": "shared_groups_8x8", "op": "shared", "groups": 8, "each": 8, "n": 1, "pre_lo": 1500, "pre_hi": 6000,
         "own_lo": 0, "own_hi": 900, "Hq": 64, "Hkv": 8, "D": 64, "page": 16, "layers": 1, "graph": False, "told": True},
        # The same instructions before requests whose draft tokens are verified.
        {"name": "shared_verify_24", "op": "shared", "groups": 1, "each": 24, "n": 5, "pre_lo": 12001, "pre_hi": 12001,
         "own_lo": 200, "own_hi": 1500, "Hq": 32, "Hkv": 4, "D": 128, "page": 32, "layers": 1, "graph": False, "told": True},
        # Many questions about one long document.
        {"name": "shared_document_256", "op": "shared", "groups": 1, "each": 256, "n": 1, "pre_lo": 32768, "pre_hi": 32768,
         "own_lo": 10, "own_hi": 1000, **gqa, "layers": 1, "graph": False, "told": False},
    ]


def draw(rng):
    def log(lo, hi):
        return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))

    op = rng.choice(["rope", "norm_rope", "append", "shared", "shared"])
    hkv = rng.choice([1, 2, 4, 8])
    hq = hkv * rng.choice([1, 3, 4, 7, 8, 12])
    if op == "shared":
        d, page = rng.choice([64, 128, 128, 256]), rng.choice([16, 32, 64, 128])
        groups, n = log(1, 16), rng.choice([1, 1, 2, 5])
        each = log(2, max(2, 256 // groups // n))
        layers = 4 if groups * each < 32 else 1
        tail = log(1, min(2000, (1 << 27) // (groups * each * hkv * d)))
        rows = groups * each * n * hq
        hi = log(64, min(32768, (1 << 28) // (groups * hkv * d * layers), (1 << 35) // (rows * d * layers) - tail - n))
        return {"op": op, "groups": groups, "each": each, "n": n, "pre_lo": rng.randint(hi // 3, hi), "pre_hi": hi,
                "own_lo": rng.randint(0, tail), "own_hi": tail, "Hq": hq, "Hkv": hkv, "D": d, "page": page,
                "layers": layers, "graph": n == 1, "told": groups > 1 or rng.random() < 0.5}
    d = rng.choice([64, 128, 128, 256]) if op == "append" else rng.choice([48, 64, 80, 96, 128, 128, 192, 256])
    rot = rng.choice([d, d, d // 2, d // 4])
    turn = {"D": d, "first": rng.choice([0, d - rot]), "rot": rot, "interleaved": rng.random() < 0.5,
            "base": rng.choice([10000.0, 500000.0, 1000000.0]), "factor": 1.0, "orig": 0}
    if rng.random() < 0.5:
        turn.update(factor=rng.choice([2.0, 8.0, 40.0]), orig=rng.choice([2048, 8192]))
    if op == "append":
        decode = rng.random() < 0.5
        return {"op": op, "B": log(1, 256) if decode else log(1, 6), "n": 1 if decode else log(2, 3000),
                "chunk": 0 if decode else log(2, 5000), "ctx_lo": rng.randint(0, 60),
                "ctx_hi": log(60, 5000 if decode else 600), "Hq": hq, "Hkv": hkv, "page": rng.choice([16, 32, 64, 128]), **turn,
                "layers": 8 if decode else 1, "graph": decode}
    few = rng.random() < 0.5
    case = {"op": op, "rows": log(1, 128) if few else log(128, 8192), **turn, "far": log(1, 1000000), "layers": 8 if few else 1,
            "graph": few}
    return {**case, "heads": hq, "inverse": rng.random() < 0.3} if op == "rope" else {**case, "Hq": hq, "Hkv": hkv}


# ---- sizes -----------------------------------------------------------------------------------------------------------
def spread(b, lo, hi):
    """b lengths over lo .. hi, both ends of the range among them for a large b."""
    return [hi if b == 1 else lo + int((i * 0.6180339887 + 0.999) % 1.0 * (hi - lo + 0.999)) for i in range(b)]


def rows_of(c):
    if c["op"] == "shared":
        return [c["n"]] * (c["groups"] * c["each"])
    return [c["chunk"]] + [c["n"]] * (c["B"] - 1) if c["chunk"] else [c["n"]] * c["B"]


def prefixes(c):
    """Tokens that each group begins with; sequence b is one of group b % groups."""
    return spread(c["groups"], c["pre_lo"], c["pre_hi"])


def lens_of(c):
    if c["op"] == "shared":
        pre = prefixes(c) * c["each"]
        return [p + o + c["n"] for p, o in zip(pre, spread(len(pre), c["own_lo"], c["own_hi"]))]
    return [a + n for a, n in zip(spread(c["B"], c["ctx_lo"], c["ctx_hi"]), rows_of(c))]


def mscale(c):
    return 0.1 * math.log(c["factor"]) + 1.0 if c["factor"] > 1.0 else 1.0


# ---- inputs ----------------------------------------------------------------------------------------------------------
def int32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def frequencies(c):
    """Radians a position for each pair, float64. Scaled: pairs that turn 32 times or more over the trained length keep their
    frequency, those that turn once or less are slowed by the factor, those between in proportion."""
    f = torch.arange(0, c["rot"], 2, dtype=torch.float64, device="cuda") / c["rot"]
    f = torch.exp(-math.log(c["base"]) * f)
    if c["orig"]:
        keep = ((f * (c["orig"] / (2 * math.pi)) - 1.0) / 31.0).clamp(0.0, 1.0)
        f = f * (keep + (1.0 - keep) / c["factor"])
    return f


def caches(gen, layers, pages, c):
    """Layers of a cache whose every slot holds a token: k, v, ks, vs, of [layers, pages, Hkv, ...]. The scales differ
    by block as they do where tokens differ."""
    h, p, d = c["Hkv"], c["page"], c["D"]

    def codes(*shape):
        x = torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)
        return (x * 64.0).to(torch.float8_e4m3fn).view(torch.uint8)

    def scales():
        return torch.randint(120, 123, (layers, pages, h), dtype=torch.uint8, generator=gen, device="cuda")

    k = torch.stack([codes(pages, h, p, d) for _ in range(layers)])
    v = torch.stack([codes(pages, h, d, p) for _ in range(layers)])
    return {"k": k, "v": v, "ks": scales(), "vs": scales()}


def tables(gen, lens, shared, group, page):
    """Pages for sequences of `lens` tokens in no order: the first shared[g] blocks of all sequences of group g are the same
    pages. A table [B, width] with -1 behind each sequence's blocks, and the number of pages."""
    blocks, shared, group = -(-lens // page), torch.tensor(shared, device="cuda"), torch.tensor(group, device="cuda")
    alone = blocks - shared[group]
    at, start = torch.cumsum(shared, 0) - shared, shared.sum() + torch.cumsum(alone, 0) - alone
    pages = int(shared.sum() + alone.sum()) + 3
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    blk = torch.arange(int(blocks.max()) + 1, device="cuda")
    mine = start[:, None] + blk - shared[group][:, None]
    index = torch.where(blk < shared[group][:, None], at[group][:, None] + blk, mine)
    table = torch.where(blk < blocks[:, None], order[index.clamp(0, pages - 1)], -1)
    return table.to(torch.int32).contiguous(), pages


def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    s = {"case": c, "graph": None}

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda").to(torch.bfloat16)

    if c["op"] in ("rope", "norm_rope"):
        s["rows"] = c["rows"]
        start = torch.randint(0, c["far"] + 1, (c["rows"],), generator=gen, device="cuda")
        s["pos"] = (start if c["far"] else torch.arange(c["rows"], device="cuda")).to(torch.int32)
    else:
        rows, lens = rows_of(c), lens_of(c)
        s.update(rows=sum(rows), most=max(rows), lens=int32(lens), cu=int32([sum(rows[:i]) for i in range(len(rows) + 1)]))
        groups = c["groups"] if c["op"] == "shared" else len(lens)
        shared = [p // c["page"] for p in prefixes(c)] if c["op"] == "shared" else [0] * groups
        group = [b % groups for b in range(len(lens))]
        s["table"], s["pages"] = tables(gen, s["lens"].long(), shared, group, c["page"])
        s["cache"] = caches(gen, c["layers"], s["pages"], c)
    if c["op"] == "shared":
        # what the program knows of where its sequences came from: each group's first one
        s.update(shared=shared, leader=int32(group) if c["told"] else None, q=normal(c["layers"], s["rows"], c["Hq"], c["D"]))
        s.update(out=torch.zeros_like(s["q"]), plan=torch.zeros(1 << 20, dtype=torch.uint8, device="cuda"))
        s["ws"] = torch.zeros(256 << 20, dtype=torch.uint8, device="cuda")
        return s
    s["freq"] = frequencies(c)
    if c["op"] == "rope":
        s["x"] = normal(c["layers"], c["rows"], c["heads"], c["D"])
        s["y"] = torch.zeros_like(s["x"])
        return s
    hq, hkv, d = c["Hq"], c["Hkv"], c["D"]
    heads = hq + 2 * hkv if c["op"] == "append" else hq + hkv
    # the rows of one projection: queries, keys (and values); tokens of different magnitude, as they come
    size = torch.exp2(torch.randn((c["layers"], s["rows"], heads, 1), generator=gen, device="cuda"))
    s["x"] = (normal(c["layers"], s["rows"], heads, d) * size).to(torch.bfloat16)
    s["wq"], s["wk"] = ((1.0 + 0.2 * normal(d).float()).to(torch.bfloat16) for _ in range(2))
    s["qo"] = torch.zeros((c["layers"], s["rows"], hq, d), dtype=torch.bfloat16, device="cuda")
    if c["op"] == "norm_rope":
        s["ko"] = torch.zeros((c["layers"], s["rows"], hkv, d), dtype=torch.bfloat16, device="cuda")
    return s


# ---- the plain forms -------------------------------------------------------------------------------------------------
def rotate32(c, x, pos, freq, inverse=False):
    """x [rows, heads, D] float32, rotated; angles in 64 bits."""
    angle = pos.double()[:, None] * (-freq if inverse else freq)
    cos, sin = ((f(angle) * mscale(c)).float()[:, None] for f in (torch.cos, torch.sin))
    lo, half, hi = c["first"], c["first"] + c["rot"] // 2, c["first"] + c["rot"]
    if c["interleaved"]:
        a, b = x[..., lo:hi:2], x[..., lo + 1:hi:2]
        turned = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
    else:
        a, b = x[..., lo:half], x[..., half:hi]
        turned = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
    return torch.cat((x[..., :lo], turned, x[..., hi:]), -1)


def norm32(x, w):
    x = x.float()
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.float()


def plain_norm_rope(c, s, layer):
    x, hq, hkv = s["x"][layer], c["Hq"], c["Hkv"]
    s["qo"][layer] = rotate32(c, norm32(x[:, :hq], s["wq"]), s["pos"], s["freq"]).to(torch.bfloat16)
    s["ko"][layer] = rotate32(c, norm32(x[:, hq:], s["wk"]), s["pos"], s["freq"]).to(torch.bfloat16)


def scale32(e):
    return torch.ldexp(torch.ones_like(e, dtype=torch.float32), e.to(torch.int32) - 127)


def values32(codes, e):
    """The values of e4m3 codes [..., x, y] with one scale byte for each leading index."""
    return codes.view(torch.float8_e4m3fn).float() * scale32(e)[..., None, None]


def quantize32(x, old, old_e, fresh):
    """x [blocks, Hkv, page, D] with zeros where there is no new token, and the codes that stay there (old, zeros where
    none), old_e [blocks, Hkv] their scale bytes; fresh [blocks]: the block held nothing. Codes of all and scale bytes."""
    a = x.abs().amax((2, 3)).clamp(min=1e-4)
    m, e = torch.frexp(a)  # a = m 2^e, m in [0.5, 1): a <= 448 2^(e - 9) where m <= 448 / 512
    e = ((e - 9 + (m > 0.875).int()).clamp(max=119) + 127).to(torch.uint8)
    e = torch.where(fresh[:, None], e, torch.maximum(e, old_e))
    moved = torch.ldexp(old.view(torch.float8_e4m3fn).float(), (old_e.int() - e.int())[..., None, None])
    return (moved + (x / scale32(e)[..., None, None]).clamp(-448.0, 448.0)).to(torch.float8_e4m3fn).view(torch.uint8), e


def plain_store(c, s, cache, new, f, e, seq, pos, page, used, where):
    """The rows `new` [rows, Hkv, D] into their slots of cache[f], scales cache[e]."""
    p, first = c["page"], s["lens"].long() - (s["cu"][1:] - s["cu"][:-1]).long()  # tokens that each sequence had
    held = torch.zeros(len(used), dtype=torch.long, device="cuda")  # tokens that stay in each page
    held[where] = (first[seq] - pos // p * p).clamp(min=0)
    for_old = (torch.arange(p, device="cuda") < held[:, None])[:, None, :, None]
    x = torch.zeros((len(used), c["Hkv"], p, c["D"]), device="cuda")
    x[where, :, pos % p] = new.float()
    wide = cache[f][used] if f == "k" else cache[f][used].transpose(2, 3)
    filled = for_old.clone()
    filled[where, :, pos % p] = True
    codes, scale = quantize32(x, torch.where(for_old, wide, 0), cache[e][used], held == 0)
    codes = torch.where(filled, codes, wide)
    cache[f][used] = codes if f == "k" else codes.transpose(2, 3)
    cache[e][used] = scale


def plain_append(c, s, layer):
    hq, hkv, x = c["Hq"], c["Hkv"], s["x"][layer]
    row = torch.arange(s["rows"], dtype=torch.int32, device="cuda")
    seq = torch.searchsorted(s["cu"][1:].contiguous(), row, right=True)
    pos = s["lens"].long()[seq] - s["cu"][1:].long()[seq] + row
    s["qo"][layer] = rotate32(c, norm32(x[:, :hq], s["wq"]), pos, s["freq"]).to(torch.bfloat16)
    k = rotate32(c, norm32(x[:, hq:hq + hkv], s["wk"]), pos, s["freq"]).to(torch.bfloat16)
    page = s["table"].long()[seq, pos // c["page"]]
    used, where = torch.unique(page, return_inverse=True)
    cache = {f: s["cache"][f][layer] for f in ("k", "v", "ks", "vs")}
    plain_store(c, s, cache, k, "k", "ks", seq, pos, page, used, where)
    plain_store(c, s, cache, x[:, hq + hkv:], "v", "vs", seq, pos, page, used, where)


def plain_shared(c, s, layer):
    """The common blocks of each group in one product with all of its rows, the other blocks sequence by sequence, and one
    softmax over both."""
    G, S, n, hkv, g, d, p = c["groups"], c["each"], c["n"], c["Hkv"], c["Hq"] // c["Hkv"], c["D"], c["page"]
    slot = torch.arange(G * S, device="cuda").view(S, G).t()  # [G, S]
    row = s["cu"][:-1].long()[slot][..., None] + torch.arange(n, device="cuda")  # [G, S, n]
    pos = (s["lens"].long() - n)[slot][..., None] + torch.arange(n, device="cuda")
    x = s["q"][layer][row].float().view(G, S, n, hkv, g, d).permute(0, 3, 1, 2, 4, 5) * d ** -0.5  # [G, hkv, S, n, g, d]
    shared, table = torch.tensor(s["shared"], device="cuda"), s["table"].clamp(min=0).long()
    k, v, ks, vs = (s["cache"][f][layer] for f in ("k", "v", "ks", "vs"))

    at = table[:G, :max(s["shared"] + [1])]  # sequence b < G is one of group b
    t = at.shape[1] * p
    w1 = torch.matmul(x.reshape(G, hkv, -1, d), values32(k[at], ks[at]).permute(0, 2, 4, 1, 3).reshape(G, hkv, d, t))
    w1.masked_fill_((torch.arange(t, device="cuda") >= shared[:, None] * p)[:, None, None], -math.inf)
    blk = shared[:, None] + torch.arange(int((table.shape[1] - shared).max()), device="cuda")  # [G, own blocks]
    mine = table[slot[..., None], blk.clamp(max=table.shape[1] - 1)[:, None]]  # [G, S, own blocks]
    u = mine.shape[2] * p
    own_k = values32(k[mine], ks[mine]).permute(0, 1, 3, 5, 2, 4).reshape(G, S, hkv, d, u)
    w2 = torch.matmul(x.permute(0, 2, 1, 3, 4, 5).reshape(G, S, hkv, n * g, d), own_k).view(G, S, hkv, n, g, u)
    token = (blk[..., None] * p + torch.arange(p, device="cuda")).view(G, u)
    w2.masked_fill_((token[:, None, None] > pos[..., None])[:, :, None, :, None], -math.inf)
    top = torch.maximum(w1.amax(-1).view(G, hkv, S, n, g).permute(0, 2, 1, 3, 4), w2.amax(-1))  # [G, S, hkv, n, g]
    w1 = w1.sub_(top.permute(0, 2, 1, 3, 4).reshape(G, hkv, -1, 1)).exp_()
    w2 = w2.sub_(top[..., None]).exp_()
    total = w1.sum(-1).view(G, hkv, S, n, g).permute(0, 2, 1, 3, 4) + w2.sum(-1)
    y = torch.matmul(w1, values32(v[at], vs[at]).permute(0, 2, 1, 4, 3).reshape(G, hkv, t, d))
    own_v = values32(v[mine], vs[mine]).permute(0, 1, 3, 2, 5, 4).reshape(G, S, hkv, u, d)
    y2 = torch.matmul(w2.view(G, S, hkv, n * g, u), own_v).view(G, S, hkv, n, g, d)
    y = (y.view(G, hkv, S, n, g, d).permute(0, 2, 1, 3, 4, 5) + y2) / total[..., None]
    s["out"][layer][row] = y.permute(0, 1, 3, 2, 4, 5).reshape(G, S, n, -1, d).to(torch.bfloat16)


def plain_layer(c, s, layer):
    if c["op"] == "rope":
        s["y"][layer] = rotate32(c, s["x"][layer].float(), s["pos"], s["freq"], c["inverse"]).to(torch.bfloat16)
    else:
        {"norm_rope": plain_norm_rope, "append": plain_append, "shared": plain_shared}[c["op"]](c, s, layer)


# ---- the library's calls ---------------------------------------------------------------------------------------------
_stream = None


def stream():
    """The stream that steps are captured on. Nothing runs there: a captured step is replayed on torch's current stream."""
    global _stream
    if _stream is None:
        from unholy_amd.device import Stream
        _stream = Stream()
    return _stream


def own_turn(c, s):
    return s["freq"].data_ptr(), c["first"], c["rot"], int(c["interleaved"]), mscale(c)


def own_layers(s, st):
    from unholy_amd import call
    c = s["case"]
    if c["op"] == "rope":
        ld = c["heads"] * c["D"]
        for i in range(c["layers"]):
            call("uh_rope", s["x"][i].data_ptr(), ld, s["y"][i].data_ptr(), ld, s["pos"].data_ptr(), s["rows"], c["heads"],
                 c["D"], *own_turn(c, s), int(c["inverse"]), st)
        return
    hq, hkv, d = c["Hq"], c["Hkv"], c["D"]
    if c["op"] == "norm_rope":
        ld = (hq + hkv) * d
        for i in range(c["layers"]):
            q = s["x"][i].data_ptr()
            call("uh_qk_norm_rope", q, ld, s["qo"][i].data_ptr(), hq * d, hq, s["wq"].data_ptr(), q + 2 * hq * d, ld,
                 s["ko"][i].data_ptr(), hkv * d, hkv, s["wk"].data_ptr(), EPS, s["pos"].data_ptr(), s["rows"], d,
                 *own_turn(c, s), st)
        return
    b = len(s["lens"])
    step = (s["cu"].data_ptr(), s["rows"], s["most"], s["lens"].data_ptr(), s["table"].data_ptr(), s["table"].shape[1], b)
    shape = (s["pages"], c["page"])
    if c["op"] == "append":
        ld = (hq + 2 * hkv) * d
        for i in range(c["layers"]):
            q, cache = s["x"][i].data_ptr(), [s["cache"][f][i].data_ptr() for f in ("k", "v", "ks", "vs")]
            call("uh_kv_append_rope", q, ld, s["qo"][i].data_ptr(), hq * d, hq, s["wq"].data_ptr(), q + 2 * hq * d, ld,
                 s["wk"].data_ptr(), EPS, q + 2 * (hq + hkv) * d, ld, *step, *own_turn(c, s), *cache, *shape, hkv, d, st)
        return
    plan = (s["plan"].data_ptr(), s["plan"].numel())
    leader = None if s["leader"] is None else s["leader"].data_ptr()
    call("uh_kv_share", leader, *step, *shape, *plan, st)
    ld = hq * d
    for i in range(c["layers"]):
        cache = [s["cache"][f][i].data_ptr() for f in ("k", "v", "ks", "vs")]
        call("uh_kv_attend_shared", s["q"][i].data_ptr(), ld, *step, *cache, *shape, hq, hkv, d, d ** -0.5, 0, 0,
             s["out"][i].data_ptr(), ld, None, *plan, s["ws"].data_ptr(), s["ws"].numel(), st)


def own_step(s):
    """A step through the layers: call by call the first time, and captured then where the program replays it in the next
    ones. All of it runs on torch's current stream, so that it comes after what writes its inputs, zeroes its workspace or
    used their memory before, and what reads its results, or is given its memory, comes after it."""
    from unholy_amd import call
    now = torch.cuda.current_stream().cuda_stream
    if s["graph"] is not None:
        call("uh_graph_launch", s["graph"].handle, now)
        return
    own_layers(s, now)
    if s["case"]["graph"]:
        from unholy_amd.device import Graph
        s["graph"] = Graph(stream(), lambda: own_layers(s, stream().handle))


def run(state):
    s, c = state, state["case"]
    if own:
        own_step(s)
    else:
        for layer in range(c["layers"]):
            plain_layer(c, s, layer)
    if c["op"] == "rope":
        return s["y"]
    if c["op"] == "shared":
        return s["out"]
    if c["op"] == "norm_rope":
        return {"q": s["qo"], "k": s["ko"]}
    return {"q": s["qo"], "k": s["cache"]["k"].view(torch.float8_e4m3fn), "v": s["cache"]["v"].view(torch.float8_e4m3fn),
            "ks": s["cache"]["ks"].view(torch.float8_e8m0fnu), "vs": s["cache"]["vs"].view(torch.float8_e8m0fnu)}


# ---- what a pass cannot do without -----------------------------------------------------------------------------------
def work(case):
    c = case
    if c["op"] in ("rope", "norm_rope"):
        heads = c["heads"] if c["op"] == "rope" else c["Hq"] + c["Hkv"]
        values = c["rows"] * heads * c["D"]
        small = 4.0 * c["rows"] + 4.0 * c["rot"]  # positions, frequencies
        return {"bytes": c["layers"] * (4.0 * values + small),
                "flops": c["layers"] * c["rows"] * heads * (3.0 * c["rot"] + (4.0 * c["D"] if c["op"] == "norm_rope" else 0.0))}
    token = c["Hkv"] * 2 * (c["D"] + 2 / c["page"])  # a token's codes and its share of the scales
    n = sum(rows_of(c))
    if c["op"] == "append":
        values = c["Hq"] + 2.0 * c["Hkv"]
        return {"bytes": c["layers"] * n * (2.0 * values * c["D"] + 2.0 * c["Hq"] * c["D"] + token),
                "flops": c["layers"] * n * c["D"] * (7.0 * (c["Hq"] + c["Hkv"]) + 4.0 * c["Hkv"])}
    pre = [x // c["page"] * c["page"] for x in prefixes(c)]
    lens = lens_of(c)
    read = sum(pre) + sum(lens) - c["each"] * sum(pre)
    pairs = sum(c["n"] * x - c["n"] * (c["n"] - 1) / 2 for x in lens)
    values = 1.0 * c["Hq"] * c["D"]
    return {"bytes": c["layers"] * (read * token + 4.0 * n * values), "flops": c["layers"] * pairs * 4.0 * values}


# ---- the same in 64 bits ---------------------------------------------------------------------------------------------
def exact(case, seed):
    c, s = case, prepare(case, seed)

    def turned(x, pos):
        """x [rows, heads, D], its pairs as complex numbers times e^(i angle)."""
        part = x[..., c["first"]:c["first"] + c["rot"]].double()
        if c["interleaved"]:
            z = torch.view_as_complex(part.unflatten(-1, (-1, 2)).contiguous())
        else:
            z = torch.complex(*part.chunk(2, -1))
        angle = torch.outer(pos.double(), s["freq"])
        z = z * torch.polar(torch.full_like(angle, mscale(c)), -angle if c.get("inverse") else angle)[:, None]
        y = x.double().clone()
        z = torch.view_as_real(z).flatten(-2) if c["interleaved"] else torch.cat((z.real, z.imag), -1)
        y[..., c["first"]:c["first"] + c["rot"]] = z
        return y

    def normed(x, w):
        return x.double() / (x.double().square().sum(-1, keepdim=True) / c["D"] + EPS).sqrt() * w.double()

    if c["op"] == "rope":
        return torch.stack([turned(x, s["pos"]) for x in s["x"]])
    if c["op"] == "norm_rope":
        return {"q": torch.stack([turned(normed(x[:, :c["Hq"]], s["wq"]), s["pos"]) for x in s["x"]]),
                "k": torch.stack([turned(normed(x[:, c["Hq"]:], s["wk"]), s["pos"]) for x in s["x"]])}
    cache, p, hq, hkv, d = s["cache"], c["page"], c["Hq"], c["Hkv"], c["D"]
    double = {"k": cache["k"].view(torch.float8_e4m3fn).double(), "v": cache["v"].view(torch.float8_e4m3fn).double(),
              "ks": cache["ks"].view(torch.float8_e8m0fnu).double(), "vs": cache["vs"].view(torch.float8_e8m0fnu).double()}
    cu, lens, table = s["cu"].tolist(), s["lens"].tolist(), s["table"]
    if c["op"] == "shared":
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        for layer in range(c["layers"]):
            for b in range(len(lens)):
                n, t = cu[b + 1] - cu[b], lens[b]
                at = table[b, : -(-t // p)].long()
                k = (double["k"][layer][at] * double["ks"][layer][at][:, :, None, None]).permute(1, 0, 2, 3)
                v = (double["v"][layer][at] * double["vs"][layer][at][:, :, None, None]).permute(1, 0, 3, 2)
                k, v = (x.reshape(hkv, -1, d)[:, :t].contiguous() for x in (k, v))
                hidden = torch.arange(t, device="cuda") > torch.arange(t - n, t, device="cuda")[:, None]
                x = s["q"][layer, cu[b]:cu[b + 1]].double().unflatten(1, (hkv, -1)).permute(1, 2, 0, 3)  # [hkv, g, n, d]
                w = torch.matmul(x.flatten(1, 2), k.transpose(1, 2).contiguous()).unflatten(1, (-1, n)) / math.sqrt(d)
                y = torch.matmul(torch.softmax(w.masked_fill(hidden, -math.inf), -1).flatten(1, 2), v)
                out[layer, cu[b]:cu[b + 1]] = y.unflatten(1, (-1, n)).permute(2, 0, 1, 3).flatten(1, 2)
        return out

    def e4m3(x):
        """Nearest e4m3 value, ties to even: steps of 2^-9 up to 2^-6, of an eighth of the power of two above."""
        step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
        return torch.round(x / step) * step

    pos = torch.cat([torch.arange(lens[b] - (cu[b + 1] - cu[b]), lens[b], device="cuda") for b in range(len(lens))])
    queries = []
    for layer in range(c["layers"]):
        x = s["x"][layer]
        queries.append(turned(normed(x[:, :hq], s["wq"]), pos))
        keys = turned(normed(x[:, hq:hq + hkv], s["wk"]), pos).to(torch.bfloat16)
        for b in range(len(lens)):
            had = lens[b] - (cu[b + 1] - cu[b])
            for block in range(had // p, -(-lens[b] // p)):
                lo, hi = max(had, block * p), min(lens[b], block * p + p)
                rows, page = slice(cu[b] + lo - had, cu[b] + hi - had), int(table[b, block])
                kept, put = slice(0, lo - block * p), slice(lo - block * p, hi - block * p)
                for new, f, e in ((keys, "k", "ks"), (x[:, hq + hkv:], "v", "vs")):
                    y = new[rows].double()  # [tokens, Hkv, D]
                    scale = torch.exp2(torch.ceil(torch.log2(y.abs().amax((0, 2)).clamp(min=1e-4) / 448)).clamp(max=119))
                    codes = double[f][layer, page] if f == "k" else double[f][layer, page].transpose(1, 2)
                    if lo > block * p:
                        old = double[e][layer, page]
                        scale = torch.maximum(scale, old)
                        codes[:, kept] = e4m3(codes[:, kept] * (old / scale)[:, None, None])
                    codes[:, put] = e4m3((y.transpose(0, 1) / scale[:, None, None]).clamp(-448, 448))
                    double[e][layer, page] = scale
    return {"q": torch.stack(queries), **double}

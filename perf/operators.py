"""The 8-bit paged key / value cache: what writes it, reads it and manages its pages, in plain torch and by this library.

One layer's cache holds pages of `page` tokens. Per page and key / value head: e4m3 codes of the keys [page, D], e4m3
codes of the values [D, page] (transposed), and a power-of-two scale (e8m0) for each of the two. Position t of sequence b
lies in slot t % page of page table[b][t // page]. Sequence b brings rows cu[b] .. cu[b + 1] of a step; lens[b] counts its
tokens, the new ones included, so that row i of its n has position lens[b] - n + i.

- append: the new rows' keys and values quantized into their pages. A block's scale is the smallest power of two that
  fits its tokens; where earlier tokens of the sequence are in the block it only grows, and their codes move with it.
- attend: causal softmax attention of the new rows over their sequences' cached tokens, for query heads that share
  key / value heads; with `window`, over the last `window` tokens and the first `sinks` ones.
- fork: sequences that are given up, new ones that share another's pages, and pages for their next tokens, with a copy
  of a page that is shared and not full.
- compact: the pages in use moved to the lowest numbers, with the tables that name them.
"""
import math

import torch

own = False


def listed():
    gqa = {"Hq": 32, "Hkv": 8, "D": 128, "page": 64, "window": 0, "sinks": 0}
    return [
        # Single-user generation: one token, one sequence, through the layers of a model; latency and launches.
        {"name": "attend_decode_1", "op": "attend", "B": 1, "n": 1, "chunk": 0, "ctx_lo": 4096, "ctx_hi": 4096, **gqa,
         "layers": 16, "graph": True},
        # An ordinary serving batch: sequences of every length up to 8k, one token each.
        {"name": "attend_decode_64", "op": "attend", "B": 64, "n": 1, "chunk": 0, "ctx_lo": 0, "ctx_hi": 8190, **gqa,
         "layers": 1, "graph": False},
        # A few very long contexts; twelve query heads for each key / value head.
        {"name": "attend_decode_long", "op": "attend", "B": 4, "n": 1, "chunk": 0, "ctx_lo": 90001, "ctx_hi": 131070,
         "Hq": 96, "Hkv": 8, "D": 128, "page": 128, "window": 0, "sinks": 0, "layers": 1, "graph": False},
        # Speculative verification: five draft tokens a sequence.
        {"name": "attend_verify_16", "op": "attend", "B": 16, "n": 5, "chunk": 0, "ctx_lo": 700, "ctx_hi": 5000, "Hq": 32,
         "Hkv": 4, "D": 128, "page": 32, "window": 0, "sinks": 0, "layers": 4, "graph": True},
        # The largest prompt chunk from scratch.
        {"name": "attend_prefill_8192", "op": "attend", "B": 1, "n": 8192, "chunk": 0, "ctx_lo": 0, "ctx_hi": 0, **gqa,
         "layers": 1, "graph": False},
        # A step that mixes decode rows with a chunk of one long prompt.
        {"name": "attend_mixed_9", "op": "attend", "B": 9, "n": 1, "chunk": 1000, "ctx_lo": 900, "ctx_hi": 4003, **gqa,
         "layers": 1, "graph": False},
        # Long contexts under a window with four sinks, small heads and small pages.
        {"name": "window_decode_32", "op": "attend", "B": 32, "n": 1, "chunk": 0, "ctx_lo": 10, "ctx_hi": 30000, "Hq": 64,
         "Hkv": 8, "D": 64, "page": 16, "window": 1024, "sinks": 4, "layers": 4, "graph": True},
        # A long prompt under the same kind of window.
        {"name": "window_prefill_7001", "op": "attend", "B": 1, "n": 7001, "chunk": 0, "ctx_lo": 1000, "ctx_hi": 1000,
         "Hq": 32, "Hkv": 4, "D": 64, "page": 64, "window": 1024, "sinks": 4, "layers": 1, "graph": False},
        # One token of each sequence of a batch into its layers' caches.
        {"name": "append_decode_64", "op": "append", "B": 64, "n": 1, "chunk": 0, "ctx_lo": 1, "ctx_hi": 500, "Hkv": 8,
         "D": 128, "page": 64, "layers": 8, "graph": True},
        # Three prompts of different lengths.
        {"name": "append_prompt_3", "op": "append", "B": 3, "n": 2001, "chunk": 8000, "ctx_lo": 0, "ctx_hi": 90, "Hkv": 8,
         "D": 128, "page": 64, "layers": 1, "graph": False},
        # Parallel sampling: half of the slots are started again from the other half and go on by a few tokens.
        {"name": "fork_64", "op": "fork", "B": 64, "grow": 3, "ctx_lo": 100, "ctx_hi": 2000, "Hkv": 8, "D": 128,
         "page": 64, "layers": 16},
        # A pool after many sequences have come and gone.
        {"name": "compact_4096", "op": "compact", "B": 40, "pages": 4096, "live": 2400, "Hkv": 8, "D": 128, "page": 64,
         "layers": 4},
    ]


def draw(rng):
    def log(lo, hi):
        return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))

    op = rng.choice(["attend"] * 4 + ["window"] * 2 + ["append"] * 2 + ["fork", "compact"])
    d, page = rng.choice([64, 128, 128, 256]), rng.choice([16, 32, 64, 64, 128])
    hkv = rng.choice([1, 2, 4, 8])
    if op in ("attend", "window"):
        hq = hkv * rng.choice([1, 3, 4, 7, 8, 12, 16])
        window, sinks = (log(16, 4096), rng.choice([0, 1, 4, 64])) if op == "window" else (0, 0)
        kind = rng.choice(["decode", "decode", "verify", "prefill", "mixed"])
        if kind in ("decode", "verify"):
            b, n, chunk = log(1, 128), 1 if kind == "decode" else rng.randint(2, 9), 0
            most = min(131072, (1 << 28) // (b * hkv * d), (1 << 26) // (b * n * hq))
        else:
            b = log(1, 4) if kind == "prefill" else log(2, 12)
            rows = log(16, min(4096, math.isqrt((1 << 29) // (b * hq))))
            n, chunk = (rows, 0) if kind == "prefill" else (1, rows)
            most = min(16384, (1 << 30) // (b * rows * hq) - rows)
        hi = log(16, max(16, most))
        return {"op": "attend", "B": b, "n": n, "chunk": chunk, "ctx_lo": rng.randint(0, hi), "ctx_hi": hi, "Hq": hq,
                "Hkv": hkv, "D": d, "page": page, "window": window, "sinks": sinks,
                "layers": 4 if b * n < 64 and not chunk else 1, "graph": n < 10 and not chunk}
    if op == "append":
        decode = rng.random() < 0.5
        b = log(1, 256) if decode else log(1, 6)
        return {"op": op, "B": b, "n": 1 if decode else log(2, 3000), "chunk": 0 if decode else log(2, 5000),
                "ctx_lo": rng.randint(0, 60), "ctx_hi": log(60, 600), "Hkv": hkv, "D": d, "page": page,
                "layers": 8 if decode else 1, "graph": decode}
    if op == "fork":
        return {"op": op, "B": 2 * log(1, 64), "grow": rng.randint(1, 200), "ctx_lo": rng.randint(1, 100),
                "ctx_hi": log(100, 4000), "Hkv": hkv, "D": d, "page": page, "layers": rng.randint(1, 16)}
    pages = log(64, 4096)
    return {"op": op, "B": min(pages // 8, log(1, 64)), "pages": pages, "live": rng.randint(pages // 4, pages * 3 // 4),
            "Hkv": hkv, "D": d if page < 128 else 128, "page": page, "layers": rng.randint(1, 4)}


# ---- sizes -----------------------------------------------------------------------------------------------------------
def spread(b, lo, hi):
    """b lengths over lo .. hi, both ends of the range among them for a large b."""
    return [hi if b == 1 else lo + int((i * 0.6180339887 + 0.999) % 1.0 * (hi - lo + 0.999)) for i in range(b)]


def rows_of(c):
    return [c["chunk"]] + [c["n"]] * (c["B"] - 1) if c["chunk"] else [c["n"]] * c["B"]


def lens_of(c):
    return [a + n for a, n in zip(spread(c["B"], c["ctx_lo"], c["ctx_hi"]), rows_of(c))]


def shares(total, b):
    """`total` pages over b sequences, unequal and each with one at least."""
    at = [total * i * i // (b * b) for i in range(b)] + [total]
    at = [max(x, i) for i, x in enumerate(at)]
    return [y - x for x, y in zip(at, at[1:])]


# ---- inputs ----------------------------------------------------------------------------------------------------------
def int32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


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


def tables(gen, blocks, pages, width):
    """A table of `width` entries a sequence: blocks[b] pages for sequence b in no order, then -1; and the pages' uses."""
    take = torch.randperm(pages, generator=gen, device="cuda")[: sum(blocks)].to(torch.int32)
    table = torch.full((len(blocks), width), -1, dtype=torch.int32, device="cuda")
    at = torch.arange(width, device="cuda")[None, :] < int32(blocks)[:, None]
    table[at] = take
    refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
    refs[take.long()] = 1
    return table, refs


def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    if c["op"] in ("attend", "append"):
        rows, lens = rows_of(c), lens_of(c)
        blocks = [-(-n // c["page"]) for n in lens]
        pages, total = sum(blocks) + 3, sum(rows)
        table, _ = tables(gen, blocks, pages, max(blocks) + 1)
        s = {"case": c, "pages": pages, "rows": total, "most": max(rows), "table": table, "lens": int32(lens),
             "cu": int32([sum(rows[:i]) for i in range(len(rows) + 1)]), "cache": caches(gen, c["layers"], pages, c),
             "graph": None}

        def normal(*shape):
            return torch.randn((c["layers"], total) + shape, generator=gen, device="cuda").to(torch.bfloat16)

        if c["op"] == "attend":
            s["q"], s["out"] = normal(c["Hq"], c["D"]), torch.zeros_like(normal(c["Hq"], c["D"]))
            s["ws"] = torch.zeros(128 << 20, dtype=torch.uint8, device="cuda")
        else:  # tokens of different magnitude, as they come; some of them make a block's scale grow
            size = torch.exp2(torch.randn((c["layers"], total, c["Hkv"], 1), generator=gen, device="cuda"))
            s["knew"], s["vnew"] = ((normal(c["Hkv"], c["D"]) * size).to(torch.bfloat16) for _ in range(2))
        return s
    if c["op"] == "fork":
        b = c["B"]
        lens = spread(b // 2, c["ctx_lo"], c["ctx_hi"]) + [0] * (b // 2)
        blocks = [-(-n // c["page"]) for n in lens]
        width = max(blocks) + -(-c["grow"] // c["page"]) + 1
        pages = sum(blocks) + b * (2 + c["grow"] // c["page"])
        table, refs = tables(gen, blocks, pages, width)
        parents = torch.randperm(b // 2, generator=gen, device="cuda").to(torch.int32)
        none = torch.full_like(parents, -1)
        return {"case": c, "pages": pages, "table": table, "refs": refs, "lens": int32(lens),
                "cache": caches(gen, c["layers"], pages, c), "keep": int32(lens), "from": torch.cat((none, parents)),
                "grow": int32([0] * (b // 2) + [c["grow"]] * (b // 2)), "ok": int32([0] * b), "done": int32([0] * b),
                "ws": torch.zeros(16 << 20, dtype=torch.uint8, device="cuda")}
    blocks = shares(c["live"], c["B"])
    table, refs = tables(gen, blocks, c["pages"], max(blocks) + 1)
    return {"case": c, "pages": c["pages"], "table": table, "refs": refs, "table_out": torch.zeros_like(table),
            "refs_out": torch.zeros_like(refs), "live": int32([0]), "cache": caches(gen, c["layers"], c["pages"], c),
            "ws": torch.zeros(16 << 20, dtype=torch.uint8, device="cuda")}


# ---- the plain forms -------------------------------------------------------------------------------------------------
def scale32(e):
    return torch.ldexp(torch.ones_like(e, dtype=torch.float32), e.to(torch.int32) - 127)


def values32(codes, e):
    """The values of e4m3 codes [..., x, y] with one scale byte for each leading index."""
    return codes.view(torch.float8_e4m3fn).float() * scale32(e)[..., None, None]


def plain_attend(c, s, layer):
    q, hkv, d, p = s["q"][layer], c["Hkv"], c["D"], c["page"]
    b, g, most, dev = c["B"], c["Hq"] // c["Hkv"], s["most"], q.device
    n = (s["cu"][1:] - s["cu"][:-1]).long()
    i = torch.arange(most, device=dev)
    row = (s["cu"][:-1].long()[:, None] + i).clamp(max=q.shape[0] - 1)  # [b, most]
    live = i < n[:, None]
    x = q[row].float().view(b, most, hkv, g, d).permute(0, 2, 3, 1, 4).reshape(b, hkv, g * most, d)
    at = s["table"].clamp(min=0).long()
    t = at.shape[1] * p
    k, v, ks, vs = (s["cache"][f][layer][at] for f in ("k", "v", "ks", "vs"))
    k = values32(k, ks).permute(0, 2, 4, 1, 3).reshape(b, hkv, d, t)
    w = torch.matmul(x, k) * d ** -0.5
    del k
    pos = (s["lens"].long() - n)[:, None, None] + i[:, None]  # [b, most, 1]
    far = pos - torch.arange(t, device=dev)
    seen = (far >= 0) & (s["table"] >= 0).repeat_interleave(p, 1)[:, None, :]
    if c["window"]:
        seen &= (far < c["window"]) | (torch.arange(t, device=dev) < c["sinks"])
    w = w.view(b, hkv, g, most, t).masked_fill_(~seen[:, None, None], -math.inf)
    top = w.amax(-1, keepdim=True)
    w = w.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = w.sum(-1, keepdim=True).view(b, hkv, g * most, 1)
    v = values32(v, vs).permute(0, 2, 1, 4, 3).reshape(b, hkv, t, d)
    y = torch.matmul(w.view(b, hkv, g * most, t), v)
    y = torch.where(total > 0, y / total, 0.0).view(b, hkv, g, most, d).permute(0, 3, 1, 2, 4).reshape(b, most, -1, d)
    out = s["out"][layer]
    out[row[live]] = y[live].to(torch.bfloat16)
    return out


def quantize32(x, old, old_e, fresh):
    """x [blocks, Hkv, page, D] with zeros where there is no new token, and the codes that stay there (old, zeros where
    none), old_e [blocks, Hkv] their scale bytes; fresh [blocks]: the block held nothing. Codes of all and scale bytes."""
    a = x.abs().amax((2, 3)).clamp(min=1e-4)
    m, e = torch.frexp(a)  # a = m 2^e, m in [0.5, 1): a <= 448 2^(e - 9) where m <= 448 / 512
    e = ((e - 9 + (m > 0.875).int()).clamp(max=119) + 127).to(torch.uint8)
    e = torch.where(fresh[:, None], e, torch.maximum(e, old_e))
    moved = torch.ldexp(old.view(torch.float8_e4m3fn).float(), (old_e.int() - e.int())[..., None, None])
    return (moved + (x / scale32(e)[..., None, None]).clamp(-448.0, 448.0)).to(torch.float8_e4m3fn).view(torch.uint8), e


def plain_append(c, s, layer):
    p, hkv, d = c["page"], c["Hkv"], c["D"]
    dev, cache = s["cu"].device, {f: s["cache"][f][layer] for f in ("k", "v", "ks", "vs")}
    total = s["rows"]
    seq = torch.searchsorted(s["cu"][1:].contiguous(), torch.arange(total, dtype=torch.int32, device=dev), right=True)
    pos = s["lens"].long()[seq] - s["cu"][1:].long()[seq] + torch.arange(total, device=dev)
    page = s["table"].long()[seq, pos // p]
    first = s["lens"].long() - (s["cu"][1:] - s["cu"][:-1]).long()  # tokens that each sequence had
    used, where = torch.unique(page, return_inverse=True)
    held = torch.zeros(len(used), dtype=torch.long, device=dev)  # tokens that stay in each page
    held[where] = (first[seq] - pos // p * p).clamp(min=0)
    for_old = (torch.arange(p, device=dev) < held[:, None])[:, None, :, None]
    for new, f, e in ((s["knew"][layer], "k", "ks"), (s["vnew"][layer], "v", "vs")):
        x = torch.zeros((len(used), hkv, p, d), device=dev)
        x[where, :, pos % p] = new.float()
        wide = cache[f][used] if f == "k" else cache[f][used].transpose(2, 3)
        filled = for_old.clone()
        filled[where, :, pos % p] = True
        codes, scale = quantize32(x, torch.where(for_old, wide, 0), cache[e][used], held == 0)
        codes = torch.where(filled, codes, wide)
        cache[f][used] = codes if f == "k" else codes.transpose(2, 3)
        cache[e][used] = scale
    return cache


def plain_free(s):
    page = s["case"]["page"]
    left = torch.minimum(s["lens"], s["keep"].clamp(min=0))
    block = torch.arange(s["table"].shape[1], device="cuda")
    gone = (block >= ((left + page - 1) // page)[:, None]) & (s["table"] >= 0)
    s["refs"].index_add_(0, s["table"][gone].long(), torch.full_like(s["table"][gone], -1))
    s["table"].masked_fill_(gone, -1)
    s["lens"].copy_(left)


def plain_fork(s):
    src = s["from"].long()
    done = (s["lens"] == 0) & (src >= 0) & (src < len(src)) & (s["lens"][src.clamp(0, len(src) - 1)] > 0)
    shared = s["table"][src.clamp(0, len(src) - 1)][done]
    s["table"][done], s["lens"][done] = shared, s["lens"][src[done]]
    s["refs"].index_add_(0, shared[shared >= 0].long(), torch.ones_like(shared[shared >= 0]))
    s["done"].copy_(done)


def plain_reserve(s):
    page, table, refs, lens = s["case"]["page"], s["table"], s["refs"], s["lens"]
    grow, slot = s["grow"].clamp(min=0), torch.arange(len(lens), device="cuda")
    held, wanted = (lens + page - 1) // page, (lens + grow + page - 1) // page
    tail = table[slot, (held - 1).clamp(min=0).long()].clamp(min=0).long()
    copied = (grow > 0) & (lens % page != 0) & (refs[tail] > 1)
    fits = wanted <= table.shape[1]
    need = torch.where(fits, wanted - held + copied, 0)
    upto = torch.cumsum(need, 0)
    free = torch.sort((refs != 0).int(), stable=True).indices.int()
    ok = fits & ((upto <= (refs == 0).sum()) | (need == 0))
    copied &= ok
    begin = upto - need
    block = torch.arange(table.shape[1], device="cuda")[None, :]
    new = ok[:, None] & (block >= held[:, None]) & (block < wanted[:, None])
    which = (begin + copied)[:, None] + block - held[:, None]
    pages = free[which[new].long()]
    to = free[begin[copied].long()]
    for x in s["cache"].values():
        x[:, to.long()] = x[:, tail[copied]]
    refs.index_add_(0, tail[copied], torch.full_like(to, -1))
    refs[pages.long()], refs[to.long()] = 1, 1
    table[new] = pages
    table[slot[copied], (held - 1)[copied].long()] = to
    lens += torch.where(ok, grow, 0)
    s["ok"].copy_(ok)


def plain_compact(s):
    refs, used = s["refs"], s["refs"] > 0
    live, page = used.sum(), torch.arange(len(refs), device="cuda")
    src, dst = page[used & (page >= live)], page[~used & (page < live)]
    for x in s["cache"].values():
        x[:, dst] = x[:, src]
    to = page.clone()
    to[src] = dst
    s["table_out"].copy_(torch.where(s["table"] >= 0, to[s["table"].clamp(min=0).long()].int(), -1))
    s["refs_out"].copy_(refs)
    s["refs_out"][dst] = refs[src]
    s["refs_out"][src] = 0
    s["live"].copy_(live[None])


# ---- the library's calls ---------------------------------------------------------------------------------------------
_stream = None


def stream():
    """The stream that steps are captured on. Nothing runs there: a captured step is replayed on torch's current stream."""
    global _stream
    if _stream is None:
        from unholy_amd.device import Stream
        _stream = Stream()
    return _stream


def arrays(s, layer=None):
    return [(s["cache"][f] if layer is None else s["cache"][f][layer]).data_ptr() for f in ("k", "v", "ks", "vs")]


def own_layers(s, st):
    from unholy_amd import call
    c, b = s["case"], s["case"]["B"]
    cu, lens, table, width = s["cu"].data_ptr(), s["lens"].data_ptr(), s["table"].data_ptr(), s["table"].shape[1]
    shape = (s["pages"], c["page"])
    if c["op"] == "append":
        ld = c["Hkv"] * c["D"]
        for i in range(c["layers"]):
            call("uh_kv_append", s["knew"][i].data_ptr(), ld, s["vnew"][i].data_ptr(), ld, cu, s["rows"], s["most"], lens,
                 table, width, b, *arrays(s, i), *shape, c["Hkv"], c["D"], st)
        return
    ld = c["Hq"] * c["D"]
    for i in range(c["layers"]):
        call("uh_kv_attend", s["q"][i].data_ptr(), ld, cu, s["rows"], s["most"], lens, table, width, b, *arrays(s, i),
             *shape, c["Hq"], c["Hkv"], c["D"], c["D"] ** -0.5, c["window"], c["sinks"], s["out"][i].data_ptr(), ld, None,
             s["ws"].data_ptr(), s["ws"].numel(), st)


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


def own_pages(s):
    from unholy_amd import call
    c, st = s["case"], torch.cuda.current_stream().cuda_stream
    shape = (c["layers"], s["pages"], c["page"], c["Hkv"], c["D"])
    ws, width = (s["ws"].data_ptr(), s["ws"].numel()), s["table"].shape[1]
    if c["op"] == "compact":
        call("uh_kv_compact", s["table"].data_ptr(), s["table_out"].data_ptr(), width, c["B"], s["refs"].data_ptr(),
             s["refs_out"].data_ptr(), *arrays(s), *shape, s["live"].data_ptr(), *ws, st)
        return
    seqs = (s["table"].data_ptr(), width, s["lens"].data_ptr())
    pool = (s["refs"].data_ptr(), s["pages"], c["page"])
    call("uh_kv_free", *seqs, s["keep"].data_ptr(), c["B"], *pool, st)
    call("uh_kv_fork", *seqs, s["from"].data_ptr(), c["B"], *pool, s["done"].data_ptr(), st)
    call("uh_kv_reserve", *seqs, s["grow"].data_ptr(), c["B"], s["refs"].data_ptr(), *arrays(s), *shape,
         s["ok"].data_ptr(), *ws, st)


def own_run(s):
    (own_step if s["case"]["op"] in ("attend", "append") else own_pages)(s)


def plain_run(s):
    c = s["case"]
    if c["op"] == "attend":
        return [plain_attend(c, s, i) for i in range(c["layers"])]
    if c["op"] == "append":
        return [plain_append(c, s, i) for i in range(c["layers"])]
    return plain_compact(s) if c["op"] == "compact" else [plain_free(s), plain_fork(s), plain_reserve(s)]


def run(state):
    s, op = state, state["case"]["op"]
    if own:
        own_run(s)
    else:
        plain_run(s)
    if op == "attend":
        return s["out"]
    cache = {"k": s["cache"]["k"].view(torch.float8_e4m3fn), "v": s["cache"]["v"].view(torch.float8_e4m3fn),
             "ks": s["cache"]["ks"].view(torch.float8_e8m0fnu), "vs": s["cache"]["vs"].view(torch.float8_e8m0fnu)}
    if op == "append":
        return cache
    if op == "compact":
        return {**cache, "table": s["table_out"], "refs": s["refs_out"], "live": s["live"]}
    return {**cache, "table": s["table"], "refs": s["refs"], "lens": s["lens"], "ok": s["ok"], "done": s["done"]}


# ---- what a pass cannot do without -----------------------------------------------------------------------------------
def work(case):
    c = case
    token = c["Hkv"] * 2 * (c["D"] + 2 / c["page"])  # a token's codes and its share of the scales
    if c["op"] == "append":
        n = sum(rows_of(c))
        return {"bytes": c["layers"] * n * (4.0 * c["Hkv"] * c["D"] + token), "flops": c["layers"] * n * 4.0 * c["Hkv"] * c["D"]}
    if c["op"] == "attend":
        read = pairs = 0
        w = c["window"] or 1 << 40
        for n, length in zip(rows_of(c), lens_of(c)):
            first = length - n  # position of the first row
            read += length if first < w else min(length, length - (first - w + 1) + min(c["sinks"], first - w + 1))
            for lo, hi in ((first, min(length, w)), (max(first, w), length)):  # positions that see all, or w and the sinks
                if hi > lo:
                    pairs += (hi * (hi + 1) - lo * (lo + 1)) // 2 if hi <= w else (hi - lo) * (w + min(c["sinks"], lo - w + 1))
        rows = 4.0 * sum(rows_of(c)) * c["Hq"] * c["D"]
        return {"bytes": c["layers"] * (read * token + rows), "flops": c["layers"] * pairs * 4.0 * c["Hq"] * c["D"]}
    if c["op"] == "fork":
        lens = spread(c["B"] // 2, c["ctx_lo"], c["ctx_hi"])
        copied = sum(n % c["page"] != 0 for n in lens)
        ints = sum(8 * -(-n // c["page"]) for n in lens) + 40 * c["B"]
        return {"bytes": copied * c["layers"] * 2.0 * token * c["page"] + ints, "flops": 0.0}
    moved = c["live"] * (c["pages"] - c["live"]) / c["pages"]  # on average
    return {"bytes": moved * c["layers"] * 2 * token * c["page"] + 8.0 * c["pages"] + 8.0 * c["live"], "flops": 0.0}


# ---- the same in 64 bits ---------------------------------------------------------------------------------------------
def exact(case, seed):
    c, s = case, prepare(case, seed)
    cache, p, hkv, d = s["cache"], c["page"], c["Hkv"], c["D"]
    double = {"k": cache["k"].view(torch.float8_e4m3fn).double(), "v": cache["v"].view(torch.float8_e4m3fn).double(),
              "ks": cache["ks"].view(torch.float8_e8m0fnu).double(), "vs": cache["vs"].view(torch.float8_e8m0fnu).double()}

    def e4m3(x):
        """Nearest e4m3 value, ties to even: steps of 2^-9 up to 2^-6, of an eighth of the power of two above."""
        step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
        return torch.round(x / step) * step

    if c["op"] == "attend":
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        cu, lens = s["cu"].tolist(), s["lens"].tolist()
        for layer in range(c["layers"]):
            for b in range(c["B"]):
                n, t = cu[b + 1] - cu[b], lens[b]
                at = s["table"][b, : -(-t // p)].long()
                k = (double["k"][layer][at] * double["ks"][layer][at][:, :, None, None]).permute(1, 0, 2, 3)
                v = (double["v"][layer][at] * double["vs"][layer][at][:, :, None, None]).permute(1, 0, 3, 2)
                k, v = (x.reshape(hkv, -1, d)[:, :t].contiguous() for x in (k, v))
                pos = torch.arange(t - n, t, device="cuda")[:, None]
                key = torch.arange(t, device="cuda")[None, :]
                hidden = key > pos
                if c["window"]:
                    hidden = hidden | ((pos - key >= c["window"]) & (key >= c["sinks"]))
                for h in range(c["Hq"]):
                    j = h // (c["Hq"] // hkv)
                    x = s["q"][layer, cu[b]:cu[b + 1], h].double() @ k[j].t().contiguous() / math.sqrt(d)
                    out[layer, cu[b]:cu[b + 1], h] = torch.softmax(x.masked_fill(hidden, -math.inf), 1) @ v[j]
        return out
    if c["op"] == "append":
        cu, lens, table = s["cu"].tolist(), s["lens"].tolist(), s["table"].tolist()
        for layer in range(c["layers"]):
            for b in range(c["B"]):
                had = lens[b] - (cu[b + 1] - cu[b])
                for block in range(had // p, -(-lens[b] // p)):
                    lo, hi = max(had, block * p), min(lens[b], block * p + p)
                    rows, page = slice(cu[b] + lo - had, cu[b] + hi - had), table[b][block]
                    kept, put = slice(0, lo - block * p), slice(lo - block * p, hi - block * p)
                    for new, f, e in ((s["knew"], "k", "ks"), (s["vnew"], "v", "vs")):
                        x = new[layer, rows].double()  # [tokens, Hkv, D]
                        scale = torch.exp2(torch.ceil(torch.log2(x.abs().amax((0, 2)).clamp(min=1e-4) / 448)).clamp(max=119))
                        codes = double[f][layer, page] if f == "k" else double[f][layer, page].transpose(1, 2)
                        if lo > block * p:
                            old = double[e][layer, page]
                            scale = torch.maximum(scale, old)
                            codes[:, kept] = e4m3(codes[:, kept] * (old / scale)[:, None, None])
                        codes[:, put] = e4m3((x.transpose(0, 1) / scale[:, None, None]).clamp(-448, 448))
                        double[e][layer, page] = scale
        return double
    table, refs = s["table"].tolist(), s["refs"].tolist()
    if c["op"] == "compact":
        live = sum(r > 0 for r in refs)
        src = [i for i, r in enumerate(refs) if r > 0 and i >= live]
        dst = [i for i, r in enumerate(refs) if r == 0 and i < live]
        to = dict(zip(src, dst))
        for x in double.values():
            x[:, dst] = x[:, src]
        new = [refs[i] if i < live and refs[i] else 0 for i in range(len(refs))]
        for i, j in to.items():
            new[j] = refs[i]
        return {**double, "table": int32([[to.get(i, i) for i in row] for row in table]), "refs": int32(new),
                "live": int32([live])}
    lens, grow, done, ok = s["lens"].tolist(), s["grow"].tolist(), [0] * c["B"], [0] * c["B"]
    before = list(lens)  # nothing is given up in a first pass: keep is what there is
    for b, j in enumerate(s["from"].tolist()):
        if j >= 0 and before[b] == 0 and before[j] > 0:
            table[b], lens[b], done[b] = list(table[j]), lens[j], 1
            for i in table[b][: -(-lens[b] // p)]:
                refs[i] += 1
    shared, free, out_of_pages = list(refs), [i for i, r in enumerate(refs) if r == 0], False
    for b in range(c["B"]):
        had, want = -(-lens[b] // p), -(-(lens[b] + grow[b]) // p)
        tail = table[b][had - 1] if lens[b] % p and grow[b] else -1
        split = tail >= 0 and shared[tail] > 1
        need = want - had + split
        out_of_pages |= want <= len(table[b]) and need > len(free)
        if want > len(table[b]) or (need and out_of_pages):
            continue
        ok[b] = 1
        if split:
            i = free.pop(0)
            for x in double.values():
                x[:, i] = x[:, tail]
            table[b][had - 1], refs[i] = i, 1
            refs[tail] -= 1
        for block in range(had, want):
            table[b][block] = free.pop(0)
            refs[table[b][block]] = 1
        lens[b] += grow[b]
    return {**double, "table": int32(table), "refs": int32(refs), "lens": int32(lens), "ok": int32(ok), "done": int32(done)}

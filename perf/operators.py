"""Operators behind several scored completions of one prompt: keys and values held in 8 bits, attention over them, copies of
cache pages, and the scores of tokens.

With ``own`` false ``run`` computes them from elementary torch operations; with ``own`` true it makes the calls of this
repository's operator set.  ``exact`` restates them in 64 bits.

Keys and values in 8 bits: a block is 16 consecutive positions of a page and one kv head, keys and values apart.  ``codes`` is
uint8 [pages, 2 (k, v), kv_heads, page, d], ``words`` int32 [pages, kv_heads, page / 16, 2 (k, v)].  A word's bits 0..7 are E,
its bits 16..31 mark tokens with a number that is not finite.  With E = 0 every value of the block is 0, else a code u
stands for (u - 127.5) * 2^(E - 133); E is the biased binary exponent of the largest magnitude in the block, at least 16.  A token
written at a block's first position starts it anew; any other leaves E or raises it, and the codes that are there go by it.
"""
from __future__ import annotations

import math

import torch

own = False
F64 = torch.float64
BLOCK = 16
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


# ----------------------------------------------------------------------------- the cases
def listed():
    return [
        # a full server decodes: one token of each of 64 requests goes into a partly filled block
        {"name": "write_64", "kind": "write", "type": "bf16", "requests": 64, "shortest": 1, "longest": 1, "held": 7,
         "kv_heads": 8, "dim": 64, "page": 16},
        # prompts come in: four of up to 1,021 tokens, the first tokens in blocks that are there
        {"name": "write_prompts", "kind": "write", "type": "bf16", "requests": 4, "shortest": 301, "longest": 1021, "held": 37,
         "kv_heads": 8, "dim": 128, "page": 32},
        # one user chats at a context of 4,000: latency
        {"name": "attend_1", "kind": "attend", "type": "bf16", "singles": 1, "shortest": 4000, "longest": 4000, "prompts": 0,
         "portion": 0, "cached": 0, "heads": 32, "kv_heads": 8, "dim": 64, "page": 16, "window": 0},
        # 64 requests of different ages
        {"name": "attend_64", "kind": "attend", "type": "bf16", "singles": 64, "shortest": 256, "longest": 2560, "prompts": 0,
         "portion": 0, "cached": 0, "heads": 32, "kv_heads": 8, "dim": 64, "page": 16, "window": 0},
        # eight long documents, heads of 128
        {"name": "attend_long", "kind": "attend", "type": "bf16", "singles": 8, "shortest": 20011, "longest": 30011, "prompts": 0,
         "portion": 0, "cached": 0, "heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "window": 0},
        # the 32-bit path
        {"name": "attend_f32", "kind": "attend", "type": "f32", "singles": 8, "shortest": 1000, "longest": 4096, "prompts": 0,
         "portion": 0, "cached": 0, "heads": 32, "kv_heads": 8, "dim": 64, "page": 16, "window": 0},
        # a prompt of 2,048 tokens
        {"name": "attend_prompt", "kind": "attend", "type": "bf16", "singles": 0, "shortest": 0, "longest": 0, "prompts": 1,
         "portion": 2048, "cached": 0, "heads": 32, "kv_heads": 8, "dim": 64, "page": 16, "window": 0},
        # the next turns of three chats beside twelve that decode
        {"name": "attend_mixed", "kind": "attend", "type": "bf16", "singles": 12, "shortest": 900, "longest": 1100, "prompts": 3,
         "portion": 131, "cached": 3001, "heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "window": 0},
        # eight completions of one prompt: its last page, seven times in 16 layers
        {"name": "fork_8", "kind": "copy", "entries": 16, "pages": 256, "pairs": 7, "fan": 7, "page_bytes": 32768, "state_bytes": 0},
        # a pool made smaller: 1,500 pages move to the front
        {"name": "compact", "kind": "copy", "entries": 16, "pages": 4096, "pairs": 1500, "fan": 1, "page_bytes": 16384,
         "state_bytes": 0},
        # five alternatives of the next token for eight requests
        {"name": "score_8", "kind": "score", "rows": 8, "vocab": 128256, "top": 5},
        # a prompt of 500 tokens scored, with twenty alternatives each
        {"name": "score_500", "kind": "score", "rows": 500, "vocab": 128256, "top": 20},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["write", "attend", "attend", "attend", "copy", "score", "score"])
    if kind == "write":
        n = _log(rng, 1, 64)
        longest = 1 if rng.random() < 0.4 else _log(rng, 1, max(2, 2600 // n))
        return {"kind": kind, "type": rng.choice(["bf16", "bf16", "f32"]), "requests": n, "shortest": max(1, longest // 3), "longest": longest,
                "held": rng.randrange(0, 100), "kv_heads": rng.choice([1, 2, 3, 8]), "dim": rng.choice([64, 128]), "page": rng.choice([16, 32, 64])}
    if kind == "attend":
        dim = rng.choice([64, 128])
        kv_heads = rng.choice([1, 2, 5, 8])
        heads = kv_heads * rng.choice([1, 3, 4, 4, 8])
        form = rng.choice(["singles", "singles", "prompt", "mixed"])
        singles = _log(rng, 1, 64) if form != "prompt" else 0
        longest = _log(rng, 1, min(30000, 100000 // singles)) if singles else 0
        portion = _log(rng, 2, 1500) if form != "singles" else 0
        prompts = 1 if portion > 200 else rng.choice([1, 2, 4])
        if rng.random() < 0.2:
            heads, kv_heads, dim = rng.choice([(6, 6, 96), (5, 5, 48), (20, 1, 64), (4, 1, 256)])
            longest, portion = min(longest, 1000), min(portion, 100)
        return {"kind": kind, "type": rng.choice(["bf16", "bf16", "f32"]) if portion <= 300 else "bf16", "singles": singles,
                "shortest": max(1, longest // rng.choice([1, 2, 10])) if singles else 0, "longest": longest,
                "prompts": prompts if portion else 0, "portion": portion, "cached": rng.choice([0, _log(rng, 1, 2000)]) if portion else 0,
                "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": rng.choice([16, 16, 32, 64]),
                "window": rng.choice([0, 0, 0, _log(rng, 1, 4000)])}
    if kind == "copy":
        pairs = _log(rng, 1, 1000)
        entries = rng.choice([1, 3, 16])
        page_bytes = 16 * _log(rng, 8, 2048)
        return {"kind": kind, "entries": entries, "pages": 2 * pairs + rng.randrange(1, 50), "pairs": pairs, "fan": rng.choice([1, 1, min(pairs, 5)]),
                "page_bytes": page_bytes, "state_bytes": rng.choice([0, 0, 4 * _log(rng, 3, 30000)])}
    rows = _log(rng, 1, 500)
    return {"kind": kind, "rows": rows, "vocab": _log(rng, 50, 128256), "top": rng.choice([0, 1, 5, 20, 32])}


def _spread(n, lo, hi):
    """n whole numbers from lo to hi, the largest first."""
    return [hi - (hi - lo) * i // max(1, n - 1) for i in range(n)]


def _lengths(case):
    """(new tokens, tokens held afterwards) of each request of a step."""
    if case["kind"] == "write":
        q = _spread(case["requests"], case["shortest"], case["longest"])
        return [(n, n + (case["held"] + 5 * i) % 100) for i, n in enumerate(q)]
    out = [(1, c) for c in _spread(case["singles"], case["shortest"], case["longest"])]
    for i, n in enumerate(_spread(case["prompts"], (case["portion"] + 1) // 2, case["portion"])):
        out.insert(2 * i, (n, n + case["cached"] // (i + 1)))
    return out


# ----------------------------------------------------------------------------- what a program has in hand
def _paging(case, lens, g):
    """A shuffled pool: table [requests, widest], the tokens' slots, requests and positions."""
    page = case["page"]
    blocks = [-(-c // page) for _, c in lens]
    pages = sum(blocks) + 3
    order = torch.randperm(pages, generator=g)
    table = torch.full((len(lens), max(blocks)), -1, dtype=torch.int32)
    at = 0
    slots, req, pos = [], [], []
    for r, ((n, c), b) in enumerate(zip(lens, blocks)):
        table[r, :b] = order[at:at + b].int()
        at += b
        p = torch.arange(c - n, c)
        slots.append(table[r, p // page] * page + p % page)
        req.append(torch.full((n,), r))
        pos.append(p)
    flat = [torch.cat(x).int().cuda() for x in (slots, req, pos)]
    return pages, table.cuda(), flat


def _random_cache(case, pages, g):
    G, d, page = case["kv_heads"], case["dim"], case["page"]
    codes = torch.empty((pages, 2, G, page, d), dtype=torch.uint8, device="cuda")
    for part in codes.split(max(1, (1 << 25) // (2 * G * page * d))):
        part.copy_((torch.randn(part.shape, generator=g, device="cuda") * 36 + 128).clamp_(0, 255))
    words = torch.randint(125, 129, (pages, G, page // BLOCK, 2), generator=g, device="cuda", dtype=torch.int32)
    return codes, words


def prepare(case, seed):
    g = torch.Generator().manual_seed(seed)
    gc = torch.Generator("cuda").manual_seed(seed)
    st = {"case": case}
    if own:
        from pytriton_llama_b200.ops.cuda import CudaOps
        st["ops"] = CudaOps("cuda:0")
    kind = case["kind"]
    if kind in ("write", "attend"):
        lens = _lengths(case)
        pages, table, (slots, req, pos) = _paging(case, lens, g)
        codes, words = _random_cache(case, pages, gc)
        G, d, T, dtype = case["kv_heads"], case["dim"], slots.numel(), DTYPES[case["type"]]
        st.update(lens=lens, table=table, slots=slots, req=req, pos=pos, codes=codes, words=words)
        st["contexts"] = [c for _, c in lens]
        if kind == "write":
            size = torch.exp2(torch.randint(-2, 3, (T, 1), generator=gc, device="cuda").float())
            st["kv"] = (torch.randn((T, 2 * G * d), generator=gc, device="cuda") * size).to(dtype)
        else:
            st["q"] = (torch.randn((T, case["heads"] * d), generator=gc, device="cuda") * 1.5).to(dtype)
            if own:
                st["hints"] = st["ops"].hints_for([n for n, _ in lens], st["contexts"])
    elif kind == "copy":
        # 32-bit words, so that the pages of any compute type are stood for
        st["tensors"] = [torch.randint(-2**31, 2**31 - 1, (case["pages"], case["page_bytes"] // 4), generator=gc, device="cuda", dtype=torch.int32)
                         for _ in range(case["entries"])]
        if case["state_bytes"]:
            st["tensors"].append(torch.randn((case["pages"], case["state_bytes"] // 4), generator=gc, device="cuda"))
        order = torch.randperm(case["pages"], generator=g).tolist()
        st["dst"] = order[:case["pairs"]]
        st["src"] = [order[case["pairs"] + i // case["fan"]] for i in range(case["pairs"])]
    else:
        rows, vocab = case["rows"], case["vocab"]
        st["logits"] = torch.randn((rows, vocab), generator=gc, device="cuda") * 2.5
        st["logits"][:, : max(1, vocab // 50)] += 3
        # numbers of few bits meet one another: ties
        st["logits"][rows // 2:] = (st["logits"][rows // 2:] * 64).round() / 64
        st["tokens"] = torch.randint(0, vocab, (rows,), generator=gc, device="cuda", dtype=torch.int32)
    return st


# ----------------------------------------------------------------------------- plain forms
def _values(codes, words, dtype):
    """What codes [..., 2, G, page, d] of whole pages stand for."""
    e = (words & 255).permute(0, 3, 1, 2).repeat_interleave(BLOCK, dim=-1)[..., None]       # [pages, 2, G, page, 1]
    step = torch.exp2((e - 133).to(dtype))
    return torch.where(e > 0, (codes.to(dtype) - 127.5) * step, torch.zeros((), dtype=dtype, device=codes.device))


def _exponent(amax):
    e = (amax.view(torch.int32) >> 23) & 255
    return torch.where(amax > 0, e.clamp(min=16), torch.zeros_like(e))


def _plain_write(st):
    case, codes, words = st["case"], st["codes"], st["words"]
    G, d, page = case["kv_heads"], case["dim"], case["page"]
    x = st["kv"].float().view(-1, 2, G, d)                           # [T, (k, v), G, d]
    slots = st["slots"].long()
    block = slots // BLOCK                                           # page by page, page / BLOCK of them in each
    ids, at = torch.unique(block, return_inverse=True)
    pg, sub = ids // (page // BLOCK), ids % (page // BLOCK)
    amax = torch.zeros((ids.numel(), 2, G), device=x.device).scatter_reduce(
        0, at[:, None, None].expand(-1, 2, G), x.abs().amax(-1), "amax")
    anew = torch.zeros(ids.numel(), dtype=torch.bool, device=x.device)
    anew[at[slots % BLOCK == 0]] = True
    old = (words[pg, :, sub] & 255).transpose(1, 2)                  # [blocks, 2, G]
    old = torch.where(anew[:, None, None], torch.zeros_like(old), old)
    new = torch.maximum(old, _exponent(amax))
    held = codes.view(-1, 2, G, page // BLOCK, BLOCK, d)
    was = held[pg, :, :, sub]                                        # [blocks, 2, G, BLOCK, d]
    shift = torch.where(old > 0, new - old, torch.full_like(old, 31)).clamp(max=31)[..., None, None]
    held[pg, :, :, sub] = (((was.int() - 128) >> shift) + 128).to(torch.uint8)
    words[pg, :, sub] = new.transpose(1, 2).to(torch.int32)
    step = torch.exp2((new[at] - 133).float())[..., None]
    u = torch.where(new[at][..., None] > 0, torch.floor(x / step) + 128, torch.full_like(x, 128))
    codes[slots // page, :, :, slots % page] = u.to(torch.uint8)


def _plain_read(st):
    """Keys and values of every request's tokens, one after the other: [tokens, 2, G, d] in the compute type."""
    case = st["case"]
    page, out = case["page"], []
    for r, c in enumerate(st["contexts"]):
        pages = st["table"][r, : -(-c // page)].long()
        v = _values(st["codes"][pages], st["words"][pages], torch.float32)        # [pages, 2, G, page, d]
        out.append(v.permute(0, 3, 1, 2, 4).flatten(0, 1)[:c])
    return torch.cat(out).to(DTYPES[case["type"]])


def _plain_attend(st):
    case, page, d, G, H = st["case"], st["case"]["page"], st["case"]["dim"], st["case"]["kv_heads"], st["case"]["heads"]
    out, t0 = [], 0
    for r, (n, c) in enumerate(st["lens"]):
        lo = max(0, c - n - case["window"] + 1) // page if case["window"] else 0
        pages = st["table"][r, lo: -(-c // page)].long()
        kv = _values(st["codes"][pages], st["words"][pages], torch.float32).transpose(0, 1).transpose(1, 2).flatten(2, 3)   # [2, G, keys, d]
        q = st["q"][t0:t0 + n].float().view(n, G, H // G, d).permute(1, 2, 0, 3)
        key = torch.arange(kv.shape[2], device=q.device) + lo * page
        p = st["pos"][t0:t0 + n].long()[:, None]
        seen = (key <= p) & (key > p - case["window"]) if case["window"] else key <= p
        s = (q @ kv[0][:, None].transpose(-1, -2) * d ** -0.5).masked_fill(~seen, -math.inf)
        w = torch.exp(s - s.amax(-1, keepdim=True))
        o = (w / w.sum(-1, keepdim=True)).masked_fill(~seen, 0.0) @ kv[1][:, None].masked_fill((key >= c)[None, None, :, None], 0.0)
        out.append(o.permute(2, 0, 1, 3).reshape(n, H * d))
        t0 += n
    return torch.cat(out).to(st["q"].dtype)


def _plain_score(st):
    x, tokens, top = st["logits"], st["tokens"].long(), st["case"]["top"]
    z = x - x.amax(-1, keepdim=True)
    e = torch.exp(z)
    total = e.sum(-1)
    lse = torch.log(total)
    logprob = z.gather(1, tokens[:, None])[:, 0] - lse
    entropy = lse - (e * z).sum(-1) / total
    k = min(top, x.shape[1])
    order = torch.sort(x, dim=-1, descending=True, stable=True)[1][:, :k]
    return logprob, entropy, z.gather(1, order) - lse[:, None], order.int()


def run(st):
    kind = st["case"]["kind"]
    if own:
        ops, case = st["ops"], st["case"]
        if kind == "write":
            ops.rope_kv8_write(st["kv"], st["pos"], None, 0, st["slots"], st["codes"], st["words"], 0, case["kv_heads"], case["dim"], case["page"])
            return ops.read_kv8(st["codes"], st["words"], st["table"], st["contexts"], DTYPES[case["type"]])
        if kind == "attend":
            return ops.paged_attention8(st["q"], st["codes"], st["words"], st["table"], st["req"], st["pos"], case["heads"], case["kv_heads"],
                                        case["dim"], case["page"], case["dim"] ** -0.5, window=case["window"], hints=st["hints"])
        if kind == "copy":
            ops.copy_pages(st["tensors"], st["src"], st["dst"])
            return st["tensors"]
        return ops.token_scores(st["logits"], st["tokens"], case["top"])
    if kind == "write":
        _plain_write(st)
        return _plain_read(st)
    if kind == "attend":
        return _plain_attend(st)
    if kind == "copy":
        src, dst = (torch.tensor(x, device="cuda") for x in (st["src"], st["dst"]))
        for t in st["tensors"]:
            t[dst] = t[src]
        return st["tensors"]
    return _plain_score(st)


# ----------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    kind = case["kind"]
    if kind == "copy":
        return {"bytes": 2 * case["pairs"] * (case["entries"] * case["page_bytes"] + case["state_bytes"]), "flops": 0}
    if kind == "score":
        n = case["rows"] * case["vocab"]
        return {"bytes": 4 * n + case["rows"] * (12 + 8 * min(case["top"], case["vocab"])), "flops": 4 * n}
    lens = _lengths(case)
    esize = 2 if case["type"] == "bf16" else 4
    row = 2 * case["kv_heads"] * case["dim"]
    if kind == "write":
        new, held = sum(n for n, _ in lens), sum(c for _, c in lens)
        return {"bytes": new * row * (esize + 1) + held * row * (esize + 1), "flops": 2 * new * row}
    seen = pairs = 0
    for n, c in lens:
        first = c - n
        w = case["window"] or c
        seen += c - max(0, first - w + 1)
        pairs += sum(min(p + 1, w) for p in range(first, c))
    rows = sum(n for n, _ in lens) * case["heads"] * case["dim"]
    return {"bytes": seen * row + seen * row // (case["dim"] * BLOCK) * 4 + 2 * rows * esize, "flops": 4 * case["heads"] * case["dim"] * pairs}


# ----------------------------------------------------------------------------- 64 bits
def _exact_cache(st):
    """Values of the whole pool in 64 bits, [pages, 2, G, page, d]."""
    c, w = st["codes"], st["words"]
    pages, _, G, page, d = c.shape
    out = torch.zeros(c.shape, dtype=F64, device="cuda")
    for b in range(page // BLOCK):
        for part in range(2):
            e = (w[:, :, b, part] & 255).to(F64)[:, :, None, None]
            tile = slice(b * BLOCK, (b + 1) * BLOCK)
            out[:, part, :, tile] = torch.where(e > 0, (2.0 * c[:, part, :, tile].to(F64) - 255.0) * torch.pow(torch.tensor(2.0, dtype=F64, device="cuda"), e - 134.0),
                                                torch.zeros((), dtype=F64, device="cuda"))
    return out


def _exact_write(st):
    """A block's last state from all its values: what it held, in the middle of its codes' steps, beside what is written."""
    case = st["case"]
    page, G, d = case["page"], case["kv_heads"], case["dim"]
    held = _exact_cache(st).cpu()
    words = (st["words"] & 255).cpu()
    x = st["kv"].to(F64).cpu().view(-1, 2, G, d)
    touched = {}
    for t, s in enumerate(st["slots"].tolist()):
        touched.setdefault(s // BLOCK, {})[s % BLOCK] = t
    for b, rows in touched.items():
        pg, first = b // (page // BLOCK), b % (page // BLOCK) * BLOCK
        tile = held[pg, :, :, first:first + BLOCK].clone()               # [2, G, BLOCK, d]
        offs, toks = list(rows), list(rows.values())
        tile[:, :, offs] = x[toks].permute(1, 2, 0, 3)
        e = torch.frexp(x[toks].abs().amax((0, 3)))[1] - 1 + 127         # [2, G]
        e = torch.where(x[toks].abs().amax((0, 3)) > 0, e.clamp(min=16), torch.zeros_like(e))
        if 0 not in rows:
            e = torch.maximum(e, words[pg, :, first // BLOCK].T)
        step = torch.ldexp(torch.ones((), dtype=F64), e - 133)[..., None, None]
        held[pg, :, :, first:first + BLOCK] = torch.where(e[..., None, None] > 0, (torch.floor(tile / step) + 0.5) * step, torch.zeros((), dtype=F64))
    out = []
    for r, c in enumerate(st["contexts"]):
        table = st["table"][r].tolist()
        for b in range(-(-c // page)):
            out.append(held[table[b]].permute(2, 0, 1, 3)[: min(page, c - b * page)])
    return torch.cat(out).cuda()


def _exact_attend(st):
    case = st["case"]
    page, d, G, H = case["page"], case["dim"], case["kv_heads"], case["heads"]
    q = st["q"].to(F64).view(-1, H, d)
    out = torch.zeros_like(q)
    two = torch.tensor(2.0, dtype=F64, device="cuda")
    t0 = 0
    for r, (n, c) in enumerate(st["lens"]):
        table = st["table"][r, : -(-c // page)].long()
        pos = torch.arange(c - n, c, device="cuda")
        key = torch.arange(c, device="cuda")
        hidden = key[None, :] > pos[:, None]
        if case["window"]:
            hidden |= pos[:, None] - key[None, :] >= case["window"]
        for h in range(G):
            kv = []
            for part in range(2):
                e = (st["words"][table][:, h, :, part] & 255).to(F64).flatten().repeat_interleave(BLOCK)[:c, None]
                u = st["codes"][table][:, part, h].to(F64).flatten(0, 1)[:c]
                kv.append(torch.where(e > 0, (u * 2 - 255) * torch.pow(two, e - 134), torch.zeros((), dtype=F64, device="cuda")))
            for j in range(h * (H // G), (h + 1) * (H // G)):
                s = torch.matmul(q[t0:t0 + n, j], kv[0].T) / math.sqrt(d)
                s[hidden] = -math.inf
                out[t0:t0 + n, j] = torch.softmax(s, -1) @ kv[1]
        t0 += n
    return out.view(-1, H * d)


def exact(case, seed):
    if case["kind"] == "copy":
        return None
    st = prepare(case, seed)
    if case["kind"] == "write":
        return _exact_write(st)
    if case["kind"] == "attend":
        return _exact_attend(st)
    lp, ent, alt = [], [], []
    for row, t in zip(st["logits"], st["tokens"].tolist()):
        full = torch.log_softmax(row.to(F64), -1)
        lp.append(full[t])
        ent.append(-(full.exp() * full).sum())
        alt.append(full.sort(descending=True)[0][: case["top"]])
    return torch.stack(lp), torch.stack(ent), torch.stack(alt), None

"""Operators of a packed step: the new tokens of many requests, of one or of thousands each, over a key / value cache in pages.

A case names an operator and its sizes:

* "extend":   page tables, positions and cache slots of a step's tokens, from the requests' lengths and a list of free pages;
* "rotary":   queries turned to their positions, and for most cases keys turned and written with their values to their slots;
* "chunk":    attention of every request's newest tokens over its pages, later ones hidden from earlier ones;
* "logprobs": log probabilities of given tokens, for some cases with the distribution's entropy and its most likely tokens.

With `own` false `run` computes them from elementary torch operations, else through the package's entry points.  Both take
the same state: device tensors that a serving program holds before the call.
"""
import math
import random

import torch

own = False

_DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


# ---------------------------------------------------------------------------------------------------------- the cases
def _extend(batch, longest, new, single, page, spare):
    return {"op": "extend", "batch": batch, "longest": longest, "new": new, "single": single, "page": page, "spare": spare}


def _rotary(dtype, tokens, heads, kv_heads, head_dim, dims, layout, farthest, base, stretch, page, write):
    return {"op": "rotary", "dtype": dtype, "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "dims": dims,
            "layout": layout, "farthest": farthest, "base": base, "stretch": stretch, "page": page, "write": write}


def _chunk(dtype, batch, heads, kv_heads, head_dim, before, new, single, page):
    return {"op": "chunk", "dtype": dtype, "batch": batch, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "before": before,
            "new": new, "single": single, "page": page}


def _logprobs(dtype, rows, vocab, top, entropy, banned):
    return {"op": "logprobs", "dtype": dtype, "rows": rows, "vocab": vocab, "top": top, "entropy": entropy, "banned": banned}


def listed():
    return [
        # a decode step of 32 users, one token each: the call that latency decides
        dict(_extend(32, 2000, 1, 0.0, 16, 0), name="extend-step"),
        # a mixed step of 301 requests, prompts and single tokens in one packed batch, padded behind the last
        dict(_extend(301, 8000, 180, 0.6, 16, 97), name="extend-mixed"),
        # a decode step of 32 users, 8B attention shape, Llama's layout of neighbouring pairs
        dict(_rotary("bfloat16", 32, 32, 8, 128, 128, "pairs", 8000, 500000.0, 1.0, 16, True), name="rotary-step"),
        # 8191 prompt tokens, 8B attention shape, halves, frequencies stretched for positions far beyond training
        dict(_rotary("bfloat16", 8191, 32, 8, 128, 128, "halves", 131072, 500000.0, 8.0, 16, True), name="rotary-prompts"),
        # a quarter of every head turned, fp32, queries alone
        dict(_rotary("float32", 1001, 16, 16, 96, 24, "halves", 4000, 10000.0, 1.0, 16, False), name="rotary-part-fp32"),
        # five drafted tokens of one user checked at once over a short chat, 8B attention shape: latency
        dict(_chunk("bfloat16", 1, 32, 8, 128, 1500, 5, 0.0, 16), name="chunk-draft"),
        # a served step: 48 requests, most with one token, some with a portion of a prompt, 1B attention shape
        dict(_chunk("float16", 48, 32, 8, 64, 3001, 300, 0.7, 32), name="chunk-mixed"),
        # the small fp32 model (6 heads of 48): 64 prompts within its 256 positions
        dict(_chunk("float32", 64, 6, 6, 48, 30, 220, 0.0, 16), name="chunk-small-fp32"),
        # a portion of 511 tokens of a document of 65536, 8B attention shape
        dict(_chunk("bfloat16", 1, 32, 8, 128, 65000, 511, 0.0, 64), name="chunk-document"),
        # six prompts of up to 4096 tokens read at once, 8B attention shape, the largest
        dict(_chunk("bfloat16", 6, 32, 8, 128, 0, 4096, 0.0, 16), name="chunk-prompts"),
        # the sampled tokens of 48 users with the 20 most likely ones beside them, Llama 3 vocabulary, some tokens banned
        dict(_logprobs("float32", 48, 128256, 20, True, True), name="logprobs-step"),
        # a prompt of 2047 tokens scored, Llama 3 vocabulary
        dict(_logprobs("bfloat16", 2047, 128256, 0, True, False), name="logprobs-prompt"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["extend", "rotary", "rotary", "chunk", "chunk", "chunk", "logprobs", "logprobs"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    page = rng.choice([1, 8, 16, 16, 32, 64, 128])
    head_dim = rng.choice([32, 48, 64, 64, 96, 128, 128])
    kv_heads = rng.choice([1, 2, 3, 4, 6, 8, 8])
    heads = kv_heads * rng.choice([1, 1, 2, 3, 4, 4, 7, 8])
    if op == "extend":
        batch = _log(rng, 1, 1000)
        return _extend(batch, _log(rng, 16, 30000), _log(rng, 1, max(2, min(4000, 100000 // batch))), rng.choice([0.0, 0.5, 0.9]), page,
                       rng.choice([0, 0, rng.randint(1, 500)]))
    if op == "rotary":
        dims = rng.choice([head_dim, head_dim, head_dim // 2, head_dim // 4 * 2 + 2])
        return _rotary(dtype, _log(rng, 1, 8192 * 40 // max(heads + 2 * kv_heads, 40)), heads, kv_heads, head_dim, dims,
                       rng.choice(["pairs", "halves"]), _log(rng, 100, 1000000), rng.choice([10000.0, 500000.0]), rng.choice([1.0, 4.0, 8.0]),
                       page, rng.random() < 0.6)
    if op == "chunk":
        batch = _log(rng, 1, 64)
        most = 4e10 if dtype == "float32" else 5e11     # products and sums, padded
        new = _log(rng, 1, 2000)
        room = most / (4.0 * batch * new * heads * head_dim)
        while room < new + 1:
            new = max(1, new // 2)
            room = most / (4.0 * batch * new * heads * head_dim)
        before = min(int(room) - new, (1 << 28) // (batch * kv_heads * head_dim))
        return _chunk(dtype, batch, heads, kv_heads, head_dim, rng.choice([0, _log(rng, 1, max(2, before))]) if before > 0 else 0, new,
                      rng.choice([0.0, 0.0, 0.5, 0.8]), page)
    top = rng.choice([0, 0, 1, 5, 20, 33])
    vocab = _log(rng, 500, 151936)
    rows = _log(rng, 1, max(2, min(2047, (60 if top else 2047) * 128256 // vocab)))
    return _logprobs(dtype, rows, vocab, top, rng.random() < 0.6, rng.random() < 0.4)


# ------------------------------------------------------------------------------------------------------------- inputs
def _spread(b):
    return math.modf(b * 0.6180339887498949 + 0.1)[0]


def _requests(case):
    """(tokens before the step, new ones) of every request; a function of the case, so that work() can count them."""
    n, before = case["batch"], case["longest" if case["op"] == "extend" else "before"]
    new, single = case["new"], case["single"]
    got = []
    for b in range(n):
        was = before if b == 0 else int(before * _spread(b))
        fresh = new if b == 0 else 1 if _spread(3 * b + 1) < single else 1 + int((new - 1) * _spread(2 * b + 1))
        got.append((was, fresh))
    return got


def _starts(counts):
    at = [0]
    for c in counts:
        at.append(at[-1] + c)
    return at


def _shuffled(rng, n):
    ids = list(range(n))
    rng.shuffle(ids)
    return ids


def _table(rng, page_counts, spare):
    """Page tables whose pages lie in any order, as an allocator leaves them after many requests; unused entries are -1."""
    total = sum(page_counts) + spare
    ids, wide, at, rows = _shuffled(rng, total), max(max(page_counts), 1), 0, []
    for c in page_counts:
        rows.append(ids[at:at + c] + [-1] * (wide - c))
        at += c
    return torch.tensor(rows, dtype=torch.int32, device="cuda"), total


def _frequencies(dims, base, stretch):
    """Radians a position of each pair; with stretch > 1, slow ones divided by it and those between faded, as for long contexts."""
    f = base ** (-torch.arange(0, dims, 2, dtype=torch.float64) / dims)
    if stretch > 1:
        turns = 8192 * f / (2 * math.pi)        # within the positions of training
        part = ((turns - 1) / (4 - 1)).clamp(0, 1)
        f = f * (part + (1 - part) / stretch)
    return f


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed) * 7919 + 17)
    rng = random.Random(int(seed) * 104729 + 5)
    op = case["op"]
    kind = _DTYPES.get(case.get("dtype"))

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(kind)

    def ints(values, to=torch.int32):
        return torch.tensor(values, dtype=to, device="cuda")

    if op == "extend":
        page, req = case["page"], _requests(case)
        had, need = [-(-w // page) for w, _ in req], [-(-(w + n) // page) for w, n in req]
        ids, wide, at, rows = _shuffled(rng, sum(need) + 9), max(need) + 2, 0, []
        for h in had:
            rows.append(ids[at:at + h] + [-1] * (wide - h))
            at += h
        st = {"table": ints(rows), "lengths": ints([w for w, _ in req]), "counts": ints([n for _, n in req]), "free": ints(ids[at:]),
              "page": page, "tokens": sum(n for _, n in req) + case["spare"]}
    elif op == "rotary":
        n, H, G, D, page = case["tokens"], case["heads"], case["kv_heads"], case["head_dim"], case["page"]
        st = {"q": normal(n, H, D), "positions": torch.randint(0, case["farthest"], (n,), generator=gen, device="cuda", dtype=torch.int32),
              "frequencies": _frequencies(case["dims"], case["base"], case["stretch"]).cuda(), "layout": case["layout"], "write": case["write"]}
        if case["write"]:
            total = -(-n // page) + 5
            st |= {"k": normal(n, G, D), "v": normal(n, G, D), "k_pages": normal(total, G, page, D), "v_pages": normal(total, G, page, D),
                   "slots": torch.randperm(total * page, generator=gen, device="cuda")[:n].contiguous()}
    elif op == "chunk":
        page, G, D, req = case["page"], case["kv_heads"], case["head_dim"], _requests(case)
        table, total = _table(rng, [-(-(w + n) // page) for w, n in req], 3)
        st = {"q": normal(sum(n for _, n in req), case["heads"], D), "k_pages": normal(total, G, page, D), "v_pages": normal(total, G, page, D),
              "table": table, "lengths": ints([w + n for w, n in req]), "starts": ints(_starts([n for _, n in req])),
              "longest": max(n for _, n in req)}
    else:
        x = normal(case["rows"], case["vocab"], scale=2.5)
        if case["banned"]:
            x[:, torch.arange(7, case["vocab"], 11, device="cuda")] = float("-inf")
        tokens = torch.randint(0, case["vocab"] // 11, (case["rows"],), generator=gen, device="cuda") * 11     # none that is banned
        st = {"logits": x, "tokens": tokens.to(torch.int32), "top": case["top"], "entropy": case["entropy"]}
    st["op"] = op
    return st


# --------------------------------------------------------------------------------------------------------- plain forms
def _plain_extend(st):
    table, was, new, free, page = st["table"], st["lengths"].long(), st["counts"].long(), st["free"], st["page"]
    B, wide = table.shape
    zero = torch.zeros(1, dtype=torch.long, device=table.device)
    had, pages = (was + page - 1) // page, (was + new + page - 1) // page
    first = torch.cat([zero, (pages - had).cumsum(0)])
    starts = torch.cat([zero, new.cumsum(0)])
    j = torch.arange(wide, device=table.device)
    at = first[:-1, None] + j - had[:, None]
    got = torch.where((at >= 0) & (at < len(free)), free[at.clamp(0, len(free) - 1)], -1)
    table.copy_(torch.where((j >= had[:, None]) & (j < pages[:, None]), got, table))
    t = torch.arange(st["tokens"], device=table.device)
    b = torch.searchsorted(starts[1:], t, right=True)
    real, b = b < B, b.clamp(max=B - 1)
    position = was[b] + t - starts[b]
    of = table[b, (position // page).clamp(0, wide - 1)].long()
    slots = torch.where(real & (of >= 0), of * page + position % page, -1)
    return {"table": table, "lengths": (was + new).int(), "starts": starts.int(), "positions": torch.where(real, position, -1).int(),
            "slots": slots, "used": first[-1:].int()}


def _plain_turn(x, positions, frequencies, layout):
    angle = positions.double()[:, None] * frequencies
    c, s = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    d, y = 2 * len(frequencies), x.float()
    if layout == "pairs":
        a, b = y[..., 0:d:2], y[..., 1:d:2]
        turned = torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
    else:
        a, b = y[..., :d // 2], y[..., d // 2:d]
        turned = torch.cat([a * c - b * s, b * c + a * s], -1)
    return torch.cat([turned, y[..., d:]], -1).to(x.dtype)


def _plain_rotary(st):
    res = {"q": _plain_turn(st["q"], st["positions"], st["frequencies"], st["layout"])}
    if st["write"]:
        page = st["k_pages"].shape[2]
        ids, off = st["slots"] // page, st["slots"] % page
        st["k_pages"][ids, :, off] = _plain_turn(st["k"], st["positions"], st["frequencies"], st["layout"])
        st["v_pages"][ids, :, off] = st["v"]
        res |= {"k_pages": st["k_pages"], "v_pages": st["v_pages"]}
    return res


def _plain_chunk(st):
    q, kp, vp, table, lens, starts = st["q"], st["k_pages"], st["v_pages"], st["table"].long(), st["lengths"].long(), st["starts"].long()
    B, (T, H, D), G, page = len(lens), q.shape, kp.shape[1], kp.shape[2]
    R, L = H // G, st["longest"]
    count = starts[1:] - starts[:-1]
    i = torch.arange(L, device=q.device)
    rows = (starts[:-1, None] + i).clamp(max=T - 1)                                  # a padded batch of the packed rows
    real = i < count[:, None]
    at = (lens - count)[:, None] + i                                                 # their positions
    pos = torch.arange(table.shape[1] * page, device=q.device)
    ids = table.clamp(min=0)
    k = kp[ids].permute(0, 2, 1, 3, 4).reshape(B, G, -1, D).float()                  # [B, G, positions, D]
    v = vp[ids].permute(0, 2, 1, 3, 4).reshape(B, G, -1, D).float()
    x = q[rows].float().reshape(B, L, G, R, D).permute(0, 2, 3, 1, 4).reshape(B, G, R * L, D)
    s = torch.matmul(x, k.transpose(2, 3)) * D ** -0.5
    s = s.reshape(B, G, R, L, -1).masked_fill_((pos > at[..., None])[:, None, None], float("-inf"))
    top = s.amax(-1, keepdim=True)
    e = s.sub_(top).exp_()
    total = e.sum(-1, keepdim=True)
    o = torch.matmul(e.reshape(B, G, R * L, -1), v).reshape(B, G, R, L, D) / total
    lse = (top + torch.log(total))[..., 0]
    o, lse = o.permute(0, 3, 1, 2, 4)[real].reshape(T, H, D), lse.permute(0, 3, 1, 2)[real].reshape(T, H)
    return {"out": o.to(q.dtype), "lse": lse}


def _plain_logprobs(st):
    x, tokens = st["logits"].float(), st["tokens"].long()
    top = x.amax(-1, keepdim=True)
    d = x - top
    e = torch.exp(d)
    total = e.sum(-1, keepdim=True)
    log = torch.log(total)
    res = {"logprobs": (d.gather(1, tokens[:, None]) - log)[:, 0]}
    if st["entropy"]:
        res["entropy"] = log[:, 0] - torch.where(e > 0, e * d, 0).sum(-1) / total[:, 0]
    if st["top"]:
        val, idx = x.sort(dim=1, descending=True, stable=True)     # stable: ties go to the lowest index
        res["top_logprobs"] = val[:, :st["top"]] - top - log
        res["top_tokens"] = idx[:, :st["top"]].to(torch.int32)
    return res


def run(st):
    op = st["op"]
    if own:
        import llama3_np_b200 as l3
    if op == "extend":
        if not own:
            return _plain_extend(st)
        step = l3.paged_extend(st["table"], st["lengths"], st["counts"], st["free"], page_size=st["page"], tokens=st["tokens"])
        return {"table": st["table"], "lengths": step.lengths, "starts": step.starts, "positions": step.positions, "slots": step.slots,
                "used": step.used}
    if op == "rotary":
        if not own:
            return _plain_rotary(st)
        if not st["write"]:
            return {"q": l3.rotary(st["q"], st["positions"], st["frequencies"], layout=st["layout"])}
        q = l3.paged_rotary_write(st["q"], st["k"], st["v"], st["positions"], st["slots"], st["k_pages"], st["v_pages"], st["frequencies"],
                                  layout=st["layout"])
        return {"q": q, "k_pages": st["k_pages"], "v_pages": st["v_pages"]}
    if op == "chunk":
        if not own:
            return _plain_chunk(st)
        out, lse = l3.paged_chunk_attention(st["q"], st["k_pages"], st["v_pages"], st["table"], st["lengths"], st["starts"], return_lse=True)
        return {"out": out, "lse": lse}
    if not own:
        return _plain_logprobs(st)
    got = l3.token_logprobs(st["logits"], st["tokens"], top=st["top"], entropy=st["entropy"])
    res = {"logprobs": got.logprobs}
    if st["entropy"]:
        res["entropy"] = got.entropy
    if st["top"]:
        res["top_logprobs"], res["top_tokens"] = got.top_logprobs, got.top_tokens
    return res


# -------------------------------------------------------------------------------------------------- work and definition
def _seen(was, new):
    """Keys that the new tokens of a request see, over all of them."""
    return new * was + new * (new + 1) // 2


def work(case):
    op = case["op"]
    size = 2 if case.get("dtype") in ("bfloat16", "float16") else 4
    if op == "extend":
        req, page = _requests(case), case["page"]
        pages = sum(-(-(w + n) // page) - -(-w // page) for w, n in req)
        return {"bytes": 16 * case["batch"] + 8 + 8 * pages + 12 * (sum(n for _, n in req) + case["spare"]), "flops": 0}
    if op == "rotary":
        rows = case["heads"] + (2 * case["kv_heads"] if case["write"] else 0)
        turned = case["heads"] + (case["kv_heads"] if case["write"] else 0)
        return {"bytes": case["tokens"] * (2 * rows * case["head_dim"] * size + (12 if case["write"] else 4)) + 4 * case["dims"],
                "flops": 3 * case["tokens"] * turned * case["dims"]}
    if op == "chunk":
        req, H, G, D = _requests(case), case["heads"], case["kv_heads"], case["head_dim"]
        new, tokens = sum(n for _, n in req), sum(w + n for w, n in req)
        return {"bytes": 2 * new * H * D * size + 4 * new * H + 2 * tokens * G * D * size + 8 * case["batch"] + 4 * tokens // case["page"],
                "flops": 4 * H * D * sum(_seen(w, n) for w, n in req)}
    return {"bytes": case["rows"] * (case["vocab"] * size + 8 + (4 if case["entropy"] else 0) + 8 * case["top"]),
            "flops": (5 if case["entropy"] else 3) * case["rows"] * case["vocab"]}


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op == "extend":
        page, free, wide = case["page"], st["free"].tolist(), st["table"].shape[1]
        table, at, starts, positions, slots = st["table"].tolist(), 0, [0], [], []
        for row, (was, new) in zip(table, _requests(case)):
            for j in range(-(-was // page), -(-(was + new) // page)):
                row[j] = free[at]
                at += 1
            starts.append(starts[-1] + new)
            positions += range(was, was + new)
            slots += [row[p // page] * page + p % page for p in range(was, was + new)]
        pad = [-1] * case["spare"]
        return {"table": torch.tensor(table, dtype=torch.int32), "lengths": torch.tensor([w + n for w, n in _requests(case)], dtype=torch.int32),
                "starts": torch.tensor(starts, dtype=torch.int32), "positions": torch.tensor(positions + pad, dtype=torch.int32),
                "slots": torch.tensor(slots + pad), "used": torch.tensor([at], dtype=torch.int32)}
    if op == "rotary":
        f = st["frequencies"]
        n, d = len(f), 2 * len(f)
        turn = torch.polar(torch.ones(case["tokens"], n, dtype=torch.float64, device="cuda"), st["positions"].double()[:, None] * f)[:, None]
        first = torch.arange(0, d, 2, device="cuda") if case["layout"] == "pairs" else torch.arange(n, device="cuda")
        second = first + (1 if case["layout"] == "pairs" else n)

        def turned(x):
            y = x.double()
            z = torch.complex(y[..., first], y[..., second]) * turn
            y[..., first], y[..., second] = z.real, z.imag
            return y

        res = {"q": turned(st["q"])}
        if case["write"]:
            k, v = st["k_pages"].double().transpose(1, 2).contiguous(), st["v_pages"].double().transpose(1, 2).contiguous()
            k.flatten(0, 1)[st["slots"]] = turned(st["k"])
            v.flatten(0, 1)[st["slots"]] = st["v"].double()
            res |= {"k_pages": k.transpose(1, 2), "v_pages": v.transpose(1, 2)}
        return res
    if op == "chunk":
        H, G, D, page, at = case["heads"], case["kv_heads"], case["head_dim"], case["page"], 0
        if 4 * H * D * sum(_seen(w, n) for w, n in _requests(case)) > 6e11:
            return None
        out, lse = st["q"].double(), torch.empty(st["q"].shape[:2], dtype=torch.float64, device="cuda")
        for b, (was, new) in enumerate(_requests(case)):
            ids = st["table"][b, :-(-(was + new) // page)].long()
            for g in range(G):
                k, v = (p[ids, g].reshape(-1, D)[:was + new].double() for p in (st["k_pages"], st["v_pages"]))
                for first in range(0, new, 512):
                    n = min(512, new - first)
                    rows, heads, seen = slice(at + first, at + first + n), slice(g * (H // G), (g + 1) * (H // G)), was + first + n
                    s = torch.einsum("thd,kd->thk", st["q"][rows, heads].double(), k[:seen]) / math.sqrt(D)
                    hidden = torch.arange(seen, device="cuda") > was + first + torch.arange(n, device="cuda")[:, None]
                    s[hidden[:, None].expand_as(s)] = -math.inf
                    lse[rows, heads] = torch.logsumexp(s, -1)
                    out[rows, heads] = torch.einsum("thk,kd->thd", torch.softmax(s, -1), v[:seen])
            at += new
        return {"out": out, "lse": lse}
    res = {"logprobs": [], "entropy": [], "top_logprobs": [], "top_tokens": []}
    for x, token in zip(st["logits"], st["tokens"].tolist()):
        p = torch.log_softmax(x.double(), -1)
        res["logprobs"].append(p[token])
        if case["entropy"]:
            res["entropy"].append(-torch.where(p > -math.inf, p.exp() * p, 0).sum())
        if case["top"]:
            least = torch.topk(p, case["top"]).values[-1]
            at = torch.nonzero(p >= least)[:, 0]
            at = at[torch.argsort(p[at], descending=True, stable=True)][:case["top"]]
            res["top_logprobs"].append(p[at])
            res["top_tokens"].append(at.to(torch.int32))
    return {name: torch.stack(rows) for name, rows in res.items() if rows}

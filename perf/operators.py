"""Operators of a paged key / value cache and of beam search, as cases that can be timed and compared.

A case names an operator and its sizes:

* "attend":  attention of one new token per sequence over a cache in pages, for some cases with the new key and value written
             into the cache by the same call;
* "write":   keys and values of a padded batch of prompts (or of one token each) into their pages;
* "copy":    whole pages of a list of pools (a layer's keys, a layer's values, ...) to other pages;
* "select":  the best continuations over beams and vocabulary, from logits and the beams' scores;
* "reorder": rows of a list of states exchanged in place so that every beam has its parent's.

With `own` false `run` computes them from elementary torch operations, else through the package's entry points.  Both take
the same state: device tensors that a serving program holds before the call.
"""
import math
import random

import torch

own = False

_DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


# ---------------------------------------------------------------------------------------------------------- the cases
def _attend(dtype, batch, heads, kv_heads, head_dim, longest, page, ragged, append):
    return {"op": "attend", "dtype": dtype, "batch": batch, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim,
            "longest": longest, "page": page, "ragged": ragged, "append": append}


def _write(dtype, batch, tokens, kv_heads, head_dim, page):
    return {"op": "write", "dtype": dtype, "batch": batch, "tokens": tokens, "kv_heads": kv_heads, "head_dim": head_dim, "page": page}


def _copy(dtype, pools, pages, moved, page, kv_heads, head_dim):
    return {"op": "copy", "dtype": dtype, "pools": pools, "pages": pages, "moved": moved, "page": page, "kv_heads": kv_heads,
            "head_dim": head_dim}


def _select(dtype, batch, beams, vocab, best, done):
    return {"op": "select", "dtype": dtype, "batch": batch, "beams": beams, "vocab": vocab, "best": best, "done": done}


def _reorder(dtype, tensors, batch, beams, kept, heads, rows, width):
    return {"op": "reorder", "dtype": dtype, "tensors": tensors, "batch": batch, "beams": beams, "kept": kept, "heads": heads,
            "rows": rows, "width": width}


def listed():
    return [
        # one user's next token behind a short chat, 8B attention shape: the call that latency decides
        dict(_attend("bfloat16", 1, 32, 8, 128, 701, 16, False, True), name="attend-one-short"),
        # a served batch of unequal lengths, 1B attention shape, the new token's key and value written by the call
        dict(_attend("float16", 48, 32, 8, 64, 4001, 32, True, True), name="attend-batch-ragged"),
        # one document of 131072 tokens, 8B attention shape: a single sequence has to fill the machine
        dict(_attend("bfloat16", 1, 32, 8, 128, 131072, 64, False, False), name="attend-one-long"),
        # the small fp32 model (6 heads of 48) served to 256 users, every context within its 256 positions
        dict(_attend("float32", 256, 6, 6, 48, 256, 16, True, True), name="attend-small-fp32"),
        # a decode step's keys and values of 32 users
        dict(_write("bfloat16", 32, 1, 8, 128, 16), name="write-step"),
        # prompts of unequal lengths, padded into one batch
        dict(_write("bfloat16", 7, 2047, 8, 128, 16), name="write-prompts"),
        # copy-on-write: beams that share a half-filled page each get their own, both pools of one layer
        dict(_copy("bfloat16", 2, 512, 24, 16, 8, 128), name="copy-shared-pages"),
        # compaction: the pools of eight layers close the gaps that finished sequences left
        dict(_copy("bfloat16", 16, 3001, 1201, 16, 8, 128), name="copy-compact"),
        # one prompt, four beams, the small model's vocabulary
        dict(_select("float32", 1, 4, 32000, 4, False), name="select-one-prompt"),
        # thirty-two prompts of eight beams over the Llama 3 vocabulary, some beams finished
        dict(_select("float32", 32, 8, 128256, 8, True), name="select-batch"),
        # what beam search moves when its cache is in pages: tables and token histories of a few beams
        dict(_reorder("int32", 2, 4, 5, 3, 1, 1, 511), name="reorder-tables"),
        # recurrent states (16 heads of 128 x 128) of six layers, sixteen prompts of four beams
        dict(_reorder("float32", 6, 16, 4, 2, 16, 128, 128), name="reorder-states"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "write", "copy", "select", "reorder"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    if op in ("attend", "write", "copy"):
        head_dim = rng.choice([32, 48, 64, 64, 96, 128, 128])
        kv_heads = rng.choice([1, 2, 3, 4, 6, 8, 8])
        page = rng.choice([1, 8, 16, 16, 32, 64, 128])
        size = 4 if dtype == "float32" else 2
        token = kv_heads * head_dim * size      # bytes of one token's keys
    if op == "attend":
        group = rng.choice([1, 1, 2, 3, 4, 4, 7, 8])
        batch = _log(rng, 1, 256)
        most = max(2, min(40000, (1 << 28) // (token * batch * 2)))
        return _attend(dtype, batch, kv_heads * group, kv_heads, head_dim, _log(rng, 1, most), page, rng.random() < 0.7,
                       rng.random() < 0.5)
    if op == "write":
        batch = _log(rng, 1, 64)
        return _write(dtype, batch, _log(rng, 1, max(2, min(4000, (1 << 25) // (token * batch)))), kv_heads, head_dim, page)
    if op == "copy":
        page = max(page, 8)
        pools = 2 * _log(rng, 1, 8)
        pages = _log(rng, 16, max(17, min(4000, (1 << 28) // (page * token * pools))))
        return _copy(dtype, pools, pages, _log(rng, 1, pages // 2 - 1), page, kv_heads, head_dim)
    if op == "select":
        beams = _log(rng, 1, 16)
        return _select(dtype, _log(rng, 1, max(2, 128 // beams)), beams, _log(rng, 500, 128256), rng.choice([beams, beams, 2 * beams]),
                       beams > 1 and rng.random() < 0.5)
    beams = _log(rng, 2, 16)
    heads, rows, width = rng.choice([(1, 1, _log(rng, 1, 4000)), (_log(rng, 1, 16), _log(rng, 1, 128), 8 * _log(rng, 1, 24)),
                                     (_log(rng, 1, 16), _log(rng, 1, 100), _log(rng, 1, 150))])
    return _reorder(rng.choice(["float32", "bfloat16", "int32"]), _log(rng, 1, 6), _log(rng, 1, max(2, 64 // beams)), beams,
                    rng.randint(1, beams - 1), heads, rows, width)


# ------------------------------------------------------------------------------------------------------------- inputs
def _lengths(case):
    """Tokens per sequence, the new one included; a function of the case, so that work() can count them."""
    n, top = case["batch"], case["longest"]
    if not case["ragged"]:
        return [top] * n
    return [top if b == 0 else 1 + int((top - 1) * math.modf(b * 0.6180339887498949)[0]) for b in range(n)]


def _counts(case):
    """Real tokens per row of a padded batch of prompts."""
    n, top = case["batch"], case["tokens"]
    return [top if b == 0 else 1 + int((top - 1) * math.modf(b * 0.6180339887498949)[0]) for b in range(n)]


def _tables(rng, page_counts, spare):
    """Page tables whose pages lie in any order, as an allocator leaves them after many requests; unused entries are -1."""
    total = sum(page_counts) + spare
    ids = list(range(total))
    rng.shuffle(ids)
    wide, at, rows = max(max(page_counts), 1), 0, []
    for c in page_counts:
        rows.append(ids[at:at + c] + [-1] * (wide - c))
        at += c
    return torch.tensor(rows, dtype=torch.int32, device="cuda"), total


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed) * 7919 + 17)
    rng = random.Random(int(seed) * 104729 + 5)
    op = case["op"]
    kind = _DTYPES.get(case["dtype"])

    def normal(*shape, to=kind, scale=1.0):
        return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(to)

    if op == "attend":
        lens, page, G, D = _lengths(case), case["page"], case["kv_heads"], case["head_dim"]
        table, total = _tables(rng, [-(-n // page) for n in lens], 3)
        st = {"q": normal(case["batch"], case["heads"], D), "k_pages": normal(total, G, page, D), "v_pages": normal(total, G, page, D),
              "table": table, "lengths": torch.tensor(lens, dtype=torch.int32, device="cuda"), "k_new": None, "v_new": None}
        if case["append"]:
            st["k_new"], st["v_new"] = normal(case["batch"], G, D), normal(case["batch"], G, D)
    elif op == "write":
        counts, page, G, D = _counts(case), case["page"], case["kv_heads"], case["head_dim"]
        starts = [rng.randint(0, 3 * page) for _ in counts]   # behind an earlier portion of the prompt
        table, total = _tables(rng, [3 + -(-n // page) for n in counts], 2)
        st = {"k": normal(case["batch"], case["tokens"], G, D), "v": normal(case["batch"], case["tokens"], G, D),
              "k_pages": normal(total, G, page, D), "v_pages": normal(total, G, page, D), "table": table,
              "start": torch.tensor(starts, dtype=torch.int32, device="cuda"),
              "count": torch.tensor(counts, dtype=torch.int32, device="cuda")}
    elif op == "copy":
        ids = list(range(case["pages"]))
        rng.shuffle(ids)
        n = case["moved"]
        st = {"pools": [normal(case["pages"], case["kv_heads"], case["page"], case["head_dim"]) for _ in range(case["pools"])],
              "src": torch.tensor(ids[:n], dtype=torch.int32, device="cuda"),
              "dst": torch.tensor(ids[n:2 * n], dtype=torch.int32, device="cuda")}
    elif op == "select":
        B, K = case["batch"], case["beams"]
        done = None
        if case["done"]:
            done = (torch.arange(B * K, device="cuda") % 7 == 3).reshape(B, K)
        scores = (-torch.rand(B, K, generator=gen, device="cuda") * 3 - 9).sort(dim=1, descending=True).values.contiguous()
        st = {"logits": normal(B, K, case["vocab"], scale=2.5), "scores": scores, "best": case["best"], "done": done, "eos": 2}
    else:
        B, K, keep = case["batch"], case["beams"], case["kept"]
        shape = (B * K, case["heads"], case["rows"], case["width"])
        # the beams that live on keep their rows, the others' rows become copies of theirs: a second pass changes nothing
        parents = []
        for _ in range(B):
            order = list(range(K))
            rng.shuffle(order)
            live, row = order[:keep], list(range(K))
            for i, j in enumerate(order[keep:]):
                row[j] = live[i % keep]
            parents.append(row)
        if kind is None:
            tensors = [torch.randint(0, 1 << 20, shape, generator=gen, device="cuda", dtype=torch.int32) for _ in range(case["tensors"])]
        else:
            tensors = [normal(*shape) for _ in range(case["tensors"])]
        st = {"states": tensors, "parents": torch.tensor(parents, dtype=torch.int32, device="cuda")}
    st["op"] = op
    return st


# --------------------------------------------------------------------------------------------------------- plain forms
def _plain_attend(st):
    q, kp, vp, table, lens = st["q"], st["k_pages"], st["v_pages"], st["table"].long(), st["lengths"].long()
    B, H, D = q.shape
    G, page = kp.shape[1], kp.shape[2]
    if st["k_new"] is not None:
        at = lens - 1
        ids = table.gather(1, (at // page)[:, None])[:, 0]
        kp[ids, :, at % page] = st["k_new"]
        vp[ids, :, at % page] = st["v_new"]
    pos = torch.arange(table.shape[1] * page, device=q.device)
    ids = table.clamp(min=0)
    k = kp[ids].permute(0, 2, 1, 3, 4).reshape(B, G, -1, D).float()     # [B, G, positions, D]
    v = vp[ids].permute(0, 2, 1, 3, 4).reshape(B, G, -1, D).float()
    s = torch.matmul(q.reshape(B, G, H // G, D).float(), k.transpose(2, 3)) * D ** -0.5
    s = s.masked_fill((pos[None] >= lens[:, None])[:, None, None], float("-inf"))
    top = s.amax(-1, keepdim=True)
    e = torch.exp(s - top)
    total = e.sum(-1, keepdim=True)
    out = (torch.matmul(e, v) / total).reshape(B, H, D).to(q.dtype)
    return out, (top + torch.log(total)).reshape(B, H)


def _plain_write(st):
    k, v, table, start, count = st["k"], st["v"], st["table"].long(), st["start"].long(), st["count"].long()
    page = st["k_pages"].shape[2]
    t = torch.arange(k.shape[1], device=k.device)
    b, t = torch.nonzero(t[None] < count[:, None], as_tuple=True)
    at = start[b] + t
    ids = table[b, at // page]
    st["k_pages"][ids, :, at % page] = k[b, t]
    st["v_pages"][ids, :, at % page] = v[b, t]


def _plain_select(st):
    # in 64 bits: the order of two candidates hangs on the last bits of their sums
    B, K, V = st["logits"].shape
    x = st["logits"].double()
    top = x.amax(-1, keepdim=True)
    logp = x - (top + torch.log(torch.exp(x - top).sum(-1, keepdim=True)))
    s = st["scores"].double()[..., None] + logp
    if st["done"] is not None:
        rest = torch.full_like(s, float("-inf"))
        rest[..., st["eos"]] = st["scores"].double()
        s = torch.where(st["done"][..., None], rest, s)
    val, idx = s.reshape(B, K * V).sort(dim=1, descending=True, stable=True)   # stable: ties go to the lowest index
    val, idx = val[:, :st["best"]], idx[:, :st["best"]]
    parents, tokens = idx // V, idx % V
    over = tokens == st["eos"]
    if st["done"] is not None:
        over = over | st["done"].gather(1, parents)
    return val.float(), tokens.to(torch.int32), parents.to(torch.int32), over


def run(st):
    op = st["op"]
    if own:
        import llama3_np_b200 as l3
    if op == "attend":
        if own:
            out, lse = l3.paged_attention(st["q"], st["k_pages"], st["v_pages"], st["table"], st["lengths"], k_new=st["k_new"],
                                          v_new=st["v_new"], return_lse=True)
        else:
            out, lse = _plain_attend(st)
        res = {"out": out, "lse": lse}
        if st["k_new"] is not None:
            res["k_pages"], res["v_pages"] = st["k_pages"], st["v_pages"]
        return res
    if op == "write":
        if own:
            l3.paged_write(st["k"], st["v"], st["k_pages"], st["v_pages"], st["table"], st["start"], st["count"])
        else:
            _plain_write(st)
        return {"k_pages": st["k_pages"], "v_pages": st["v_pages"]}
    if op == "copy":
        if own:
            l3.copy_pages(st["pools"], st["src"], st["dst"])
        else:
            src, dst = st["src"].long(), st["dst"].long()
            for p in st["pools"]:
                p[dst] = p[src]
        return {"pools": st["pools"]}
    if op == "select":
        if own:
            scores, tokens, parents, done = l3.beam_select(st["logits"], st["scores"], st["best"], done=st["done"], eos_id=st["eos"])
        else:
            scores, tokens, parents, done = _plain_select(st)
        return {"scores": scores, "tokens": tokens, "parents": parents, "done": done}
    if own:
        l3.beam_reorder(st["states"], st["parents"])
    else:
        B, K = st["parents"].shape
        rows = (st["parents"].long() + torch.arange(0, B * K, K, device=st["parents"].device)[:, None]).reshape(-1)
        for x in st["states"]:
            x.copy_(x[rows])
    return {"states": st["states"]}


# -------------------------------------------------------------------------------------------------- work and definition
def work(case):
    op = case["op"]
    size = 2 if case["dtype"] in ("bfloat16", "float16") else 4
    if op == "attend":
        n, B, H, G, D = sum(_lengths(case)), case["batch"], case["heads"], case["kv_heads"], case["head_dim"]
        moved = 2 * n * G * D * size + 2 * B * H * D * size + 4 * B * (1 + -(-case["longest"] // case["page"])) + 4 * B * H
        if case["append"]:
            moved += 2 * B * G * D * size       # the new rows are written; read, they stand for the cache's own last rows
        return {"bytes": moved, "flops": 4 * n * H * D}
    if op == "write":
        n = sum(_counts(case))
        return {"bytes": 4 * n * case["kv_heads"] * case["head_dim"] * size + 4 * n // case["page"] + 8 * case["batch"], "flops": 0}
    if op == "copy":
        return {"bytes": 2 * case["pools"] * case["moved"] * case["page"] * case["kv_heads"] * case["head_dim"] * size + 8 * case["moved"],
                "flops": 0}
    if op == "select":
        rows = case["batch"] * case["beams"]
        live = rows - (len([i for i in range(rows) if i % 7 == 3]) if case["done"] else 0)
        return {"bytes": live * case["vocab"] * size + 5 * rows + 13 * case["batch"] * case["best"], "flops": 3 * live * case["vocab"]}
    row = case["heads"] * case["rows"] * case["width"] * size
    dead, read = case["beams"] - case["kept"], min(case["kept"], case["beams"] - case["kept"])
    return {"bytes": case["tensors"] * case["batch"] * (dead + read) * row + 4 * case["batch"] * case["beams"], "flops": 0}


def _slot(table, b, position, page):
    return int(table[b][position // page]), position % page


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op == "attend":
        table, lens, page = st["table"].tolist(), st["lengths"].tolist(), case["page"]
        kp, vp = st["k_pages"], st["v_pages"]
        if case["append"]:
            for b, n in enumerate(lens):
                p, o = _slot(table, b, n - 1, page)
                kp[p, :, o], vp[p, :, o] = st["k_new"][b], st["v_new"][b]
        H, G, D = case["heads"], case["kv_heads"], case["head_dim"]
        out = torch.empty(case["batch"], H, D, dtype=torch.float64, device="cuda")
        lse = torch.empty(case["batch"], H, dtype=torch.float64, device="cuda")
        for b, n in enumerate(lens):
            ids = st["table"][b, :-(-n // page)].long()
            for g in range(G):
                k = kp[ids, g].reshape(-1, D)[:n].double()
                v = vp[ids, g].reshape(-1, D)[:n].double()
                heads = slice(g * (H // G), (g + 1) * (H // G))
                s = (st["q"][b, heads].double() @ k.T) / math.sqrt(D)
                lse[b, heads] = torch.logsumexp(s, -1)
                out[b, heads] = torch.softmax(s, -1) @ v
        res = {"out": out, "lse": lse}
        if case["append"]:
            res["k_pages"], res["v_pages"] = kp, vp
        return res
    if op == "write":
        table, page = st["table"].tolist(), case["page"]
        for b, (s, n) in enumerate(zip(st["start"].tolist(), st["count"].tolist())):
            t = 0
            while t < n:                        # as far as the page goes
                p, o = _slot(table, b, s + t, page)
                m = min(page - o, n - t)
                st["k_pages"][p, :, o:o + m] = st["k"][b, t:t + m].transpose(0, 1)
                st["v_pages"][p, :, o:o + m] = st["v"][b, t:t + m].transpose(0, 1)
                t += m
        return {"k_pages": st["k_pages"], "v_pages": st["v_pages"]}
    if op == "copy":
        moves = list(zip(st["src"].tolist(), st["dst"].tolist()))
        res = []
        for p in st["pools"]:
            order = list(range(case["pages"]))
            for a, b in moves:
                order[b] = a
            res.append(p.index_select(0, torch.tensor(order, device="cuda")))
        return {"pools": res}
    if op == "select":
        B, K, V = st["logits"].shape
        scores, tokens, parents, done = [], [], [], []
        was = st["done"].tolist() if st["done"] is not None else [[False] * K] * B
        for b in range(B):
            every = []
            for j in range(K):
                if was[b][j]:
                    every.append((-float(st["scores"][b, j]), j, st["eos"]))
                    continue
                logp = torch.log_softmax(st["logits"][b, j].double(), -1) + st["scores"][b, j].double()
                least = torch.topk(logp, min(V, case["best"])).values[-1]
                for t in torch.nonzero(logp >= least)[:, 0].tolist():
                    every.append((-float(logp[t]), j, t))
            every = sorted(every)[:case["best"]]
            scores.append([-e[0] for e in every])
            parents.append([e[1] for e in every])
            tokens.append([e[2] for e in every])
            done.append([was[b][e[1]] or e[2] == st["eos"] for e in every])
        if any(len(r) != case["best"] for r in scores):
            return None
        return {"scores": torch.tensor(scores, dtype=torch.float64), "tokens": torch.tensor(tokens, dtype=torch.int32),
                "parents": torch.tensor(parents, dtype=torch.int32), "done": torch.tensor(done)}
    K = case["beams"]
    rows = [b * K + p for b, row in enumerate(st["parents"].tolist()) for p in row]
    return {"states": [torch.stack([x[r] for r in rows]) for x in st["states"]]}

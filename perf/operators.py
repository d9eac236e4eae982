"""Cases of the operators over the paged K/V cache: the page plan of a ragged batch,
the store of new key and value rows, attention of new tokens over the cached ones,
and beam search's selection and cache reordering.

``run`` with ``own`` false computes each in elementary torch operations (fp32, or 64
bits for the beam totals); with ``own`` true it makes the calls of ``tie_b200.ops``.
"""
import math
import os
import random
import sys

import torch

own = False

PAGE = 16          # positions of a page
D = 64             # head dimension of the engine
VOCAB = 50257      # GPT-2's vocabulary
ERR_CAPACITY = 8   # MODEL_ERR_CAPACITY


def _ops():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    pkg = os.path.join(root, "transformer-inference-engine_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from tie_b200 import ops
    return ops


# ------------------------------------------------------------------ the cases

def listed():
    return [
        # a decode step of 256 sequences: one new position each, GPT-2's context
        {"name": "plan_decode_256", "op": "plan", "n_seq": 256, "ctx_max": 1023, "new_min": 1, "new_max": 1},
        # a serving step of many requests, prompts of up to 96 tokens among them
        {"name": "plan_ragged_1500", "op": "plan", "n_seq": 1500, "ctx_max": 4000, "new_min": 0, "new_max": 96},
        # the K/V rows of a decode step (GPT-2 small, fp32 pages)
        {"name": "store_decode_256", "op": "store", "rows": 256, "kv_heads": 12, "kv": "f32"},
        # the K/V rows of a large prompt batch into bf16 pages (GPT-2 medium's width)
        {"name": "store_prompt_bf16", "op": "store", "rows": 16391, "kv_heads": 16, "kv": "bf16"},
        # one sequence, one token: latency (GPT-2 small at its full context)
        {"name": "attn_decode_1", "op": "attention", "n_seq": 1, "ctx_max": 1023, "new_min": 1, "new_max": 1,
         "heads": 12, "kv_heads": 12, "kv": "f32"},
        # a decode batch of ragged contexts
        {"name": "attn_decode_256", "op": "attention", "n_seq": 256, "ctx_max": 1000, "new_min": 1, "new_max": 1,
         "heads": 12, "kv_heads": 12, "kv": "f32"},
        # a step that mixes decoding sequences with prompt chunks (GPT-2 XL's 25 heads)
        {"name": "attn_mixed_48", "op": "attention", "n_seq": 48, "ctx_max": 900, "new_min": 0, "new_max": 117,
         "heads": 25, "kv_heads": 25, "kv": "f32"},
        # a long prompt's next chunk over bf16 pages, four query heads to a K/V head
        {"name": "attn_chunk_long_bf16", "op": "attention", "n_seq": 1, "ctx_max": 14336, "new_min": 2048,
         "new_max": 2048, "heads": 32, "kv_heads": 8, "kv": "bf16"},
        # one request, four beams: latency
        {"name": "select_1x4", "op": "select", "n_req": 1, "beams": 4, "vocab": VOCAB},
        # a batch of requests, six beams each
        {"name": "select_96x6", "op": "select", "n_req": 96, "beams": 6, "vocab": VOCAB},
        # a few generated positions of one request (GPT-2 small, every layer)
        {"name": "reorder_2x4", "op": "reorder", "n_req": 2, "beams": 4, "layers": 12, "kv_heads": 12, "kv": "f32",
         "first": 61, "length": 98},
        # long generations of a batch of beams
        {"name": "reorder_24x5", "op": "reorder", "n_req": 24, "beams": 5, "layers": 12, "kv_heads": 12, "kv": "f32",
         "first": 64, "length": 401},
    ]


def _log(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["plan", "store", "attention", "attention", "select", "reorder"])
    if op == "plan":
        lo = rng.choice([0, 1])
        return {"op": op, "n_seq": _log(rng, 1, 1500), "ctx_max": _log(rng, 1, 4000), "new_min": lo,
                "new_max": max(lo, _log(rng, 1, 96))}
    if op == "store":
        return {"op": op, "rows": _log(rng, 1, 16391), "kv_heads": rng.choice([1, 2, 5, 8, 12, 16]),
                "kv": rng.choice(["f32", "bf16"])}
    if op == "attention":
        group = rng.choice([1, 1, 2, 4, 8])
        kv_heads = rng.choice([1, 2, 8, 12, 16, 25]) if group == 1 else rng.choice([1, 2, 3, 8])
        kind = rng.choice(["decode", "chunk", "mixed"])
        c = {"op": op, "heads": group * kv_heads, "kv_heads": kv_heads, "kv": rng.choice(["f32", "bf16"])}
        if kind == "decode":
            c |= {"n_seq": _log(rng, 1, 256), "ctx_max": _log(rng, 1, 4000), "new_min": 1, "new_max": rng.choice([1, 1, 2])}
        elif kind == "chunk":
            new = _log(rng, 3, 1500)
            c |= {"n_seq": rng.choice([1, 2, 4]), "ctx_max": _log(rng, 1, 7000), "new_min": new, "new_max": new}
        else:
            c |= {"n_seq": _log(rng, 2, 48), "ctx_max": _log(rng, 16, 1500), "new_min": rng.choice([0, 1]),
                  "new_max": _log(rng, 8, 300)}
        # no dearer than the largest listed case: shorter contexts, then fewer sequences
        while _attention_cost(c) > 1.0 and c["ctx_max"] > 64:
            c["ctx_max"] = c["ctx_max"] * 2 // 3
        while _attention_cost(c) > 1.0 and c["n_seq"] > 1:
            c["n_seq"] = c["n_seq"] * 2 // 3
        return c
    if op == "select":
        beams = rng.choice([1, 2, 3, 4, 5, 8])
        return {"op": op, "n_req": _log(rng, 1, 576 // beams), "beams": beams, "vocab": rng.choice([VOCAB, 32000, 16411, 999])}
    beams = rng.choice([2, 3, 4, 5])
    first = rng.randrange(0, 300)
    return {"op": op, "n_req": _log(rng, 1, 24), "beams": beams, "layers": rng.choice([1, 4, 12]),
            "kv_heads": rng.choice([2, 8, 12]), "kv": rng.choice(["f32", "bf16"]), "first": first,
            "length": first + _log(rng, 1, 330)}


def _attention_cost(c):
    """Work of a case against the largest listed one's, by products and by cache bytes."""
    pairs = c["n_seq"] * c["new_max"] * (c["ctx_max"] + c["new_max"]) * c["heads"]
    cache = c["n_seq"] * (c["ctx_max"] + c["new_max"]) * c["kv_heads"]
    return max(pairs / (2048 * 16384 * 32), cache / (256 * 1001 * 12))


def _lengths(case):
    """Each sequence's cached and new positions: a part of the case, the same for every seed."""
    r = random.Random(str(sorted(case.items())))
    n = case["n_seq"]
    if n == 1:
        return [case["ctx_max"]], [case["new_max"]]
    ctx = [r.randint(0, case["ctx_max"]) for _ in range(n)]
    new = [r.randint(case["new_min"], case["new_max"]) for _ in range(n)]
    ctx[r.randrange(n)] = case["ctx_max"]
    new[r.randrange(n)] = case["new_max"]
    return ctx, new


def _parents(case):
    """Each beam's parent (as beam_select places them: a beam with children keeps its own place)."""
    r = random.Random(str(sorted(case.items())))
    k, out = case["beams"], []
    for q in range(case["n_req"]):
        alive = sorted(r.sample(range(k), r.randint(1, k)))
        out += [q * k + (b if b in alive else r.choice(alive)) for b in range(k)]
    return out


def _pages_of(length):
    return (length + PAGE - 1) // PAGE


# ------------------------------------------------------------------ the inputs

def _rand(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 1000003 + len(str(case)))
    return g


def _int32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _kv_type(case):
    return torch.bfloat16 if case["kv"] == "bf16" else torch.float32


def _normal(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device="cuda", dtype=dtype)


def prepare(case, seed):
    return {"plan": _plan_inputs, "store": _store_inputs, "attention": _attention_inputs, "select": _select_inputs,
            "reorder": _reorder_inputs}[case["op"]](case, seed)


def _tables(counts, width, n_pages, g):
    """Page tables whose pages lie anywhere in the pool; unused entries name the pool's last page."""
    used = sum(counts)
    perm = torch.randperm(n_pages - 1, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(counts), width), n_pages - 1, dtype=torch.int32, device="cuda")
    mask = torch.arange(width, device="cuda")[None, :] < _int32(counts)[:, None]
    table[mask] = perm[:used]
    return table, perm[used:]


def _plan_inputs(case, seed):
    g = _rand(case, seed)
    ctx, new = _lengths(case)
    width = max(_pages_of(c + n) for c, n in zip(ctx, new))
    have = [_pages_of(c) for c in ctx]
    need = sum(_pages_of(c + n) for c, n in zip(ctx, new)) - sum(have)
    n_pages = sum(have) + need + 1 + max(8, need // 4)
    table, free = _tables(have, width, n_pages, g)
    # a fixed-size step: rows behind the last sequence's stay marked as none
    rows = max(1, sum(new) + max(1, sum(new) // 16))
    out = lambda n: torch.empty(n, dtype=torch.int32, device="cuda")  # noqa: E731
    return {"op": "plan", "ctx": _int32(ctx), "new": _int32(new), "table": table, "n_pages": n_pages,
            "free": free.contiguous(), "n_free": _int32([free.numel()]), "n_free_out": out(1), "row_start": out(len(ctx) + 1),
            "seq_of": out(rows), "pos_of": out(rows), "slots": out(rows), "status": out(1), "rows": rows}


def _store_inputs(case, seed):
    g = _rand(case, seed)
    rows, w = case["rows"], case["kv_heads"] * D
    n_pages = _pages_of(rows) + 4
    k_pages = _normal(g, n_pages, PAGE, w).to(_kv_type(case))
    v_pages = _normal(g, n_pages, PAGE, w).to(_kv_type(case))
    # the rows of a fused projection: query, key and value side by side
    qkv = _normal(g, rows, 3 * w)
    slots = torch.randperm(n_pages * PAGE, generator=g, device="cuda")[:rows].to(torch.int32)
    return {"op": "store", "k_pages": k_pages, "v_pages": v_pages, "k": qkv[:, w:2 * w], "v": qkv[:, 2 * w:],
            "slots": slots}


def _attention_inputs(case, seed):
    g = _rand(case, seed)
    ctx, new = _lengths(case)
    counts = [_pages_of(c + n) for c, n in zip(ctx, new)]
    n_pages = sum(counts) + 2
    w = case["kv_heads"] * D
    table, _ = _tables(counts, max(counts), n_pages, g)
    k_pages = _normal(g, n_pages, PAGE, w).to(_kv_type(case))
    v_pages = _normal(g, n_pages, PAGE, w).to(_kv_type(case))
    rows = sum(new)
    start = [0]
    for n in new:
        start.append(start[-1] + n)
    seq_of = torch.repeat_interleave(torch.arange(len(new), device="cuda"), torch.tensor(new, device="cuda"))
    off = torch.arange(rows, device="cuda") - torch.tensor(start, device="cuda")[seq_of]
    # scores of a trained model are sharper than random rows': a standard deviation of 2
    q = 2.0 * _normal(g, rows, case["heads"] * D)
    return {"op": "attention", "q": q, "k_pages": k_pages, "v_pages": v_pages, "table": table, "heads": case["heads"],
            "kv_heads": case["kv_heads"], "ctx": _int32(ctx), "row_start": _int32(start), "seq_of": seq_of, "off": off,
            "new_max": max(new), "n_pages": n_pages, "out": torch.empty_like(q),
            "work": torch.empty(96 << 20, dtype=torch.uint8, device="cuda"), "status": torch.zeros(1, dtype=torch.int32, device="cuda")}


def _select_inputs(case, seed):
    g = _rand(case, seed)
    n = case["n_req"] * case["beams"]
    logits = 3.0 * _normal(g, n, case["vocab"])
    scores = -20.0 * torch.rand(n, generator=g, device="cuda")
    done = (torch.rand(n, generator=g, device="cuda") < 0.1).to(torch.int32)
    out = lambda t: torch.empty(n, dtype=t, device="cuda")  # noqa: E731
    return {"op": "select", "logits": logits, "scores": scores, "done": done, "beams": case["beams"],
            "eos": case["vocab"] - 1, "next": out(torch.int32), "parent": out(torch.int32), "scores_out": out(torch.float32),
            "done_out": out(torch.int32), "work": torch.empty(64 << 20, dtype=torch.uint8, device="cuda")}


def _reorder_inputs(case, seed):
    g = _rand(case, seed)
    n, w, layers = case["n_req"] * case["beams"], case["kv_heads"] * D, case["layers"]
    per = _pages_of(case["length"])
    n_pages = n * per + 1
    table, _ = _tables([per] * n, per, n_pages, g)
    return {"op": "reorder", "k_pages": _normal(g, layers, n_pages, PAGE, w).to(_kv_type(case)),
            "v_pages": _normal(g, layers, n_pages, PAGE, w).to(_kv_type(case)), "table": table, "beams": case["beams"],
            "parent": _int32(_parents(case)), "first": _int32([case["first"]] * case["n_req"]),
            "length": _int32([case["length"]] * case["n_req"])}


# ------------------------------------------------------------------ one pass

def run(s):
    op = s["op"]
    if own:
        return _own(op, s, _ops())
    return {"plan": _plain_plan, "store": _plain_store, "attention": _plain_attention, "select": _plain_select,
            "reorder": _plain_reorder}[op](s)


def _own(op, s, ops):
    if op == "plan":
        ops.page_plan(s["ctx"], s["new"], s["table"], s["n_pages"], s["row_start"], s["seq_of"], s["pos_of"], s["slots"],
                      s["status"], free_pages=s["free"], n_free=s["n_free"], n_free_out=s["n_free_out"])
        return [s["table"], s["n_free_out"], s["row_start"], s["seq_of"], s["pos_of"], s["slots"], s["status"]]
    if op == "store":
        ops.kv_store(s["k"], s["v"], s["slots"], s["k_pages"], s["v_pages"])
        return [s["k_pages"], s["v_pages"]]
    if op == "attention":
        ops.attention_paged(s["q"], s["k_pages"], s["v_pages"], s["table"], s["row_start"], s["ctx"], s["new_max"],
                            s["out"], s["work"], status=s["status"])
        return s["out"]
    if op == "select":
        ops.beam_select(s["logits"], s["scores"], s["beams"], s["next"], s["parent"], s["scores_out"], s["work"],
                        done=s["done"], done_out=s["done_out"], eos_id=s["eos"])
        return [s["next"], s["parent"], s["scores_out"], s["done_out"]]
    ops.kv_reorder(s["k_pages"], s["v_pages"], s["table"], s["parent"], s["first"], s["length"], s["beams"])
    return [s["k_pages"], s["v_pages"]]


def _plain_plan(s):
    ctx, new, table = s["ctx"].long(), s["new"].long(), s["table"]
    width, rows = table.shape[1], s["rows"]
    have, want = (ctx + PAGE - 1) // PAGE, (ctx + new + PAGE - 1) // PAGE
    need = want - have
    last = torch.cumsum(need, 0)
    n_free = s["n_free"].long()
    ends = torch.cumsum(new, 0)
    ok = (last[-1:] <= n_free) & (want.max() <= width) & (ends[-1:] <= rows)
    col = torch.arange(width, device=table.device)[None, :]
    at = n_free - 1 - ((last - need)[:, None] + col - have[:, None])
    fresh = (col >= have[:, None]) & (col < want[:, None]) & ok
    table = torch.where(fresh, s["free"][at.clamp(0, s["free"].numel() - 1)], table)
    start = torch.cat([torch.zeros_like(ends[:1]), ends]) * ok
    r = torch.arange(rows, device=table.device)
    seq = torch.searchsorted(start[1:], r, right=True)
    live = r < start[-1]
    at_seq = seq.clamp(max=len(ctx) - 1)
    pos = ctx[at_seq] + r - start[at_seq]
    page = table[at_seq, (pos // PAGE).clamp(0, width - 1)].long()
    mapped = live & (page >= 0) & (page < s["n_pages"])
    slot = torch.where(mapped, page * PAGE + pos % PAGE, -1)
    status = torch.where(ok, 0, ERR_CAPACITY)
    whole = lambda t: t.to(torch.int32)  # noqa: E731
    return [table, whole(n_free - last[-1:] * ok), whole(start), whole(torch.where(live, seq, -1)),
            whole(torch.where(live, pos, -1)), whole(slot), whole(status)]


def _plain_store(s):
    slots = s["slots"].long()
    for_type = s["k_pages"].dtype
    w = s["k_pages"].shape[-1]
    s["k_pages"].view(-1, w)[slots] = s["k"].to(for_type)
    s["v_pages"].view(-1, w)[slots] = s["v"].to(for_type)
    return [s["k_pages"], s["v_pages"]]


def _plain_attention(s):
    table, heads, kv_heads = s["table"].long(), s["heads"], s["kv_heads"]
    n_seq, width = table.shape
    group = heads // kv_heads
    k = s["k_pages"][table].float().view(n_seq, width * PAGE, kv_heads, D)
    v = s["v_pages"][table].float().view(n_seq, width * PAGE, kv_heads, D)
    start, ctx = s["row_start"].long(), s["ctx"].long()
    step = torch.arange(s["new_max"], device=k.device)
    rows = (start[:-1, None] + step).clamp(max=s["q"].shape[0] - 1)
    q = s["q"][rows].view(n_seq, s["new_max"], kv_heads, group, D)
    scores = torch.matmul(q.permute(0, 2, 3, 1, 4), k.permute(0, 2, 3, 1)[:, :, None]) * (1.0 / math.sqrt(D))
    seen = torch.arange(width * PAGE, device=k.device) <= (ctx[:, None] + step)[..., None]
    scores = scores.masked_fill(~seen[:, None, None], float("-inf"))
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    out = torch.matmul(p, v.permute(0, 2, 1, 3)[:, :, None]) / p.sum(-1, keepdim=True)
    out = out.permute(0, 3, 1, 2, 4).reshape(n_seq, s["new_max"], heads * D)
    return out[s["seq_of"], s["off"]]


def _placed(parent, k, *ranked):
    """The best candidates by rank ([requests, k]) put in their places: the first child of a beam in
    that beam's place, the others in the free places in order."""
    same = parent[:, :, None] == parent[:, None, :]
    heir = ~(same & torch.ones(k, k, dtype=torch.bool, device=parent.device).tril(-1)).any(-1)
    taken = torch.zeros_like(parent, dtype=torch.int32).scatter_add(1, parent, heir.to(torch.int32))
    free = torch.argsort(taken, dim=1, stable=True)               # the free places first, in order
    nth = torch.cumsum((~heir).long(), 1) - 1
    place = torch.where(heir, parent, free.gather(1, nth.clamp(min=0)))
    return [torch.empty_like(x).scatter_(1, place, x) for x in ranked]


def _plain_select(s):
    k, vocab = s["beams"], s["logits"].shape[1]
    x = s["logits"].double()
    top = x.amax(1, keepdim=True)
    x = x - (top + torch.log(torch.exp(x - top).sum(1, keepdim=True)))
    done = s["done"].bool()[:, None]
    is_eos = torch.arange(vocab, device=x.device)[None] == s["eos"]
    x = torch.where(done, torch.where(is_eos, 0.0, float("-inf")), x) + s["scores"].double()[:, None]
    best, at = torch.topk(x.view(-1, k * vocab), k, dim=1)
    parent, token = at // vocab, at % vocab
    finished = done.view(-1, k).gather(1, parent) | (token == s["eos"])
    base = torch.arange(parent.shape[0], device=x.device)[:, None] * k
    token, whole, best, finished = _placed(parent, k, token, parent + base, best, finished.long())
    return [token.to(torch.int32).view(-1), whole.to(torch.int32).view(-1), best.float().view(-1),
            finished.to(torch.int32).view(-1)]


def _plain_reorder(s):
    table, parent, k = s["table"].long(), s["parent"].long(), s["beams"]
    n, width = table.shape
    pos = torch.arange(width * PAGE, device=table.device)[None]
    first, length = (s[x].long().repeat_interleave(k)[:, None] for x in ("first", "length"))
    to = table.repeat_interleave(PAGE, 1) * PAGE + pos % PAGE
    moved = (pos >= first) & (pos < length) & (parent != torch.arange(n, device=table.device))[:, None]
    src, to = torch.where(moved, to[parent], to).view(-1), to.view(-1)
    for pages in (s["k_pages"], s["v_pages"]):
        flat = pages.view(pages.shape[0], -1, pages.shape[-1])
        flat[:, to] = flat[:, src]
    return [s["k_pages"], s["v_pages"]]


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    op = case["op"]
    size = 2 if case.get("kv") == "bf16" else 4
    w = case.get("kv_heads", 0) * D
    if op == "plan":
        ctx, new = _lengths(case)
        fresh = sum(_pages_of(c + n) - _pages_of(c) for c, n in zip(ctx, new))
        rows = max(1, sum(new) + max(1, sum(new) // 16))
        return {"bytes": 4 * (3 * len(ctx) + 2 * fresh + 3 * rows), "flops": 0}
    if op == "store":
        return {"bytes": case["rows"] * (2 * w * (4 + size) + 4), "flops": 0}
    if op == "attention":
        ctx, new = _lengths(case)
        cache = sum(c + n for c, n in zip(ctx, new) if n)
        pairs = sum(n * c + n * (n + 1) // 2 for c, n in zip(ctx, new))
        return {"bytes": 2 * cache * w * size + 2 * sum(new) * case["heads"] * D * 4, "flops": 4 * D * case["heads"] * pairs}
    if op == "select":
        n = case["n_req"] * case["beams"]
        return {"bytes": n * (4 * case["vocab"] + 24), "flops": 4 * n * case["vocab"]}
    moved = sum(p != i for i, p in enumerate(_parents(case))) * (case["length"] - case["first"])
    return {"bytes": max(64, 4 * case["layers"] * moved * w * size), "flops": 0}


# ------------------------------------------------------------------ the definitions in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "plan":
        return None                       # whole numbers only
    if op == "store":
        out = []
        for pages, x in ((s["k_pages"], s["k"]), (s["v_pages"], s["v"])):
            flat = pages.double().reshape(-1, pages.shape[-1])
            flat.index_copy_(0, s["slots"].long(), x.double())
            out.append(flat.view(pages.shape))
        return out
    if op == "reorder":
        out = []
        for pages in (s["k_pages"], s["v_pages"]):
            new = pages.double()
            old = new.clone()
            for i, p in enumerate(s["parent"].tolist()):
                for j in range(case["first"] // PAGE, _pages_of(case["length"])) if p != i else ():
                    lo, hi = max(0, case["first"] - PAGE * j), min(PAGE, case["length"] - PAGE * j)
                    new[:, s["table"][i, j], lo:hi] = old[:, s["table"][p, j], lo:hi]
            out.append(new)
        return out
    if op == "select":
        return [None, None, _exact_scores(s), None]
    return _exact_attention(s)


def _exact_scores(s):
    k, (n, vocab) = s["beams"], s["logits"].shape
    out = torch.empty(n, dtype=torch.float64, device="cuda")
    for q in range(n // k):
        cand = []
        for b in range(k):
            i, score = q * k + b, float(s["scores"][q * k + b])
            if int(s["done"][i]):
                cand.append((-score, b * vocab + s["eos"]))
                continue
            x = torch.log_softmax(s["logits"][i].double(), 0)
            v, at = torch.topk(x, min(k, vocab))
            cand += [(-(score + a), b * vocab + t) for a, t in zip(v.tolist(), at.tolist())]
        kept, rest, places = {}, [], set(range(k))
        for c in sorted(cand)[:k]:
            b = c[1] // vocab
            if b in kept:
                rest.append(c)
            else:
                kept[b] = c
                places.discard(b)
        for place, c in zip(sorted(places), rest):
            kept[place] = c
        for b, c in kept.items():
            out[q * k + b] = -c[0]
    return out


def _exact_attention(s):
    heads, kv_heads = s["heads"], s["kv_heads"]
    start, ctx = s["row_start"].tolist(), s["ctx"].tolist()
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for i, c in enumerate(ctx):
        lo, hi = start[i], start[i + 1]
        if hi == lo:
            continue
        n = c + hi - lo
        at = s["table"][i, :_pages_of(n)].long()
        k, v = (p[at].double().reshape(-1, kv_heads, D)[:n] for p in (s["k_pages"], s["v_pages"]))
        hidden = torch.arange(n, device="cuda")[None] > torch.arange(c, n, device="cuda")[:, None]
        for h in range(heads):
            g = h // (heads // kv_heads)
            t = s["q"][lo:hi, h * D:(h + 1) * D].double() @ k[:, g].T / math.sqrt(D)
            t[hidden] = -math.inf
            out[lo:hi, h * D:(h + 1) * D] = torch.softmax(t, 1) @ v[:, g]
    return out

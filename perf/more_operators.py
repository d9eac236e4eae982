"""Cases of the operators for serving from fewer bytes: the 8-bit K/V cache (rows quantised
as they are stored, and read back), attention of a batch whose sequences share their first
positions (over fp32, bf16 or 8-bit pages), 4-bit weights with group scales (made, read back)
and their matrix-vector products.

``run`` with ``own`` false computes each in elementary torch operations (fp32, levels in 64
bits); with ``own`` true it makes the calls of ``tie_b200.ops``. What is held in 8 or 4 bits
comes back as the values it stands for.
"""
import math
import os
import random
import sys

import torch

own = False

PAGE = 16          # positions of a page
D = 64             # head dimension of the engine
BLOCK = 128        # weights of a row that lie together in 64 bytes (4 bits each)


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
        # the K/V rows of a decode step into 8-bit pages, and out again (GPT-2 small)
        {"name": "cache_q8_256", "op": "cache", "rows": 256, "kv_heads": 12},
        # a large prompt batch's rows, read back as a whole to move them (GPT-2 medium's width)
        {"name": "cache_q8_prompt", "op": "cache", "rows": 16391, "kv_heads": 16},
        # one request of four beams, a token each, behind its prompt: latency (GPT-2 small)
        {"name": "shared_beams_1x4", "op": "attention", "n_seq": 4, "n_group": 1, "prefix_max": 512, "ctx_max": 24,
         "new_min": 1, "new_max": 1, "heads": 12, "kv_heads": 12, "kv": "f32"},
        # a decode step of 256 answers to one long prompt, up to GPT-2's full context
        {"name": "shared_prompt_256", "op": "attention", "n_seq": 256, "n_group": 1, "prefix_max": 700, "ctx_max": 300,
         "new_min": 1, "new_max": 1, "heads": 12, "kv_heads": 12, "kv": "f32"},
        # beams of many requests, each request with its own prompt, over 8-bit pages (GPT-2 XL's 25 heads)
        {"name": "shared_groups_q8", "op": "attention", "n_seq": 120, "n_group": 24, "prefix_max": 1500, "ctx_max": 337,
         "new_min": 1, "new_max": 1, "heads": 25, "kv_heads": 25, "kv": "q8"},
        # a decode batch of long ragged contexts that share nothing, over 8-bit pages
        {"name": "decode_q8_64", "op": "attention", "n_seq": 64, "n_group": 0, "prefix_max": 0, "ctx_max": 4000,
         "new_min": 1, "new_max": 1, "heads": 32, "kv_heads": 8, "kv": "q8"},
        # a few guessed tokens of each of 64 answers, checked behind one very long shared text
        {"name": "shared_long_bf16", "op": "attention", "n_seq": 64, "n_group": 1, "prefix_max": 14336, "ctx_max": 500,
         "new_min": 1, "new_max": 4, "heads": 32, "kv_heads": 8, "kv": "bf16"},
        # making 4-bit weights of one layer's matrix (GPT-2 small's fused projection)
        {"name": "q4_make_qkv", "op": "quantize", "n": 2304, "k": 768, "group": 64},
        # and of the largest matrix, the tied head (GPT-2 XL)
        {"name": "q4_make_head", "op": "quantize", "n": 50257, "k": 1600, "group": 128},
        # one token through one projection: latency (GPT-2 small)
        {"name": "q4_qkv_1", "op": "matvec", "rows": 1, "n": 2304, "k": 768, "group": 64, "bias": True, "residual": False,
         "gelu": False},
        # five sequences through an up-projection and its activation (GPT-2 XL)
        {"name": "q4_fc_5", "op": "matvec", "rows": 5, "n": 6400, "k": 1600, "group": 32, "bias": True, "residual": False,
         "gelu": True},
        # eight sequences' logits (GPT-2 XL)
        {"name": "q4_head_8", "op": "matvec", "rows": 8, "n": 50257, "k": 1600, "group": 128, "bias": False,
         "residual": False, "gelu": False},
    ]


def _log(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["cache", "attention", "attention", "attention", "quantize", "matvec", "matvec"])
    if op == "cache":
        return {"op": op, "rows": _log(rng, 1, 16391), "kv_heads": rng.choice([1, 2, 5, 8, 12, 16])}
    if op == "quantize":
        return {"op": op, "n": _log(rng, 1, 50257), "k": _log(rng, 33, 1600), "group": rng.choice([32, 64, 128])}
    if op == "matvec":
        epilogue = rng.choice(["none", "bias", "gelu", "residual"])
        return {"op": op, "rows": rng.choice([1, 1, 2, 3, 4, 5, 7, 8]), "n": _log(rng, 33, 50257), "k": _log(rng, 33, 1600),
                "group": rng.choice([32, 64, 128]), "bias": epilogue != "none", "residual": epilogue == "residual",
                "gelu": epilogue == "gelu"}
    group = rng.choice([1, 1, 2, 4, 8])
    kv_heads = rng.choice([1, 2, 8, 12, 16, 25]) if group == 1 else rng.choice([1, 2, 3, 8])
    c = {"op": op, "n_seq": _log(rng, 1, 256), "ctx_max": _log(rng, 1, 1500), "new_min": 1,
         "new_max": rng.choice([1, 1, 1, 2, 5, 17]), "heads": group * kv_heads, "kv_heads": kv_heads,
         "kv": rng.choice(["f32", "bf16", "q8"])}
    kind = rng.choice(["none", "one", "one", "many"])
    c["n_group"] = 0 if kind == "none" else 1 if kind == "one" else min(c["n_seq"], _log(rng, 1, 40))
    c["prefix_max"] = 0 if kind == "none" else _log(rng, 16, 14336 if kind == "one" else 2000)
    # no dearer than the largest listed case: shorter texts, then fewer sequences
    while _attention_cost(c) > 1.0 and max(c["prefix_max"], c["ctx_max"]) > 64:
        for part in ("prefix_max", "ctx_max"):
            c[part] = c[part] * 3 // 4 if c[part] > 16 else c[part]
    while _attention_cost(c) > 1.0 and c["n_seq"] > 1:
        c["n_seq"] = c["n_seq"] * 2 // 3
        c["n_group"] = min(c["n_group"], c["n_seq"])
    return c


def _attention_cost(c):
    """Work of a case against the largest listed ones', by products and by cache bytes."""
    rows = c["n_seq"] * (c["new_min"] + c["new_max"]) / 2
    pairs = rows * (c["prefix_max"] + c["ctx_max"] / 2 + c["new_max"]) * c["heads"]
    cache = (c["n_group"] * c["prefix_max"] + c["n_seq"] * (c["ctx_max"] / 2 + c["new_max"])) * c["kv_heads"]
    size = {"f32": 4, "bf16": 2, "q8": 1.0625}[c["kv"]]
    return max(pairs / (64 * 2.5 * 14588 * 32), cache * size / (256 * 200 * 12 * 4))


def _lengths(case):
    """Each sequence's cached and new positions: a part of the case, the same for every seed."""
    r = random.Random(str(sorted(case.items())))
    n = case["n_seq"]
    ctx = [r.randint(0, case["ctx_max"]) for _ in range(n)]
    new = [r.randint(case["new_min"], case["new_max"]) for _ in range(n)]
    ctx[r.randrange(n)] = case["ctx_max"]
    new[r.randrange(n)] = case["new_max"]
    return ctx, new


def _groups(case):
    """First sequence of each group (and the end of the last), and the positions each group shares."""
    n, m = case["n_seq"], case["n_group"]
    r = random.Random("groups" + str(sorted(case.items())))
    cuts = [0] + sorted(r.sample(range(1, n), m - 1)) + [n] if m else []
    shared = [r.randint(case["prefix_max"] // 3, case["prefix_max"]) for _ in range(m)]
    if m:
        shared[r.randrange(m)] = case["prefix_max"]
    return cuts, shared


def _pages_of(length):
    return (length + PAGE - 1) // PAGE


# ------------------------------------------------------------------ the inputs

def _rand(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 1000003 + len(str(case)))
    return g


def _int32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def prepare(case, seed):
    return {"cache": _cache_inputs, "attention": _attention_inputs, "quantize": _quantize_inputs,
            "matvec": _matvec_inputs}[case["op"]](case, seed)


def _pool(g, n_pages, kv_heads, kind):
    """Key and value pages (and scales) of a pool in use."""
    out = {}
    for name in ("k", "v"):
        if kind == "q8":
            out[name + "_pages"] = torch.randint(-127, 128, (n_pages, PAGE, kv_heads * D), generator=g, device="cuda",
                                                 dtype=torch.int8)
            # rows of a standard deviation of about 1
            out[name + "_scales"] = (0.5 + torch.rand(n_pages, kv_heads, PAGE, generator=g, device="cuda")) / 73.0
        else:
            dtype = torch.bfloat16 if kind == "bf16" else torch.float32
            out[name + "_pages"] = _normal(g, n_pages, PAGE, kv_heads * D).to(dtype)
            out[name + "_scales"] = None
    return out


def _cache_inputs(case, seed):
    g = _rand(case, seed)
    rows, heads = case["rows"], case["kv_heads"]
    w, n_pages = heads * D, _pages_of(rows) + 4
    # the rows of a fused projection: query, key and value side by side
    qkv = _normal(g, rows, 3 * w)
    slots = torch.randperm(n_pages * PAGE, generator=g, device="cuda")[:rows].to(torch.int32)
    return {"op": "cache", "heads": heads, "k": qkv[:, w:2 * w], "v": qkv[:, 2 * w:], "slots": slots,
            **_pool(g, n_pages, heads, "q8"), "k_out": torch.empty(rows, w, device="cuda"),
            "v_out": torch.empty(rows, w, device="cuda")}


def _attention_inputs(case, seed):
    g = _rand(case, seed)
    ctx, new = _lengths(case)
    cuts, shared = _groups(case)
    counts = [_pages_of(c + n) for c, n in zip(ctx, new)]
    firsts = [_pages_of(n) for n in shared]
    n_pages = sum(counts) + sum(firsts) + 2
    perm = torch.randperm(n_pages - 1, generator=g, device="cuda").to(torch.int32)

    def table(of, at):
        t = torch.full((len(of), max(of)), n_pages - 1, dtype=torch.int32, device="cuda")
        t[torch.arange(max(of), device="cuda")[None, :] < _int32(of)[:, None]] = perm[at:at + sum(of)]
        return t

    start = [0]
    for n in new:
        start.append(start[-1] + n)
    rows = start[-1]
    seq_of = torch.repeat_interleave(torch.arange(len(new), device="cuda"), torch.tensor(new, device="cuda"))
    off = torch.arange(rows, device="cuda") - torch.tensor(start, device="cuda")[seq_of]
    # scores of a trained model are sharper than random rows': a standard deviation of 2
    q = 2.0 * _normal(g, rows, case["heads"] * D)
    s = {"op": "attention", "q": q, **_pool(g, n_pages, case["kv_heads"], case["kv"]), "table": table(counts, 0),
         "heads": case["heads"], "kv_heads": case["kv_heads"], "ctx": _int32(ctx), "row_start": _int32(start),
         "seq_of": seq_of, "off": off, "new_max": max(new), "prefix_table": None, "prefix_lens": None, "group_start": None,
         "out": torch.empty_like(q),
         "work": torch.empty((160 << 20) + rows * case["heads"] * 1024, dtype=torch.uint8, device="cuda")}
    if cuts:
        group_rows = [start[b] - start[a] for a, b in zip(cuts, cuts[1:])]
        s |= {"prefix_table": table(firsts, sum(counts)), "prefix_lens": _int32(shared), "group_start": _int32(cuts),
              "group_rows": max(group_rows), "group_of": torch.repeat_interleave(
                  torch.arange(len(shared), device="cuda"), torch.tensor(group_rows, device="cuda"))}
    return s


def _quantize_inputs(case, seed):
    g = _rand(case, seed)
    n, k, group = case["n"], case["k"], case["group"]
    return {"op": "quantize", "w": 0.02 * _normal(g, n, k), "group": group,
            "packed": torch.empty(n, -(-k // BLOCK) * (BLOCK // 2), dtype=torch.uint8, device="cuda"),
            "scales": torch.empty(n, -(-k // group), dtype=torch.bfloat16, device="cuda"),
            "w_out": torch.empty(n, k, device="cuda")}


def _matvec_inputs(case, seed):
    g = _rand(case, seed)
    rows, n, k, group = case["rows"], case["n"], case["k"], case["group"]
    levels = torch.randint(-7, 8, (n, k), generator=g, device="cuda", dtype=torch.int8)
    scales = ((0.5 + torch.rand(n, -(-k // group), generator=g, device="cuda")) * (0.02 / 3.5)).to(torch.bfloat16)
    x = _normal(g, rows, -(-k // 4) * 4)[:, :k]
    return {"op": "matvec", "x": x, "packed": _pack(levels), "scales": scales, "group": group,
            "bias": 0.1 * _normal(g, n) if case["bias"] else None,
            "residual": _normal(g, rows, n) if case["residual"] else None, "gelu": case["gelu"],
            "y": torch.empty(rows, n, device="cuda")}


def _pack(levels):
    """Levels -7 .. 7 [n, k] as they lie in memory: blocks of 128 weights of a row, filled up with zeros;
    the 32-bit word 4 t + j of a block holds its weights 32 j + 8 t .. + 7, the level + 8 of weight
    32 j + 8 t + i in bits 4 i .. 4 i + 3."""
    n, k = levels.shape
    blocks = -(-k // BLOCK)
    u = torch.full((n, blocks * BLOCK), 8, dtype=torch.uint8, device=levels.device)
    u[:, :k] = (levels + 8).to(torch.uint8)
    u = u.view(n, blocks, 4, 4, 4, 2).transpose(2, 3)         # block, j, t, byte, half -> block, t, j, ...
    return (u[..., 0] | (u[..., 1] << 4)).reshape(n, blocks * (BLOCK // 2))


def _levels(packed, k):
    """The levels that packed bytes hold, in order."""
    n, blocks = packed.shape[0], packed.shape[1] // (BLOCK // 2)
    u = packed.view(n, blocks, 4, 4, 4).transpose(2, 3)
    return torch.stack([u & 15, u >> 4], -1).reshape(n, blocks * BLOCK)[:, :k].to(torch.int32) - 8


# ------------------------------------------------------------------ one pass

def run(s):
    op = s["op"]
    if own:
        return _own(op, s, _ops())
    return {"cache": _plain_cache, "attention": _plain_attention, "quantize": _plain_quantize, "matvec": _plain_matvec}[op](s)


def _own(op, s, ops):
    if op == "cache":
        ops.kv_store_q8(s["k"], s["v"], s["slots"], s["k_pages"], s["v_pages"], s["k_scales"], s["v_scales"])
        ops.kv_load(s["slots"], s["k_pages"], s["v_pages"], s["k_out"], s["v_out"], s["k_scales"], s["v_scales"])
        return [s["k_out"], s["v_out"]]
    if op == "attention":
        ops.attention_shared(s["q"], s["k_pages"], s["v_pages"], s["table"], s["row_start"], s["ctx"], s["new_max"],
                             s["out"], s["work"], k_scales=s["k_scales"], v_scales=s["v_scales"],
                             prefix_table=s["prefix_table"], prefix_lens=s["prefix_lens"], group_start=s["group_start"])
        return s["out"]
    if op == "quantize":
        ops.quantize_q4(s["w"], s["packed"], s["scales"], s["group"])
        ops.dequantize_q4(s["packed"], s["scales"], s["group"], s["w_out"])
        return s["w_out"]
    ops.matvec_q4(s["x"], s["packed"], s["scales"], s["group"], s["y"], bias=s["bias"], residual=s["residual"],
                  gelu=s["gelu"])
    return s["y"]


def _plain_cache(s):
    slots, heads = s["slots"].long(), s["heads"]
    page, row = slots // PAGE, slots % PAGE
    out = []
    for name in ("k", "v"):
        x = s[name].reshape(-1, heads, D)
        scale = (x.abs().amax(-1).double() / 127.0).float()
        # (64 bits: a quotient next to the border of two levels)
        level = torch.where(scale[..., None] > 0, torch.round(x.double() / scale[..., None].double()).clamp(-127, 127), 0.0)
        pages, scales = s[name + "_pages"], s[name + "_scales"]
        pages.view(-1, heads * D)[slots] = level.to(torch.int8).view(-1, heads * D)
        scales[page, :, row] = scale
        got = pages.view(-1, heads, D)[slots].float() * scales[page, :, row][..., None]
        out.append(got.view(-1, heads * D))
    return out


def _rows_of(s, name, table):
    """The fp32 rows that a table's pages hold: [sequences, positions, kv_heads, D]."""
    x = s[name + "_pages"][table.long()].float().view(table.shape[0], -1, PAGE, s["kv_heads"], D)
    if s[name + "_scales"] is not None:
        x = x * s[name + "_scales"][table.long()].transpose(2, 3)[..., None]
    return x.reshape(table.shape[0], -1, s["kv_heads"], D)


def _partial(s, q, table, seen):
    """Maximum, sum and weighted values of rows q [sequences, rows, kv_heads, group, D] over the keys `seen`
    [sequences, rows, positions]."""
    k, v = _rows_of(s, "k", table), _rows_of(s, "v", table)
    scores = torch.matmul(q.permute(0, 2, 3, 1, 4), k.permute(0, 2, 3, 1)[:, :, None]) * (1.0 / math.sqrt(D))
    scores = scores.masked_fill(~seen[:, None, None], float("-inf"))
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == float("-inf"), 0.0, top))
    total, o = p.sum(-1, keepdim=True), torch.matmul(p, v.permute(0, 2, 1, 3)[:, :, None])
    return [x.permute(0, 3, 1, 2, 4) for x in (top, total, o)]


def _plain_attention(s):
    heads, kv_heads = s["heads"], s["kv_heads"]
    group, rows = heads // kv_heads, s["q"].shape[0]
    start, ctx = s["row_start"].long(), s["ctx"].long()
    step = torch.arange(s["new_max"], device=ctx.device)
    at = (start[:-1, None] + step).clamp(max=rows - 1)
    q = s["q"].view(rows, kv_heads, group, D)
    seen = torch.arange(s["table"].shape[1] * PAGE, device=ctx.device) <= (ctx[:, None] + step)[..., None]
    top, total, o = (x[s["seq_of"], s["off"]] for x in _partial(s, q[at], s["table"], seen))
    if s["prefix_table"] is not None:
        first = start[s["group_start"].long()[:-1]]
        step = torch.arange(s["group_rows"], device=ctx.device)
        at = (first[:, None] + step).clamp(max=rows - 1)
        seen = torch.arange(s["prefix_table"].shape[1] * PAGE, device=ctx.device) < s["prefix_lens"].long()[:, None]
        off = torch.arange(rows, device=ctx.device) - first[s["group_of"]]
        top2, total2, o2 = (x[s["group_of"], off] for x in _partial(s, q[at], s["prefix_table"], seen[:, None].expand(
            -1, s["group_rows"], -1)))
        both = torch.maximum(top, top2)
        a, b = torch.exp(top - both), torch.exp(top2 - both)
        total, o = total * a + total2 * b, o * a + o2 * b
    return (o / total).reshape(rows, heads * D)


def _plain_quantize(s):
    w, group = s["w"], s["group"]
    n, k = w.shape
    groups = -(-k // group)
    x = torch.zeros(n, groups * group, device=w.device)
    x[:, :k] = w
    x = x.view(n, groups, group)
    scale = (x.abs().amax(-1).double() / 7.0).float().to(torch.bfloat16)
    wide = scale.double()[..., None]          # 64 bits: a quotient next to the border of two levels
    level = torch.where(wide > 0, torch.round(x.double() / wide).clamp(-7, 7), 0.0)
    s["packed"].copy_(_pack(level.view(n, -1)[:, :k].to(torch.int8)))
    s["scales"].copy_(scale)
    return _weights(s["packed"], s["scales"], group, k)


def _weights(packed, scales, group, k):
    return _levels(packed, k).float() * scales.float().repeat_interleave(group, 1)[:, :k]


def _plain_matvec(s):
    y = torch.matmul(s["x"], _weights(s["packed"], s["scales"], s["group"], s["x"].shape[1]).T)
    if s["bias"] is not None:
        y = y + s["bias"]
    if s["gelu"]:
        y = 0.5 * y * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (y + 0.044715 * y * y * y)))
    if s["residual"] is not None:
        y = y + s["residual"]
    return y


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    op = case["op"]
    if op == "cache":
        w = case["kv_heads"] * D
        # two rows in, stored in 8 bits with their scales, read, two rows out
        return {"bytes": 2 * case["rows"] * (2 * 4 * w + 2 * (w + 4 * case["kv_heads"])) + 8 * case["rows"], "flops": 0}
    if op in ("quantize", "matvec"):
        n, k = case["n"], case["k"]
        small = n * (-(-k // BLOCK) * (BLOCK // 2) + 2 * -(-k // case["group"]))
        if op == "quantize":
            return {"bytes": 8 * n * k + 2 * small, "flops": 0}
        rows = case["rows"]
        more = 4 * n * (case["bias"] + rows * case["residual"])
        return {"bytes": small + 4 * rows * (n + k) + more, "flops": 2 * rows * n * k}
    ctx, new = _lengths(case)
    cuts, shared = _groups(case)
    row = 2 * case["kv_heads"] * {"f32": 4 * D, "bf16": 2 * D, "q8": D + 4}[case["kv"]]
    pairs = sum(n * c + n * (n + 1) // 2 for c, n in zip(ctx, new))
    pairs += sum(p * sum(new[a:b]) for p, a, b in zip(shared, cuts, cuts[1:]))
    return {"bytes": (sum(ctx) + sum(new) + sum(shared)) * row + 2 * sum(new) * case["heads"] * D * 4,
            "flops": 4 * D * case["heads"] * pairs}


# ------------------------------------------------------------------ the definitions in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    return {"cache": _exact_cache, "attention": _exact_attention, "quantize": _exact_quantize,
            "matvec": _exact_matvec}[case["op"]](case, s)


def _nearest_level(x, most):
    """x [..., n] (64 bits) and its scale [...] in the type it is kept in, as the values that its levels stand for."""
    def values(scale):
        t = scale.double().unsqueeze(-1)
        level = torch.clamp(torch.round(x / torch.where(t > 0, t, torch.ones_like(t))), -most, most)
        return level * t
    return values


def _exact_cache(case, s):
    out = []
    for x in (s["k"], s["v"]):
        x = x.double().reshape(case["rows"], case["kv_heads"], D)
        out.append(_nearest_level(x, 127)((x.abs().max(-1).values / 127).float()).reshape(case["rows"], -1))
    return out


def _exact_quantize(case, s):
    out = torch.empty(case["n"], case["k"], dtype=torch.float64, device="cuda")
    for a in range(0, case["k"], case["group"]):
        x = s["w"][:, a:a + case["group"]].double()
        out[:, a:a + case["group"]] = _nearest_level(x, 7)((x.abs().max(-1).values / 7).float().to(torch.bfloat16))
    return out


def _exact_matvec(case, s):
    n, k, group = case["n"], case["k"], case["group"]
    word = s["packed"].view(torch.int32).view(n, -1, 16)      # blocks of 16 words
    y = torch.zeros(case["rows"], n, dtype=torch.float64, device="cuda")
    x = s["x"].double()
    for i in range(k):
        b, r = divmod(i, BLOCK)
        j, t, nibble = r // 32, r % 32 // 8, r % 8
        level = (word[:, b, 4 * t + j] >> (4 * nibble) & 15) - 8
        y += x[:, i:i + 1] * (level.double() * s["scales"][:, i // group].double())[None]
    if s["bias"] is not None:
        y = y + s["bias"].double()
    if s["gelu"]:
        y = y / 2 * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3)))
    if s["residual"] is not None:
        y = y + s["residual"].double()
    return y


def _exact_attention(case, s):
    heads, kv_heads = case["heads"], case["kv_heads"]
    group = heads // kv_heads
    ctx, new = _lengths(case)
    cuts, shared = _groups(case)

    def rows(name, entries, n):
        at = entries[:_pages_of(n)].long()
        x = s[name + "_pages"][at].double().view(len(at), PAGE, kv_heads, D)
        if s[name + "_scales"] is not None:
            x = x * s[name + "_scales"][at].double().permute(0, 2, 1)[..., None]
        return x.reshape(-1, kv_heads, D)[:n].transpose(0, 1)     # [kv_heads, n, D]

    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lo, g, before = 0, -1, None
    for i, (c, m) in enumerate(zip(ctx, new)):
        while cuts and g + 1 < len(shared) and cuts[g + 1] <= i:
            g += 1
            before = [rows(name, s["prefix_table"][g], shared[g]) for name in ("k", "v")] if shared[g] else None
        k, v = (rows(name, s["table"][i], c + m) for name in ("k", "v"))
        n0 = 0
        if before is not None:
            n0 = before[0].shape[1]
            k, v = torch.cat([before[0], k], 1), torch.cat([before[1], v], 1)
        q = s["q"][lo:lo + m].double().view(m, kv_heads, group, D).permute(1, 2, 0, 3).reshape(kv_heads, group * m, D)
        t = (q @ k.transpose(1, 2) / math.sqrt(D)).view(kv_heads, group, m, -1)
        hidden = torch.arange(n0 + c + m, device="cuda")[None] > n0 + torch.arange(c, c + m, device="cuda")[:, None]
        t = torch.softmax(t.masked_fill(hidden, -math.inf), -1).view(kv_heads, group * m, -1)
        o = (t @ v).view(kv_heads, group, m, D).permute(2, 0, 1, 3)
        out[lo:lo + m] = o.reshape(m, heads * D)
        lo += m
    return out

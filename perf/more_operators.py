"""Timed cases of the 4-bit paged KV cache: appending to it (and reading it back), attention over it, with or without
the attention weights that its slots receive, and eviction down to a budget by those weights.

``own`` selects what ``run`` calls: the framework's operators, or their plain form in elementary torch operations
(fp32 arithmetic, one rounding at the end).  Ragged lengths are a fixed function of the case, so the work of a case
is known without its inputs; every tensor value comes from the seed.

The cache of a layer is one byte tensor (P, G, page / 16, 18 D): for each 16 tokens of a page and KV head the keys'
codes (16, D / 2), two dims to a byte with the even one in the low half, the keys' parameters (16, D / 32) of 16 bits, and
the same for the values.  Group j holds the 32 dims d with (d / 4) % (D / 32) == j.  A parameter is the f16 pattern of
the group's scale s, its low 4 bits replaced by the zero point z, and a code n stands for s (n - z).
"""

import math

import torch

own = False

GOLDEN = 0.6180339887498949


# ---- ragged lengths -------------------------------------------------------------------------------
def ragged(n, lo, hi, shift=0.0):
    """n lengths spread evenly, in scrambled order, over [lo, hi]."""
    return [lo + int((hi - lo + 1) * math.modf((i + 1) * GOLDEN + shift)[0]) for i in range(n)]


def lengths(c):
    """(new tokens, cached length after the append) of each sequence of an append / attention case."""
    new = ragged(c["batch"], c["new_lo"], c["new_hi"], 0.37)
    past = ragged(c["batch"], c["past_lo"], c["past_hi"])
    return new, [p + n for p, n in zip(past, new)]


# ---- cases ----------------------------------------------------------------------------------------
def append_case(name, batch, new_lo, new_hi, past_lo, past_hi, heads, kv_heads, head_dim, page, queries, dtype):
    return {"name": name, "op": "append", "batch": batch, "new_lo": new_lo, "new_hi": new_hi, "past_lo": past_lo,
            "past_hi": past_hi, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "page": page,
            "queries": queries, "dtype": dtype}


def attention_case(name, batch, new_lo, new_hi, past_lo, past_hi, heads, kv_heads, head_dim, page, diff, window,
                   weights, dtype):
    return {"name": name, "op": "attention", "batch": batch, "new_lo": new_lo, "new_hi": new_hi, "past_lo": past_lo,
            "past_hi": past_hi, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "page": page,
            "diff": diff, "window": window, "weights": weights, "dtype": dtype}


def evict_case(name, batch, past_lo, past_hi, kv_heads, head_dim, page, budget, recent):
    return {"name": name, "op": "evict", "batch": batch, "past_lo": past_lo, "past_hi": past_hi, "kv_heads": kv_heads,
            "head_dim": head_dim, "page": page, "budget": budget, "recent": recent}


def listed():
    return [
        # one token of one conversation: the latency of a decode step of the smaller model shapes
        append_case("append one token", 1, 1, 1, 700, 700, 16, 4, 128, 64, 1, "bf16"),
        # ragged prompts enter the cache, some behind a cached prefix; both query tensors of the differential layer
        append_case("append prompts", 24, 37, 1600, 0, 130, 32, 8, 128, 32, 2, "bf16"),
        # one token of one conversation over a short cache
        attention_case("decode one", 1, 1, 1, 700, 700, 16, 4, 128, 64, False, 0, False, "bf16"),
        # a rollout batch in the middle of its answers, differential attention
        attention_case("decode 64 rollouts", 64, 1, 1, 300, 8191, 32, 8, 128, 64, True, 0, False, "bf16"),
        # the same step of a single-softmax model whose cache is going to be evicted from
        attention_case("decode 64 with weights", 64, 1, 1, 300, 8191, 32, 8, 128, 64, False, 0, True, "bf16"),
        # one long document, one token: the cache's length is the only parallelism
        attention_case("decode long", 1, 1, 1, 131000, 131000, 32, 8, 128, 128, False, 0, False, "bf16"),
        # a few drafted tokens a sequence, small heads and small pages, sliding window, f16
        attention_case("drafts in a window", 30, 1, 5, 100, 7000, 8, 2, 64, 16, False, 4096, False, "f16"),
        # a chunk of a long prompt on its cached prefix, beside sequences that decode
        attention_case("prompt chunks", 6, 1, 2048, 900, 14000, 32, 8, 128, 64, True, 0, False, "bf16"),
        # chunks of prompts that are evicted from once they are in: every key's weight over all of its queries
        attention_case("prompts with weights", 4, 700, 1024, 2000, 8192, 32, 8, 128, 64, False, 0, True, "bf16"),
        # a conversation that has just outgrown its budget
        evict_case("evict one", 1, 700, 700, 4, 128, 64, 512, 64),
        # a rollout batch is cut to its budget; the short ones stay as they are
        evict_case("evict 64 rollouts", 64, 300, 8191, 8, 128, 64, 2048, 256),
        # a long document is cut to a quarter
        evict_case("evict long", 1, 131000, 131000, 8, 128, 128, 32000, 1000),
    ]


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kind = rng.choice(["append", "attention", "attention", "attention", "evict", "evict"])
    heads, kv_heads, head_dim = rng.choice([(32, 8, 128), (16, 4, 128), (8, 2, 64), (16, 16, 64), (12, 4, 128)])
    page = rng.choice([16, 32, 64, 128])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    if kind == "append":
        batch, new = spread(1, 200), rng.choice([1, 1, spread(2, 1500)])
        batch = max(1, min(batch, 30000 // new))
        past = spread(1, 4000)
        return unnamed(append_case("", batch, max(1, new // 4), new, past // 8, past, heads, kv_heads, head_dim, page,
                                   rng.choice([0, 1, 2]), dtype))
    if kind == "evict":
        past = spread(20, 60000)
        batch = max(1, min(spread(1, 64), 520000 // past))
        budget = min(32000, max(1, int(past * rng.uniform(0.1, 1.05))))
        return unnamed(evict_case("", batch, past // 3, past, kv_heads, head_dim, page, budget,
                                  int(budget * rng.choice([0.0, 0.1, 0.5, 1.0]))))
    new = rng.choice([1, 1, 1, spread(2, 12), spread(16, 1500)])
    past = spread(1, 14000) if new > 1 else spread(1, 60000)
    batch = spread(1, 64)
    batch = max(1, min(batch, 520000 // (past + new), 3000 // new))
    return unnamed(attention_case("", batch, max(1, new // 4), new, past // 6, past, heads, kv_heads, head_dim, page,
                                  rng.random() < 0.5, rng.choice([0, 0, 1 + past // 3]), rng.random() < 0.5, dtype))


def unnamed(c):
    return {k: v for k, v in c.items() if k != "name"}


# ---- work -----------------------------------------------------------------------------------------
ITEM = {"bf16": 2, "f16": 2}


def work(c):
    G, D = c["kv_heads"], c["head_dim"]
    token = 9 * D // 8                                      # bytes of a token's keys and values of one head
    if c["op"] == "evict":
        total = ragged(c["batch"], c["past_lo"], c["past_hi"])
        # a sequence within its budget is copied whole, without a look at its weights
        look = sum(L for L in total if L > c["budget"]) * G
        kept = sum(min(L, c["budget"]) for L in total) * G
        return {"bytes": 4 * look + kept * 2 * (token + 4) + 4 * c["batch"] * G * c["budget"], "flops": look}
    new, total = lengths(c)
    H, e = c["heads"], ITEM[c["dtype"]]
    if c["op"] == "append":
        T = sum(new)
        kv = T * G * (2 * D * e + token)                    # in, and read back out
        qs = 2 * c["queries"] * T * H * D * e
        return {"bytes": 2 * kv + qs + T * D * 4, "flops": 3 * T * D * (G + c["queries"] * H) + 8 * T * G * D}
    maps = 2 if c["diff"] else 1
    W = c["window"] or (1 << 40)
    read = sum(min(L, W + n - 1) for n, L in zip(new, total)) * G
    pairs = sum(min(L - n + i + 1, W) for n, L in zip(new, total) for i in range(n))
    return {"bytes": read * (token + (8 if c["weights"] else 0)) + sum(new) * H * D * e * (maps + 1),
            "flops": 4.0 * pairs * H * D * maps}


# ---- inputs ---------------------------------------------------------------------------------------
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
DEV = "cuda"


def quantised(x):
    """fp32 (.., D) -> codes (.., D / 2) uint8 and parameters (.., D / 32) int16."""
    D = x.shape[-1]
    x = torch.nan_to_num(x, nan=0.0).clamp(-65504.0, 65504.0).unflatten(-1, (8, D // 32, 4))
    lo, hi = x.amin((-3, -1)).clamp(max=0.0), x.amax((-3, -1)).clamp(min=0.0)
    s = (hi - lo) * 0.06666666                              # a fifteenth, rounded down; then up to 7 significant bits
    up = ((s.view(torch.int32) + 0x1FFFF) & ~0x1FFFF).view(torch.float32)
    s = torch.where(s < 2.0 ** -14, torch.ceil(s * 2.0 ** 20) * 2.0 ** -20, up).clamp(min=2.0 ** -20)
    z = torch.round(-lo * (1.0 / s)).clamp(0.0, 15.0)
    s = s.clamp(max=4352.0)
    n = (torch.round(x * (1.0 / s)[..., None, :, None]) + z[..., None, :, None]).clamp(0.0, 15.0)
    n = n.to(torch.uint8).flatten(-3)
    return n[..., 0::2] | n[..., 1::2] << 4, s.half().view(torch.int16) | z.to(torch.int16)


def held(codes, params):
    """The values that codes and parameters stand for, fp32."""
    D = 2 * codes.shape[-1]
    n = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).unflatten(-1, (8, D // 32, 4)).float()
    s = (params & -16).view(torch.float16).float()
    return (s[..., None, :, None] * (n - (params & 15).float()[..., None, :, None])).flatten(-3)


def parts(blocks):
    """Views of a cache (P, G, page / 16, 18 D): key codes, key parameters, value codes, value parameters, (.., 16, ..)."""
    D = blocks.shape[-1] // 18
    out = []
    for x in (blocks[..., : 9 * D], blocks[..., 9 * D:]):
        out += [x[..., : 8 * D].unflatten(-1, (16, D // 2)), x[..., 8 * D:].view(torch.int16).unflatten(-1, (16, D // 32))]
    return out


def scrambled(need, P, g):
    """A block table for sequences of `need` pages in a pool of P, in no order."""
    perm = torch.randperm(P, generator=g, device=DEV).to(torch.int32)
    table = torch.full((len(need), max(max(need), 1)), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = torch.arange(at, at + n, dtype=torch.int32)
        at += n
    table = table.to(DEV)
    return torch.where(table >= 0, perm[table.clamp(min=0).long()], table)


def cache_for(c, g, total, past, spare=0):
    """A pool whose pages hold `past` tokens of each sequence in scrambled pages; slots past the end hold any bytes."""
    G, D, ps = c["kv_heads"], c["head_dim"], c["page"]
    need = [-(-L // ps) for L in total]
    P = sum(need) + 3
    table = scrambled(need, P, g)
    count = torch.zeros(P + 1, dtype=torch.long, device=DEV)        # tokens that each page holds
    inside = (torch.tensor(past, device=DEV)[:, None] - torch.arange(table.shape[1], device=DEV)[None] * ps).clamp(0, ps)
    count[torch.where(table >= 0, table, P).long()] = inside
    stale = torch.arange(ps, device=DEV)[None] >= count[:P, None]                     # (P, ps)
    blocks = torch.empty(P + spare, G, ps // 16, 18 * D, dtype=torch.uint8, device=DEV)
    blocks[P:] = 0xFF
    at = parts(blocks[:P])
    for i, name in enumerate("kv"):
        x = torch.randn(P, G, ps, D, generator=g, device=DEV)
        if name == "k":                                             # keys have a few strong channels, and channel means
            x *= torch.where(torch.rand(D, generator=g, device=DEV) < 0.05, 6.0, 1.0)
            x += 0.5 * torch.randn(D, generator=g, device=DEV)
        for to, y in zip(at[2 * i: 2 * i + 2], quantised(x)):
            to.copy_(y.masked_fill_(stale[:, None, :, None], 0xFF if y.dtype == torch.uint8 else -1).unflatten(2, (-1, 16)))
    # weights received so far: few tokens have most, some none at all; behind the end anything
    mass = torch.randn(P + spare, G, ps, generator=g, device=DEV).mul_(2.0).exp_()
    mass *= torch.rand(P + spare, G, ps, generator=g, device=DEV) < 0.8
    if c["op"] == "attention":                                      # of the size of what a pass adds
        mass *= c["heads"] // G * max(lengths(c)[0]) / (8.0 * max(total))
    mass[:P].masked_fill_(stale[:, None], 40.0 if c["op"] == "evict" else 0.0)
    return blocks, mass, table


def prepare(c, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    G, D, ps = c["kv_heads"], c["head_dim"], c["page"]
    if c["op"] == "evict":
        total = ragged(c["batch"], c["past_lo"], c["past_hi"])
        out = [-(-min(L, c["budget"]) // ps) for L in total]
        # the kept tokens go to pages of their own, so that a shared prompt stays whole for the other rollouts
        blocks, mass, table = cache_for(c, g, total, total, sum(out) + 1)
        to = scrambled(out, sum(out) + 1, g)
        to = torch.where(to >= 0, to + blocks.shape[0] - sum(out) - 1, to)
        return {"c": c, "blocks": blocks, "mass": mass, "table": table, "to": to,
                "lens": torch.tensor(total, dtype=torch.int32, device=DEV)}
    dt = TYPES[c["dtype"]]
    new, total = lengths(c)
    H, T = c["heads"], sum(new)
    blocks, mass, table = cache_for(c, g, total, [L - n for n, L in zip(new, total)] if c["op"] == "append" else total)
    cu = torch.tensor([0] + new).cumsum(0).to(torch.int32).to(DEV)
    st = {"c": c, "blocks": blocks, "mass": mass, "table": table, "cu": cu,
          "lens": torch.tensor(total, dtype=torch.int32, device=DEV), "max_new": max(new)}
    rand = lambda *s: torch.randn(*s, generator=g, device=DEV).to(dt)  # noqa: E731
    if c["op"] == "append":
        st["k"], st["v"] = rand(T, G, D), rand(T, G, D)
        st["queries"] = [rand(T, H, D) for _ in range(c["queries"])]
        st["pos"] = torch.cat([torch.arange(L - n, L) for n, L in zip(new, total)]).to(DEV)
        ang = torch.outer(torch.arange(max(total), device=DEV, dtype=torch.float32),
                          1.0 / 10000.0 ** (torch.arange(0, D, 2, device=DEV, dtype=torch.float32) / D))
        st["cos"], st["sin"] = ang.cos(), ang.sin()
        return st
    st["q"] = rand(T, H, D)
    if c["diff"]:
        st["q2"] = rand(T, H, D)
        st["lam"] = (0.5 + 0.45 * torch.rand(H, generator=g, device=DEV))
    return st


# ---- the operators --------------------------------------------------------------------------------
def run(st):
    return {"append": run_append, "attention": run_attention, "evict": run_evict}[st["c"]["op"]](st)


def run_append(st):
    """New tokens go in; what the cache then holds of them comes back out, in the inputs' type."""
    if own:
        from mamformer_b200 import ops
        cache = ops.PagedKV4(st["blocks"])
        qs = ops.kv_append(st["k"], st["v"], cache, st["table"], st["cu"], st["lens"], st["max_new"], st["cos"], st["sin"],
                           st["pos"], st["queries"])
        k, v = ops.kv_read(cache, st["table"], st["cu"], st["lens"], st["k"].shape[0], st["k"].dtype)
        return {"k": k, "v": v, "queries": list(qs)}
    cos, sin = st["cos"][st["pos"]][:, None], st["sin"][st["pos"]][:, None]
    ps, cu, T = st["c"]["page"], st["cu"].long(), st["k"].shape[0]
    t = torch.arange(T, device=DEV)
    b = torch.searchsorted(cu[1:], t, right=True)
    slot = t - cu[1:][b] + st["lens"].long()[b]
    page = st["table"].long()[b, slot // ps]
    block, row = slot % ps // 16, slot % 16
    at = parts(st["blocks"])
    out = {"queries": [rotated(q.float(), cos, sin).to(q.dtype) for q in st["queries"]]}
    for i, (name, x) in enumerate((("k", rotated(st["k"].float(), cos, sin)), ("v", st["v"].float()))):
        for to, y in zip(at[2 * i: 2 * i + 2], quantised(x)):
            to[page, :, block, row] = y
        out[name] = held(*(y[page, :, block, row] for y in at[2 * i: 2 * i + 2])).to(st["k"].dtype)
    return out


def rotated(x, cos, sin):
    a, b = x[..., : x.shape[-1] // 2], x[..., x.shape[-1] // 2:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def run_attention(st):
    """A layer's attention; with `weights` each slot's received weights grow (from a copy, so that a pass can be repeated)."""
    c = st["c"]
    mass = st["mass"].clone() if c["weights"] else None
    if own:
        from mamformer_b200 import ops
        o = ops.paged_attention(st["q"], ops.PagedKV4(st["blocks"], mass), st["table"], st["cu"], st["lens"], st["max_new"],
                                q2=st.get("q2"), lam=st.get("lam"), window=c["window"])
        return {"out": o, "mass": mass}
    B, G, D, ps = c["batch"], c["kv_heads"], c["head_dim"], c["page"]
    table = st["table"].long()
    L, N = table.shape[1] * ps, st["max_new"]
    cu, lens = st["cu"].long(), st["lens"].long()
    slot = torch.arange(L, device=DEV)
    i = torch.arange(N, device=DEV)
    at = (lens - (cu[1:] - cu[:-1]))[:, None] + i                                     # (B, N) slot of each query
    see = (slot <= at[..., None]) & (slot < lens[:, None, None])
    if c["window"]:
        see = see & (slot > at[..., None] - c["window"])
    see = see[:, None, None]                                                          # (B, 1, 1, N, L)
    pieces = parts(st["blocks"])

    def cached(codes, params):
        x = held(codes[table.clamp(min=0)], params[table.clamp(min=0)])              # (B, W, G, ps / 16, 16, D)
        x = x.transpose(1, 2).reshape(B, G, 1, L, D)
        return torch.where((slot < lens[:, None])[:, None, None, :, None], x, 0.0)

    k, v = cached(*pieces[:2]), cached(*pieces[2:])
    token = (cu[:-1, None] + i).clamp(max=st["q"].shape[0] - 1)
    real = i < (cu[1:] - cu[:-1])[:, None]                                            # (B, N)

    def one(q):
        x = q[token].float().unflatten(2, (G, -1)).permute(0, 2, 3, 1, 4)             # (B, G, H / G, N, D)
        s = (x @ k.transpose(-1, -2)).mul_(D ** -0.5).masked_fill_(~see, -math.inf)
        m = s.amax(-1, keepdim=True)
        p = s.sub_(torch.where(m == -math.inf, 0.0, m)).exp_()
        d = p.sum(-1, keepdim=True)
        d = torch.where(d > 0, d, 1.0)
        w = p.mul(real[:, None, None, :, None] / d).sum((2, 3)) if c["weights"] else 0.0      # (B, G, L)
        return ((p @ v) / d).permute(0, 3, 1, 2, 4).flatten(2, 3), w

    o, w = one(st["q"])
    if c["diff"]:
        lam = st["lam"][:, None]
        o2, w2 = one(st["q2"])
        o, w = (o - lam * o2) / (1.0 - lam + 1e-8), w + w2
    if c["weights"]:
        used = table >= 0
        mass[table[used]] += torch.where(slot < lens[:, None, None], w, 0.0).unflatten(2, (-1, ps)).transpose(1, 2)[used]
    return {"out": o[real].to(st["q"].dtype), "mass": mass}


def run_evict(st):
    """Returns the kept slots of each sequence and head (-1: none), the new lengths, and the cache; its bytes move as they are."""
    c, budget, recent = st["c"], st["c"]["budget"], st["c"]["recent"]
    blocks, mass = st["blocks"], st["mass"]
    if own:
        from mamformer_b200 import ops
        kept, lens = ops.kv_evict(ops.PagedKV4(blocks, mass), st["table"], st["lens"], budget, recent, out_table=st["to"])
        return {"kept": kept, "lens": lens, "blocks": blocks, "mass": mass}
    B, G, ps = c["batch"], c["kv_heads"], c["page"]
    table, lens = st["table"].long(), st["lens"].long()
    L = table.shape[1] * ps
    slot = torch.arange(L, device=DEV)
    m = mass[table.clamp(min=0)].transpose(1, 2).reshape(B, G, L)
    bits = (m + 0.0).view(torch.int32).long()
    key = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits) * (1 << 20) - slot      # ties to the lower slot
    key = torch.where((slot >= (lens - recent)[:, None, None]), 1 << 60, key)
    key = torch.where((slot < lens[:, None, None]), key, -(1 << 60) - slot)
    n = min(budget, L)
    kept = torch.topk(key, n, dim=2).indices
    left = lens.clamp(max=budget)
    kept = torch.where(kept < lens[:, None, None], kept, L).sort(dim=2).values
    out = torch.full((B, G, budget), -1, dtype=torch.int32, device=DEV)
    out[:, :, :n] = torch.where(kept < L, kept, -1)
    b, g, r = torch.nonzero(out >= 0, as_tuple=True)
    src = out[b, g, r].long()
    frm = (table[b, src // ps], g, src % ps // 16, src % 16)
    to = (st["to"].long()[b, r // ps], g, r % ps // 16, r % 16)
    for x in parts(blocks) + [mass.unflatten(2, (-1, 16))]:
        x[to] = x[frm]
    return {"kept": out, "lens": left.to(torch.int32), "blocks": blocks, "mass": mass}


# ---- the definitions in 64 bits -------------------------------------------------------------------
def exact(c, seed):
    st = prepare(c, seed)
    return {"append": exact_append, "attention": exact_attention, "evict": exact_evict}[c["op"]](c, st)


def exact_evict(c, st):
    """Whole numbers but for the weights, which move unchanged: sequence by sequence, head by head."""
    mass, ps = st["mass"].double(), c["page"]
    for b, L in enumerate(ragged(c["batch"], c["past_lo"], c["past_hi"])):
        slot = torch.arange(L, device=DEV)
        page, to = st["table"][b].long()[slot // ps], st["to"][b].long()
        for g in range(c["kv_heads"]):
            m = st["mass"][page, g, slot % ps].double()
            keep = slot
            if L > c["budget"]:
                old = L - c["recent"]
                first = torch.sort(m[:old], descending=True, stable=True).indices[: c["budget"] - c["recent"]]
                keep = torch.cat([torch.sort(first).values, slot[old:]])
            r = torch.arange(len(keep), device=DEV)
            mass[to[r // ps], g, r % ps] = m[keep]
    return {"kept": None, "lens": None, "blocks": None, "mass": mass}


def level(x):
    """x (.., D) in 64 bits rounded to the sixteen levels of its groups, group by group."""
    D = x.shape[-1]
    out = torch.empty_like(x)
    for j in range(D // 32):
        dims = [d for d in range(D) if d // 4 % (D // 32) == j]
        y = x[..., dims]
        lo, hi = y.amin(-1, keepdim=True).clamp(max=0), y.amax(-1, keepdim=True).clamp(min=0)
        s = (hi - lo) / 15
        unit = torch.exp2(torch.floor(torch.log2(s.clamp(min=2.0 ** -14)))) / 64
        s = (torch.ceil(s / unit) * unit).clamp(min=2.0 ** -20)
        z = torch.round(-lo / s)
        s = s.clamp(max=4352)
        out[..., dims] = s * ((torch.round(y / s) + z).clamp(0, 15) - z)
    return out


def exact_append(c, st):
    """The rotation as a complex product, then the levels."""
    D = c["head_dim"]
    turn = torch.complex(st["cos"].double(), st["sin"].double())[st["pos"]][:, None]

    def turned(x):
        z = torch.complex(x[..., : D // 2].double(), x[..., D // 2:].double()) * turn
        return torch.cat([z.real, z.imag], -1)

    return {"queries": [turned(q) for q in st["queries"]], "k": level(turned(st["k"])), "v": level(st["v"].double())}


def exact_attention(c, st):
    new, total = lengths(c)
    H, G, D, ps, W = c["heads"], c["kv_heads"], c["head_dim"], c["page"], c["window"]
    out = torch.zeros(sum(new), H, D, dtype=torch.float64, device=DEV)
    mass = st["mass"].double() if c["weights"] else None
    at = 0
    for b, (n, L) in enumerate(zip(new, total)):
        pages = st["table"][b, : -(-L // ps)].long()
        mine = st["blocks"][pages]
        where = torch.arange(L - n, L, device=DEV)[:, None] - torch.arange(L, device=DEV)[None]
        hide = (where < 0) | (where >= W) if W else where < 0
        slot = torch.arange(L, device=DEV)
        for g in range(G):
            kv = []
            for x in (mine[:, g, :, : 9 * D], mine[:, g, :, 9 * D:]):
                code = x[..., : 8 * D].reshape(-1, D // 2).long()
                word = x[..., 8 * D:].reshape(-1, D // 32, 2).long()
                word = word[..., 0] + 256 * word[..., 1]
                s = (word - word % 16).to(torch.int16).view(torch.float16).double()
                y = torch.zeros(len(code), D, dtype=torch.float64, device=DEV)
                y[:, 0::2], y[:, 1::2] = (code % 16).double(), (code // 16).double()
                of = torch.arange(D, device=DEV) // 4 % (D // 32)
                kv.append((s[:, of] * (y - (word % 16).double()[:, of]))[:L])
            for h in range(g * (H // G), (g + 1) * (H // G)):
                maps = []
                for q in [st["q"]] + ([st["q2"]] if c["diff"] else []):
                    s = (q[at: at + n, h].double() @ kv[0].T) / math.sqrt(D)
                    p = torch.softmax(s.masked_fill(hide, -math.inf), -1)
                    maps.append(p @ kv[1])
                    if mass is not None:
                        mass[pages[slot // ps], g, slot % ps] += p.sum(0)
                if c["diff"]:
                    lam = st["lam"][h].double()
                    maps[0] = (maps[0] - lam * maps[1]) / (1.0 - lam + 1e-8)
                out[at: at + n, h] = maps[0]
        at += n
    return {"out": out, "mass": mass}

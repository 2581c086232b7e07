"""Timed cases of the rollout-and-scoring operators: appending to the paged 8-bit KV cache, attention over that
cache, and the scores (log probability, entropy, top alternatives, gradient) of given tokens.

``own`` selects what ``run`` calls: the framework's operators, or their plain form in elementary torch operations
(fp32 arithmetic, one rounding at the end).  Ragged lengths are a fixed function of the case, so the work of a case
is known without its inputs; every tensor value comes from the seed.
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


def attention_case(name, batch, new_lo, new_hi, past_lo, past_hi, heads, kv_heads, head_dim, page, diff, window, dtype):
    return {"name": name, "op": "attention", "batch": batch, "new_lo": new_lo, "new_hi": new_hi, "past_lo": past_lo,
            "past_hi": past_hi, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "page": page,
            "diff": diff, "window": window, "dtype": dtype}


def scores_case(name, rows, vocab, top_k, temperature, ignored, backward, dtype):
    return {"name": name, "op": "scores", "rows": rows, "vocab": vocab, "top_k": top_k, "temperature": temperature,
            "ignored": ignored, "backward": backward, "dtype": dtype}


def listed():
    return [
        # one token of one conversation: the latency of a decode step of the smaller model shapes
        append_case("append one token", 1, 1, 1, 700, 700, 16, 4, 128, 64, 1, "bf16"),
        # one decode step of a rollout batch, both query tensors of the differential layer rotated
        append_case("append 200 rollouts", 200, 1, 1, 17, 4096, 32, 8, 128, 64, 2, "bf16"),
        # ragged prompts enter the cache, some behind a cached prefix
        append_case("append prompts", 24, 37, 1600, 0, 130, 32, 8, 128, 32, 2, "bf16"),
        # one token of one conversation over a short cache
        attention_case("decode one", 1, 1, 1, 700, 700, 16, 4, 128, 64, False, 0, "bf16"),
        # a rollout batch in the middle of its answers, differential attention
        attention_case("decode 64 rollouts", 64, 1, 1, 300, 8191, 32, 8, 128, 64, True, 0, "bf16"),
        # one long document, one token: the cache's length is the only parallelism
        attention_case("decode long", 1, 1, 1, 131000, 131000, 32, 8, 128, 128, False, 0, "bf16"),
        # a few drafted tokens a sequence, small heads and small pages, sliding window, f16
        attention_case("drafts in a window", 30, 1, 5, 100, 7000, 8, 2, 64, 16, False, 4096, "f16"),
        # a chunk of a long prompt on its cached prefix, beside sequences that decode
        attention_case("prompt chunks", 6, 1, 2048, 900, 14000, 32, 8, 128, 64, True, 0, "bf16"),
        # a sampling step's scores with its alternatives; fp32 logits
        scores_case("score 7 rows", 7, 32000, 8, 0.8, 0.0, False, "f32"),
        # the scores of a rollout batch's step over the full vocabulary
        scores_case("score 200 rows", 200, 128000, 20, 0.9, 0.0, False, "bf16"),
        # scoring sequences whose prompt positions are ignored, odd vocabulary, with gradient
        scores_case("train 1500 odd", 1500, 64003, 5, 1.0, 0.3, True, "f16"),
        # the training pass of a policy update: gradient of log probabilities and entropies
        scores_case("train 4096", 4096, 128000, 0, 1.0, 0.1, True, "bf16"),
    ]


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kind = rng.choice(["append", "attention", "attention", "scores"])
    if kind == "scores":
        backward, vocab = rng.random() < 0.5, spread(1000, 128000)
        rows = spread(1, min(4096, 4096 * 128000 // vocab // 2))
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        return unnamed(scores_case("", rows, vocab, rng.choice([0, 1, 5, 20, 32]), rng.choice([1.0, 0.7, 1.3]),
                                   rng.choice([0.0, 0.4]), backward, dtype))
    heads, kv_heads, head_dim = rng.choice([(32, 8, 128), (16, 4, 128), (8, 2, 64), (16, 16, 64), (12, 4, 128)])
    page = rng.choice([16, 32, 64, 128])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    if kind == "append":
        batch, new = spread(1, 200), rng.choice([1, 1, spread(2, 1500)])
        batch = max(1, min(batch, 30000 // new))
        past = spread(1, 4000)
        return unnamed(append_case("", batch, max(1, new // 4), new, past // 8, past, heads, kv_heads, head_dim, page,
                                   rng.choice([0, 1, 2]), dtype))
    new = rng.choice([1, 1, 1, spread(2, 12), spread(16, 1500)])
    past = spread(1, 14000) if new > 1 else spread(1, 60000)
    batch = spread(1, 64)
    batch = max(1, min(batch, 520000 // (past + new), 3000 // new))
    return unnamed(attention_case("", batch, max(1, new // 4), new, past // 6, past, heads, kv_heads, head_dim, page,
                                  rng.random() < 0.5, rng.choice([0, 0, 1 + past // 3]), dtype))


def unnamed(c):
    return {k: v for k, v in c.items() if k != "name"}


# ---- work -----------------------------------------------------------------------------------------
ITEM = {"bf16": 2, "f16": 2, "f32": 4}


def work(c):
    e = ITEM[c["dtype"]]
    if c["op"] == "scores":
        n = c["rows"] * (1.0 - c["ignored"]) * c["vocab"]
        write = c["rows"] * c["vocab"] * e if c["backward"] else 0
        return {"bytes": n * e + write, "flops": n * (14 if c["backward"] else 7)}
    new, total = lengths(c)
    H, G, D = c["heads"], c["kv_heads"], c["head_dim"]
    if c["op"] == "append":
        T = sum(new)
        kv = 2 * T * G * D * (e + 1)
        qs = 2 * c["queries"] * T * H * D * e
        return {"bytes": kv + qs + T * D * 4, "flops": 3 * T * D * (G + c["queries"] * H) + 2 * T * G * D}
    maps = 2 if c["diff"] else 1
    W = c["window"] or (1 << 40)
    read = sum(min(L, W + n - 1) for n, L in zip(new, total)) * G * D * 2
    pairs = sum(min(L - n + i + 1, W) for n, L in zip(new, total) for i in range(n))
    return {"bytes": read + sum(new) * H * D * e * (maps + 1), "flops": 4.0 * pairs * H * D * maps}


# ---- inputs ---------------------------------------------------------------------------------------
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
DEV = "cuda"


def block_scale(amax):
    """The power of two 2^e with the least e for which amax <= 448 * 2^e (448 = 0.875 * 2^9), e in [-100, 119]."""
    m, x = torch.frexp(amax)
    e = torch.where(m > 0.875, x - 8, x - 9)
    e = torch.where(amax > 0, e, torch.full_like(e, -100)).clamp(-100, 119)
    return torch.ldexp(torch.ones_like(amax), e)


def cache_for(c, g, past):
    """A pool whose pages hold `past` tokens of each sequence in scrambled pages; slots past the end hold NaN codes."""
    new, total = lengths(c)
    G, D, ps, B = c["kv_heads"], c["head_dim"], c["page"], c["batch"]
    need = [-(-L // ps) for L in total]
    P = sum(need) + 3
    perm = torch.randperm(P, generator=g, device=DEV).to(torch.int32)
    table = torch.full((B, max(need)), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = torch.arange(at, at + n, dtype=torch.int32)
        at += n
    table = table.to(DEV)
    table = torch.where(table >= 0, perm[table.clamp(min=0).long()], table)
    held = torch.zeros(P + 1, dtype=torch.long, device=DEV)          # tokens that each page holds
    first = torch.arange(max(need), device=DEV) * ps
    inside = (torch.tensor(past, device=DEV)[:, None] - first[None]).clamp(0, ps)
    held[torch.where(table >= 0, table, P).long()] = inside
    stale = torch.arange(ps, device=DEV)[None] >= held[:P, None]                      # (P, ps)
    out = {}
    for name in ("k", "v"):
        x = torch.randn(P, G, ps, D, generator=g, device=DEV)
        if name == "k":                                             # keys have a few strong channels
            x *= torch.where(torch.rand(D, generator=g, device=DEV) < 0.05, 6.0, 1.0)
        x.masked_fill_(stale[:, None, :, None], 0.0)
        s = block_scale(x.abs().amax((2, 3)))
        codes = (x / s[..., None, None]).to(torch.float8_e4m3fn).view(torch.uint8)
        codes.masked_fill_(stale[:, None, :, None], 0x7F)
        out[name], out[name + "_scale"] = codes.view(torch.float8_e4m3fn), s
    return out, table


def prepare(c, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    dt = TYPES[c["dtype"]]
    if c["op"] == "scores":
        R, V = c["rows"], c["vocab"]
        x = torch.randn(R, V, generator=g, device=DEV, dtype=torch.float32 if R * V < 1 << 28 else dt).mul_(2.0)
        lift = torch.randint(0, V, (R, 12), generator=g, device=DEV)   # a few likely continuations
        x.scatter_add_(1, lift, (4.0 + 8.0 * torch.rand(R, 12, generator=g, device=DEV)).to(x.dtype))
        x = x.to(dt)
        target = torch.where(torch.rand(R, generator=g, device=DEV) < 0.7, lift[:, 0],
                             torch.randint(0, V, (R,), generator=g, device=DEV))
        n = round(R * c["ignored"])                                    # prompt positions
        target[:n] = -100
        st = {"c": c, "logits": x, "target": target}
        if c["backward"]:
            x.requires_grad_(True)
            st["g_lp"] = torch.randn(R, generator=g, device=DEV)
            st["g_ent"] = 0.1 * torch.randn(R, generator=g, device=DEV)
        return st
    new, total = lengths(c)
    H, G, D, B, T = c["heads"], c["kv_heads"], c["head_dim"], c["batch"], sum(new)
    cache, table = cache_for(c, g, [L - n for n, L in zip(new, total)] if c["op"] == "append" else total)
    cu = torch.tensor([0] + new).cumsum(0).to(torch.int32).to(DEV)
    st = {"c": c, "cache": cache, "table": table, "cu": cu, "lens": torch.tensor(total, dtype=torch.int32, device=DEV),
          "max_new": max(new)}
    rand = lambda *s: torch.randn(*s, generator=g, device=DEV).to(dt)  # noqa: E731
    if c["op"] == "append":
        st["k"], st["v"] = rand(T, G, D), rand(T, G, D)
        st["queries"] = [rand(T, H, D) for _ in range(c["queries"])]
        pos = torch.cat([torch.arange(L - n, L) for n, L in zip(new, total)])
        st["pos"] = pos.to(DEV)
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
    return {"append": run_append, "attention": run_attention, "scores": run_scores}[st["c"]["op"]](st)


def run_append(st):
    c, kv = st["c"], st["cache"]
    if own:
        from mamformer_b200 import ops
        qs = ops.kv_append(st["k"], st["v"], ops.PagedKV(kv["k"], kv["v"], kv["k_scale"], kv["v_scale"]), st["table"],
                           st["cu"], st["lens"], st["max_new"], st["cos"], st["sin"], st["pos"], st["queries"])
    else:
        cos, sin = st["cos"][st["pos"]][:, None], st["sin"][st["pos"]][:, None]
        qs = [rotated(q.float(), cos, sin).to(q.dtype) for q in st["queries"]]
        plain_append(st, "k", rotated(st["k"].float(), cos, sin))
        plain_append(st, "v", st["v"].float())
    return {"k": kv["k"], "v": kv["v"], "k_scale": kv["k_scale"], "v_scale": kv["v_scale"], "queries": list(qs)}


def rotated(x, cos, sin):
    a, b = x[..., : x.shape[-1] // 2], x[..., x.shape[-1] // 2:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def plain_append(st, name, x):
    """Every touched page: take its held tokens, lay the new ones over them, choose the scale, quantise, put it back."""
    c, codes, scales, cu = st["c"], st["cache"][name], st["cache"][name + "_scale"], st["cu"].long()
    ps = c["page"]
    end = st["lens"].long()
    start = end - (cu[1:] - cu[:-1])
    n = (st["max_new"] + ps - 2) // ps + 1
    which = start[:, None] // ps + torch.arange(n, device=x.device)                   # (B, n) page of the sequence
    b, _ = touched = torch.nonzero((which * ps < end[:, None]) & (end > start)[:, None], as_tuple=True)
    which = which[touched]
    page = st["table"][b, which].long()
    slot = which[:, None] * ps + torch.arange(ps, device=x.device)                    # (U, ps) slot of the sequence
    fresh = (slot >= start[b][:, None]) & (slot < end[b][:, None])
    old = slot < start[b][:, None]
    new = x[(cu[b][:, None] + slot - start[b][:, None]).clamp(0, x.shape[0] - 1)].transpose(1, 2)   # (U, G, ps, D)
    new = torch.where(fresh[:, None, :, None], new, 0.0)
    need = block_scale(torch.where(torch.isfinite(new), new.abs(), 0.0).amax((2, 3)))
    had = scales[page]
    s = torch.where(old[:, :1], torch.maximum(had, need), need)
    kept = codes.view(torch.uint8)[page]
    value = torch.where(fresh[:, None, :, None], new / s[..., None, None],
                        kept.view(torch.float8_e4m3fn).float() * (had / s)[..., None, None]).clamp(-448.0, 448.0)
    put = torch.where((fresh | old)[:, None, :, None], value.to(torch.float8_e4m3fn).view(torch.uint8), kept)
    codes.view(torch.uint8)[page] = put
    scales[page] = s


def run_attention(st):
    c, kv = st["c"], st["cache"]
    if own:
        from mamformer_b200 import ops
        return ops.paged_attention(st["q"], ops.PagedKV(kv["k"], kv["v"], kv["k_scale"], kv["v_scale"]), st["table"],
                                   st["cu"], st["lens"], st["max_new"], q2=st.get("q2"), lam=st.get("lam"),
                                   window=c["window"])
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

    def held(name):
        x = kv[name].view(torch.uint8)[table.clamp(min=0)].view(torch.float8_e4m3fn).float()
        x = x * kv[name + "_scale"][table.clamp(min=0)][..., None, None]
        x = x.transpose(1, 2).reshape(B, G, 1, L, D)
        return torch.where((slot < lens[:, None])[:, None, None, :, None], x, 0.0)

    k, v = held("k"), held("v")
    token = (cu[:-1, None] + i).clamp(max=st["q"].shape[0] - 1)
    real = i < (cu[1:] - cu[:-1])[:, None]                                            # (B, N)

    def one(q):
        x = q[token].float().unflatten(2, (G, -1)).permute(0, 2, 3, 1, 4)             # (B, G, H / G, N, D)
        s = (x @ k.transpose(-1, -2)).mul_(D ** -0.5).masked_fill_(~see, -math.inf)
        m = s.amax(-1, keepdim=True)
        p = s.sub_(torch.where(m == -math.inf, 0.0, m)).exp_()
        d = p.sum(-1, keepdim=True)
        return ((p @ v) / torch.where(d > 0, d, 1.0)).permute(0, 3, 1, 2, 4).flatten(2, 3)

    o = one(st["q"])
    if c["diff"]:
        lam = st["lam"][:, None]
        o = (o - lam * one(st["q2"])) / (1.0 - lam + 1e-8)
    return o[real].to(st["q"].dtype)


def run_scores(st):
    c, x = st["c"], st["logits"]
    if own:
        from mamformer_b200 import ops
        s = ops.token_scores(x, st["target"], top_k=c["top_k"], temperature=c["temperature"])
        out = {"log_probs": s.log_probs.detach(), "entropy": s.entropy.detach(), "top_log_probs": s.top_log_probs.detach(),
               "top_ids": s.top_ids}
        if c["backward"]:
            out["grad"], = torch.autograd.grad((s.log_probs, s.entropy), x, (st["g_lp"], st["g_ent"]))
        return out
    x = x.detach().float()
    live = st["target"] != -100
    u = (x - x.amax(1, keepdim=True)) / c["temperature"]
    e = u.exp()
    z = e.sum(1, keepdim=True)
    lse = z.log()
    ent = lse - (u * e).sum(1, keepdim=True) / z
    t = st["target"].clamp(min=0)[:, None]
    out = {"log_probs": torch.where(live, (u.gather(1, t) - lse)[:, 0], 0.0), "entropy": torch.where(live, ent[:, 0], 0.0)}
    ids = top_ids(x, c["top_k"])
    out["top_log_probs"] = torch.where(live[:, None], u.gather(1, ids) - lse, 0.0)
    out["top_ids"] = torch.where(live[:, None], ids, -1)
    if c["backward"]:
        g1, g2 = (torch.where(live, g, 0.0)[:, None] for g in (st["g_lp"], st["g_ent"]))
        p = e / z
        d = (u - lse + ent).mul_(g2).add_(g1).mul_(p).neg_()
        d.scatter_add_(1, t, g1)
        out["grad"] = (d / c["temperature"]).to(st["logits"].dtype)
    return out


def top_ids(x, k):
    """The k largest of each row in descending order, ties to the lowest index: one whole number for value and index."""
    if k == 0:
        return torch.zeros(x.shape[0], 0, dtype=torch.long, device=x.device)
    bits = (x + 0.0).view(torch.int32).long()
    key = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits) * (1 << 20) - torch.arange(x.shape[1], device=x.device)
    return torch.topk(key, k, dim=1).indices


# ---- the definitions in 64 bits -------------------------------------------------------------------
def exact(c, seed):
    st = prepare(c, seed)
    return {"append": exact_append, "attention": exact_attention, "scores": exact_scores}[c["op"]](c, st)


def exact_append(c, st):
    """Token by token rotation as a complex product; page by page quantisation of what the page then holds."""
    ps, D = c["page"], c["head_dim"]
    new, total = lengths(c)
    turn = torch.complex(st["cos"].double(), st["sin"].double())[st["pos"]][:, None]

    def turned(x):
        z = torch.complex(x[..., : D // 2].double(), x[..., D // 2:].double()) * turn
        return torch.cat([z.real, z.imag], -1)

    out = {"queries": [turned(q) for q in st["queries"]]}
    for name, x in (("k", turned(st["k"])), ("v", st["v"].double())):
        codes, scale = st["cache"][name].double(), st["cache"][name + "_scale"].double()
        table, at = st["table"].tolist(), 0
        for b, (n, L) in enumerate(zip(new, total)):
            start = L - n
            for j in range(start // ps, -(-L // ps)):
                lo, hi = max(start, j * ps), min(L, (j + 1) * ps)
                block = x[at + lo - start: at + hi - start].transpose(0, 1)             # (G, tokens, D)
                s = 2.0 ** torch.ceil(torch.log2(block.abs().amax((1, 2)) / 448.0))
                p, keep = table[b][j], lo - j * ps
                if keep:
                    s = torch.maximum(s, scale[p])
                    codes[p, :, :keep] = e4m3(codes[p, :, :keep] * (scale[p] / s)[:, None, None])
                codes[p, :, keep: hi - j * ps] = e4m3(block / s[:, None, None])
                scale[p] = s
            at += n
        out[name], out[name + "_scale"] = codes, scale
    return out


def e4m3(x):
    """x rounded to 4 significant bits (spacing 2^-9 below 2^-6), ties to even, within +-448; 64 bits throughout."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3.0)
    return (torch.round(x / step) * step).clamp(-448.0, 448.0)


def exact_attention(c, st):
    new, total = lengths(c)
    H, G, D, ps, W = c["heads"], c["kv_heads"], c["head_dim"], c["page"], c["window"]
    out = torch.zeros(sum(new), H, D, dtype=torch.float64, device=DEV)
    at = 0
    for b, (n, L) in enumerate(zip(new, total)):
        pages = st["table"][b, : -(-L // ps)].long()
        kv = [(st["cache"][x].view(torch.uint8)[pages].view(torch.float8_e4m3fn).double()
               * st["cache"][x + "_scale"].double()[pages][..., None, None]).transpose(0, 1).reshape(G, -1, D)[:, :L]
              for x in ("k", "v")]
        where = torch.arange(L - n, L, device=DEV)[:, None] - torch.arange(L, device=DEV)[None]
        hide = (where < 0) | (where >= W) if W else where < 0
        for h in range(H):
            k, v = (x[h // (H // G)] for x in kv)
            maps = []
            for q in [st["q"]] + ([st["q2"]] if c["diff"] else []):
                s = (q[at: at + n, h].double() @ k.T) / math.sqrt(D)
                maps.append(torch.softmax(s.masked_fill(hide, -math.inf), -1) @ v)
            if c["diff"]:
                lam = st["lam"][h].double()
                maps[0] = (maps[0] - lam * maps[1]) / (1.0 - lam + 1e-8)
            out[at: at + n, h] = maps[0]
        at += n
    return out


def exact_scores(c, st):
    R, V, T = c["rows"], c["vocab"], c["temperature"]
    keys = ["log_probs", "entropy", "top_log_probs"] + (["grad"] if c["backward"] else [])
    parts = {k: [] for k in keys}
    for r in range(0, R, 512):
        x, t = st["logits"].detach()[r: r + 512].double() / T, st["target"][r: r + 512]
        live = (t != -100)[:, None]
        lp = torch.log_softmax(x, -1)
        p = lp.exp()
        ent = -(p * lp).sum(-1, keepdim=True)
        parts["log_probs"].append(torch.where(live, lp.gather(1, t.clamp(min=0)[:, None]), 0.0)[:, 0])
        parts["entropy"].append(torch.where(live, ent, 0.0)[:, 0])
        parts["top_log_probs"].append(torch.where(live, lp.sort(-1, descending=True).values[:, : c["top_k"]], 0.0))
        if c["backward"]:
            g1, g2 = (st[k][r: r + 512].double()[:, None] for k in ("g_lp", "g_ent"))
            hot = torch.zeros_like(p).scatter_(1, t.clamp(min=0)[:, None], 1.0)
            parts["grad"].append(torch.where(live, (g1 * (hot - p) - g2 * p * (lp + ent)) / T, 0.0))
    out = {k: torch.cat(v) for k, v in parts.items()}
    out["top_ids"] = None
    return out

"""The paged 8-bit cache in the models: PagedKVCache's bookkeeping, attention modules decoding on it against the same
module on the values the cache holds, generate(kv_cache="paged") and a GRPO step that rolls out on it and scores its
tokens with entropies.

Tolerances: a stored value is within 2^-4 of itself, so an attention output, a weighted mean of values under weights
exp(score) whose scores move by at most the sum of |q_d k_d| 2^-4 sqrt(1 / hd), is compared on the stored values
(difference: roundings of the layers only) rather than on the exact ones."""

import math
import os

import pytest
import torch

from mamformer_b200 import ops
from mamformer_b200.config import MamformerConfig
from mamformer_b200.models.attention import GroupedQueryAttention
from mamformer_b200.models.kda_diff import FullDiffAttention
from mamformer_b200.models.model import MamformerForCausalLM
from mamformer_b200.paged_cache import PagedKVCache

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DEVICES = [("cpu", torch.float32), pytest.param("cuda", torch.bfloat16, marks=pytest.mark.gpu)]


def test_bookkeeping():
    c = PagedKVCache(2, 2, 64, batch=3, max_len=100, page_size=16, n_pages=12, device="cpu")
    c.extend([20, 0, 33])
    assert c.lens == [20, 0, 33] and c.kv_lens.tolist() == [20, 0, 33] and c.cu_seqlens.tolist() == [0, 20, 20, 53]
    assert c.max_new == 33 and c.tokens == 53
    used = c.block_table[c.block_table >= 0].tolist()
    assert len(used) == 5 and len(set(used)) == 5
    c.extend(1)
    assert c.lens == [21, 1, 34] and c.cu_seqlens.tolist() == [0, 1, 2, 3] and (c.block_table >= 0).sum() == 6
    c.release(2)
    assert c.kv_lens.tolist() == [21, 1, 0] and (c.block_table[2] == -1).all() and len(c._free) == 12 - 3
    c.extend([0, 0, 100])
    assert (c.block_table[2] >= 0).sum() == 7
    held = c.block_table[c.block_table >= 0].tolist()
    assert len(held) == len(set(held))
    with pytest.raises(ValueError, match="room"):
        c.extend([0, 0, 20])
    with pytest.raises(RuntimeError, match="free"):
        c.extend([70, 50, 0])
    with pytest.raises(ValueError):
        c.extend([1, 2])
    assert c.lens == [21, 1, 100]                                # a refused step changes nothing
    for kw in ({"page_size": 24}, {"head_dim": 80}):
        with pytest.raises(ValueError):
            PagedKVCache(**{**dict(n_layers=1, n_kv_heads=1, head_dim=64, batch=1, max_len=9, device="cpu"), **kw})


def stored(layer, owner, b):
    page = owner.page_size
    pages = owner.block_table[b, :-(-owner.lens[b] // page)].long()
    out = []
    for x, s in ((layer.kv.k, layer.kv.k_scale), (layer.kv.v, layer.kv.v_scale)):
        x = x.view(torch.uint8)[pages].view(torch.float8_e4m3fn).double() * s[pages].double()[..., None, None]
        out.append(x.transpose(0, 1).reshape(owner.n_kv_heads, -1, owner.head_dim)[:, :owner.lens[b]])
    return out


@pytest.mark.parametrize("dev,dtype", DEVICES)
@pytest.mark.parametrize("kind", ["gqa", "diff"])
@pytest.mark.parametrize("window", [0, 24])
def test_modules_attend_to_what_the_cache_holds(dev, dtype, kind, window):
    torch.manual_seed(0)
    B, S, H, G, hd, d = 2, 37, 4, 2, 64, 256
    kw = dict(n_heads=H, n_kv_heads=G, head_dim=hd, sliding_window=window, window_mode="causal")
    mod = (GroupedQueryAttention(d, **kw) if kind == "gqa" else FullDiffAttention(d, latent_dim=64, use_state_injection=False, **kw))
    mod = mod.to(dev, dtype)
    for p in mod.parameters():                                   # outputs of the size of their inputs
        if p.dim() == 2:
            torch.nn.init.normal_(p, std=p.shape[1] ** -0.5)
    if kind == "diff":
        mod.lambda_raw.data = mod.lambda_raw.data.float()
    owner = PagedKVCache(1, G, hd, B, S + 3, page_size=16, device=dev)
    layer = owner.layer(0)
    x = torch.randn(B, S + 3, d).to(dev, dtype)
    seen = {}
    mod.o_proj.register_forward_pre_hook(lambda m, args: seen.update(out=args[0]))
    if kind == "diff":                                           # the attention itself, before its norm
        mod._norm_and_project = lambda o: mod.o_proj(o.reshape(o.shape[0], o.shape[1], -1))
    at = 0
    for n in (S, 1, 2):
        owner.extend(n)
        with torch.no_grad():
            y, cache = mod(x[:, at:at + n], use_cache=True, cache={"attn_type": "full", "paged": layer})
        assert cache["paged"] is layer and y.shape == (B, n, d)
        xs = x[:, at:at + n]
        cos, sin = (t[0, 0, :, :hd // 2] for t in mod.rope(n, xs.device, 0))
        qs = [mod.q_proj] if kind == "gqa" else [mod.q1_proj, mod.q2_proj]
        qs = [ops.rope(p(xs).view(B, n, H, hd), cos, sin).double() for p in qs]
        at += n
        for b in range(B):
            k, v = (t.repeat_interleave(H // G, 0) for t in stored(layer, owner, b))
            i, j = torch.arange(at - n, at, device=dev)[:, None], torch.arange(at, device=dev)
            see = (j <= i) & (j > i - window) if window else j <= i
            maps = [torch.softmax((q[b].transpose(0, 1) @ k.transpose(1, 2) / math.sqrt(hd)).masked_fill(~see, -math.inf), -1) @ v
                    for q in qs]
            want, gain = maps[0], 1.0
            if kind == "diff":
                lam = torch.sigmoid(mod.lambda_raw.double()).clamp(max=0.99)[:, None, None]
                want, gain = (maps[0] - lam * maps[1]) / (1 - lam + 1e-8), 9.0
            got = seen["out"][b].view(n, H, hd).transpose(0, 1).double()
            unit = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -20
            # rotated queries are rounded once more than here: a score moves by |s| times the type's rounding
            tol = unit * want.abs() + gain * v.abs().amax() * ((2.0 ** -8 * 3 if dtype == torch.bfloat16 else 2.0 ** -18) + 2.0 ** -11)
            assert ((got - want).abs() <= tol).all()


def small_config(hd=64):
    d = MamformerConfig.from_yaml(os.path.join(ROOT, "configs", "ultra-7b.yaml")).to_dict()
    d.update(d_model=2 * hd, n_heads=2, n_kv_heads=1, head_dim=hd, n_layers=4, vocab_size=259, moe_enabled=False,
             interleave_fusion_layers=[3], interleave_last_layers_dense=1, kda_diff_kernel_dim=hd, kda_diff_latent_dim=32,
             kda_diff_linear_ratio=0, kda_diff_use_dynamic_ratio=False, use_sliding_window=False, d_ff=128, mamba_d_state=32, mtp_enabled=False)
    return MamformerConfig.from_dict(d)


@pytest.mark.parametrize("dev,dtype", DEVICES)
def test_generate_on_the_paged_cache(dev, dtype):
    torch.manual_seed(1)
    model = MamformerForCausalLM(small_config()).eval()
    if dtype == torch.bfloat16:
        from mamformer_b200.utils.precision import to_compute_dtype
        to_compute_dtype(model, dtype)
    model = model.to(dev)
    ids = torch.randint(0, 259, (2, 21), generator=torch.Generator().manual_seed(2)).to(dev)
    calls = []
    real = ops.paged_attention
    try:
        ops.paged_attention = lambda *a, **k: calls.append(a[0].shape[0]) or real(*a, **k)
        out = model.generate(ids, max_new_tokens=6, temperature=0.0, kv_cache="paged")
    finally:
        ops.paged_attention = real
    assert out.shape == (2, 27) and torch.equal(out[:, :21], ids)
    assert calls and calls[0] == 42 and set(calls[1:]) <= {42, 2}
    dense = model.generate(ids, max_new_tokens=6, temperature=0.0)
    assert dense.shape == out.shape
    with pytest.raises(ValueError):
        model.generate(ids, max_new_tokens=2, kv_cache="other")


@pytest.mark.parametrize("dev,dtype", DEVICES)
def test_prompt_logits_on_both_caches(dev, dtype):
    """The first forward differs only by the stored values' rounding (2^-4 of each, averaged over keys and dims)."""
    torch.manual_seed(1)
    model = MamformerForCausalLM(small_config()).eval()
    if dtype == torch.bfloat16:
        from mamformer_b200.utils.precision import to_compute_dtype
        to_compute_dtype(model, dtype)
    model = model.to(dev)
    ids = torch.randint(0, 259, (2, 40), generator=torch.Generator().manual_seed(2)).to(dev)
    paged = PagedKVCache.for_model(model, 2, 50)
    paged.extend(40)
    with torch.no_grad():
        a = model(ids, use_cache=True, cache=paged.layer_caches(), return_logits=True)["logits"].double()
        b = model(ids, use_cache=True, return_logits=True)["logits"].double()
    assert (a - b).norm() <= 2.0 ** -4 * b.norm()


@pytest.mark.parametrize("dev,dtype", DEVICES)
def test_token_scores_of_a_model(dev, dtype):
    torch.manual_seed(1)
    model = MamformerForCausalLM(small_config())
    if dtype == torch.bfloat16:
        from mamformer_b200.utils.precision import to_compute_dtype
        to_compute_dtype(model, dtype)
    model = model.to(dev)
    ids = torch.randint(0, 259, (2, 19), generator=torch.Generator().manual_seed(2)).to(dev)
    labels = ids.clone()
    labels[:, :7] = -100
    s = model.get_token_scores(ids, labels=labels, top_k=3)
    assert s.log_probs.shape == s.entropy.shape == (2, 18) and s.top_ids.shape == (2, 18, 3)
    assert (s.log_probs[:, :6] == 0).all() and (s.top_ids[:, :6] == -1).all()
    with torch.no_grad():
        lp = torch.log_softmax(model(ids, return_logits=True)["logits"].double(), -1)[:, :-1]
    assert (s.log_probs[:, 6:].double() - lp.gather(-1, ids[:, 1:, None])[..., 0][:, 6:]).abs().max() < 1e-5
    assert (s.entropy[:, 6:].double() + (lp.exp() * lp).sum(-1)[:, 6:]).abs().max() < 1e-5
    mean = model.get_log_probs(ids, labels=labels)
    assert torch.allclose(mean, s.log_probs[:, 6:].mean(1), atol=1e-5)
    (s.log_probs.sum() + s.entropy.sum()).backward()
    assert model.model.embed_tokens.weight.grad.isfinite().all()


@pytest.mark.parametrize("dev,dtype", DEVICES)
def test_grpo_step_on_the_paged_cache(dev, dtype):
    from mamformer_b200.grpo import GRPOConfig, GRPOTrainer
    from mamformer_b200.tokenizer import MamformerTokenizer
    torch.manual_seed(1)
    tok = MamformerTokenizer()
    cfg = small_config()
    cfg.vocab_size = max(cfg.vocab_size, len(tok) if hasattr(tok, "__len__") else 259)
    model = MamformerForCausalLM(cfg).to(dev)
    trainer = GRPOTrainer(model, tok, GRPOConfig(group_size=2, gen_max_tokens=5, gen_kv_cache="paged", entropy_beta=0.01),
                          compute_dtype=dtype)
    batch = {"input_ids": torch.randint(0, 200, (2, 9)), "ground_truth": ["4", "5"], "reward_type": ["math", "math"],
             "test_cases": [[], []], "reward_weights": [None, None]}
    m = trainer.step(batch)
    assert torch.isfinite(m["loss"]) and m["entropy"] > 0


def test_refusals():
    cfg = small_config()
    torch.manual_seed(0)
    model = MamformerForCausalLM(cfg)
    cfg.use_sliding_window = True
    windowed = FullDiffAttention(128, 2, 1, 64, sliding_window=8, window_mode="reference")
    model.model.layers[3].attention.full_attn = windowed
    with pytest.raises(ValueError, match="window"):
        PagedKVCache.for_model(model, 1, 10)
    owner = PagedKVCache(1, 1, 64, 1, 10, device="cpu")
    owner.extend(2)
    att = FullDiffAttention(128, 2, 1, 64, latent_dim=16, use_state_injection=False)
    x = torch.randn(1, 2, 128)
    cache = {"attn_type": "full", "paged": owner.layer(0)}
    with torch.no_grad(), pytest.raises(ValueError, match="attention_mask"):
        att(x, attention_mask=torch.zeros(1, 1, 2, 2), use_cache=True, cache=cache)
    with pytest.raises(RuntimeError, match="no gradient"):
        att(x, use_cache=True, cache=cache)
    with torch.no_grad(), pytest.raises(ValueError, match="rows"):
        att(x[:, :1], use_cache=True, cache=cache)


@pytest.mark.gpu
def test_errors_on_the_device_reach_the_caller(monkeypatch):
    """A page outside the pool is raised by generate and by a GRPO step, which leaves the weights alone."""
    from mamformer_b200.fault import PagedCacheError, check_device_status
    from mamformer_b200.grpo import GRPOConfig, GRPOTrainer
    from mamformer_b200.tokenizer import MamformerTokenizer
    from mamformer_b200.utils.precision import to_compute_dtype
    torch.manual_seed(1)
    check_device_status()
    cfg = small_config()
    model = MamformerForCausalLM(cfg).eval().cuda()
    trainer = GRPOTrainer(model, MamformerTokenizer(), GRPOConfig(group_size=2, gen_max_tokens=3), compute_dtype=torch.bfloat16)
    before = [p.detach().clone() for p in trainer.policy.parameters()]
    batch = {"input_ids": torch.randint(0, 200, (2, 9)), "ground_truth": ["4", "5"], "reward_type": ["math", "math"],
             "test_cases": [[], []], "reward_weights": [None, None]}
    score = trainer.score
    spoiled = PagedKVCache(1, 1, 64, 1, 10)

    def spoil(*args):
        spoiled.extend(1)
        q = torch.zeros(1, 1, 2, 64, dtype=torch.bfloat16, device="cuda")
        spoiled.block_table.fill_(-1)
        with torch.no_grad():
            spoiled.layer(0).attend(q, q[:, :, :1], q[:, :, :1], torch.ones(1, 32, device="cuda"), torch.zeros(1, 32, device="cuda"))
        return score(*args)

    monkeypatch.setattr(trainer, "score", spoil)
    with pytest.raises(PagedCacheError, match="page of the pool"):
        trainer.step(batch)
    assert all(torch.equal(a, b) for a, b in zip(before, trainer.policy.parameters()))
    extend = PagedKVCache.extend

    def broken(self, new):
        extend(self, new)
        self.block_table.fill_(-1)

    monkeypatch.setattr(PagedKVCache, "extend", broken)
    half = to_compute_dtype(MamformerForCausalLM(cfg).eval(), torch.bfloat16).cuda()
    with pytest.raises(PagedCacheError, match="page of the pool"):
        half.generate(torch.randint(0, 200, (2, 9), device="cuda"), max_new_tokens=2, temperature=0.0, kv_cache="paged")
    check_device_status()


def test_a_tensor_parallel_rank_holds_its_heads():
    model = MamformerForCausalLM(small_config())
    for layer in model.model.layers:
        att = getattr(layer, "attention", None)
        if att is not None:
            att.full_attn.n_kv_heads = 7                              # what sharding leaves on the module
    assert PagedKVCache.for_model(model, 1, 10).n_kv_heads == 7
    model.model.layers[0].attention.full_attn.n_kv_heads = 3
    with pytest.raises(ValueError, match="one number"):
        PagedKVCache.for_model(model, 1, 10)


@pytest.mark.gpu
def test_fp32_models_are_refused_before_anything_is_cached():
    model = MamformerForCausalLM(small_config()).eval().cuda()
    ids = torch.randint(0, 200, (1, 5), device="cuda")
    with pytest.raises(ValueError, match="bf16"):
        model.generate(ids, max_new_tokens=2, kv_cache="paged")
    with torch.autocast("cuda", dtype=torch.bfloat16):
        PagedKVCache.for_model(model, 1, 10)


@pytest.mark.parametrize("extra", [["--num_beams", "2"], ["--thinking", "FastThink"]])
def test_the_script_refuses_what_the_paged_cache_does_not_do(extra):
    import sys
    sys.path.insert(0, os.path.join(ROOT, "scripts"))
    try:
        import generate as script
    finally:
        sys.path.pop(0)
    from mamformer_b200.tokenizer import MamformerTokenizer
    args = script.build_parser().parse_args(["--config", "x", "--kv_cache", "paged", "--max_new_tokens", "2"] + extra)
    model = MamformerForCausalLM(small_config()).eval()
    with pytest.raises(ValueError, match="paged"):
        script.generate_text(model, MamformerTokenizer(), "a", args)


def test_configs_set_the_window_mode(tmp_path):
    for name in ("pro-7b", "ultra-7b", "ultra-37b"):
        c = MamformerConfig.from_yaml(os.path.join(ROOT, "configs", f"{name}.yaml"))
        assert c.use_sliding_window and c.window_mode == "reference" and "window_mode" not in c.to_dict()
    cfg = small_config()
    d = cfg.to_dict()
    d.update(use_sliding_window=True, sliding_window=8)
    with pytest.raises(ValueError, match="window_mode"):
        PagedKVCache.for_model(MamformerForCausalLM(MamformerConfig.from_dict(d)), 1, 10)
    with pytest.raises(ValueError, match="window_mode"):
        MamformerConfig.from_dict({**d, "window_mode": "both"})
    path = str(tmp_path / "c.yaml")
    for nested in (False, True):
        MamformerConfig.from_dict({**d, "window_mode": "causal"}).to_yaml(path, nested)
        cfg = MamformerConfig.from_yaml(path)
        assert cfg.window_mode == "causal"
    torch.manual_seed(0)
    model = MamformerForCausalLM(cfg).eval()
    ids = torch.randint(0, 200, (2, 21))
    paged = PagedKVCache.for_model(model, 2, 30)
    paged.extend(21)
    with torch.no_grad():
        a = model(ids, use_cache=True, cache=paged.layer_caches(), return_logits=True)["logits"].double()
        b = model(ids, use_cache=True, return_logits=True)["logits"].double()
    assert (a - b).norm() <= 2.0 ** -4 * b.norm()
    assert model.generate(ids, max_new_tokens=3, temperature=0.0, kv_cache="paged").shape == (2, 24)


@pytest.mark.parametrize("dev,dtype", DEVICES)
def test_a_gated_layer_stays_on_the_paged_cache(dev, dtype, monkeypatch):
    """full, linear, full: as on the dense cache, the layer attends to what comes after the last turn, and stays paged."""
    from mamformer_b200.models.kda_diff import KDADiffAttention
    torch.manual_seed(0)
    B, H, G, hd, d = 2, 4, 2, 64, 256
    mod = KDADiffAttention(d, H, G, hd, kernel_dim=64, latent_dim=64, use_state_injection=False, use_dynamic_ratio=True).to(dev, dtype)
    for p in mod.parameters():
        if p.dim() == 2:
            torch.nn.init.normal_(p, std=p.shape[1] ** -0.5)
    for m in (mod.full_attn, mod.linear_attn):
        m.lambda_raw.data = m.lambda_raw.data.float()
    turns = [True, True, False, False, True, True, False, True]
    counts = [18, 1, 1, 1, 1, 1, 1, 1]
    x = torch.randn(B, sum(counts), d).to(dev, dtype)
    h = torch.zeros(B, 1, 4, device=dev)
    owner = PagedKVCache(1, G, hd, B, sum(counts), page_size=16, device=dev)
    calls = []
    real = ops.paged_attention
    monkeypatch.setattr(ops, "paged_attention", lambda *a, **k: calls.append(a[4].tolist()) or real(*a, **k))
    paged, dense, at = {"attn_type": "full", "paged": owner.layer(0)}, None, 0
    for full, n in zip(turns, counts):
        monkeypatch.setattr(mod, "choose_full", lambda h: full)
        owner.extend(n)
        with torch.no_grad():
            a, paged = mod(x[:, at:at + n], use_cache=True, cache=paged, h_states=h)
            b, dense = mod(x[:, at:at + n], use_cache=True, cache=dense, h_states=h)
        assert paged["attn_type"] == ("full" if full else "linear") and paged["paged"] is owner.layer(0)
        at += n
        # the stored values' rounding, 2^-4 of each, on the full turns
        assert (a - b).double().norm() <= (2.0 ** -3 if full else 2.0 ** -20) * b.double().norm(), (full, at)
    assert calls == [[18, 18], [19, 19], [1, 1], [2, 2], [1, 1]]
    owner.release(0)
    owner.extend([3, 0])
    assert owner.layer(0)._skipped.tolist()[0] == 0

"""The 4-bit cache in the models: PagedKVCache(bits=4) with eviction, generate(kv_cache="paged4", kv_budget=..), GRPO rollouts
on it.  Attention over the cache is compared on the values that it holds (see test_paged4)."""

import pytest
import torch

from mamformer_b200 import ops
from mamformer_b200.models.model import MamformerForCausalLM
from mamformer_b200.paged_cache import PagedKVCache
from test_paged4 import close, held, plain
from test_paged_cache import rand
from test_paged_generate import DEVICES, small_config


def cache_of(dev, batch=3, max_len=100, layers=2, **kw):
    return PagedKVCache(layers, 2, 64, batch, max_len, page_size=16, device=dev, bits=4, weights=True, **kw)


@pytest.mark.parametrize("dev,dtype", DEVICES)
def test_layers_attend_evict_and_go_on(dev, dtype):
    c = cache_of(dev)
    cos, sin = torch.ones(1, 32, device=dev), torch.zeros(1, 32, device=dev)
    seen = []
    for step, new in enumerate(([70, 5, 33], [1, 1, 1], [1, 1, 1], [3, 0, 20], [1, 1, 1])):
        if step in (2, 4):
            before = [[held(x.kv, c.block_table, c.lens, b) for b in range(3)] for x in c.layers]
            pages = c._free[:]
            c.evict(24, 8)
            assert c.lens == [min(n, 24) for n in seen] and c.kv_lens.tolist() == c.lens and len(c._free) > len(pages)
            used = c.block_table[c.block_table >= 0].tolist()
            assert sorted(used + c._free) == list(range(c.n_pages)) and [len(p) for p in c._pages] == [-(-n // 16) for n in c.lens]
            for x, was in zip(c.layers, before):
                for b, n in enumerate(c.lens):
                    for got, had in zip(held(x.kv, c.block_table, c.lens, b), was[b]):
                        for g in range(2):                            # tokens of before, in order, the last 8 among them
                            at = [next(i for i in range(had.shape[1]) if torch.equal(had[g, i], y)) for y in got[g]]
                            assert at == sorted(set(at)) and at[-min(n, 8):] == list(range(had.shape[1]))[-min(n, 8):]
        c.extend(new)
        seen = c.lens[:]
        T = sum(new)
        for i in range(2):
            q, k, v = (rand((T, h, 64), dtype, dev, 10 * step + i + j) for j, h in ((0, 4), (3, 2), (6, 2)))
            layer = c.layer(i)
            mass = None if layer.kv is None else layer.kv.mass.double()
            got = layer.attend(q, k, v, cos.expand(T, -1), sin.expand(T, -1))
            want, tol, m, mt = plain(q, layer.kv, c.block_table, new, c.lens)
            close(got, want, tol + (2.0 ** -18 if dtype == torch.float32 else 0.0))
            if mass is not None:
                for b, n in enumerate(c.lens):
                    slot = torch.arange(n - new[b], device=dev)
                    at = c.block_table[b].long()[slot // 16], slice(None), slot % 16
                    close(layer.kv.mass[at], (mass + m)[at], (mt + 2.0 ** -23 * (mass + m))[at])
    with pytest.raises(ValueError, match="window"):
        c.extend(1)
        c.layer(0).attend(rand((3, 4, 64), dtype, dev, 1), *(rand((3, 2, 64), dtype, dev, 1) for _ in range(2)), cos.expand(3, -1), sin.expand(3, -1), window=5)
    c.check()


def test_a_layer_that_takes_part_later_keeps_its_own_length():
    c = cache_of("cpu")
    cos, sin = torch.ones(1, 32), torch.zeros(1, 32)

    def attend(i, T, seed):
        c.layer(i).attend(rand((T, 4, 64), torch.float32, "cpu", seed), *(rand((T, 2, 64), torch.float32, "cpu", seed + j) for j in (1, 2)),
                          cos.expand(T, -1), sin.expand(T, -1))

    c.extend([40, 9, 30])
    attend(0, 79, 1)
    c.extend([20, 0, 3])
    attend(0, 23, 2)
    c.layer(1).restart()
    attend(1, 23, 3)                                              # 20, 0 and 3 tokens of its own
    before = [held(c.layer(1).kv, c.block_table, [20, 0, 3], b) for b in (0, 2)]
    c.evict(24, 4)
    assert c.lens == [24, 9, 24] and (c.kv_lens - c.layer(1)._skipped).tolist() == [20, 0, 3]
    for was, b in zip(before, (0, 2)):
        for x, y in zip(was, held(c.layer(1).kv, c.block_table, [20, 0, 3], b)):
            assert torch.equal(x, y)
    c.evict(10, 4)
    assert c.lens == [10, 9, 10] and (c.kv_lens - c.layer(1)._skipped).tolist() == [10, 0, 3]


def test_refusals():
    for kw in ({"bits": 5}, {"bits": 8, "weights": True}):
        with pytest.raises(ValueError):
            PagedKVCache(1, 1, 64, 1, 9, device="cpu", **kw)
    c = PagedKVCache(1, 1, 64, 1, 99, device="cpu", bits=4)
    with pytest.raises(ValueError, match="weights"):
        c.evict(5)
    c = cache_of("cpu")
    c.extend([40, 3, 3])
    for args in ((0,), (5, 6), (5, -1)):
        with pytest.raises(ValueError):
            c.evict(*args)
    assert c.lens == [40, 3, 3]


@pytest.mark.parametrize("dev,dtype", DEVICES)
@pytest.mark.parametrize("budget", [None, 16])
def test_generate(dev, dtype, budget, monkeypatch):
    torch.manual_seed(1)
    model = MamformerForCausalLM(small_config()).eval()
    if dtype == torch.bfloat16:
        from mamformer_b200.utils.precision import to_compute_dtype
        to_compute_dtype(model, dtype)
    model = model.to(dev)
    ids = torch.randint(0, 259, (2, 100), generator=torch.Generator().manual_seed(2)).to(dev)
    cuts = []
    evict = PagedKVCache.evict
    monkeypatch.setattr(PagedKVCache, "evict", lambda self, *a: (cuts.append((self.lens[0], a)), evict(self, *a)))
    out = model.generate(ids, max_new_tokens=70, temperature=0.0, kv_cache="paged4", kv_budget=budget)
    assert out.shape == (2, 170) and torch.equal(out[:, :100], ids)
    # after the prompt, and whenever a page more than the budget is there
    assert cuts == ([] if budget is None else [(100, (16, 4)), (80, (16, 4))])
    assert torch.equal(out, model.generate(ids, max_new_tokens=70, temperature=0.0, kv_cache="paged4", kv_budget=budget))
    for kw in ({"kv_cache": "paged", "kv_budget": 9}, {"kv_budget": 9}, {"kv_cache": "paged4", "kv_budget": 0}):
        with pytest.raises(ValueError, match="kv_budget"):
            model.generate(ids, max_new_tokens=2, **kw)


@pytest.mark.parametrize("dev,dtype", DEVICES)
def test_first_tokens_agree_with_the_dense_cache_on_sharp_logits(dev, dtype):
    """A budget that nothing outgrows changes nothing."""
    torch.manual_seed(3)
    model = MamformerForCausalLM(small_config()).eval()
    if dtype == torch.bfloat16:
        from mamformer_b200.utils.precision import to_compute_dtype
        to_compute_dtype(model, dtype)
    model = model.to(dev)
    ids = torch.randint(0, 259, (1, 30), generator=torch.Generator().manual_seed(2)).to(dev)
    a = model.generate(ids, max_new_tokens=8, temperature=0.0, kv_cache="paged4")
    b = model.generate(ids, max_new_tokens=8, temperature=0.0, kv_cache="paged4", kv_budget=1000)
    assert torch.equal(a, b)


def test_windows_do_not_go_with_a_budget():
    cfg = small_config()
    cfg.use_sliding_window, cfg.sliding_window, cfg.window_mode = True, 16, "causal"
    model = MamformerForCausalLM(cfg)
    if any(getattr(getattr(x.attention, "full_attn", x.attention), "sliding_window", 0) for x in model.model.layers if x.attention is not None):
        with pytest.raises(ValueError, match="window"):
            PagedKVCache.for_model(model, 1, 50, bits=4, weights=True)


def test_rollouts(tmp_path):
    """GRPO's rollouts reach the cache with its settings."""
    from mamformer_b200.grpo import GRPOConfig, GRPOTrainer
    got = []

    class Policy(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.w = torch.nn.Parameter(torch.zeros(2))

        def generate(self, ids, **kw):
            got.append((kw["kv_cache"], kw["kv_budget"]))
            return torch.cat([ids, ids], 1)

    trainer = GRPOTrainer.__new__(GRPOTrainer)
    trainer.cfg, trainer.policy = GRPOConfig(group_size=2, gen_kv_cache="paged4", gen_kv_budget=32), Policy()
    assert len(trainer.rollouts(torch.zeros(1, 3, dtype=torch.long))) == 2
    assert got == [("paged4", 32)] * 2


@pytest.mark.parametrize("name,flags", [("generate", ["--kv_cache", "paged4", "--kv_budget", "64"]), ("train_grpo", ["--gen_kv_cache", "paged4", "--gen_kv_budget", "64"])])
def test_scripts_take_the_flags(name, flags):
    import importlib
    script = importlib.import_module(f"scripts.{name}")
    parser = script.build_parser()
    need = [x for a in parser._actions if a.required for x in (a.option_strings[0], "x")]
    args = parser.parse_args(need + flags)
    assert "paged4" in vars(args).values() and 64 in vars(args).values()

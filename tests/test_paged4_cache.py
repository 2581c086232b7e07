"""The 4-bit cache behind the models' and scripts' entry points: what an eviction leaves behind, what is refused and what is not."""

import pytest
import torch

from mamformer_b200.paged_cache import PagedKVCache
from test_paged4 import close, plain
from test_paged_cache import rand
from test_paged_generate import DEVICES


def attend(c, dtype, dev, seed, window=0):
    """A step of layer 0 with the tokens that extend() announced: its queries and results."""
    T = c.tokens
    cos, sin = torch.ones(T, 32, device=dev), torch.zeros(T, 32, device=dev)
    q, k, v = (rand((T, h, 64), dtype, dev, seed + j) for j, h in ((0, 4), (3, 2), (6, 2)))
    return q, c.layer(0).attend(q, k, v, cos, sin, window=window)


@pytest.mark.parametrize("dev,dtype", DEVICES)
def test_windows_after_the_evicted_sequences_were_released(dev, dtype):
    """Windows count slots, which are positions again once no sequence is left that was evicted from."""
    c = PagedKVCache(1, 2, 64, 3, 200, page_size=16, device=dev, bits=4, weights=True)
    c.extend([70, 5, 33])
    attend(c, dtype, dev, 1)
    c.evict(20, 4)                                       # sequences 0 and 2
    for b, refused in ((1, True), (0, True), (2, False)):
        c.release(b)
        assert c.evicted == refused
        new = [1 if n else 0 for n in c.lens]
        new[b] = 40
        c.extend(new)
        if refused:
            with pytest.raises(ValueError, match="window"):
                attend(c, dtype, dev, 1, window=9)
            attend(c, dtype, dev, 2)                     # the step itself
        else:
            q, got = attend(c, dtype, dev, 3, window=9)
            want, tol, _, _ = plain(q, c.layer(0).kv, c.block_table, new, c.lens, window=9)
            close(got, want, tol + (2.0 ** -18 if dtype == torch.float32 else 0.0))
    c.check()


@pytest.mark.parametrize("flags", [["--num_beams", "2"], ["--thinking", "FastThink"], []])
@pytest.mark.parametrize("kv", ["dense", "paged"])
def test_generate_script_refuses_a_budget_that_it_would_not_keep(flags, kv):
    from mamformer_b200.models.model import MamformerForCausalLM
    from mamformer_b200.tokenizer import MamformerTokenizer
    from scripts.generate import build_parser, generate_text
    from test_paged_generate import small_config
    parser = build_parser()
    need = [x for a in parser._actions if a.required for x in (a.option_strings[0], "x")]
    args = parser.parse_args(need + flags + ["--kv_cache", kv, "--kv_budget", "64", "--max_new_tokens", "1"])
    model = MamformerForCausalLM(small_config()).eval()
    with pytest.raises(ValueError, match="kv_budget" if kv == "dense" or not flags else "kv_"):
        generate_text(model, MamformerTokenizer(), "x", args)


def test_rollouts_of_a_policy_without_a_budget():
    """A policy of one's own whose generate() knows no budget goes on as before where none is set."""
    from mamformer_b200.grpo import GRPOConfig, GRPOTrainer

    class Policy(torch.nn.Module):
        def generate(self, ids, max_new_tokens, temperature, top_k, top_p, kv_cache):
            return torch.cat([ids, ids], 1)

    trainer = GRPOTrainer.__new__(GRPOTrainer)
    trainer.cfg, trainer.policy = GRPOConfig(group_size=2), Policy()
    assert len(trainer.rollouts(torch.zeros(1, 3, dtype=torch.long))) == 2


def test_decodes_as_the_dense_cache_does_on_the_values_that_it_holds(monkeypatch):
    """Greedy tokens and every step's logits, against the dense cache with keys and values rounded to the 4-bit levels.  In fp32 both differ in the
    order of sums of up to 60 terms alone: far less than 2^-10 of the logits' size."""
    from mamformer_b200 import ops
    from mamformer_b200.models.model import MamformerForCausalLM
    from mamformer_b200.ops import reference as ref
    from test_paged_generate import small_config
    torch.manual_seed(3)
    model = MamformerForCausalLM(small_config()).eval()
    ids = torch.randint(0, 259, (2, 50), generator=torch.Generator().manual_seed(2))
    seen, calls = [], []
    sample = model._sample_from_logits
    monkeypatch.setattr(model, "_sample_from_logits", lambda logits, *a: (seen.append(logits), sample(logits, *a))[1])
    out = model.generate(ids, max_new_tokens=8, temperature=0.0, kv_cache="paged4")
    paged = seen[:]
    del seen[:]
    levels = lambda x: ref.kv4_values(*ref.kv4_levels(x.float())).to(x.dtype)  # noqa: E731
    for name, at in (("diff_attention", 2), ("attention", 1)):
        plain_form = getattr(ops, name)
        monkeypatch.setattr(ops, name, lambda *a, f=plain_form, at=at, **kw: (calls.append(1), f(*a[:at], levels(a[at]), levels(a[at + 1]), *a[at + 2:], **kw))[1])
    dense = model.generate(ids, max_new_tokens=8, temperature=0.0)
    assert calls and len(seen) == len(paged) == 8
    assert torch.equal(out, dense)
    for a, b in zip(paged, seen):
        assert (a - b).abs().max() <= 2.0 ** -10 * b.abs().max()


@pytest.mark.parametrize("word", ["kv_append_error", "paged_attention_error", "kv4_error", "paged4_attention_error", None])
def test_every_word_of_the_paged_kernels_is_read(monkeypatch, word):
    """Of an extension with the 4-bit cache's words; one without them is checked for those that it has.  (The words are fakes.)"""
    from mamformer_b200 import fault
    from mamformer_b200.ops import _ext
    words = {n: 0 for n in ("kv_append_error", "paged_attention_error", "kv4_error", "paged4_attention_error")}
    if word:
        words[word] = 1 << 2

    class Fake:
        pass

    for n in words if word else ("kv_append_error", "paged_attention_error"):
        setattr(Fake, n, staticmethod(lambda clear=True, n=n: words.update({n: 0}) or 1 << 2 if words[n] and clear else words[n]))
    monkeypatch.setattr(_ext, "ext", lambda: Fake)
    monkeypatch.setattr(torch.cuda, "is_available", lambda: True)
    if word:
        for clear in (False, True):
            with pytest.raises(fault.PagedCacheError, match="length"):
                fault.check_paged_status(clear)
    fault.check_paged_status()

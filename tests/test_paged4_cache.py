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

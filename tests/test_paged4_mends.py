"""The 4-bit paged cache in calls at the edge of what its documentation allows: entries below a window that name other
sequences' pages, bad pages, groups as wide as f16, offsets out of order, tables and pools of unlike sizes, large budgets.
Tolerances are those of test_paged4."""

import math

import pytest
import torch

from mamformer_b200 import ops
from test_paged4 import CASES, check, close, filled, group_of, half_step, held, kept_slots, pair, plain, pool, some_mass
from test_paged_cache import DEVICES, i32, offsets, rand, rotation, tables


# ---- windows -------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("page,window", [(16, 40), (64, 70)])
@pytest.mark.parametrize("new,lens", [([1, 2], [300, 170]), ([90, 150], [300, 470]), ([90, 1, 100], [2500, 300, 700])])
def test_entries_below_a_window_may_name_live_pages(dev, page, window, new, lens):
    """Pages that were given back and are another sequence's now, or a later one of the same: their weights grow by what their
    owner's rows give them and nothing else, the same every time."""
    cache, table = filled(lens, page, 2, 128, dev)
    q = rand((sum(new), 4, 128), torch.bfloat16, dev, 3)
    gone = [max(0, L - n + 1 - window) // page for n, L in zip(new, lens)]
    live = [table[b, gone[b]:-(-L // page)].tolist() for b, L in enumerate(lens)]
    assert max(gone) > 0
    for shift in range(len(lens)):                                    # 0: the sequence's own later pages
        t = table.clone()
        for b, n in enumerate(gone):
            pages = live[(b + shift) % len(lens)]
            t[b, :n] = i32([pages[j % len(pages)] for j in range(n)], dev)
        check(q, cache, t, new, lens, window=window)
        mass = cache.mass.clone()
        for _ in range(3):
            check(q, cache, t, new, lens, window=window)
            assert torch.equal(mass, cache.mass)

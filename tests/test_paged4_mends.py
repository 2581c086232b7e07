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


# ---- eviction ------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("hd,page", [(64, 16), (128, 32)])
@pytest.mark.parametrize("gone", [-1, 1 << 30])
def test_evicted_tokens_of_a_bad_page_leave_their_new_slots_alone(in_place, hd, page, gone):
    """Nothing but what a slot held, or the token that it is to hold, is in it afterwards, whatever memory held before."""
    from mamformer_b200.fault import PagedCacheError, check_device_status
    lens, G, budget, recent = [150, 90], 2, 70, 20
    cache, table = filled(lens, page, G, hd, "cuda")
    cache.mass.copy_(some_mass(cache.mass.shape, 1, "cuda") + 1.0)
    bad = 140 // page                                                 # of the last tokens of sequence 0, which are kept whatever their weight
    t = table.clone()
    t[0, bad] = gone
    to, P = None, cache.blocks.shape[0]
    if not in_place:
        new, extra = tables([budget] * 2, page, "cuda", 9)
        cache = ops.PagedKV4(torch.cat([cache.blocks, pool(extra, G, page, hd, "cuda").blocks]), torch.cat([cache.mass, torch.full((extra, G, page), 8.0, device="cuda")]))
        to = new + P
    # what the cache holds of each token: its bytes and its weight
    slots = lambda c: torch.cat([x.flatten(4) for x in _pieces(c)], -1).flatten(2, 3)                    # noqa: E731  (P, G, page, bytes)
    check_device_status()
    junk = [torch.full((1 << 15,), 0x5A, dtype=torch.uint8, device="cuda") for _ in range(64)]     # what a workspace may find
    before = slots(cache).clone()
    del junk
    kept, left = ops.kv_evict(cache, t, i32(lens, "cuda"), budget, recent, out_table=to)
    with pytest.raises(PagedCacheError, match="page"):
        check_device_status()
    after, where = slots(cache), t if in_place else to
    assert left.tolist() == [70, 70]
    unmoved = 0
    for b in range(2):
        for g in range(G):
            for r, s in enumerate(kept[b, g].tolist()):
                at = int(where[b, r // page])
                if not 0 <= at < cache.blocks.shape[0]:
                    continue
                from_page = int(t[b, s // page])
                ok = 0 <= from_page < P
                unmoved += not ok
                want = before[from_page, g, s % page] if ok else before[at, g, r % page]
                assert torch.equal(after[at, g, r % page], want)
    assert unmoved > 0


def _pieces(cache):
    """The bytes of each token of a cache, (P, G, page / 16, 16, ..) each: codes and parameters of keys and values, weight."""
    hd = cache.blocks.shape[-1] // 18
    out = []
    for x in (cache.blocks[..., :9 * hd], cache.blocks[..., 9 * hd:]):
        out += [x[..., :8 * hd].unflatten(-1, (16, hd // 2)), x[..., 8 * hd:].unflatten(-1, (16, hd // 16))]
    return out + [cache.mass.view(torch.uint8).unflatten(-1, (-1, 16, 4))]


# ---- the levels of wide groups -------------------------------------------------------------------------
def wide(seed=1):
    """Rows (T, 1, 64) whose two groups have any two ends within f16: both signs, one sign, symmetric, the largest."""
    g = torch.Generator().manual_seed(seed)
    x = torch.rand(600, 1, 64, generator=g)
    top, low = 65504 * torch.rand(600, 1, 64, generator=g)[..., :1] ** 0.3, 65504 * torch.rand(600, 1, 1, generator=g) ** 0.3
    top[::5], low[1::5], top[2::5], low[2::5] = 65504.0, 65504.0, 65504.0, 65504.0
    top[3::5], low[3::5] = 40000.0, 40000.0
    x = (top + low) * x - low
    x[4::50] = x[4::50].abs()
    x[9::50] = -x[9::50].abs()
    x[..., :8], x[..., 8:16] = top, -low
    return x.clamp(-65504.0, 65504.0)


@pytest.mark.parametrize("dev", DEVICES)
def test_values_of_wide_groups(dev):
    """Within half a step of the group's levels where these fit into f16 as they are; within a step for every group."""
    x = wide().to(dev)
    T = len(x)
    table, P = tables([T], 32, dev)
    cache = pool(P, 1, 32, 64, dev)
    ops.kv_append(x, -x, cache, table, offsets([T], dev), i32([T], dev), T)
    back = ops.kv_read(cache, table, offsets([T], dev), i32([T], dev), T, torch.float32)
    for got, want in zip(back, (x.double(), -x.double())):
        off, half = (got.double() - want).abs(), half_step(want)
        assert got.abs().amax() <= 65504 and (off <= 2 * half).all()
        for j in range(2):
            of = (group_of(64) == j).to(dev)
            fits = want[..., of].abs().amax(-1) <= 60900
            assert fits.any() and not fits.all() and (off[..., of][fits] <= half[..., of][fits]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_both_devices_store_the_same_bytes_of_wide_groups(dtype):
    x = wide(2).to(dtype)
    T, got = len(x), []
    for dev in ("cpu", "cuda"):
        table, P = tables([T], 32, dev)
        cache = ops.PagedKV4(torch.zeros(P, 1, 2, 18 * 64, dtype=torch.uint8, device=dev))
        ops.kv_append(x.to(dev), -x.to(dev), cache, table, offsets([T], dev), i32([T], dev), T)
        got.append(cache.blocks.cpu())
    assert torch.equal(*got)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("new", [[3], [80]])
def test_attention_over_wide_groups(dev, new):
    """The products take what the cache holds, up to f16's largest."""
    x = wide(3)[:200].to(dev)
    table, P = tables([200], 16, dev)
    cache = pool(P, 1, 16, 64, dev)
    ops.kv_append(x.flip(0) * 2.0 ** -14, x, cache, table, offsets([200], dev), i32([200], dev), 200)
    check(rand((sum(new), 2, 64), torch.bfloat16, dev, 3), cache, table, new, [200])


# ---- offsets out of order ------------------------------------------------------------------------------
def cache_of(bits, lens, page, G, hd):
    if bits == 4:
        return filled(lens, page, G, hd, "cuda")
    import test_paged_cache as eight
    table, P = tables(lens, page, "cuda")
    cache = eight.pool(P, G, page, hd, "cuda")
    k, v = rand((sum(lens), G, hd), torch.float32, "cuda", 1), rand((sum(lens), G, hd), torch.float32, "cuda", 2)
    ops.kv_append(k, v, cache, table, offsets(lens, "cuda"), i32(lens, "cuda"), max(lens))
    return cache, table


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("hd,diff", [(64, False), (128, True)])
@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("off,T,max_new", [([0, 200, 100], 200, 100), ([0, 200, 100], 600, 200), ([100, 0, 200], 200, 100), ([0, 300, 200, 600], 600, 200),
                                           ([0, 90, 900], 180, 90), ([-5, 100, 200], 200, 100)])
def test_offsets_out_of_order_give_zeros(bits, hd, diff, wide, off, T, max_new):
    """With a table so wide that the chunk kernel's CTAs share keys, and without; weights stay as they were."""
    from mamformer_b200.fault import PagedCacheError, check_device_status
    lens = [300] * (len(off) - 1)
    cache, table = cache_of(bits, lens, 64, 2, hd)
    if wide:
        table = torch.cat([table, torch.full((len(lens), 96), -1, dtype=torch.int32, device="cuda")], 1)
    q = rand((T, 4, hd), torch.bfloat16, "cuda", 4)
    check_device_status()
    for _ in range(3):
        junk = [torch.full((n,), 7.0, device="cuda") for n in (T * 4 * hd // 2, 1 << 22, 1 << 24)]      # what outputs and workspaces may find
        del junk
        got = ops.paged_attention(q, cache, table, i32(off, "cuda"), i32(lens, "cuda"), max_new, **pair(q, diff))
        with pytest.raises(PagedCacheError, match="lengths"):
            check_device_status()
        assert (got == 0).all()
        if bits == 4:
            held_by = torch.zeros(cache.mass.shape[0], dtype=torch.bool, device="cuda")
            held_by[table[table >= 0].long()] = True
            assert ((cache.mass[held_by] == 0) | (cache.mass[held_by] == 3)).all()


# ---- tables wider than the pool ------------------------------------------------------------------------
def widened(table, slots, page):
    """The same sequences in a table with room for `slots` tokens each."""
    more = max(0, slots // page - table.shape[1])
    return torch.cat([table, torch.full((table.shape[0], more), -1, dtype=torch.int32, device=table.device)], 1)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("new,lens", CASES)
@pytest.mark.parametrize("hd,page,G,rep,diff,window,dtype", [(64, 16, 2, 1, True, 0, torch.float16), (128, 16, 1, 3, False, 29, torch.bfloat16),
                                                             (128, 64, 2, 4, False, 0, torch.bfloat16), (128, 128, 1, 8, True, 64, torch.bfloat16)])
def test_short_sequences_on_a_wide_table(dev, new, lens, hd, page, G, rep, diff, window, dtype):
    """What a cache made for long sequences asks of short ones."""
    cache, table = filled([max(n, 1) for n in lens], page, G, hd, dev)
    q = rand((sum(new), G * rep, hd), dtype, dev, 3)
    check(q, cache, widened(table, 20000, page), new, lens, **pair(q, diff), window=window)


@pytest.mark.gpu
def test_received_weights_take_no_more_memory_than_the_pool_has_slots():
    """64 sequences of a few tokens in a table for 2^17 each: by the table's width the scores alone would take 2 GB."""
    lens, G, hd, page = [5 + 3 * b for b in range(64)], 8, 64, 64
    cache, table = filled(lens, page, G, hd, "cuda")
    table = widened(table, 1 << 17, page)
    for new, H in (([1] * 64, 32), ([1] * 63 + [100], 32)):
        q = rand((sum(new), H, hd), torch.bfloat16, "cuda", 3)
        torch.cuda.synchronize()
        torch.cuda.empty_cache()
        torch.cuda.reset_peak_memory_stats()
        had = torch.cuda.memory_allocated()
        ops.paged_attention(q, cache, table, offsets(new, "cuda"), i32(lens, "cuda"), max(new))
        assert torch.cuda.max_memory_allocated() - had < 1 << 28
        check(q, cache, table, new, lens)


@pytest.mark.gpu
def test_lengths_beyond_the_pool_on_a_wide_table():
    """A length whose pages are not there: reported, the other sequences as without it, weights too."""
    from mamformer_b200.fault import PagedCacheError, check_device_status
    lens, G, hd, page = [300, 90, 200], 2, 64, 16
    cache, table = filled(lens, page, G, hd, "cuda")
    table = widened(table, 1 << 15, page)
    q = rand((3, 4, hd), torch.bfloat16, "cuda", 3)
    check_device_status()
    for b in range(3):
        results = []
        for long_one in (lens[b], 20000):
            cache.mass.fill_(1.0)
            got = ops.paged_attention(q, cache, table, offsets([1] * 3, "cuda"), i32([long_one if i == b else n for i, n in enumerate(lens)], "cuda"), 1)
            results.append((got, cache.mass.clone()))
            if long_one == 20000:
                with pytest.raises(PagedCacheError):
                    check_device_status()
        (a, am), (c, cm) = results
        others = [i for i in range(3) if i != b]
        # its own row and weights are those of whatever is behind its end in its last page
        assert torch.equal(a[others], c[others])
        for i in others:
            pages = table[i, :-(-lens[i] // page)].long()
            # what does not fit is left out of the weights, never added to others'
            assert torch.equal(am[pages], cm[pages]) or (cm[pages] == 1.0).all()


# ---- append --------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("new,max_new", [([1, 5, 2], 4), ([1, 2, 1], 1), ([40, 3, 90], 64)])
def test_runs_of_more_tokens_than_were_said_are_reported(bits, new, max_new):
    """They are not appended, the other sequences' are, by either cache."""
    from mamformer_b200.fault import PagedCacheError, check_device_status
    lens, G, hd, page = [50, 70, 130], 2, 64, 16
    cache, table = cache_of(bits, lens, page, G, hd)
    tensors = [x for x in cache if x is not None]
    k, v = rand((sum(new), G, hd), torch.bfloat16, "cuda", 7), rand((sum(new), G, hd), torch.bfloat16, "cuda", 8)
    cu, ln = offsets(new, "cuda"), i32(lens, "cuda")
    start = [x.clone() for x in tensors]
    check_device_status()
    ops.kv_append(k, v, cache, table, cu, ln, max_new)
    with pytest.raises(PagedCacheError, match="length"):
        check_device_status()
    got = [x.clone() for x in tensors]
    for x, was in zip(tensors, start):
        x.copy_(was)
    at = 0
    for b, n in enumerate(new):                                       # one by one, as they were to go in
        if n <= max_new:
            ops.kv_append(k[at:at + n], v[at:at + n], cache, table[b:b + 1], offsets([n], "cuda"), ln[b:b + 1], max_new)
        at += n
    check_device_status()
    assert any(n > max_new for n in new)
    for x, y in zip(got, tensors):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))


@pytest.mark.parametrize("dev", DEVICES)
def test_weights_that_are_no_numbers_come_first_whatever_their_sign(dev):
    """An x86 host makes negative NaN of infinity less infinity, a GPU positive: the choice is the same."""
    cache, table = filled([8], 16, 1, 64, dev)
    bits = [0x7FC00000, 0xFFC00000, 0xFF800001, 0x7FFFFFFF, 0x7F800000, 0x3F800000, 0x40000000, 0xFFFFFFFF]
    cache.mass[table[0, 0].long(), 0, :8] = torch.tensor([b - (1 << 32) if b >> 31 else b for b in bits], dtype=torch.int32, device=dev).view(torch.float32)
    for budget, want in ((1, [0]), (2, [0, 1]), (4, [0, 1, 2, 3]), (5, [0, 1, 2, 3, 7]), (6, [0, 1, 2, 3, 4, 7]), (7, [0, 1, 2, 3, 4, 6, 7])):
        c = ops.PagedKV4(cache.blocks.clone(), cache.mass.clone())
        kept, _ = ops.kv_evict(c, table, i32([8], dev), budget, 0)
        assert kept[0, 0].tolist() == want


@pytest.mark.gpu
def test_a_budget_beyond_the_table_takes_no_memory_for_it():
    """Nothing is cut: the workspace is of what the table has room for, and only the kept slots are as many as was asked for."""
    lens, G, hd, page, budget = [300, 90], 2, 128, 16, 1 << 22
    cache, table = filled(lens, page, G, hd, "cuda")
    before = cache.blocks.clone()
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    torch.cuda.reset_peak_memory_stats()
    had = torch.cuda.memory_allocated()
    kept, left = ops.kv_evict(cache, table, i32(lens, "cuda"), budget, 5)
    torch.cuda.synchronize()
    assert torch.cuda.max_memory_allocated() - had < 2 * G * budget * 4 + (1 << 24)
    assert left.tolist() == lens and torch.equal(cache.blocks, before)
    for b, n in enumerate(lens):
        assert torch.equal(kept[b, 0, :n], torch.arange(n, device="cuda", dtype=torch.int32)) and (kept[b, :, n:] == -1).all()


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [4, 8])
def test_tables_of_more_slots_than_32_bits_count_are_refused(bits):
    cache, _ = cache_of(bits, [20], 128, 1, 64)
    table = torch.zeros(1, (1 << 31) // 128 - 8000, dtype=torch.int32, device="cuda")
    q = rand((1, 1, 64), torch.bfloat16, "cuda", 1)
    with pytest.raises(RuntimeError, match="sizes"):
        ops.paged_attention(q, cache, table, offsets([1], "cuda"), i32([20], "cuda"), 1)
    with pytest.raises(RuntimeError, match="sizes"):
        ops.kv_append(q, q, cache, table, offsets([1], "cuda"), i32([20], "cuda"), 1)

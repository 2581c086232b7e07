"""ops.kv_append and ops.paged_attention where they can go wrong: rows and tiles that see nothing, factors of any sign,
pages whose values differ by many orders of magnitude, pages given back below a window, what the device reports and when.

Tolerances of an attention row, from the values that this row sees: each weight is rounded once to 11 bits (2^-11 of its
share) and fp32 sums add less than 2^-14 of the shares; a weight whose share is far below the largest one's is held to
2^-24 of that instead, for each key and up to 448 times the scale of its block, which is at most twice the block's
largest value."""

import math

import pytest
import torch

from mamformer_b200 import ops
from test_paged_cache import DEVICES, ROUND, held, i32, offsets, pool, rand, tables


def plain(q, cache, table, new, lens, q2=None, lam=None, window=0, scale=None):
    """The definition in 64 bits, and each row's tolerance.  Only what some row of a sequence sees is read."""
    H, hd = q.shape[1:]
    G, page = cache.k.shape[1:3]
    scale = hd ** -0.5 if scale is None else scale
    out, tol, at = torch.zeros_like(q, dtype=torch.float64), torch.zeros_like(q, dtype=torch.float64), 0
    for b, (n, L) in enumerate(zip(new, lens)):
        if n and L:
            k, v = (x.repeat_interleave(H // G, 0) for x in held(cache, table, lens, b))
            pages = table[b, :-(-L // page)].long()
            top = (cache.v_scale[pages].double() * 448).T.repeat_interleave(page, 1)[:, :L].repeat_interleave(H // G, 0)
            i, j = torch.arange(L - n, L, device=q.device)[:, None], torch.arange(L, device=q.device)
            see = (j <= i) & (j > i - window) if window else j <= i
            used = see.any(0)
            k, v = k.masked_fill(~used[:, None], 0.0), v.masked_fill(~used[:, None], 0.0)
            maps, tols = [], []
            for x in (q,) if q2 is None else (q, q2):
                s = x[at:at + n].double().transpose(0, 1) @ k.transpose(1, 2) * scale
                p = torch.softmax(s.masked_fill(~see, -math.inf), -1).nan_to_num(0.0)
                maps.append(p @ v)
                tols.append((2.0 ** -11 + 2.0 ** -14) * (p @ v.abs()) + L * 2.0 ** -24 * (p * top[:, None]).amax(-1, keepdim=True))
            o, t = maps[0], tols[0]
            if q2 is not None:
                w = lam.double()[:, None, None]
                o, t = (maps[0] - w * maps[1]) / (1 - w + 1e-8), (tols[0] + w * tols[1]) / (1 - w)
            out[at:at + n], tol[at:at + n] = o.transpose(0, 1), t.transpose(0, 1)
        at += n
    return out, tol


def close(got, want, tol):
    tol = tol + ROUND[got.dtype] * want.abs()
    bad = ~((got.double() - want).abs() <= tol)
    assert not bad.any(), ((got.double() - want).abs() / tol)[bad].max()


def pair(q, diff):
    """The second map's arguments."""
    return {"q2": q.flip(0), "lam": torch.linspace(0.1, 0.8, q.shape[1], device=q.device)} if diff else {}


def filled(lens, page, G, hd, dev, gain=None, seed=0):
    """A cache of unit normals, values of slot j times gain[j // page]."""
    table, P = tables(lens, page, dev, seed)
    cache = pool(P, G, page, hd, dev)
    T = sum(lens)
    k, v = rand((T, G, hd), torch.float32, dev, seed + 1), rand((T, G, hd), torch.float32, dev, seed + 2)
    if gain is not None:
        slot = torch.cat([torch.arange(n) for n in lens]) // page
        v = v * torch.tensor(gain, device=dev)[slot.to(dev) % len(gain), None, None]
    ops.kv_append(k, v, cache, table, offsets(lens, dev), i32(lens, dev), max(lens))
    return cache, table


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("diff", [False, True])
@pytest.mark.parametrize("new,lens", [([300], [10]), ([280, 90], [0, 90]), ([520, 300], [1, 3])])
def test_tiles_that_see_nothing_give_zero(dev, hd, diff, new, lens):
    """Lengths so short that whole tiles of rows have no key at all."""
    cache, table = filled([max(n, 1) for n in lens], 16, 1, hd, dev)
    q = rand((sum(new), 2, hd), torch.bfloat16, dev, 1)
    kw = pair(q, diff)
    want, tol = plain(q, cache, table, new, lens, **kw)
    for _ in range(1 if dev == "cpu" else 20):
        got = ops.paged_attention(q, cache, table, offsets(new, dev), i32(lens, dev), max(new), **kw)
        at = 0
        for n, L in zip(new, lens):
            assert (got[at:at + n - L] == 0).all()
            at += n
        close(got, want, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("diff", [False, True])
@pytest.mark.parametrize("new,lens", [([1, 2], [5000, 70]), ([200], [900]), ([90, 1], [2000, 300])])
def test_waits_that_run_out_are_reported_and_wound_down(diff, new, lens):
    """Waits that give up at once: copies and products are then still under way when the kernel winds down."""
    from mamformer_b200.fault import KernelTimeoutError, check_device_status
    from mamformer_b200.ops._ext import require_native
    C = require_native()
    cache, table = filled(lens, 64, 2, 128, "cuda")
    q = rand((sum(new), 4, 128), torch.bfloat16, "cuda", 3)
    kw = pair(q, diff)
    run = lambda: ops.paged_attention(q, cache, table, offsets(new, "cuda"), i32(lens, "cuda"), max(new), **kw)  # noqa: E731
    check_device_status()
    had = C.paged_attention_wait_limit(-1)
    try:
        run()
        torch.cuda.synchronize()
    finally:
        C.paged_attention_wait_limit(had)
    with pytest.raises(KernelTimeoutError):
        check_device_status()
    close(run(), *plain(q, cache, table, new, lens, **kw))
    check_device_status()


@pytest.mark.gpu
@pytest.mark.parametrize("new,lens", [([1, 2], [60000, 70]), ([200], [9000])])
def test_a_wait_that_ran_out_is_over_with_its_call(new, lens):
    """Nobody has read the error yet: the calls after it wait as they would have."""
    from mamformer_b200.fault import KernelTimeoutError, check_device_status
    from mamformer_b200.ops._ext import require_native
    C = require_native()
    cache, table = filled(lens, 64, 2, 128, "cuda")
    q = rand((sum(new), 4, 128), torch.bfloat16, "cuda", 3)
    run = lambda: ops.paged_attention(q, cache, table, offsets(new, "cuda"), i32(lens, "cuda"), max(new))  # noqa: E731
    check_device_status()
    want = run()
    had = C.paged_attention_wait_limit(-1)
    try:
        run()
        torch.cuda.synchronize()
    finally:
        C.paged_attention_wait_limit(had)
    for _ in range(50):
        assert torch.equal(run(), want)
    with pytest.raises(KernelTimeoutError):
        check_device_status()
    assert torch.equal(run(), want)
    check_device_status()


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("first", [1, 40, 1000])
@pytest.mark.parametrize("new,lens", [([1, 1], [40, 20]), ([60, 3], [90, 3]), ([1, 90], [17, 400])])
def test_offsets_that_do_not_start_at_zero(dev, first, new, lens):
    """Rows before the first sequence belong to nobody: they are not appended, and their queries give 0."""
    table, P = tables(lens, 16, dev)
    G, hd, H, T = 2, 64, 4, sum(new)
    k, v = rand((T, G, hd), torch.bfloat16, dev, 1), rand((T, G, hd), torch.bfloat16, dev, 2)
    front = rand((first, G, hd), torch.bfloat16, dev, 5) * 100.0
    q = rand((first + T, H, hd), torch.bfloat16, dev, 3)
    caches = pool(P, G, 16, hd, dev), pool(P, G, 16, hd, dev)
    for c in caches:
        kx, vx = rand((sum(lens), G, hd), torch.bfloat16, dev, 6), rand((sum(lens), G, hd), torch.bfloat16, dev, 7)
        ops.kv_append(kx, vx, c, table, offsets(lens, dev), i32(lens, dev), max(lens))
    cu = offsets(new, dev)
    ops.kv_append(k, v, caches[0], table, cu, i32(lens, dev), max(new))
    ops.kv_append(torch.cat([front, k]), torch.cat([front, v]), caches[1], table, cu + first, i32(lens, dev), max(new))
    for a, b in zip(*caches):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    for diff in (False, True):
        kw, kw0 = pair(q, diff), pair(q[first:], diff)
        if diff:
            kw0["q2"] = kw["q2"][first:]
        got = ops.paged_attention(q, caches[0], table, cu + first, i32(lens, dev), max(new), **kw)
        assert (got[:first] == 0).all()
        close(got[first:], *plain(q[first:], caches[0], table, new, lens, **kw0))


def dirty(shape, dtype, dev):
    """Memory that the next allocation of its size gets, full of NaN."""
    torch.full(shape, math.nan, dtype=dtype, device=dev)


@pytest.mark.gpu
@pytest.mark.parametrize("diff", [False, True])
def test_rows_that_are_not_computed_are_zeros(diff):
    from mamformer_b200.fault import KernelTimeoutError, PagedCacheError, check_device_status
    from mamformer_b200.ops._ext import require_native
    C = require_native()
    check_device_status()

    def run(q, cu, lens, max_new):
        dirty(q.shape, q.dtype, "cuda")
        return ops.paged_attention(q, cache, table, cu, lens, max_new, **pair(q, diff))

    # sequence 1 has more tokens than max_new says
    new, lens = [1, 30, 2], [40, 90, 70]
    cache, table = filled(lens, 16, 2, 128, "cuda")
    q = rand((sum(new), 4, 128), torch.bfloat16, "cuda", 3)
    cu, ln = offsets(new, "cuda"), i32(lens, "cuda")
    want, tol = plain(q, cache, table, new, lens, **pair(q, diff))
    got = run(q, cu, ln, 2)
    assert (got[1:31] == 0).all()
    for rows in (slice(0, 1), slice(31, 33)):
        close(got[rows], want[rows], tol[rows])
    with pytest.raises(PagedCacheError, match="lengths"):
        check_device_status()
    # offsets that fall, or run past the queries
    q = rand((600, 4, 128), torch.bfloat16, "cuda", 4)
    for bad in ([0, 5, 3, 8], [0, 2, 4, 900], [0, 200, 100, 600], [-5, 0, 5, 9], [0, 1, 2, -1]):
        for max_new in (2, 40, 200):
            got = run(q, i32(bad, "cuda"), ln, max_new)
            assert got.isfinite().all() and (max_new == 200 or (got == 0).all())
            with pytest.raises(PagedCacheError, match="lengths"):
                check_device_status()
    # a length that the table has no room for
    ln, new, lens = i32([40, (1 << 31) - 1, 70], "cuda"), [1, 1, 2], [40, 90, 70]
    want, tol = plain(q[:4], cache, table, new, lens, **pair(q[:4], diff))
    got = run(q[:4], offsets(new, "cuda"), ln, 2)
    for rows in (slice(0, 1), slice(2, 4)):                 # the other sequences'
        close(got[rows], want[rows], tol[rows])
    with pytest.raises(PagedCacheError):
        check_device_status()
    # waits that run out
    for new, lens in (([1, 2], [60000, 70]), ([200], [9000]), ([90, 1], [2000, 300]), ([2000], [2000])):
        cache, table = filled(lens, 64, 2, 128, "cuda")
        q = rand((sum(new), 4, 128), torch.bfloat16, "cuda", 3)
        had = C.paged_attention_wait_limit(-1)
        try:
            got = run(q, offsets(new, "cuda"), i32(lens, "cuda"), max(new))
            torch.cuda.synchronize()
        finally:
            C.paged_attention_wait_limit(had)
        assert (got == 0).all()
        with pytest.raises(KernelTimeoutError):
            check_device_status()


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("scale", [0.0, -0.1, -1e-30, 0.3])
@pytest.mark.parametrize("diff", [False, True])
@pytest.mark.parametrize("new,lens", [([1, 3], [70, 33]), ([130, 70], [130, 400])])
def test_score_factors_of_any_sign(dev, scale, diff, new, lens):
    cache, table = filled(lens, 32, 2, 128, dev)
    q = rand((sum(new), 4, 128), torch.bfloat16, dev, 1)
    kw = dict(pair(q, diff), scale=scale)
    close(ops.paged_attention(q, cache, table, offsets(new, dev), i32(lens, dev), max(new), **kw), *plain(q, cache, table, new, lens, **kw))
    windowed = dict(kw, window=20)
    close(ops.paged_attention(q, cache, table, offsets(new, dev), i32(lens, dev), max(new), **windowed),
          *plain(q, cache, table, new, lens, **windowed))


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("size", [2.0 ** -60, 2.0 ** -120, 2.0 ** 40])
@pytest.mark.parametrize("new,lens", [([1, 3], [70, 33]), ([130, 70], [130, 400])])
def test_zero_keys_and_queries_of_any_size(dev, size, new, lens):
    """Keys of zeros have the smallest block scale there is: the scores' factor underflows with small queries."""
    table, P = tables(lens, 16, dev)
    cache = pool(P, 1, 16, 64, dev)
    v = rand((sum(lens), 1, 64), torch.float32, dev, 2)
    ops.kv_append(torch.zeros_like(v), v, cache, table, offsets(lens, dev), i32(lens, dev), max(lens))
    q = (rand((sum(new), 2, 64), torch.float32, dev, 1) * size).bfloat16()
    close(ops.paged_attention(q, cache, table, offsets(new, dev), i32(lens, dev), max(new)), *plain(q, cache, table, new, lens))


SPREADS = [[1.0, 2.0 ** -8], [1.0, 2.0 ** -14], [2.0 ** -26, 1.0], [1.0, 2.0 ** 20], [1e-5, 500.0], [1.0, 2.0 ** 40, 2.0 ** -40, 1.0],
           [0.0, 1.0], [1e-20, 0.0, 1e20, 3.0, 2.0 ** 55]]


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("gain", SPREADS)
@pytest.mark.parametrize("hd,page", [(64, 16), (128, 32), (128, 64)])
@pytest.mark.parametrize("diff", [False, True])
@pytest.mark.parametrize("new,lens", [([1, 1, 1], [40, 100, 150]), ([5, 3], [60, 33]), ([150, 90], [150, 200])])
def test_pages_of_values_of_any_size(dev, gain, hd, page, diff, new, lens):
    """Neighbouring pages' values differ by up to 2^120; a row is held to the values that it sees."""
    cache, table = filled(lens, page, 1, hd, dev, gain)
    q = rand((sum(new), 4, hd), torch.bfloat16, dev, 3)
    kw = pair(q, diff)
    got = ops.paged_attention(q, cache, table, offsets(new, dev), i32(lens, dev), max(new), **kw)
    close(got, *plain(q, cache, table, new, lens, **kw))


@pytest.mark.gpu
@pytest.mark.parametrize("gain", SPREADS)
@pytest.mark.parametrize("new,lens", [([1], [9000]), ([70], [4000])])
def test_parts_of_values_of_any_size(gain, new, lens):
    """The same where several CTAs share a row's keys."""
    cache, table = filled(lens, 16, 2, 64, "cuda", gain)
    q = rand((sum(new), 4, 64), torch.bfloat16, "cuda", 3)
    close(ops.paged_attention(q, cache, table, offsets(new, "cuda"), i32(lens, "cuda"), max(new)), *plain(q, cache, table, new, lens))


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("new,window", [([3], 120), ([16], 130), ([60], 130)])
@pytest.mark.parametrize("hd", [64, 128])
def test_a_window_hides_huge_values(dev, new, window, hd):
    """The first rows of a tile see the end of a page of huge values, the others do not."""
    lens = [new[0] + 134]
    cache, table = filled(lens, 16, 1, hd, dev, [2.0 ** 90] + [1.0, 2.0 ** -10] * 6)
    q = rand((sum(new), 2, hd), torch.bfloat16, dev, 3)
    got = ops.paged_attention(q, cache, table, offsets(new, dev), i32(lens, dev), max(new), window=window)
    close(got, *plain(q, cache, table, new, lens, window=window))


@pytest.mark.parametrize("dev", DEVICES)
def test_keys_without_weight_have_huge_values(dev):
    """Scores push the pages of huge values below fp32's smallest weight; what is left are the other pages' values."""
    lens, hd = [150], 64
    table, P = tables(lens, 16, dev)
    cache = pool(P, 1, 16, hd, dev)
    k, v = rand((150, 1, hd), torch.float32, dev, 1), rand((150, 1, hd), torch.float32, dev, 2)
    k[:64], v[:64] = -20.0, v[:64] * 2.0 ** 100
    ops.kv_append(k, v, cache, table, offsets(lens, dev), i32(lens, dev), 150)
    q = torch.full((1, 2, hd), 1.0, dtype=torch.bfloat16, device=dev)
    close(ops.paged_attention(q, cache, table, offsets([1], dev), i32(lens, dev), 1), *plain(q, cache, table, [1], lens))


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("page,window", [(16, 40), (32, 33), (64, 70)])
@pytest.mark.parametrize("diff", [False, True])
@pytest.mark.parametrize("new,lens", [([1, 2], [300, 170]), ([90, 150], [300, 170]), ([90], [2500])])
def test_pages_below_a_window_may_be_given_back(dev, page, window, diff, new, lens):
    """Pages that no query sees: another sequence's now, here full of NaN, or no page at all."""
    from mamformer_b200.fault import check_device_status
    cache, table = filled(lens, page, 2, 128, dev)
    P = cache.k.shape[0]
    unused = min(set(range(P)) - set(table.flatten().tolist()))
    q = rand((sum(new), 4, 128), torch.bfloat16, dev, 3)
    kw = dict(pair(q, diff), window=window)
    want, tol = plain(q, cache, table, new, lens, **kw)
    check_device_status()
    for gone in (unused, -1, P + 5):
        t = table.clone()
        for b, (n, L) in enumerate(zip(new, lens)):
            t[b, :max(0, L - n + 1 - window) // page] = gone
        close(ops.paged_attention(q, cache, t, offsets(new, dev), i32(lens, dev), max(new), **kw), want, tol)
        check_device_status()


@pytest.mark.gpu
def test_one_check_reads_every_word():
    """The append and both attention kernels have recorded something; with clear=False it stays."""
    from mamformer_b200.fault import KernelTimeoutError, PagedCacheError, check_device_status
    from mamformer_b200.ops._ext import require_native
    C = require_native()
    check_device_status()
    cache, table = filled([40, 300], 16, 1, 64, "cuda")
    q = rand((101, 2, 64), torch.bfloat16, "cuda", 1)
    kv = rand((2, 1, 64), torch.bfloat16, "cuda", 2)
    bad = table.clone()
    bad[:, 2] = -1
    two, both = offsets([1, 1], "cuda"), i32([40, 300], "cuda")

    had = C.paged_attention_wait_limit(0)
    C.paged_attention_wait_limit(had)
    for timeout, error in ((False, PagedCacheError), (True, KernelTimeoutError)):
        ops.kv_append(kv, kv, cache, bad, two, i32([40, 40], "cuda"), 1)
        ops.paged_attention(q[:2], cache, bad, two, both, 1)
        if timeout:
            C.paged_attention_wait_limit(-1)
        try:
            ops.paged_attention(q, cache, table, offsets([1, 100], "cuda"), both, 100)
            torch.cuda.synchronize()
        finally:
            C.paged_attention_wait_limit(had)
        for _ in range(2):
            with pytest.raises(error, match="page of the pool"):
                check_device_status(clear=False)
        with pytest.raises(error, match="page of the pool"):
            check_device_status()
        check_device_status()


@pytest.mark.parametrize("comm,gemm", [(101, 0), (0, 7)])
def test_an_earlier_error_leaves_the_paged_words(monkeypatch, comm, gemm):
    """Another kernel's error is raised first; the paged ones are there for the next check.  (The words are fakes.)"""
    from mamformer_b200 import fault
    from mamformer_b200.ops import _ext
    words = {"comm": comm, "gemm": gemm, "append": 1 << 1, "attention": 1 << 4}

    class Fake:
        comm_error = staticmethod(lambda: words["comm"])
        gemm_error = staticmethod(lambda: words["gemm"])
        comm_clear_error = staticmethod(lambda: words.update(comm=0))
        gemm_clear_error = staticmethod(lambda: words.update(gemm=0))

    def read(name):
        def f(clear=True):
            v = words[name]
            if clear:
                words[name] = 0
            return v
        return staticmethod(f)

    Fake.kv_append_error, Fake.paged_attention_error = read("append"), read("attention")
    monkeypatch.setattr(_ext, "ext", lambda: Fake)
    monkeypatch.setattr(torch.cuda, "is_available", lambda: True)
    with pytest.raises(fault.CommTimeoutError if comm else fault.KernelTimeoutError, match="peer 1" if comm else "GEMM"):
        fault.check_device_status()
    for clear in (False, True):
        with pytest.raises(fault.KernelTimeoutError, match="timed out; a block table entry"):
            fault.check_device_status(clear)
    fault.check_device_status()


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("size", [60.0, 1e-4, 2.0 ** -20, 3e4])
@pytest.mark.parametrize("diff", [False, True])
def test_large_and_tiny_scores_of_many_rows(dev, size, diff):
    """Scores of several hundred and more, and of next to nothing, in chunks of a prompt."""
    new, lens = [130, 70], [130, 400]
    cache, table = filled(lens, 32, 2, 128, dev, seed=7)
    q = (rand((sum(new), 4, 128), torch.float32, dev, 3) * size).bfloat16()
    kw = pair(q, diff)
    got = ops.paged_attention(q, cache, table, offsets(new, dev), i32(lens, dev), max(new), **kw)
    assert got.isfinite().all()
    # a score of size s carries 2^-24 s of rounding in each of its 128 products, and the weights carry that much; values
    # are below 5, times (1 + lam) / (1 - lam)
    slack = 2.0 ** -24 * 128 * size * 12
    if slack < 0.1:
        want, tol = plain(q, cache, table, new, lens, **kw)
        close(got, want, tol + slack * 5.0 * (9.0 if diff else 1.0))


@pytest.mark.gpu
def test_score_factors_that_are_not_numbers_are_refused():
    cache, table = filled([9], 16, 1, 64, "cuda")
    q = rand((1, 2, 64), torch.bfloat16, "cuda", 1)
    for scale in (math.nan, math.inf, -math.inf, 1e39):
        with pytest.raises(RuntimeError, match="scale"):
            ops.paged_attention(q, cache, table, offsets([1], "cuda"), i32([9], "cuda"), 1, scale=scale)

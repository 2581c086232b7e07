"""ops.kv_append and ops.paged_attention (csrc/paged_kv.cu, csrc/paged_attn*.cu on CUDA, the eager forms on CPU) against
plain 64-bit forms: every head size, page size and type, ragged batches from no token to several pages, windows, the
differential form, what earlier owners left in the pages, strides, streams, and the refusals.

Tolerances, from the arithmetic.  A stored value is within half a step of e4m3 (2^-4 of itself, 2^-10 of the scale below
the normal range) of the rotated one, and once more that where its block's scale grew later.  Attention over given codes
rounds each weight once to 11 bits and the result to its type; fp32 sums add less than 2^-14 of the largest value, so a
map is within 2^-11 + 2^-14 of max |v| plus the type's rounding, and the differential form within (1 + lam) / (1 - lam)
of a map's."""

import math

import pytest
import torch

from mamformer_b200 import ops

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
ROUND = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}      # half a step, relative


def pool(P, G, page, hd, dev):
    """A pool whose memory earlier owners left full of NaN codes and strange scales."""
    nan = torch.full((P, G, page, hd), 0x7F, dtype=torch.uint8)
    return ops.PagedKV(*(nan.clone().to(dev).view(torch.float8_e4m3fn) for _ in range(2)),
                       *(torch.full((P, G), 2.0 ** 60, device=dev) for _ in range(2)))


def tables(lens, page, dev, seed=0, spare=2):
    """A block table with scrambled pages; entries past a sequence's last page are -1."""
    need = [-(-n // page) for n in lens]
    order = torch.randperm(sum(need) + spare, generator=torch.Generator().manual_seed(seed)).tolist()
    t = torch.full((len(lens), max(need + [1])), -1, dtype=torch.int32)
    for b, n in enumerate(need):
        t[b, :n] = torch.tensor([order.pop() for _ in range(n)], dtype=torch.int32)
    return t.to(dev), sum(need) + spare


def i32(xs, dev):
    return torch.tensor(list(xs), dtype=torch.int32, device=dev)


def offsets(new, dev):
    return i32([0] + torch.tensor(new).cumsum(0).tolist(), dev)


def held(cache, table, lens, b):
    """k, v (G, len, hd) of a sequence in 64 bits."""
    page = cache.k.shape[2]
    pages = table[b, :-(-lens[b] // page)].long()
    out = []
    for x, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        x = x.view(torch.uint8)[pages].view(torch.float8_e4m3fn).double() * s[pages].double()[..., None, None]
        out.append(x.transpose(0, 1).reshape(x.shape[1], -1, x.shape[3])[:, :lens[b]])
    return out


def rotation(n, hd, dev):
    ang = torch.outer(torch.arange(n, dtype=torch.float32), 1.0 / 10000.0 ** (torch.arange(0, hd, 2).float() / hd))
    return ang.cos().to(dev), ang.sin().to(dev)


def turned(x, cos, sin, pos):
    c, s = cos.double()[pos][:, None], sin.double()[pos][:, None]
    a, b = x.double().chunk(2, -1)
    return torch.cat([a * c - b * s, b * c + a * s], -1)


def rand(shape, dtype, dev, seed):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(dev)


def step_of(x, scale):
    """Half a step of e4m3 around x."""
    return torch.maximum(x.abs() * 2.0 ** -4, scale * 2.0 ** -10) * (1 + 1e-5)


# ---- append ------------------------------------------------------------------------------------------
STEPS = [[[1]], [[5, 0, 130], [1, 1, 1], [3, 40, 0], [0, 0, 0]], [[16, 15, 17, 1], [16, 16, 16, 16], [1, 2, 300, 1]]]


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("hd,page,G", [(64, 16, 2), (64, 128, 1), (128, 32, 2), (128, 64, 3), (128, 128, 1)])
@pytest.mark.parametrize("steps", STEPS)
def test_append_stores_the_rotated_values(dev, dtype, hd, page, G, steps):
    B, H = len(steps[0]), 2 * G
    total = [sum(s[b] for s in steps) for b in range(B)]
    table, P = tables(total, page, dev)
    cache = pool(P, G, page, hd, dev)
    cos, sin = rotation(max(total) + 1, hd, dev)
    lens = [0] * B
    want = [[[], []] for _ in range(B)]
    for i, new in enumerate(steps):
        lens = [a + n for a, n in zip(lens, new)]
        T = sum(new)
        k, v, q1, q2 = (rand((T, h, hd), dtype, dev, 10 * i + j) for j, h in enumerate((G, G, H, H)))
        k, v = k * 3.0 ** i, v * 0.3 ** i                       # later keys raise their block's scale
        pos = torch.tensor([p for n, L in zip(new, lens) for p in range(L - n, L)], dtype=torch.long, device=dev)
        r1, r2 = ops.kv_append(k, v, cache, table, offsets(new, dev), i32(lens, dev), max(new), cos, sin, pos, [q1, q2])
        for r, q in ((r1, q1), (r2, q2)):
            w = turned(q, cos, sin, pos)
            assert r.dtype == dtype and ((r.double() - w).abs() <= (ROUND[dtype] + 2.0 ** -22) * w.abs() + 2.0 ** -22).all()
        kt, at = turned(k, cos, sin, pos), 0
        for b, n in enumerate(new):
            want[b][0].append(kt[at:at + n]), want[b][1].append(v[at:at + n].double())
            at += n
    for b in range(B):
        if not total[b]:
            continue
        pages = table[b, :-(-total[b] // page)].long()
        for got, parts, s in zip(held(cache, table, total, b), want[b], (cache.k_scale, cache.v_scale)):
            x = torch.cat(parts).transpose(0, 1)
            scale = s[pages].double().T.repeat_interleave(page, 1)[:, :total[b], None]
            assert (torch.frexp(scale)[0] == 0.5).all()
            once = step_of(x, scale)
            assert ((got - x).abs() <= 2 * once * (1 + 2.0 ** -4)).all()
            for j in range(len(pages)):                          # no larger scale than the block's values ask for
                block = x[:, j * page:(j + 1) * page].abs().amax((1, 2))
                assert (s[pages[j]].double() * 224 <= block * (1 + 1e-5)).all()
                assert (s[pages[j]].double() * 448 >= block * (1 - 1e-5)).all()


@pytest.mark.parametrize("dev", DEVICES)
def test_append_rounds_once_where_the_scale_stays(dev):
    new, page, G, hd = [70, 33], 32, 2, 128
    table, P = tables(new, page, dev)
    cache = pool(P, G, page, hd, dev)
    k, v = rand((103, G, hd), torch.float32, dev, 1), rand((103, G, hd), torch.float32, dev, 2)
    assert ops.kv_append(k, v, cache, table, offsets(new, dev), i32(new, dev), 70) == []
    for b, (lo, hi) in enumerate(((0, 70), (70, 103))):
        pages = table[b, :-(-new[b] // page)].long()
        for got, x, s in zip(held(cache, table, new, b), (k, v), (cache.k_scale, cache.v_scale)):
            x = x[lo:hi].double().transpose(0, 1)
            scale = s[pages].double().T.repeat_interleave(page, 1)[:, :new[b], None]
            assert ((got - x).abs() <= step_of(x, scale)).all()


@pytest.mark.parametrize("dev", DEVICES)
def test_append_of_zeros_infinities_and_nan(dev):
    table, P = tables([3, 3, 3], 16, dev)
    cache = pool(P, 1, 16, 64, dev)
    k = torch.zeros(9, 1, 64, device=dev)
    v = torch.ones(9, 1, 64, device=dev)
    v[3, 0, 5], v[4, 0, 6], v[5, 0, 7] = math.inf, -math.inf, math.nan
    k[6:] = torch.finfo(torch.float32).max
    ops.kv_append(k, v, cache, table, offsets([3, 3, 3], dev), i32([3, 3, 3], dev), 3)
    k0, v1, k2 = held(cache, table, [3] * 3, 0)[0], held(cache, table, [3] * 3, 1)[1], held(cache, table, [3] * 3, 2)[0]
    assert (k0 == 0).all()
    s = cache.v_scale[table[1, 0].long()].item()
    assert v1[0, 0, 5] == 448 * s and v1[0, 1, 6] == -448 * s and v1[0, 2, 7].isnan()
    keep = torch.ones(3, 64, dtype=torch.bool, device=dev)
    keep[0, 5] = keep[1, 6] = keep[2, 7] = False
    assert (v1[0][keep] == 1).all()
    assert k2.isfinite().all() and (k2 > 2.9e38).all()


@pytest.mark.parametrize("dev", DEVICES)
def test_append_leaves_other_slots_alone(dev):
    table, P = tables([20, 40], 16, dev)
    cache = pool(P, 2, 16, 64, dev)
    before = [x.view(torch.uint8).clone() for x in cache[:2]]
    k = rand((3, 2, 64), torch.bfloat16, dev, 3)
    ops.kv_append(k, k, cache, table, offsets([0, 3], dev), i32([20, 40], dev), 3)      # slots 37..39: page 2 from slot 5
    for x, y in zip(cache[:2], before):
        changed = (x.view(torch.uint8) != y).any(-1).any(1)                               # (P, page)
        want = torch.zeros_like(changed)
        want[table[1, 2].long(), 5:8] = True
        assert torch.equal(changed & ~want, torch.zeros_like(want))


@pytest.mark.parametrize("dev", DEVICES)
def test_append_from_strided_tensors(dev):
    T, G, hd = 21, 2, 128
    table, P = tables([T], 16, dev)
    packed = rand((T, 3 * G, hd), torch.bfloat16, dev, 4)
    odd = rand((T, G, hd + 1), torch.bfloat16, dev, 5)[..., 1:]
    a, b = pool(P, G, 16, hd, dev), pool(P, G, 16, hd, dev)
    cos, sin = rotation(T, hd, dev)
    pos = torch.arange(T, device=dev)
    args = (table, offsets([T], dev), i32([T], dev), T, cos, sin, pos)
    ra = ops.kv_append(packed[:, :G], odd, a, *args, [packed[:, G:]])
    rb = ops.kv_append(packed[:, :G].contiguous(), odd.contiguous(), b, *args, [packed[:, G:].contiguous()])
    assert torch.equal(ra[0], rb[0])
    for x, y in zip(a, b):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))


# ---- attention ---------------------------------------------------------------------------------------
def plain_attention(q, cache, table, new, lens, q2=None, lam=None, window=0):
    H, hd = q.shape[1:]
    out, tol, at = torch.zeros_like(q, dtype=torch.float64), torch.zeros_like(q, dtype=torch.float64), 0
    for b, (n, L) in enumerate(zip(new, lens)):
        k, v = (x.repeat_interleave(H // x.shape[0], 0) for x in held(cache, table, lens, b))
        i, j = torch.arange(L - n, L, device=q.device)[:, None], torch.arange(L, device=q.device)
        see = (j <= i) & (j > i - window) if window else j <= i
        maps = []
        for x in (q,) if q2 is None else (q, q2):
            s = x[at:at + n].double().transpose(0, 1) @ k.transpose(1, 2) / math.sqrt(hd)
            p = torch.softmax(s.masked_fill(~see, -math.inf), -1).nan_to_num(0.0)
            maps.append(p @ v)
        o, t = maps[0], (2.0 ** -11 + 2.0 ** -14) * v.abs().amax((1, 2), keepdim=True).expand_as(maps[0]) if L else maps[0]
        if q2 is not None:
            w = lam.double()[:, None, None]
            o, t = (maps[0] - w * maps[1]) / (1 - w + 1e-8), t * (1 + w) / (1 - w)
        out[at:at + n], tol[at:at + n] = o.transpose(0, 1), t.transpose(0, 1)
        at += n
    return out, tol


def filled(lens, page, G, hd, dev, seed=0):
    table, P = tables(lens, page, dev, seed)
    cache = pool(P, G, page, hd, dev)
    T = sum(lens)
    k, v = rand((T, G, hd), torch.float32, dev, seed + 1), rand((T, G, hd), torch.float32, dev, seed + 2)
    k[..., :3] *= 6.0
    ops.kv_append(k, v, cache, table, offsets(lens, dev), i32(lens, dev), max(lens + [0]))
    return cache, table


def check_attention(dev, dtype, hd, page, H, G, new, lens, diff, window=0, seed=0):
    cache, table = filled(lens, page, G, hd, dev, seed)
    q, q2 = rand((sum(new), H, hd), dtype, dev, seed + 3), rand((sum(new), H, hd), dtype, dev, seed + 4)
    lam = torch.linspace(0.1, 0.9, H, device=dev)
    kw = {"q2": q2, "lam": lam} if diff else {}
    got = ops.paged_attention(q, cache, table, offsets(new, dev), i32(lens, dev), max(new + [0]), window=window, **kw)
    want, tol = plain_attention(q, cache, table, new, lens, window=window, **kw)
    assert got.dtype == dtype and got.shape == q.shape
    bad = (got.double() - want).abs() > tol + ROUND[dtype] * want.abs()
    assert not bad.any(), ((got.double() - want).abs() / (tol + ROUND[dtype] * want.abs()))[bad].max()


HEADS = [(4, 2), (8, 1), (6, 2), (3, 3), (32, 1)]


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hd,page", [(64, 16), (64, 64), (128, 32), (128, 64), (128, 128)])
@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("diff", [False, True])
def test_single_tokens(dev, dtype, hd, page, heads, diff):
    lens = [1, 300, 17, 64, 65, 129]
    check_attention(dev, dtype, hd, page, *heads, [1] * len(lens), lens, diff, seed=hd + page)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("hd,page", [(64, 16), (128, 64)])
@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("diff", [False, True])
@pytest.mark.parametrize("new,lens", [([3, 0, 1, 5], [3, 40, 200, 133]), ([70, 1, 33], [70, 500, 290]),
                                      ([150], [260]), ([1, 130, 2], [700, 130, 2])])
def test_several_tokens(dev, hd, page, heads, diff, new, lens):
    check_attention(dev, torch.bfloat16, hd, page, *heads, new, lens, diff, seed=len(new))


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("window", [1, 16, 100, 257, 100000])
@pytest.mark.parametrize("diff", [False, True])
def test_windows(dev, window, diff):
    check_attention(dev, torch.bfloat16, 128, 32, 8, 2, [1, 40, 2], [400, 300, 2], diff, window)
    check_attention(dev, torch.float16, 64, 16, 4, 2, [1, 2, 1], [400, 300, 2], diff, window)


@pytest.mark.gpu
@pytest.mark.parametrize("diff", [False, True])
def test_long_caches(diff):
    check_attention("cuda", torch.bfloat16, 128, 64, 8, 2, [1], [40001], diff)
    check_attention("cuda", torch.bfloat16, 128, 64, 8, 2, [1, 1, 1], [9000, 5, 20011], diff)
    check_attention("cuda", torch.float16, 64, 16, 4, 4, [4, 1], [30011, 12000], diff)
    check_attention("cuda", torch.bfloat16, 128, 128, 4, 1, [300, 1], [9000, 5000], diff)


@pytest.mark.gpu
def test_many_sequences():
    lens = [1 + (37 * i) % 900 for i in range(300)]
    check_attention("cuda", torch.bfloat16, 128, 64, 8, 2, [1] * 300, lens, True)
    check_attention("cuda", torch.bfloat16, 64, 16, 4, 2, [min(L, 1 + i % 3) for i, L in enumerate(lens)], lens, False)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("diff", [False, True])
def test_large_and_tiny_scores(dev, diff):
    """Scores of several hundred (one key takes all the weight) and queries far from 1 in size."""
    lens, H, G, hd = [200, 90], 4, 2, 128
    cache, table = filled(lens, 32, G, hd, dev, 7)
    lam = torch.full((H,), 0.5, device=dev)
    for size in (60.0, 1e-4, 2.0 ** -20, 3e4):
        q = (rand((2, H, hd), torch.float32, dev, 3) * size).bfloat16()
        kw = {"q2": q.flip(0), "lam": lam} if diff else {}
        # a score of size s carries 2^-24 s of rounding in its sum of 128 products, so the weights carry that much
        slack = 2.0 ** -24 * 128 * size * 12
        got = ops.paged_attention(q, cache, table, offsets([1, 1], dev), i32(lens, dev), 1, **kw)
        want, tol = plain_attention(q, cache, table, [1, 1], lens, **kw)
        if slack < 0.1:
            vmax = 5.0 * (3 if diff else 1)
            assert ((got.double() - want).abs() <= tol + ROUND[torch.bfloat16] * want.abs() + slack * vmax).all(), size
        assert got.isfinite().all()


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("new,lens", [([4, 2], [2, 100]), ([3], [0]), ([40, 1], [17, 60])])
@pytest.mark.parametrize("diff", [False, True])
def test_queries_that_see_nothing_give_zero(dev, new, lens, diff):
    """Lengths shorter than the new tokens leave their first queries without a key."""
    cache, table = filled(lens, 16, 1, 64, dev)
    q = rand((sum(new), 2, 64), torch.bfloat16, dev, 1)
    kw = {"q2": q.flip(0), "lam": torch.full((2,), 0.5, device=dev)} if diff else {}
    got = ops.paged_attention(q, cache, table, offsets(new, dev), i32(lens, dev), max(new), **kw)
    want, tol = plain_attention(q, cache, table, new, lens, **kw)
    assert (got[:max(0, new[0] - lens[0])] == 0).all()
    assert ((got.double() - want).abs() <= tol + ROUND[torch.bfloat16] * want.abs()).all()


@pytest.mark.parametrize("dev", DEVICES)
def test_no_sequences_and_padding_rows(dev):
    cache, table = filled([30, 5], 16, 2, 64, dev)
    q = rand((7, 4, 64), torch.bfloat16, dev, 2)
    got = ops.paged_attention(q, cache, table, offsets([2, 1], dev), i32([30, 5], dev), 2)
    want, tol = plain_attention(q[:3], cache, table, [2, 1], [30, 5])
    assert (got[3:] == 0).all() and ((got[:3].double() - want).abs() <= tol + ROUND[torch.bfloat16] * want.abs()).all()
    many = rand((90, 4, 64), torch.bfloat16, dev, 2)
    for tb, c, n, ln in ((table[:0], [0], 0, []), (table[:0], [0], 90, []), (table[:1], [0, 80], 80, [30]), (table[:1], [0, 2], 2, [30])):
        got = ops.paged_attention(many, cache, tb, i32(c, dev), i32(ln, dev), n)
        assert (got[c[-1]:] == 0).all() and got.isfinite().all()
    none = ops.paged_attention(q[:0], cache, table[:0], i32([0], dev), i32([], dev), 0)
    assert none.shape == (0, 4, 64)
    assert ops.kv_append(q[:0, :2], q[:0, :2], cache, table[:0], i32([0], dev), i32([], dev), 0) == []


@pytest.mark.parametrize("dev", DEVICES)
def test_strided_queries(dev):
    cache, table = filled([70], 16, 2, 128, dev)
    big = rand((5, 8, 128), torch.bfloat16, dev, 3)
    odd = rand((5, 4, 129), torch.bfloat16, dev, 4)[..., 1:]
    args = (cache, table, offsets([5], dev), i32([70], dev), 5)
    for q in (big[:, ::2], big[:, 4:], odd):
        assert torch.equal(ops.paged_attention(q, *args), ops.paged_attention(q.contiguous(), *args))


@pytest.mark.gpu
@pytest.mark.parametrize("new,lens", [([1, 1], [900, 65]), ([50, 60], [300, 100])])
def test_another_stream_graph_and_repeatability(new, lens):
    cache, table = filled(lens, 32, 2, 128, "cuda")
    q, q2 = (rand((sum(new), 8, 128), torch.bfloat16, "cuda", s) for s in (1, 2))
    lam = torch.full((8,), 0.4, device="cuda")
    run = lambda: ops.paged_attention(q, cache, table, cu, ln, max(new), q2=q2, lam=lam)  # noqa: E731
    cu, ln = offsets(new, "cuda"), i32(lens, "cuda")
    first = run()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = run()
    s.synchronize()
    assert torch.equal(first, other)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held_out = run()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(first, held_out)


# ---- refusals ----------------------------------------------------------------------------------------
@pytest.mark.gpu
def test_bad_pages_and_lengths_are_skipped_and_reported():
    from mamformer_b200.fault import PagedCacheError, check_device_status
    check_device_status()
    cache, table = filled([40, 40], 16, 1, 64, "cuda")
    good = table.clone()
    q = rand((2, 1, 64), torch.bfloat16, "cuda", 1)
    cu, lens = offsets([1, 1], "cuda"), i32([40, 40], "cuda")
    want = ops.paged_attention(q, cache, good, cu, lens, 1)
    for bad in (-1, cache.k.shape[0], 1 << 30):
        table[1, 1] = bad
        got = ops.paged_attention(q, cache, table, cu, lens, 1)
        assert got.isfinite().all() and torch.equal(got[0], want[0])
        with pytest.raises(PagedCacheError):
            check_device_status()
        kv = rand((2, 1, 64), torch.bfloat16, "cuda", 2)
        table[1, 2] = bad
        ops.kv_append(kv, kv, cache, table, cu, lens, 1)
        with pytest.raises(PagedCacheError):
            check_device_status()
        table[1, 2] = good[1, 2]
    ops.paged_attention(q, cache, good, cu, i32([40, 80], "cuda"), 1)       # longer than the table
    with pytest.raises(PagedCacheError):
        check_device_status()
    cos, sin = rotation(4, 64, "cuda")
    ops.kv_append(kv, kv, cache, good, cu, lens, 1, cos, sin, torch.tensor([3, 4], device="cuda"))
    with pytest.raises(PagedCacheError, match="position"):
        check_device_status()
    ops.kv_append(kv, kv, cache, good, cu, i32([0, 40], "cuda"), 1)
    with pytest.raises(PagedCacheError, match="lengths"):
        check_device_status()
    check_device_status()


@pytest.mark.gpu
def test_refusals():
    cache, table = filled([40], 16, 2, 64, "cuda")
    cu, lens = offsets([1], "cuda"), i32([40], "cuda")
    q = rand((1, 4, 64), torch.bfloat16, "cuda", 1)
    ok = (cache, table, cu, lens, 1)
    bad = [((q.float(), *ok), {}), ((q[:, :3], *ok), {}), ((q[..., :32], *ok), {}), ((q.cpu(), *ok), {}),
           ((q, cache, table.long(), cu, lens, 1), {}), ((q, cache, table, cu[:1], lens, 1), {}),
           ((q, cache._replace(k=cache.k.view(torch.uint8)), table, cu, lens, 1), {}),
           ((q, cache._replace(k_scale=cache.k_scale[:1]), table, cu, lens, 1), {}),
           ((q, cache._replace(v=cache.v.transpose(1, 2)), table, cu, lens, 1), {}),
           ((q, *ok), {"q2": q}), ((q, *ok), {"lam": torch.zeros(4, device="cuda")}),
           ((q, *ok), {"q2": q, "lam": torch.zeros(3, device="cuda")}), ((q, *ok), {"window": -1})]
    for args, kw in bad:
        with pytest.raises((RuntimeError, ValueError)):
            ops.paged_attention(*args, **kw)
    k = rand((1, 2, 64), torch.bfloat16, "cuda", 2)
    cos, sin = rotation(50, 64, "cuda")
    pos = torch.zeros(1, dtype=torch.long, device="cuda")
    for args, kw in [((k, k.half()), {}), ((k[:, :1], k[:, :1]), {}), ((k, k), {"queries": [q]}),
                     ((k, k), {"cos": cos, "sin": sin}), ((k, k), {"cos": cos.double(), "sin": sin, "positions": pos}),
                     ((k, k), {"cos": cos, "sin": sin, "positions": pos, "queries": [q, q, q]}),
                     ((k, k), {"cos": cos, "sin": sin, "positions": pos, "queries": [q.float()]})]:
        with pytest.raises((RuntimeError, ValueError)):
            ops.kv_append(*args, *ok, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("heads", [(4, 2), (8, 1)])
@pytest.mark.parametrize("diff", [False, True])
@pytest.mark.parametrize("new,lens,window", [([70], [5000], 0), ([33, 40], [4000, 61], 0), ([300], [3000], 700),
                                             ([20, 0, 90], [2100, 7, 90], 0), ([64], [64], 0)])
def test_few_tiles_share_their_keys(heads, diff, new, lens, window):
    check_attention("cuda", torch.bfloat16, 128, 64, *heads, new, lens, diff, window)
    check_attention("cuda", torch.float16, 64, 16, *heads, new, lens, diff, window)


@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 40])
def test_pages_past_32_bits_of_offset(new):
    """The same sequences in a small pool and at the end of one of over 2^32 bytes: the same codes and results."""
    G, page, hd, H, P = 8, 64, 128, 16, 66500
    lens, news = [200, 130], [new, new]
    assert P * G * page * hd > 1 << 32
    small = pool(8, G, page, hd, "cuda")
    big = ops.PagedKV(*(torch.zeros(P, G, page, hd, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn) for _ in range(2)),
                      *(torch.ones(P, G, device="cuda") for _ in range(2)))
    table = torch.tensor([[3, 0, 6, 1], [2, 7, 5, -1]], dtype=torch.int32, device="cuda")
    far = torch.where(table >= 0, table + P - 8, table)
    k, v = rand((330, G, hd), torch.bfloat16, "cuda", 1), rand((330, G, hd), torch.bfloat16, "cuda", 2)
    q, q2 = rand((2 * new, H, hd), torch.bfloat16, "cuda", 3), rand((2 * new, H, hd), torch.bfloat16, "cuda", 4)
    lam = torch.full((H,), 0.3, device="cuda")
    got = []
    for cache, t in ((small, table), (big, far)):
        ops.kv_append(k, v, cache, t, offsets(lens, "cuda"), i32(lens, "cuda"), 200)
        got.append(ops.paged_attention(q, cache, t, offsets(news, "cuda"), i32(lens, "cuda"), new, q2=q2, lam=lam))
    assert torch.equal(got[0], got[1]) and got[0].isfinite().all()
    want, tol = plain_attention(q, small, table, news, lens, q2, lam)
    assert ((got[0].double() - want).abs() <= tol + ROUND[torch.bfloat16] * want.abs()).all()
    for b in range(2):
        for x, y in zip(held(small, table, lens, b), held(big, far, lens, b)):
            assert torch.equal(x, y)

"""The 4-bit paged cache: ops.kv_append, kv_read, paged_attention and kv_evict on ops.PagedKV4 (csrc/paged_kv.cu,
csrc/paged4*.cu on CUDA, the eager forms on CPU) against plain 64-bit forms.

Tolerances, from the arithmetic.  A stored value is within half a step of its group's levels, a step being a fifteenth of
the group's range (0 in it) rounded up to 7 significant bits: at most 2^-6 more, or 2^-20.  Attention over given codes takes
them exactly, rounds each weight once to 11 bits at 2^7 or more for a row's largest (2^-11 of itself, and 2^-32 of the
largest one's for those that are subnormal then) and the result to its type; fp32 sums add less than 2^-14 of the shares.
A slot's received weight is a sum of fp32 weights, whose scores are fp32 sums of hd exact products: each rounding is
at most 2^-23 of the sum of their sizes, in the score and in the row's sum of weights."""

import math

import pytest
import torch

from mamformer_b200 import ops
from test_paged_cache import DEVICES, ROUND, i32, offsets, rand, rotation, tables, turned


def pool(P, G, page, hd, dev, mass=True):
    """A pool full of what earlier owners left: scales that are NaN or infinite, any weights."""
    g = torch.Generator().manual_seed(P)
    blocks = torch.randint(0, 256, (P, G, page // 16, 18 * hd), generator=g, dtype=torch.uint8)
    blocks.view(-1)[::3] = 0xFF
    return ops.PagedKV4(blocks.to(dev), torch.full((P, G, page), 3.0, device=dev) if mass else None)


def group_of(hd):
    """The group of each dim."""
    return torch.tensor([d // 4 % (hd // 32) for d in range(hd)])


def parts(blocks):
    """Key values and value values (P, G, page, hd) in 64 bits, read byte by byte as the layout says."""
    hd = blocks.shape[-1] // 18
    out = []
    for x in (blocks[..., :9 * hd], blocks[..., 9 * hd:]):
        code = x[..., :8 * hd].reshape(*x.shape[:3], 16, hd // 2).long()
        word = x[..., 8 * hd:].reshape(*x.shape[:3], 16, hd // 32, 2).long()
        word = word[..., 0] + 256 * word[..., 1]
        s = (word // 16 * 16).to(torch.int16).view(torch.float16).double()
        n = torch.stack([code % 16, code // 16], -1).flatten(-2).double()
        of = group_of(hd).to(x.device)
        out.append((s[..., of] * (n - (word % 16).double()[..., of])).flatten(2, 3))
    return out


def held(cache, table, lens, b):
    """k, v (G, len, hd) of a sequence in 64 bits."""
    page = 16 * cache.blocks.shape[2]
    pages = table[b, :-(-lens[b] // page)].long()
    return [x.transpose(0, 1).flatten(1, 2)[:, :lens[b]] for x in parts(cache.blocks[pages])]


def half_step(x):
    """What a stored value may be off, for x (.., hd) in 64 bits."""
    hd = x.shape[-1]
    tol = torch.empty_like(x)
    for j in range(hd // 32):
        of = (group_of(hd) == j).to(x.device)
        span = x[..., of].amax(-1, keepdim=True).clamp(min=0) - x[..., of].amin(-1, keepdim=True).clamp(max=0)
        tol[..., of] = 0.5 * torch.maximum(span / 15 * (1 + 2.0 ** -6), span / 15 + 2.0 ** -20) * (1 + 2.0 ** -12)
    return tol


def filled(lens, page, G, hd, dev, gain=1.0, seed=0, mass=True):
    table, P = tables(lens, page, dev, seed)
    cache = pool(P, G, page, hd, dev, mass)
    T = sum(lens)
    k, v = rand((T, G, hd), torch.float32, dev, seed + 1), rand((T, G, hd), torch.float32, dev, seed + 2) * gain
    ops.kv_append(k + 0.5, v, cache, table, offsets(lens, dev), i32(lens, dev), max(lens))
    return cache, table


# ---- append and read -----------------------------------------------------------------------------------
STEPS = [[[1]], [[5, 0, 130], [1, 1, 1], [3, 40, 0], [0, 0, 0]], [[16, 15, 17, 1], [16, 16, 16, 16], [1, 2, 300, 1]]]


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("hd,page,G", [(64, 16, 2), (64, 128, 1), (128, 32, 3), (128, 64, 8)])
@pytest.mark.parametrize("steps", STEPS)
def test_append_and_read(dev, dtype, hd, page, G, steps):
    B, H = len(steps[0]), 2 * G
    total = [sum(s[b] for s in steps) for b in range(B)]
    table, P = tables(total, page, dev)
    cache = pool(P, G, page, hd, dev)
    before = cache.blocks.clone()
    cos, sin = rotation(max(total) + 1, hd, dev)
    lens = [0] * B
    want = [[[], []] for _ in range(B)]
    for i, new in enumerate(steps):
        lens = [a + n for a, n in zip(lens, new)]
        T = sum(new)
        k, v, q1, q2 = (rand((T, h, hd), dtype, dev, 10 * i + j) for j, h in enumerate((G, G, H, H)))
        k, v = k * 3.0 ** i + 1.0, v * 0.3 ** i
        pos = torch.tensor([p for n, L in zip(new, lens) for p in range(L - n, L)], dtype=torch.long, device=dev)
        cu, ln = offsets(new, dev), i32(lens, dev)
        r1, r2 = ops.kv_append(k, v, cache, table, cu, ln, max(new), cos, sin, pos, [q1, q2])
        for r, q in ((r1, q1), (r2, q2)):
            w = turned(q, cos, sin, pos)
            assert r.dtype == dtype and ((r.double() - w).abs() <= (ROUND[dtype] + 2.0 ** -22) * w.abs() + 2.0 ** -22).all()
        kt, at = turned(k, cos, sin, pos), 0
        back = ops.kv_read(cache, table, cu, ln, T, torch.float32)
        for x, got in zip((kt, v.double()), back):
            assert ((got.double() - x).abs() <= half_step(x) + 2.0 ** -20 * (x.abs().amax() if T else 0.0)).all()
        for got, exact in zip(ops.kv_read(cache, table, cu, ln, T, torch.float16), back):
            assert torch.equal(got.float(), exact)                # the levels are f16 values
        for got, exact in zip(ops.kv_read(cache, table, cu, ln, T, torch.bfloat16), back):
            assert torch.equal(got, exact.bfloat16())
        for b, n in enumerate(new):
            for j in range(2):
                want[b][j].append(back[j][at:at + n])
            at += n
    used = torch.zeros(P, page, dtype=torch.bool, device=dev)
    for b in range(B):
        for got, w in zip(held(cache, table, total, b), want[b]):        # later steps left the earlier tokens alone
            assert torch.equal(got, torch.cat(w).transpose(0, 1).double())
        slot = torch.arange(total[b], device=dev)
        used[table[b].long()[slot // page], slot % page] = True
    rest = lambda x: x[..., :8 * hd].reshape(P, G, page, hd // 2).transpose(1, 2)[~used]  # noqa: E731
    assert torch.equal(rest(before), rest(cache.blocks))                  # and slots that nobody appended to
    assert (cache.mass.transpose(1, 2)[used] == 0).all() and (cache.mass.transpose(1, 2)[~used] == 3).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("size", [1.0, 1e-4, 1e-7, 300.0, 1e5])
@pytest.mark.parametrize("hd", [64, 128])
def test_both_devices_store_the_same_bytes(dtype, size, hd):
    T, G, page = 300, 3, 32
    k, v = rand((T, G, hd), torch.float32, "cpu", 1) * size, rand((T, G, hd), torch.float32, "cpu", 2) * size
    v[::7] = v[::7].abs()
    v[5], k[6] = 0.0, -0.0
    cos, sin = rotation(T, hd, "cpu")
    got = []
    for dev in ("cpu", "cuda"):
        table, P = tables([T], page, dev)
        cache = ops.PagedKV4(torch.zeros(P, G, page // 16, 18 * hd, dtype=torch.uint8, device=dev))
        ops.kv_append(k.to(dtype).to(dev), v.to(dtype).to(dev), cache, table, offsets([T], dev), i32([T], dev), T, cos.to(dev),
                      sin.to(dev), torch.arange(T, device=dev))
        got.append(cache.blocks.cpu())
    assert torch.equal(*got)


@pytest.mark.parametrize("dev", DEVICES)
def test_append_of_what_is_no_number_or_out_of_range(dev):
    table, P = tables([4], 16, dev)
    cache = pool(P, 1, 16, 64, dev)
    k, v = torch.zeros(4, 1, 64, device=dev), torch.ones(4, 1, 64, device=dev)
    v[0, 0, 5], v[1, 0, 6], v[2, 0, 7] = math.nan, math.inf, -math.inf
    k[1] = torch.finfo(torch.float32).max
    k[2, 0, :32], k[2, 0, 32:] = 65504.0, -65504.0
    k[3] = 3e-8
    ops.kv_append(k, v, cache, table, offsets([4], dev), i32([4], dev), 4)
    k0, v0 = (x[:, 0] for x in ops.kv_read(cache, table, offsets([4], dev), i32([4], dev), 4, torch.float32))
    assert (k0[0] == 0).all() and k0[1].isfinite().all() and (k0[1] > 65000).all()
    # both ends of f16 in a group: the levels stop short of them, around 0
    assert (k0[2, :32] > 30000).all() and (k0[2, 32:] < -30000).all()
    assert (k0[3].abs() <= 2.0 ** -20).all()
    other = torch.ones(64, dtype=torch.bool, device=dev)
    other[5] = False
    assert v0[0, 5] == 0 and ((v0[0][other] - 1).abs() <= 1 / 30).all()
    assert v0[1, 6] > 65000 and v0[2, 7] < -65000
    far = (group_of(64) != group_of(64)[6]).to(dev)                   # the other group's values are untouched
    assert ((v0[1][far] - 1).abs() <= 1 / 30).all()
    assert ((v0[3] - 1).abs() <= 1 / 30).all()


@pytest.mark.parametrize("dev", DEVICES)
def test_append_from_strided_tensors(dev):
    T, G, hd = 21, 2, 128
    table, P = tables([T], 16, dev)
    packed = rand((T, 3 * G, hd), torch.bfloat16, dev, 4)
    odd = rand((T, G, hd + 1), torch.bfloat16, dev, 5)[..., 1:]
    a, b = pool(P, G, 16, hd, dev), pool(P, G, 16, hd, dev)
    cos, sin = rotation(T, hd, dev)
    args = (table, offsets([T], dev), i32([T], dev), T, cos, sin, torch.arange(T, device=dev))
    ra = ops.kv_append(packed[:, :G], odd, a, *args, [packed[:, G:]])
    rb = ops.kv_append(packed[:, :G].contiguous(), odd.contiguous(), b, *args, [packed[:, G:].contiguous()])
    assert torch.equal(ra[0], rb[0]) and torch.equal(a.blocks, b.blocks)


@pytest.mark.parametrize("dev", DEVICES)
def test_read_of_more_than_there_is(dev):
    """Rows in front of a shorter sequence, of an empty one and of none are zeros."""
    cache, table = filled([5, 1, 40], 16, 2, 64, dev)
    want = [held(cache, table, [5, 1, 40], b) for b in range(3)]
    k, v = ops.kv_read(cache, table, offsets([8, 3, 2], dev) + 2, i32([5, 0, 40], dev), 17, torch.float32)
    for i, x in enumerate((k, v)):
        x = x.double()
        assert (x[:5] == 0).all() and (x[10:13] == 0).all() and (x[15:] == 0).all()
        assert torch.equal(x[5:10], want[0][i].transpose(0, 1)) and torch.equal(x[13:15], want[2][i].transpose(0, 1)[38:])


# ---- attention -----------------------------------------------------------------------------------------
def plain(q, cache, table, new, lens, q2=None, lam=None, window=0, scale=None):
    """The definition in 64 bits and each row's tolerance; the received weights and theirs."""
    H, hd = q.shape[1:]
    G, page = cache.blocks.shape[1], 16 * cache.blocks.shape[2]
    scale = hd ** -0.5 if scale is None else scale
    out, tol, at = torch.zeros_like(q, dtype=torch.float64), torch.zeros_like(q, dtype=torch.float64), 0
    mass = torch.zeros(cache.blocks.shape[0], G, page, dtype=torch.float64, device=q.device)
    mass_tol = torch.zeros_like(mass)
    for b, (n, L) in enumerate(zip(new, lens)):
        if n and L:
            i, j = torch.arange(L - n, L, device=q.device)[:, None], torch.arange(L, device=q.device)
            see = (j <= i) & (j > i - window) if window else j <= i
            used = see.any(0)
            first = int(used.long().argmax()) // page * page
            pages = table[b, first // page:-(-L // page)].long()
            k, v = (torch.zeros(G, L, hd, dtype=torch.float64, device=q.device) for _ in range(2))
            for x, y in zip((k, v), parts(cache.blocks[pages])):
                x[:, first:] = y.transpose(0, 1).flatten(1, 2)[:, :L - first]
            k, v = (x.masked_fill(~used[:, None], 0.0).repeat_interleave(H // G, 0) for x in (k, v))
            maps, tols = [], []
            for x in (q,) if q2 is None else (q, q2):
                x = x[at:at + n].double().transpose(0, 1)
                s = x @ k.transpose(1, 2) * scale
                p = torch.softmax(s.masked_fill(~see, -math.inf), -1).nan_to_num(0.0)
                maps.append(p @ v)
                most = v.abs().amax((1, 2))[:, None, None]
                tols.append((2.0 ** -11 + 2.0 ** -14) * (p @ v.abs()) + L * 2.0 ** -32 * p.amax(-1, keepdim=True) * most)
                sizes = (x.abs() @ k.transpose(1, 2).abs() * abs(scale)).masked_fill(~see, 0.0)
                off = 2 * (hd + 4) * 2.0 ** -23 * (sizes + sizes.amax(-1, keepdim=True)) + (L / 16 + 64) * 2.0 ** -23
                for to, y in ((mass, p), (mass_tol, p * off + 2.0 ** -120)):
                    y = y.sum(1).unflatten(0, (G, -1)).sum(1)                              # (G, L)
                    to[table[b].long()[j[used] // page], :, j[used] % page] += y[:, used].T
            o, t = maps[0], tols[0]
            if q2 is not None:
                w = lam.double()[:, None, None]
                o, t = (maps[0] - w * maps[1]) / (1 - w + 1e-8), (tols[0] + w * tols[1]) / (1 - w)
            out[at:at + n], tol[at:at + n] = o.transpose(0, 1), t.transpose(0, 1)
        at += n
    return out, tol, mass, mass_tol


def close(got, want, tol):
    tol = tol + ROUND[got.dtype] * want.abs()
    bad = ~((got.double() - want).abs() <= tol)
    assert not bad.any(), ((got.double() - want).abs() / tol)[bad].max()


def pair(q, diff):
    """The second map's arguments."""
    return {"q2": q.flip(0), "lam": torch.linspace(0.1, 0.8, q.shape[1], device=q.device)} if diff else {}


def check(q, cache, table, new, lens, **kw):
    """Output and received weights, which are added to what is there."""
    dev = q.device
    want, tol, mass, mass_tol = plain(q, cache, table, new, lens, **kw)
    if cache.mass is not None:
        cache.mass.copy_(torch.rand(cache.mass.shape, generator=torch.Generator().manual_seed(5)).to(dev))
        had = cache.mass.double()
    got = ops.paged_attention(q, cache, table, offsets(new, dev), i32(lens, dev), max(new), **kw)
    close(got, want, tol)
    if cache.mass is not None:
        close(cache.mass, had + mass, mass_tol + 2.0 ** -23 * (had + mass))
    return got


CASES = [
    ([1], [1]), ([1], [700]), ([1, 1, 1], [17, 1, 300]), ([0, 1, 0], [5, 33, 0]), ([3, 1, 2], [60, 64, 130]),
    ([5, 0, 7], [5, 20, 200]), ([20], [50]), ([70, 1], [90, 200]), ([40, 3, 100], [40, 3, 331]), ([300], [300]), ([130, 140], [513, 140]),
]


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("new,lens", CASES)
@pytest.mark.parametrize("hd,page,G,rep", [(64, 16, 2, 1), (64, 32, 1, 4), (128, 16, 1, 3), (128, 64, 2, 4), (128, 128, 1, 16)])
@pytest.mark.parametrize("diff,window,dtype", [(False, 0, torch.bfloat16), (True, 0, torch.float16), (False, 29, torch.float16), (True, 64, torch.bfloat16)])
def test_attention_and_received_weights(dev, new, lens, hd, page, G, rep, diff, window, dtype):
    cache, table = filled([max(n, 1) for n in lens], page, G, hd, dev)
    q = rand((sum(new), G * rep, hd), dtype, dev, 3)
    kw = dict(pair(q, diff), window=window)
    got = check(q, cache, table, new, lens, **kw)
    again = ops.paged_attention(q, ops.PagedKV4(cache.blocks), table, offsets(new, dev), i32(lens, dev), max(new), **kw)
    assert torch.equal(got, again)                                    # the same bits with and without them


@pytest.mark.gpu
@pytest.mark.parametrize("new,lens", [([1], [40000]), ([1, 1], [9000, 20]), ([2], [30000]), ([9, 1], [6000, 6000]), ([40], [9000]),
                                      ([200], [5000]), ([1] * 130, [100 + 7 * i for i in range(130)])])
@pytest.mark.parametrize("hd,diff", [(64, True), (128, False), (128, True)])
def test_long_caches_split_over_ctas(new, lens, hd, diff):
    cache, table = filled(lens, 64, 2, hd, "cuda")
    q = rand((sum(new), 8, hd), torch.bfloat16, "cuda", 3)
    a = check(q, cache, table, new, lens, **pair(q, diff))
    mass = cache.mass.clone()
    b = check(q, cache, table, new, lens, **pair(q, diff))
    assert torch.equal(a, b) and torch.equal(mass, cache.mass)        # no order of arrival in them


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("scale", [0.0, -0.1, -1e-30, 0.3, 3.0])
@pytest.mark.parametrize("diff", [False, True])
@pytest.mark.parametrize("new,lens", [([1, 3], [70, 33]), ([130, 70], [130, 400])])
def test_score_factors_of_any_sign(dev, scale, diff, new, lens):
    cache, table = filled(lens, 32, 2, 128, dev)
    q = rand((sum(new), 4, 128), torch.bfloat16, dev, 1)
    check(q, cache, table, new, lens, **pair(q, diff), scale=scale)
    check(q, cache, table, new, lens, **pair(q, diff), scale=scale, window=20)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("size", [2.0 ** -120, 2.0 ** -30, 2.0 ** 10])
@pytest.mark.parametrize("new,lens", [([1, 3], [70, 33]), ([130, 70], [130, 400])])
def test_queries_and_values_of_any_size(dev, size, new, lens):
    """Values from the smallest step to f16's largest, in neighbouring tokens; sharp and flat weights."""
    table, P = tables(lens, 16, dev)
    cache = pool(P, 1, 16, 64, dev)
    k, v = rand((sum(lens), 1, 64), torch.float32, dev, 1), rand((sum(lens), 1, 64), torch.float32, dev, 2)
    v = v * torch.tensor([1.0, 1e4, 1e-5, 30.0, 0.0, 1e-3, 2e4], device=dev)[torch.arange(sum(lens), device=dev) % 7, None, None]
    k[::5] = 0.0
    ops.kv_append(k, v, cache, table, offsets(lens, dev), i32(lens, dev), max(lens))
    q = (rand((sum(new), 2, 64), torch.float32, dev, 3) * size).bfloat16()
    check(q, cache, table, new, lens)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("diff", [False, True])
@pytest.mark.parametrize("new,lens", [([300], [10]), ([280, 90], [0, 90]), ([520, 300], [1, 3]), ([3, 2], [1, 0])])
def test_rows_that_see_nothing_give_zero(dev, hd, diff, new, lens):
    cache, table = filled([max(n, 1) for n in lens], 16, 1, hd, dev)
    q = rand((sum(new), 2, hd), torch.bfloat16, dev, 1)
    got = check(q, cache, table, new, lens, **pair(q, diff))
    at = 0
    for n, L in zip(new, lens):
        assert (got[at:at + n - L] == 0).all()
        at += n


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("page,window", [(16, 40), (64, 70)])
@pytest.mark.parametrize("new,lens", [([1, 2], [300, 170]), ([90, 150], [300, 170]), ([90], [2500])])
def test_pages_below_a_window_may_be_given_back(dev, page, window, new, lens):
    from mamformer_b200.fault import check_device_status
    cache, table = filled(lens, page, 2, 128, dev)
    P = cache.blocks.shape[0]
    unused = min(set(range(P)) - set(table.flatten().tolist()))
    q = rand((sum(new), 4, 128), torch.bfloat16, dev, 3)
    check_device_status()
    for gone in (unused, -1, P + 5):
        t = table.clone()
        for b, (n, L) in enumerate(zip(new, lens)):
            t[b, :max(0, L - n + 1 - window) // page] = gone
        check(q, cache, t, new, lens, window=window)
        check_device_status()


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("first", [1, 40])
@pytest.mark.parametrize("new,lens", [([1, 1], [40, 20]), ([60, 3], [90, 3]), ([1, 90], [17, 400])])
def test_rows_of_no_sequence(dev, first, new, lens):
    """Offsets that do not start at 0, and rows behind the last sequence: not appended, outputs 0."""
    table, P = tables(lens, 16, dev)
    G, hd, T = 2, 64, sum(new)
    k, v = rand((T, G, hd), torch.bfloat16, dev, 1), rand((T, G, hd), torch.bfloat16, dev, 2)
    caches = pool(P, G, 16, hd, dev), pool(P, G, 16, hd, dev)
    for c in caches:
        kx, vx = rand((sum(lens), G, hd), torch.bfloat16, dev, 6), rand((sum(lens), G, hd), torch.bfloat16, dev, 7)
        ops.kv_append(kx, vx, c, table, offsets(lens, dev), i32(lens, dev), max(lens))
    cu, around = offsets(new, dev), rand((first, G, hd), torch.bfloat16, dev, 5)
    ops.kv_append(k, v, caches[0], table, cu, i32(lens, dev), max(new))
    ops.kv_append(torch.cat([around, k, around]), torch.cat([around, v, around]), caches[1], table, cu + first, i32(lens, dev), max(new))
    assert torch.equal(caches[0].blocks, caches[1].blocks)
    q = rand((T, 4, hd), torch.bfloat16, dev, 3)
    want = ops.paged_attention(q, caches[0], table, cu, i32(lens, dev), max(new))
    pad = rand((first, 4, hd), torch.bfloat16, dev, 4)
    got = ops.paged_attention(torch.cat([pad, q, pad]), caches[1], table, cu + first, i32(lens, dev), max(new))
    assert (got[:first] == 0).all() and (got[first + T:] == 0).all()
    # another share of the work for each CTA may be another order of the sums: two roundings of the result
    assert ((got[first:first + T].double() - want.double()).abs() <= 2 * (2.0 ** -8 + 2.0 ** -10) * want.double().abs().amax(-1, keepdim=True)).all()
    assert ((caches[0].mass - caches[1].mass).abs() <= 2.0 ** -15 * caches[0].mass.abs()).all()


# ---- eviction ------------------------------------------------------------------------------------------
def some_mass(shape, seed, dev):
    """Heavy tails, many ties, zeros of both signs."""
    g = torch.Generator().manual_seed(seed)
    m = torch.randn(shape, generator=g).mul_(3).exp_()
    m = torch.where(torch.rand(shape, generator=g) < 0.3, m.round(), m)
    m = torch.where(torch.rand(shape, generator=g) < 0.1, -0.0, m)
    return m.to(dev)


def kept_slots(weights, L, budget, recent):
    """By hand: order by (-weight, slot)."""
    if L <= budget:
        return list(range(L))
    order = sorted(range(L - recent), key=lambda i: (-weights[i], i))
    return sorted(order[:budget - recent]) + list(range(L - recent, L))


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("hd,page,G", [(64, 16, 3), (128, 32, 2), (128, 128, 1)])
@pytest.mark.parametrize("lens,budget,recent", [([1], 1, 0), ([40, 7, 0, 100], 20, 5), ([130, 33, 64], 33, 33), ([257, 300], 200, 0), ([50, 300], 300, 17),
                                                ([300], 299, 298), ([300, 290], 1, 0), ([20], 500, 3)])
def test_evict(dev, in_place, hd, page, G, lens, budget, recent):
    cache, table = filled([max(n, 1) for n in lens], page, G, hd, dev)
    P = cache.blocks.shape[0]
    cache.mass.copy_(some_mass(cache.mass.shape, 1, dev))
    mass = cache.mass.clone()
    before = [held(cache, table, lens, b) if L else None for b, L in enumerate(lens)]
    to = None
    if not in_place:
        t, extra = tables([max(1, min(n, budget)) for n in lens], page, dev, 9)
        cache = ops.PagedKV4(torch.cat([cache.blocks, pool(extra, G, page, hd, dev).blocks]), torch.cat([mass, torch.full((extra, G, page), 8.0, device=dev)]))
        to = torch.where(t >= 0, t + P, t)
    source = cache.blocks[:P].clone()
    kept, left = ops.kv_evict(cache, table, i32(lens, dev), budget, recent, out_table=to)
    assert kept.dtype == left.dtype == torch.int32 and kept.shape == (len(lens), G, budget)
    assert left.tolist() == [min(n, budget) for n in lens]
    if not in_place:
        assert torch.equal(cache.blocks[:P], source) and torch.equal(cache.mass[:P], mass)
    where = table if in_place else to
    for b, L in enumerate(lens):
        slot = torch.arange(L, device=dev)
        for g in range(G):
            w = mass[table[b].long()[slot // page], g, slot % page]
            want = kept_slots(w.tolist(), L, budget, recent)
            assert kept[b, g].tolist() == want + [-1] * (budget - len(want))
            if not L:
                continue
            at = torch.arange(len(want), device=dev)
            assert torch.equal(cache.mass[where[b].long()[at // page], g, at % page], w[want])
            for x, y in zip(held(cache, where, left.tolist(), b), before[b]):
                assert torch.equal(x[g], y[g][want])


@pytest.mark.gpu
@pytest.mark.parametrize("L,budget,recent", [(9000, 3000, 10), (65536, 65535, 0), (70000, 12345, 777), (140000, 100, 1), (140000, 139000, 500)])
@pytest.mark.parametrize("ties", ["none", "some", "all"])
def test_evict_from_long_caches(L, budget, recent, ties):
    """Several CTAs of a cluster, and several rounds of it."""
    page, G, hd = 64, 2, 64
    table, P = tables([L], page, "cuda")
    g = torch.Generator("cuda").manual_seed(1)
    blocks = torch.randint(0, 256, (P, G, page // 16, 18 * hd), generator=g, dtype=torch.uint8, device="cuda")
    m = torch.randn(P, G, page, generator=g, device="cuda").exp()
    m = {"none": m, "some": m.round(), "all": torch.ones_like(m)}[ties]
    cache = ops.PagedKV4(blocks.clone(), m.clone())
    kept, left = ops.kv_evict(cache, table, i32([L], "cuda"), budget, recent)
    at = lambda x, g, slot: x[table[0].long()[slot // page], g, slot % page]  # noqa: E731
    code = lambda x: x[..., :8 * hd].reshape(P, G, page // 16, 16, hd // 2).flatten(2, 3)  # noqa: E731
    for g in range(G):
        w = at(m, g, torch.arange(L - recent, device="cuda"))
        want = torch.cat([torch.sort(w, descending=True, stable=True).indices[:budget - recent].sort().values, torch.arange(L - recent, L, device="cuda")])
        assert torch.equal(kept[0, g].long(), want)
        r = torch.arange(budget, device="cuda")
        assert torch.equal(at(cache.mass, g, r), at(m, g, want)) and torch.equal(at(code(cache.blocks), g, r), at(code(blocks), g, want))


@pytest.mark.parametrize("dev", DEVICES)
def test_evict_orders_any_weights(dev):
    """Infinities, NaN above them, negative weights below zero."""
    cache, table = filled([8], 16, 1, 64, dev)
    page = table[0, 0].long()
    cache.mass[page, 0, :8] = torch.tensor([0.0, math.nan, -1.0, math.inf, -math.inf, 2.0, -0.0, 2.0], device=dev)
    for budget, want in ((1, [1]), (2, [1, 3]), (3, [1, 3, 5]), (4, [1, 3, 5, 7]), (5, [0, 1, 3, 5, 7]), (7, [0, 1, 2, 3, 5, 6, 7])):
        c = ops.PagedKV4(cache.blocks.clone(), cache.mass.clone())
        kept, _ = ops.kv_evict(c, table, i32([8], dev), budget, 0)
        assert kept[0, 0].tolist() == want


@pytest.mark.parametrize("dev", DEVICES)
def test_attention_over_what_is_left(dev):
    """Append, attend, evict, append, attend: the whole turn, against attention over the kept tokens."""
    lens, G, hd, page, budget, recent = [90, 40, 130], 2, 128, 16, 48, 8
    cache, table = filled(lens, page, G, hd, dev)
    cache.mass.zero_()
    q = rand((3, 8, hd), torch.bfloat16, dev, 1)
    cu = offsets([1, 1, 1], dev)
    check(q, cache, table, [1, 1, 1], lens)
    before = [held(cache, table, lens, b) for b in range(3)]
    kept, left = ops.kv_evict(cache, table, i32(lens, dev), budget, recent)
    now = [n + 1 for n in left.tolist()]
    k, v = rand((3, G, hd), torch.bfloat16, dev, 2), rand((3, G, hd), torch.bfloat16, dev, 3)
    ops.kv_append(k, v, cache, table, cu, i32(now, dev), 1)
    for b in range(3):
        n = left[b].item()
        for x, y in zip(held(cache, table, now, b), before[b]):
            for g in range(G):
                assert torch.equal(x[g, :n], y[g][kept[b, g, :n].long()])
    check(q, cache, table, [1, 1, 1], now)


# ---- refusals ------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dev", DEVICES)
def test_refusals(dev):
    cache, table = filled([40], 16, 2, 64, dev)
    cu, ln = offsets([2], dev), i32([40], dev)
    k = rand((2, 2, 64), torch.bfloat16, dev, 1)
    q = rand((2, 4, 64), torch.bfloat16, dev, 1)
    bad = (ValueError, RuntimeError)
    with pytest.raises(bad):
        ops.kv_append(k[:, :1], k[:, :1], cache, table, cu, ln, 2)
    with pytest.raises(bad):
        ops.kv_append(k[..., :32], k[..., :32], cache, table, cu, ln, 2)
    with pytest.raises(bad):
        ops.paged_attention(q[:, :3], cache, table, cu, ln, 2)
    with pytest.raises(bad):
        ops.paged_attention(q[..., :32].contiguous(), cache, table, cu, ln, 2)
    with pytest.raises(bad):
        ops.paged_attention(q, cache, table, cu, ln, 2, q2=q)
    with pytest.raises(RuntimeError, match="gradient"):
        ops.paged_attention(q.clone().requires_grad_(True), cache, table, cu, ln, 2)
    for budget, recent in ((0, 0), (5, 6), (5, -1)):
        with pytest.raises(ValueError):
            ops.kv_evict(cache, table, ln, budget, recent)
    with pytest.raises(ValueError, match="mass"):
        ops.kv_evict(ops.PagedKV4(cache.blocks), table, ln, 5, 1)
    with pytest.raises(bad):
        ops.kv_evict(cache, table, ln, 30, 1, out_table=table[:, :1].contiguous())
    with pytest.raises(TypeError):
        ops.kv_evict((cache.blocks, cache.mass), table, ln, 5, 1)
    with pytest.raises(TypeError):
        ops.kv_read(cache.blocks, table, cu, ln, 2)
    with pytest.raises(ValueError):
        ops.kv_read(cache, table, cu, ln, 2, torch.float64)
    with pytest.raises(ValueError):
        ops.kv_read(cache, table, cu, ln, -1)
    if dev == "cuda":
        with pytest.raises(RuntimeError, match="bf16 or f16"):
            ops.paged_attention(q.float(), cache, table, cu, ln, 2)
        with pytest.raises(RuntimeError, match="int32"):
            ops.paged_attention(q, cache, table.long(), cu, ln, 2)
        with pytest.raises(RuntimeError, match="mass"):
            ops.paged_attention(q, ops.PagedKV4(cache.blocks, cache.mass.half()), table, cu, ln, 2)
        with pytest.raises(RuntimeError, match="one GPU"):
            ops.kv_evict(cache, table.cpu(), ln, 5, 1)
        with pytest.raises(RuntimeError, match="pages of"):
            ops.paged_attention(q, ops.PagedKV4(cache.blocks[:3].reshape(1, 2, 3, -1)), table, cu, ln, 2)


@pytest.mark.gpu
def test_bad_pages_lengths_and_positions_are_reported():
    from mamformer_b200.fault import PagedCacheError, check_device_status
    check_device_status()
    cache, table = filled([40, 90], 16, 2, 64, "cuda")
    P = cache.blocks.shape[0]
    k, q = rand((2, 2, 64), torch.bfloat16, "cuda", 1), rand((2, 4, 64), torch.bfloat16, "cuda", 1)
    cu, ln = offsets([1, 1], "cuda"), i32([40, 90], "cuda")
    whole = cache.blocks.clone()
    good = ops.paged_attention(q, cache, table, cu, ln, 1)

    def raises(what):
        with pytest.raises(PagedCacheError, match=what):
            check_device_status()
        check_device_status()

    for page in (-1, P, 1 << 30):
        t = table.clone()
        t[0, 2] = page
        ops.kv_append(k[:1], k[:1], cache, t, offsets([1, 0], "cuda"), ln, 1)
        raises("page")
        assert torch.equal(cache.blocks, whole)
        got = ops.paged_attention(q, cache, t, cu, ln, 1)
        raises("page")
        assert got.isfinite().all() and torch.equal(got[1], good[1])
        got = ops.paged_attention(rand((90, 4, 64), torch.bfloat16, "cuda", 1), cache, t, offsets([40, 50], "cuda"), ln, 50)
        raises("page")
        assert got.isfinite().all()
        ops.kv_read(cache, t, offsets([40, 0], "cuda"), ln, 40)
        raises("page")
        c = ops.PagedKV4(cache.blocks.clone(), cache.mass.clone())
        ops.kv_evict(c, t, ln, 36, 20)
        raises("page")
    # lengths below the new tokens, and beyond the table
    for lens in ([-3, 90], [0, 90], [1000, 90], [(1 << 31) - 1, 90]):
        ops.kv_append(k, k, ops.PagedKV4(cache.blocks.clone()), table, cu, i32(lens, "cuda"), 1)
        raises("length|page")
    for lens in ([-3, 90], [1000, 90], [(1 << 31) - 1, 90]):
        got = ops.paged_attention(q, cache, table, cu, i32(lens, "cuda"), 1)
        with pytest.raises(PagedCacheError):
            check_device_status()
        assert torch.equal(got[1], good[1])
        ops.kv_evict(ops.PagedKV4(cache.blocks.clone(), cache.mass.clone()), table, i32(lens, "cuda"), 36, 20)
        with pytest.raises(PagedCacheError):
            check_device_status()
    # offsets that fall, or run past the queries
    q = rand((600, 4, 64), torch.bfloat16, "cuda", 4)
    for off in ([0, 5, 3], [0, 2, 900], [-5, 0, 9], [0, 200, 100]):
        for max_new in (2, 40, 200):
            got = ops.paged_attention(q, cache, table, i32(off, "cuda"), ln, max_new)
            assert got.isfinite().all() and (max_new == 200 or (got == 0).all())
            raises("lengths")
        kv = rand((600, 2, 64), torch.bfloat16, "cuda", 4)
        ops.kv_append(kv, kv, ops.PagedKV4(cache.blocks.clone()), table, i32(off, "cuda"), ln, 200)
        with pytest.raises(PagedCacheError):
            check_device_status()
    cos, sin = rotation(10, 64, "cuda")
    ops.kv_append(k, k, ops.PagedKV4(cache.blocks.clone()), table, cu, ln, 1, cos, sin, torch.tensor([3, 10], device="cuda"), [])
    raises("position")


@pytest.mark.gpu
@pytest.mark.parametrize("diff", [False, True])
@pytest.mark.parametrize("new,lens", [([1, 2], [60000, 70]), ([200], [9000]), ([90, 1], [2000, 300]), ([2000], [2000])])
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
    cache.mass.zero_()
    had = C.paged_attention_wait_limit(-1)
    try:
        got = run()
        torch.cuda.synchronize()
    finally:
        C.paged_attention_wait_limit(had)
    assert (got == 0).all() and (cache.mass == 0).all()
    with pytest.raises(KernelTimeoutError):
        check_device_status()
    check(q, cache, table, new, lens, **kw)
    check_device_status()


# ---- streams, graphs, devices of calls -----------------------------------------------------------------
@pytest.mark.gpu
def test_streams_and_graphs():
    lens, G, hd, page = [70, 300, 33], 2, 128, 16
    cache, table = filled(lens, page, G, hd, "cuda")
    cache.mass.zero_()
    q = rand((3, 8, hd), torch.bfloat16, "cuda", 1)
    k = rand((3, G, hd), torch.bfloat16, "cuda", 2)
    cu, ln = offsets([1, 1, 1], "cuda"), i32(lens, "cuda")
    t, extra = tables([32] * 3, page, "cuda", 4)
    P = cache.blocks.shape[0]
    cache = ops.PagedKV4(torch.cat([cache.blocks, pool(extra, G, page, hd, "cuda").blocks]), torch.cat([cache.mass, torch.zeros(extra, G, page, device="cuda")]))
    to = t + P

    def step():
        ops.kv_append(k, k, cache, table, cu, ln, 1)
        out = ops.paged_attention(q, cache, table, cu, ln, 1)
        kept, left = ops.kv_evict(cache, table, ln, 32, 4, out_table=to)
        return out, kept, left, *ops.kv_read(cache, to, cu32, left, 96)

    cu32 = offsets([32] * 3, "cuda")
    start = cache.mass.clone()
    want = [x.clone() for x in step()]
    mass = cache.mass.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cache.mass.copy_(start)
        for a, b in zip(step(), want):
            assert torch.equal(a, b)
        cache.mass.copy_(start)
        graphs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
        outs = []
        for g in graphs:
            with torch.cuda.graph(g, stream=side):
                outs.append(step())
        for g, o in zip(graphs * 2, outs * 2):
            cache.mass.copy_(start)
            g.replay()
            for a, b in zip(o, want):
                assert torch.equal(a, b)
            assert torch.equal(cache.mass, mass)
    torch.cuda.current_stream().wait_stream(side)


@pytest.mark.gpu
def test_blocks_past_31_bits():
    """A pool whose last pages start past 2^31 bytes."""
    page, G, hd = 128, 8, 128
    P = (1 << 31) // (G * page // 16 * 18 * hd) + 40
    blocks = torch.empty(P, G, page // 16, 18 * hd, dtype=torch.uint8, device="cuda")
    mass = torch.empty(P, G, page, device="cuda")
    cache = ops.PagedKV4(blocks, mass)
    lens = [1000, 77]
    small, st = filled(lens, page, G, hd, "cuda")
    table = torch.full_like(st, -1)
    high = iter(range(P - 20, P))
    for b, n in enumerate(lens):
        for j in range(-(-n // page)):
            p = next(high)
            table[b, j] = p
            blocks[p], mass[p] = small.blocks[st[b, j]], 0.0
    for new in ([1, 1], [200, 30]):
        q = rand((sum(new), 16, hd), torch.bfloat16, "cuda", 1)
        want, tol, m, mt = plain(q, small, st, new, lens)
        mass[P - 20:] = 0.0
        close(ops.paged_attention(q, cache, table, offsets(new, "cuda"), i32(lens, "cuda"), max(new)), want, tol)
        for b, n in enumerate(lens):
            used = -(-n // page)
            close(mass[table[b, :used].long()], m[st[b, :used].long()], mt[st[b, :used].long()])
    kept, left = ops.kv_evict(cache, table, i32(lens, "cuda"), 64, 8)
    k, v = ops.kv_read(cache, table, offsets([64, 64], "cuda"), left, 128, torch.float32)
    ks, vs = held(small, st, lens, 0)
    for g in range(G):
        assert torch.equal(k[:64, g].double(), ks[g][kept[0, g].long()]) and torch.equal(v[:64, g].double(), vs[g][kept[0, g].long()])

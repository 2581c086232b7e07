"""ops.token_scores and ops.token_log_probs where they can go wrong: derivatives of other kinds than one backward pass,
function transforms, targets outside the vocabulary, shapes.

Tolerances: fp32 results of a few hundred terms of size 1, each to 2^-22: 1e-5."""

import math

import pytest
import torch
import torch.autograd.forward_ad as fwd

from mamformer_b200 import ops

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def rows(dev, R=5, V=300, dtype=torch.float32, seed=1):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(R, V, generator=g).to(dtype).to(dev)
    t = torch.randint(0, V, (R,), generator=g).to(dev)
    return x, t, torch.randn(R, V, generator=g).to(dtype).to(dev)


def plain_log_probs(x, t):
    return torch.log_softmax(x.double(), -1).gather(-1, t[..., None])[..., 0]


def near(a, b):
    assert a.shape == b.shape and ((a.double() - b.double()).abs() <= 1e-5).all()


@pytest.mark.parametrize("dev", DEVICES)
def test_forward_mode_derivatives(dev):
    x, t, dx = rows(dev)
    p = torch.softmax(x.double(), -1)
    want = dx.double().gather(-1, t[:, None])[:, 0] - (p * dx).sum(-1)
    lp = torch.log_softmax(x.double(), -1)
    want_ent = -(p * (dx - (p * dx).sum(-1, keepdim=True)) * (lp + 1)).sum(-1)
    with fwd.dual_level():
        d = fwd.make_dual(x, dx)
        near(fwd.unpack_dual(ops.token_log_probs(d, t)).tangent, want)
        s = ops.token_scores(d, t, top_k=2)
        near(fwd.unpack_dual(s.log_probs).tangent, want)
        near(fwd.unpack_dual(s.entropy).tangent, want_ent)
        near(ops.token_log_probs(x, t), plain_log_probs(x, t))
    out, tangent = torch.func.jvp(lambda z: ops.token_log_probs(z, t), (x,), (dx,))
    near(out, plain_log_probs(x, t))
    near(tangent, want)


@pytest.mark.parametrize("dev", DEVICES)
def test_function_transforms(dev):
    x, t, _ = rows(dev)
    near(torch.func.vmap(ops.token_log_probs)(x, t), plain_log_probs(x, t))
    near(torch.func.vmap(lambda a, b: ops.token_scores(a, b, top_k=3).log_probs)(x, t), plain_log_probs(x, t))
    got = torch.func.grad(lambda z: ops.token_log_probs(z, t).sum())(x)
    want, = torch.autograd.grad(plain_log_probs(z := x.double().requires_grad_(True), t).sum(), z)
    near(got, want)
    h = torch.func.hessian(lambda z: ops.token_log_probs(z, t[:1]).sum())(x[:1, :20].contiguous().clamp(-2, 2)) \
        if t[0] < 20 else torch.func.hessian(lambda z: ops.token_log_probs(z, t[:1] * 0).sum())(x[:1, :20].contiguous())
    assert h.shape == (1, 20, 1, 20) and h.isfinite().all() and h.abs().max() > 0


@pytest.mark.parametrize("dev", DEVICES)
def test_paged_operators_refuse_tangents_and_transforms(dev):
    from test_paged_cache import filled, i32, offsets
    cache, table = filled([5], 16, 1, 64, dev)
    q = torch.ones(1, 2, 64, dtype=torch.bfloat16, device=dev)
    k = torch.ones(1, 1, 64, dtype=torch.bfloat16, device=dev)
    args = cache, table, offsets([1], dev), i32([5], dev), 1
    with fwd.dual_level():
        ops.paged_attention(q, *args)
        with pytest.raises(RuntimeError, match="no gradient"):
            ops.paged_attention(fwd.make_dual(q, q), *args)
        with pytest.raises(RuntimeError, match="no gradient"):
            ops.kv_append(fwd.make_dual(k, k), k, *args)
    with pytest.raises(RuntimeError, match="no gradient"):
        torch.func.vmap(lambda x: ops.paged_attention(x, *args))(q[None])


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_second_derivatives_of_log_probs(dev, dtype):
    x, t, w = rows(dev, dtype=dtype)
    t[2] = -100
    g = torch.linspace(-1, 2, 5, device=dev)

    def second(x, g, w, f, live):
        d, = torch.autograd.grad(f(x)[live], x, g[live], create_graph=True)
        return d, *torch.autograd.grad((d * w).sum(), (x, g))

    live = t != -100
    got = second(x.clone().requires_grad_(True), g.clone().requires_grad_(True), w, lambda z: ops.token_log_probs(z, t), live)
    want = second(x.double().requires_grad_(True), g.double().requires_grad_(True), w.double(),
                  lambda z: plain_log_probs(z, t.clamp(min=0)), live)
    # bf16: the first gradient is rounded once (2^-8 of itself), and so is the second; their sums over w see sqrt(300) of those
    for a, b in zip(got, want):
        unit = 1e-5 if dtype == torch.float32 else 2.0 ** -7
        assert ((a.double() - b).abs() <= unit * (1 + b.abs())).all()


@pytest.mark.parametrize("dev", DEVICES)
def test_third_derivative_of_log_probs(dev):
    x, t, w = rows(dev, R=2, V=9)

    def third(x, f):
        for _ in range(3):
            x_, = torch.autograd.grad(f, x, create_graph=True)
            f = (x_ * w.to(x.dtype)).sum()
        return x_

    a = x.clone().requires_grad_(True)
    b = x.double().requires_grad_(True)
    near(third(a, ops.token_log_probs(a, t).sum()), third(b, plain_log_probs(b, t).sum()))


@pytest.mark.parametrize("dev", DEVICES)
def test_targets_of_another_shape_or_type_are_refused(dev):
    x = torch.randn(2, 3, 11, device=dev)
    for shape in ((6,), (3, 2), (2, 3, 1), (1, 3), ()):
        for f in (ops.token_log_probs, ops.token_scores):
            with pytest.raises(ValueError):
                f(x, torch.zeros(shape, dtype=torch.long, device=dev))
    for f in (ops.token_log_probs, ops.token_scores):
        with pytest.raises(ValueError):
            f(x, torch.zeros(2, 3, device=dev))


@pytest.mark.parametrize("dev", DEVICES)
def test_targets_outside_the_vocabulary_are_not_silent(dev):
    """NaN in that row, no gradient from it, and on the GPU an error word."""
    from mamformer_b200.fault import TargetRangeError, check_device_status
    check_device_status()
    x, t, _ = rows(dev)
    good = ops.token_scores(x, t, top_k=2)
    for bad in (300, -1, 1 << 40):
        t2 = t.clone()
        t2[3] = bad
        x.requires_grad_(True)
        s = ops.token_scores(x, t2, top_k=2)
        assert s.log_probs[3].isnan() and s.entropy[3].isnan() and s.top_log_probs[3].isnan().all() and (s.top_ids[3] == -1).all()
        keep = [0, 1, 2, 4]
        for a, b in zip(s, good):
            assert torch.equal(a[keep], b[keep])
        d, = torch.autograd.grad(s.log_probs[keep].sum(), x)
        assert (d[3] == 0).all() and d.isfinite().all()
        x.requires_grad_(False)
        if dev == "cuda":
            with pytest.raises(TargetRangeError, match="vocabulary"):
                check_device_status()
            assert ops.token_log_probs(x.double(), t2)[3].isnan()
            assert ops.token_log_probs(x, t2)[3].isnan()
            with pytest.raises(TargetRangeError, match="vocabulary"):
                check_device_status()
        else:
            with pytest.raises((RuntimeError, IndexError)):
                ops.token_log_probs(x, t2)
    t[1] = -100
    assert ops.token_scores(x, t).log_probs[1] == 0
    check_device_status()


@pytest.mark.parametrize("dev", DEVICES)
def test_temperatures_at_the_ends_of_their_range(dev):
    """Very cold: all weight on the largest logit; very hot: all that are not -inf alike, those of -inf still nothing."""
    x, t, _ = rows(dev, R=3, V=700)
    x[:, 5] = 9.0
    x[:, 100:110] = -math.inf
    t[:] = 5
    cold = ops.token_scores(x, t, top_k=2, temperature=1e-30)
    assert (cold.log_probs == 0).all() and (cold.entropy.abs() < 1e-6).all() and (cold.top_ids[:, 0] == 5).all()
    hot = ops.token_scores(x, t, temperature=1e27)
    near(hot.log_probs, torch.full((3,), -math.log(690), device=dev))
    near(hot.entropy, torch.full((3,), math.log(690), device=dev))
    for bad in (1e-31, 1e-45, 1e28, math.inf):
        with pytest.raises(ValueError):
            ops.token_scores(x, t, temperature=bad)

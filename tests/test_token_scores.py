"""ops.token_scores (csrc/token_scores.cu on CUDA, the eager form on CPU) against its definition in 64 bits: log
probabilities, entropies, alternatives and gradients, for vocabularies around the vector and segment sizes, every
type, strided rows, ignored rows, masked logits, and the refusals.

Tolerances, from the arithmetic: exp is good to 2 units in fp32's last place (2^-22), and a thread adds at most V / 512
terms to a running sum, so the two sums are off by c = (V / 512 + 40) 2^-24 relatively; a log probability by c plus
three roundings of itself; the entropy by c (1 + H + log V); a gradient by its type's rounding plus c times the size
of its terms."""

import math

import pytest
import torch

from mamformer_b200 import ops

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
ROUND = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}      # half a step, relative


def plain(x, t, k, T, ignore=-100):
    """(log_probs, entropy, top_log_probs, top_ids) in 64 bits, differentiable."""
    x = x.double()
    live = t != ignore
    lp = torch.log_softmax(x / T, -1)
    p = lp.exp()
    ent = -torch.where(p > 0, p * lp.clamp(min=-1e300), 0.0).sum(-1)
    ids = torch.sort(x.detach(), dim=-1, descending=True, stable=True).indices[..., :k]
    got = lp.gather(-1, t.clamp(min=0).unsqueeze(-1)).squeeze(-1)
    return (torch.where(live, got, 0.0), torch.where(live, ent, 0.0),
            torch.where(live.unsqueeze(-1), lp.gather(-1, ids), 0.0), torch.where(live.unsqueeze(-1), ids, -1))


def close(got, want, tol):
    assert got.shape == want.shape
    bad = (got.double() - want).abs() > tol
    assert not bad.any(), ((got.double() - want).abs()[bad].max(), bad.sum())


def c_of(V):
    return (V / 512 + 40) * 2.0 ** -24


def check(x, t, k, T, dev):
    s = ops.token_scores(x, t, top_k=k, temperature=T)
    lp, ent, top, ids = plain(x, t, k, T)
    V = x.shape[-1]
    c = c_of(V)
    assert s.log_probs.dtype == s.entropy.dtype == s.top_log_probs.dtype == torch.float32
    close(s.log_probs, lp, c + 3 * 2.0 ** -24 * lp.abs())
    close(s.entropy, ent, c * (1 + ent.abs() + math.log(V)))
    assert torch.equal(s.top_ids, ids)
    close(s.top_log_probs, top, c + 3 * 2.0 ** -24 * top.abs())
    return s


def logits(shape, dtype, dev, seed, scale=3.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype).to(dev)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("V,k", [(1, 1), (2, 1), (7, 7), (33, 32), (300, 5), (1000, 20), (4099, 32), (8191, 8),
                                 (16384, 0), (16385, 3), (33000, 17)])
def test_forward_matches_64_bits(dev, dtype, V, k):
    x = logits((5, V), dtype, dev, V)
    t = torch.arange(5, device=dev) * 7919 % V
    t[3] = -100
    check(x, t, k, 0.7, dev)


@pytest.mark.gpu
@pytest.mark.parametrize("R", [1, 3, 40, 160, 700])
@pytest.mark.parametrize("V", [8192, 64003, 65536])
def test_forward_for_few_and_many_rows(R, V):
    x = logits((R, V), torch.bfloat16, "cuda", R + V)
    check(x, torch.arange(R, device="cuda") * 104729 % V, 9, 1.0, "cuda")


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("V", [1, 5, 300, 4099, 16384, 17001])
@pytest.mark.parametrize("with_top", [False, True])
def test_gradient_matches_the_formula(dev, dtype, V, with_top):
    k, T = min(4, V), 1.3
    x = logits((2, 3, V), dtype, dev, V + 1).requires_grad_(True)
    t = (torch.arange(6, device=dev) * 31 % V).view(2, 3)
    t[1, 1] = -100
    s = ops.token_scores(x, t, top_k=k, temperature=T)
    g = torch.Generator().manual_seed(5)
    gl, ge, gt = (torch.randn(*o.shape, generator=g).to(dev) for o in (s.log_probs, s.entropy, s.top_log_probs))
    outs, grads = ([s.log_probs, s.entropy], [gl, ge])
    x64 = x.detach().double().requires_grad_(True)
    w = plain(x64, t, k, T)
    want_o = list(w[:2])
    if with_top:
        outs.append(s.top_log_probs), grads.append(gt), want_o.append(w[2])
    got, = torch.autograd.grad(outs, x, grads)
    want, = torch.autograd.grad(want_o, x64, [v.double() for v in grads])
    assert got.dtype == dtype and got.shape == x.shape
    size = gl.abs() + (gt.abs().sum(-1) if with_top else 0) + ge.abs() * (2 + 2 * math.log(V + 1))
    close(got, want, ROUND[dtype] * want.abs() + (c_of(V) + 2.0 ** -19) * size.unsqueeze(-1) + (2.0 ** -25 if dtype == torch.float16 else 0))
    assert (got[1, 1] == 0).all()


@pytest.mark.parametrize("dev", DEVICES)
def test_gradient_matches_differences(dev):
    """Central differences of the 64-bit definition, step 1e-4: error 1e-8 / 6 times the third derivative (< 10)."""
    x = logits((3, 50), torch.float32, dev, 3).requires_grad_(True)
    t = torch.tensor([4, 49, 0], device=dev)
    s = ops.token_scores(x, t, top_k=2, temperature=0.9)
    got, = torch.autograd.grad(s.log_probs.sum() + 0.5 * s.entropy.sum() + 0.25 * s.top_log_probs.sum(), x)

    def value(z):
        lp, ent, top, _ = plain(z, t, 2, 0.9)
        return lp + 0.5 * ent + 0.25 * top.sum(-1)

    base = x.detach().double()
    for j in range(50):
        d = torch.zeros_like(base)
        d[:, j] = 1e-4
        diff = (value(base + d) - value(base - d)) / 2e-4
        assert ((got[:, j].double() - diff).abs() < 1e-5).all()


@pytest.mark.parametrize("dev", DEVICES)
def test_one_missing_gradient(dev):
    x = logits((4, 1000), torch.float32, dev, 8).requires_grad_(True)
    t = torch.tensor([1, 2, -100, 999], device=dev)
    for pick in (0, 1):
        got, = torch.autograd.grad(ops.token_scores(x, t)[pick].sum(), x)
        x64 = x.detach().double().requires_grad_(True)
        want, = torch.autograd.grad(plain(x64, t, 0, 1.0)[pick].sum(), x64)
        close(got, want, ROUND[torch.float32] * want.abs() + c_of(1000) * 16)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_masked_logits(dev, dtype):
    V, low = 5000, torch.finfo(dtype).min
    x = logits((7, V), dtype, dev, 11)
    t = torch.full((7,), 17, device=dev)
    x[0, 100:] = -math.inf                    # a constrained vocabulary
    x[1, 100:] = low
    x[2] = -math.inf                          # nothing is allowed
    x[3] = low                                # everything equally unlikely
    x[4, 17] = -math.inf                      # the target is not allowed
    x[5, :] = -math.inf
    x[5, 4321] = 2.0                          # one token left
    x[6] = 0.25                               # all equal
    x.requires_grad_(True)
    s = ops.token_scores(x, t, top_k=6, temperature=0.5)
    assert not s.log_probs.isnan().any() and not s.entropy.isnan().any() and not s.top_log_probs.isnan().any()
    uniform = -math.log(V)
    assert s.log_probs[2] == -math.inf and s.entropy[2] == 0 and (s.top_log_probs[2] == -math.inf).all()
    assert s.log_probs[4] == -math.inf and s.log_probs[5] == -math.inf and abs(s.entropy[5]) < 1e-6
    for r in (3, 6):
        assert abs(s.log_probs[r] - uniform) < 1e-5 and abs(s.entropy[r] + uniform) < 1e-5
        assert s.top_ids[r].tolist() == list(range(6))
    assert s.top_ids[2].tolist() == list(range(6))
    assert s.top_ids[5].tolist() == [4321, 0, 1, 2, 3, 4] and s.top_log_probs[5, 0] == 0 and s.top_log_probs[5, 1] == -math.inf
    rows = torch.tensor([0, 4], device=dev)
    lp, ent, top, ids = plain(x.detach()[rows], t[rows], 6, 0.5)
    assert torch.equal(s.top_ids[rows], ids)
    close(s.entropy[rows], ent, c_of(V) * 20)
    close(s.log_probs[0], lp[0], c_of(V) + 3 * 2.0 ** -24 * lp[0].abs())
    got, = torch.autograd.grad((s.log_probs[[0, 1, 3, 6]].sum() + s.entropy.sum()), x)
    assert got.isfinite().all() and (got[2] == 0).all() and (got[0, 100:] == 0).all() and (got[1, 100:] == 0).all()


@pytest.mark.parametrize("dev", DEVICES)
def test_nan_and_infinity_reach_the_result(dev):
    x = logits((3, 700), torch.float32, dev, 2)
    x[0, 3], x[1, 650] = math.nan, math.inf
    s = ops.token_scores(x, torch.tensor([5, 6, 7], device=dev))
    assert s.log_probs[:2].isnan().all() and s.entropy[:2].isnan().all() and s.log_probs[2].isfinite()


@pytest.mark.parametrize("dev", DEVICES)
def test_ties_and_candidates_in_one_place(dev):
    """Alternatives that all fall to one thread, and more equal logits than are kept as candidates."""
    V = 20000
    x = logits((4, V), torch.bfloat16, dev, 4, scale=0.1)
    x[0, 8:16] = 5.0
    x[0, 4096 + 8:4096 + 16] = 5.0
    x[1, 3000:9000] = 7.0
    x[2, ::2] = 1.5
    x[3] = torch.linspace(9, -9, V).bfloat16().to(dev)
    check(x, torch.zeros(4, dtype=torch.long, device=dev), 20, 1.0, dev)


@pytest.mark.gpu
def test_negative_zero_is_zero():
    x = torch.full((1, 3000), -1.0, device="cuda")
    x[0, 7], x[0, 2], x[0, 2999] = 0.0, -0.0, 0.0
    assert ops.token_scores(x, torch.tensor([7], device="cuda"), top_k=4).top_ids.tolist() == [[2, 7, 2999, 0]]


@pytest.mark.parametrize("dev", DEVICES)
def test_strided_rows(dev):
    base = logits((3, 6, 1003), torch.bfloat16, dev, 9)
    t = torch.arange(15, device=dev).view(3, 5)
    check(base[:, :-1], t, 4, 1.0, dev)
    check(base[:, 1:, 1:], t, 4, 1.0, dev)                         # rows off the 16-byte grid
    check(base.transpose(0, 1)[:5], t.T, 4, 1.0, dev)
    check(base[..., ::2][:, :5], t, 4, 1.0, dev)
    check(base.view(3, 2, 3, 1003)[:, :, :2], t[:, :4].reshape(3, 2, 2), 2, 1.0, dev)
    x = base.detach().clone().requires_grad_(True)
    got, = torch.autograd.grad(ops.token_scores(x[:, :-1], t).log_probs.sum(), x)
    x64 = x.detach().double().requires_grad_(True)
    want, = torch.autograd.grad(plain(x64[:, :-1], t, 0, 1.0)[0].sum(), x64)
    close(got, want, ROUND[torch.bfloat16] * want.abs() + 1e-5)


@pytest.mark.parametrize("dev", DEVICES)
def test_no_rows_and_scalar_target(dev):
    s = ops.token_scores(torch.zeros(0, 9, device=dev), torch.zeros(0, dtype=torch.long, device=dev), top_k=2)
    assert s.log_probs.shape == (0,) and s.top_ids.shape == (0, 2)
    s = ops.token_scores(torch.zeros(9, device=dev), torch.tensor(4, device=dev), top_k=1)
    assert s.log_probs.shape == () and abs(s.entropy - math.log(9)) < 1e-6 and s.top_ids.tolist() == [0]


@pytest.mark.parametrize("dev", DEVICES)
def test_refusals(dev):
    x, t = torch.zeros(4, 10, device=dev), torch.zeros(4, dtype=torch.long, device=dev)
    for kw in ({"top_k": 33}, {"top_k": 11}, {"top_k": -1}, {"temperature": 0.0}, {"temperature": -1.0},
               {"temperature": math.nan}):
        with pytest.raises(ValueError):
            ops.token_scores(x, t, **kw)
    with pytest.raises(ValueError):
        ops.token_scores(x, t[:3])


def test_native_refusals_that_name_a_number_raise():
    """An error message with a number in it is an exception and does not end the process."""
    from mamformer_b200.ops._ext import ext
    if ext() is None:
        pytest.skip("native extension not built")
    with pytest.raises(RuntimeError, match="got -2"):
        ext().token_scores_fwd(torch.zeros(2, 3), torch.zeros(2, dtype=torch.long), -100, -2.0, 0)


@pytest.mark.gpu
def test_refusal_of_targets_elsewhere():
    with pytest.raises(RuntimeError, match="one GPU"):
        ops.token_scores(torch.zeros(4, 10, device="cuda"), torch.zeros(4, dtype=torch.long))


@pytest.mark.gpu
def test_another_stream_and_repeatability():
    x = logits((64, 32000), torch.bfloat16, "cuda", 1)
    t = torch.arange(64, device="cuda")
    first = ops.token_scores(x, t, top_k=8)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = ops.token_scores(x, t, top_k=8)
    s.synchronize()
    for a, b in zip(first, other):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dev", DEVICES)
def test_token_log_probs_unchanged_for_other_types(dev):
    x, t = logits((3, 77), torch.float64, dev, 6), torch.tensor([0, 5, 76], device=dev)
    close(ops.token_log_probs(x, t), plain(x, t, 0, 1.0)[0], 1e-5)


@pytest.mark.gpu
def test_kept_graph_and_second_derivative():
    """A graph may be kept and its first gradient used; the gradient itself is not differentiable."""
    x = logits((3, 40), torch.float32, "cuda", 3).requires_grad_(True)
    t = torch.tensor([1, 2, 3], device="cuda")
    s = ops.token_scores(x, t)
    a, = torch.autograd.grad(s.log_probs.sum(), x, retain_graph=True)
    b, = torch.autograd.grad(s.log_probs.sum(), x, create_graph=True)
    assert torch.equal(a, b) and b.requires_grad
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(b.sum(), x)
    assert not s.top_ids.requires_grad and not ops.token_scores(x.detach(), t).log_probs.requires_grad

"""Hot-op dispatch: native sm_100a kernels for CUDA tensors, PyTorch reference math on CPU.

Every public function here is differentiable.  For CUDA tensors it calls the in-tree
extension ``mamformer_b200._C`` (built by ``setup.py build_ext --inplace`` or
``__graft_entry__.build()``); if that extension is missing on a machine with a GPU the call
raises instead of silently running PyTorch code.  CPU tensors always take the reference path
(``ops.reference``), which is also the numerics oracle in the tests.

``NATIVE`` lists the ops that have a native kernel; ops not listed run composite PyTorch on
CUDA too (each is a documented gap).
"""

from __future__ import annotations

import math
import os
from typing import List, NamedTuple, Optional, Sequence, Tuple, Union

import torch
import torch.autograd.forward_ad as forward_ad
import torch.nn.functional as F

from mamformer_b200.ops import reference as ref
from mamformer_b200.ops._ext import ext, has_native, require_native

__all__ = [
    "rms_norm", "rope", "swiglu", "causal_conv1d_silu", "selective_scan", "mamba_inner",
    "linear_diff_attention", "diff_attention", "attention", "head_group_norm", "router_topk",
    "expert_histogram", "moe_routed", "moe_expert_outputs", "linear_cross_entropy",
    "fused_ce_available", "token_log_probs", "token_scores", "TokenScores", "PagedKV", "PagedKV4", "kv_append",
    "kv_read", "paged_attention", "kv_evict",
    "NATIVE", "has_native", "force_reference",
]

# Native-kernel coverage (op name -> kernel source file).  Filled by ops.native on import.
NATIVE: dict = {}

_FORCE_REF = os.environ.get("MAMF_FORCE_REFERENCE", "0") == "1"


def force_reference() -> bool:
    """True when MAMF_FORCE_REFERENCE=1 sends every CUDA op to its eager PyTorch form (for A/B
    debugging only; benchmarks refuse to run in this mode)."""
    return _FORCE_REF


def _native(t: torch.Tensor) -> bool:
    """True when this call should take the native path (CUDA tensor).  Raises if the
    extension is absent on CUDA, unless MAMF_FORCE_REFERENCE=1 (debug / A-B only)."""
    if not t.is_cuda or _FORCE_REF:
        return False
    require_native()
    return True


_NATIVE_MODULE = None


def _nat():
    global _NATIVE_MODULE
    if _NATIVE_MODULE is None:
        from mamformer_b200.ops import native
        _NATIVE_MODULE = native
    return _NATIVE_MODULE


# ---------------------------------------------------------------------------------------------
def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float) -> torch.Tensor:
    if _native(x) and "rms_norm" in NATIVE:
        return _nat().rms_norm(x, weight, eps)
    return ref.rms_norm(x, weight, eps)


def rope(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    """x (B, S, H, hd); cos/sin (S, hd/2) fp32 -> rotated copy."""
    if _native(x) and "rope" in NATIVE:
        return _nat().rope(x, cos, sin)
    return ref.rope(x, cos, sin)


def swiglu(gate: torch.Tensor, up: torch.Tensor) -> torch.Tensor:
    if _native(gate) and "swiglu" in NATIVE:
        return _nat().swiglu(gate, up)
    return ref.swiglu(gate, up)


def causal_conv1d_silu(x: torch.Tensor, weight: torch.Tensor) -> torch.Tensor:
    """silu(depthwise causal conv(x)); x (B, S, C) (may be a strided view), weight (C, K)."""
    if _native(x) and "causal_conv1d_silu" in NATIVE:
        return _nat().causal_conv1d_silu(x, weight)
    return F.silu(ref.causal_conv1d(x, weight))


def selective_scan(x, dt, A_log, B, C, D, return_h_states=False, return_final_state=False):
    """Reference-signature scan (dt already positive)."""
    if _native(x) and "selective_scan" in NATIVE:
        return _nat().selective_scan(x, dt, A_log, B, C, D, return_h_states, return_final_state)
    return ref.selective_scan(x, dt, A_log, B, C, D, return_h_states, return_final_state)


def mamba_inner(x_act, dt_raw, A_log, Bm, Cm, D, z, need_h_states: bool,
                return_final: bool = False):
    """softplus(dt_raw) -> scan -> y*silu(z).  Returns (y_gated, h_states|None, final|None)."""
    if _native(x_act) and "mamba_inner" in NATIVE:
        return _nat().mamba_inner(x_act, dt_raw, A_log, Bm, Cm, D, z, need_h_states, return_final)
    return ref.mamba_inner(x_act, dt_raw, A_log, Bm, Cm, D, z, need_h_states, return_final=return_final)


def linear_diff_attention(q1, q2, k, v, lam, kernel_dim: int, chunk: int = 256):
    if _native(q1) and "linear_diff_attention" in NATIVE:
        return _nat().linear_diff_attention(q1, q2, k, v, lam, kernel_dim)
    return ref.linear_diff_attention(q1, q2, k, v, lam, kernel_dim, chunk)


def _window_bounds(window: int, window_mode: str):
    """(lo, hi) on (key - query) for same-length self-attention, causal included."""
    if window <= 0:
        return -(1 << 30), 0
    if window_mode == "reference":
        return 0, 0           # causal AND 0 <= k - q < W  ->  diagonal only
    return -(window - 1), 0   # causal sliding window


def diff_attention(q1, q2, k, v, lam, window: int = 0, window_mode: str = "reference",
                   attention_mask: Optional[torch.Tensor] = None, scale: Optional[float] = None):
    same_len = q1.shape[1] == k.shape[1]
    if _native(q1) and "diff_attention" in NATIVE and attention_mask is None and same_len:
        lo, hi = _window_bounds(window, window_mode)
        return _nat().diff_attention(q1, q2, k, v, lam, lo, hi, scale)
    if window > 0 and window_mode == "causal":
        return _causal_window_diff(q1, q2, k, v, lam, window, attention_mask, scale)
    return ref.diff_attention(q1, q2, k, v, lam, window, True, scale, attention_mask)


def _causal_window_diff(q1, q2, k, v, lam, window, attention_mask, scale):
    S, Skv = q1.shape[1], k.shape[1]
    off = Skv - S
    iq = torch.arange(S, device=q1.device).unsqueeze(1) + off
    ik = torch.arange(Skv, device=q1.device).unsqueeze(0)
    valid = (ik <= iq) & (iq - ik < window)
    m = torch.zeros(S, Skv, device=q1.device, dtype=q1.dtype).masked_fill(~valid, float("-inf"))
    if attention_mask is not None:
        m = m + attention_mask
    return ref.diff_attention(q1, q2, k, v, lam, 0, False, scale, m)


def attention(q, k, v, window: int = 0, window_mode: str = "reference",
              attention_mask: Optional[torch.Tensor] = None, dropout_p: float = 0.0):
    """GQA softmax attention, reference masking semantics (see models.attention)."""
    same_len = q.shape[1] == k.shape[1]
    native_ok = attention_mask is None and same_len and dropout_p == 0.0
    if _native(q) and "attention" in NATIVE and native_ok:
        if window > 0 and window_mode == "reference":
            lo, hi = 0, window - 1          # reference GQA window: 0 <= key - query < W, no causal mask
        else:
            lo, hi = _window_bounds(window, window_mode)
        return _nat().attention(q, k, v, lo, hi)
    if window > 0 and window_mode == "causal":
        S, Skv = q.shape[1], k.shape[1]
        iq = torch.arange(S, device=q.device).unsqueeze(1) + (Skv - S)
        ik = torch.arange(Skv, device=q.device).unsqueeze(0)
        valid = (ik <= iq) & (iq - ik < window)
        m = torch.zeros(S, Skv, device=q.device, dtype=q.dtype).masked_fill(~valid, float("-inf"))
        return ref.sdpa_attention(q, k, v, 0, m if attention_mask is None else m + attention_mask, dropout_p)
    return ref.sdpa_attention(q, k, v, window, attention_mask, dropout_p)


def head_group_norm(x: torch.Tensor, n_heads: int, weight: torch.Tensor, bias: torch.Tensor,
                    eps: float) -> torch.Tensor:
    if _native(x) and "head_group_norm" in NATIVE:
        return _nat().head_group_norm(x, n_heads, weight, bias, eps)
    return ref.head_group_norm(x, n_heads, weight.to(x.dtype) if x.dtype != torch.float32 else weight,
                               bias.to(x.dtype) if x.dtype != torch.float32 else bias, eps)


def router_topk(scores: torch.Tensor, k: int):
    """(softmax over the top-k scores, indices).  scores (T, E) fp32."""
    if _native(scores) and "router_topk" in NATIVE:
        return _nat().router_topk(scores, k)
    return ref.router_topk(scores, k)


def expert_histogram(idx: torch.Tensor, n_experts: int) -> torch.Tensor:
    if _native(idx) and "expert_histogram" in NATIVE:
        return _nat().expert_histogram(idx, n_experts)
    return torch.bincount(idx.flatten().long(), minlength=n_experts)


def moe_routed(x, idx, gates, w_gate, w_up, w_down):
    if _native(x) and "moe_routed" in NATIVE:
        return _nat().moe_routed(x, idx, gates, w_gate, w_up, w_down)
    return ref.moe_routed(x, idx, gates, w_gate, w_up, w_down)


def moe_expert_outputs(x, idx, w_gate, w_up, w_down):
    """Unweighted per-slot expert outputs (T, k, d)."""
    if _native(x) and "moe_expert_outputs" in NATIVE:
        return _nat().moe_expert_outputs(x, idx, w_gate, w_up, w_down)
    return ref.moe_expert_outputs(x, idx, w_gate, w_up, w_down)


def fused_ce_available(h: torch.Tensor) -> bool:
    return h.is_cuda and not _FORCE_REF and has_native() and "linear_cross_entropy" in NATIVE


def linear_cross_entropy(h: torch.Tensor, weight: torch.Tensor, labels: torch.Tensor,
                         ignore_index: int = -100) -> torch.Tensor:
    if _native(h) and "linear_cross_entropy" in NATIVE:
        return _nat().linear_cross_entropy(h, weight, labels, ignore_index)
    return ref.linear_cross_entropy(h, weight, labels, ignore_index)


class TokenScores(NamedTuple):
    """Scores of one given token per row of logits, fp32 (ids int64)."""
    log_probs: torch.Tensor        # (..)
    entropy: torch.Tensor          # (..)
    top_log_probs: torch.Tensor    # (.., k)
    top_ids: torch.Tensor          # (.., k)


_SCORE_TYPES = (torch.bfloat16, torch.float16, torch.float32)
_func_active = torch._C._are_functorch_transforms_active


def _transformed() -> bool:
    """Inside forward-mode differentiation or a torch.func transform, whose tensors a kernel call would take for plain
    ones: their tangents would be lost."""
    return forward_ad._current_level >= 0 or _func_active()


def token_scores(logits: torch.Tensor, targets: torch.Tensor, top_k: int = 0, temperature: float = 1.0,
                 ignore_index: int = -100) -> TokenScores:
    """Under p = softmax(logits / temperature): log p of ``targets``, the entropy of p, and the ``top_k`` (at most
    32) most likely tokens with their log probabilities, ties to the lower id.

    logits (.., V) bf16 / f16 / fp32 (other types run the eager form, and so do forward-mode differentiation
    and torch.func transforms), targets (..) int64.  Differentiable once in all three scores.  Rows whose target is
    ``ignore_index`` give 0, ids -1 and no gradient, and are not read; a logit of -inf has probability 0; a row of
    -inf only gives log probabilities of -inf, entropy 0 and no gradient.  Another target outside the vocabulary
    gives NaN, ids -1 and no gradient, and on the GPU ``fault.check_device_status`` raises afterwards."""
    shape = logits.shape
    if len(shape) < 1 or targets.shape != shape[:-1]:
        raise ValueError(f"token_scores: targets {tuple(targets.shape)} for logits {tuple(shape)}")
    if targets.is_floating_point():
        raise ValueError(f"token_scores: integer targets, got {targets.dtype}")
    if not 1e-30 <= temperature <= 1e27:
        raise ValueError(f"token_scores: temperature from 1e-30 to 1e27, got {temperature}")
    if not (0 <= top_k <= 32 and top_k <= shape[-1]):
        raise ValueError(f"token_scores: top_k from 0 to {min(32, shape[-1])}, got {top_k}")
    if _native(logits) and "token_scores" in NATIVE and logits.dtype in _SCORE_TYPES and not _transformed():
        return TokenScores(*_nat().token_scores(logits, targets, top_k, temperature, ignore_index))
    return TokenScores(*ref.token_scores(logits, targets, top_k, temperature, ignore_index))


def token_log_probs(logits: torch.Tensor, targets: torch.Tensor) -> torch.Tensor:
    """log_softmax(logits)[..., target] without materialising the full log-softmax; 0 where the target is -100.
    targets (..) int64 for logits (.., V).  A target outside the vocabulary is an error: on the GPU the result is NaN and
    ``fault.check_device_status`` raises.  Differentiable any number of times; forward-mode differentiation and
    torch.func transforms run the eager form."""
    if targets.dtype != torch.int64 or targets.shape != logits.shape[:-1]:
        raise ValueError(f"token_log_probs: int64 targets {tuple(logits.shape[:-1])} for logits {tuple(logits.shape)}, "
                         f"got {targets.dtype} {tuple(targets.shape)}")
    if _native(logits) and "token_scores" in NATIVE and logits.dtype in _SCORE_TYPES and not _transformed():
        return _nat().token_log_probs(logits, targets, -100)
    lf = logits.float()
    pick = targets.masked_fill(targets == -100, 0)
    if logits.is_cuda:                                # an index out of range would fault there
        pick = pick.clamp(0, logits.shape[-1] - 1)
    lp = lf.gather(-1, pick.unsqueeze(-1)).squeeze(-1) - torch.logsumexp(lf, dim=-1)
    if logits.is_cuda:
        lp = torch.where(pick == targets, lp, math.nan)
    return lp.masked_fill(targets == -100, 0.0)


class PagedKV(NamedTuple):
    """One layer's paged 8-bit cache: e4m3 codes and a power-of-two scale per (page, KV head)."""
    k: torch.Tensor          # (P, G, page, hd) float8_e4m3fn
    v: torch.Tensor
    k_scale: torch.Tensor    # (P, G) fp32
    v_scale: torch.Tensor


class PagedKV4(NamedTuple):
    """One layer's paged 4-bit cache, and the attention weight that its slots have received where that is kept.

    A block holds 16 tokens of a KV head: key codes (16, hd / 2), key parameters (16, hd / 32) of 16 bits, and the
    same of the values.  A byte holds two dims, the even one in its low half.  Group j of hd / 32 is the 32 dims d with
    (d / 4) % (hd / 32) == j; its parameter is the f16 pattern of a scale s with the zero point z in the low 4 bits,
    and a code n stands for s (n - z), exactly an f16.  Values within a group are rounded to the nearest of sixteen even
    levels that span them and 0, a fifteenth of that range apart, 1/64 of it more at most, and 2^-20 at least.  The range
    is f16's: larger values and infinities become its largest, NaN becomes 0.  Levels stay within f16 too, so that in a
    group that has values of both signs and some above 60,900 in size the end away from those may be off by a whole step."""
    blocks: torch.Tensor                       # (P, G, page / 16, 18 hd) uint8
    mass: Optional[torch.Tensor] = None        # (P, G, page) fp32


def _no_gradient(what: str, *tensors: torch.Tensor) -> None:
    if torch.is_grad_enabled():
        for t in tensors:
            if t.requires_grad:
                raise RuntimeError(f"{what} has no gradient: call it under torch.no_grad()")
    if _transformed():
        for t in tensors:
            if torch._C._functorch.is_functorch_wrapped_tensor(t) or forward_ad.unpack_dual(t).tangent is not None:
                raise RuntimeError(f"{what} has no gradient: neither forward-mode differentiation nor torch.func transforms")


def kv_append(k: torch.Tensor, v: torch.Tensor, cache: Union[PagedKV, PagedKV4], block_table: torch.Tensor, cu_seqlens: torch.Tensor,
              kv_lens: torch.Tensor, max_new: int, cos: Optional[torch.Tensor] = None,
              sin: Optional[torch.Tensor] = None, positions: Optional[torch.Tensor] = None,
              queries: Sequence[torch.Tensor] = ()) -> List[torch.Tensor]:
    """Write packed new keys and values (T, G, hd) into the cache's pages, in place; returns the rotated ``queries``.

    Sequence b's new tokens are rows cu_seqlens[b] : cu_seqlens[b + 1] (int32, B + 1) and take the last slots of its
    kv_lens[b] (int32, the length *with* them); block_table (B, W) int32 gives the page of each block of slots;
    ``max_new`` is the largest number of new tokens of a sequence.  With ``cos`` / ``sin`` (positions, hd / 2) fp32
    and ``positions`` (T,) int64, keys and up to two query tensors (T, H, hd) are rotated on the way (halves, as
    :func:`rope`).  A page that takes new tokens must belong to one sequence only.  On the GPU a page or length out
    of range is skipped and a position is clamped to the tables, and ``fault.check_device_status`` raises
    afterwards.  No gradient.

    ``cache`` is a :class:`PagedKV` or a :class:`PagedKV4`; of the latter, the new slots' ``mass`` becomes 0."""
    _no_gradient("kv_append", k, v, *queries)
    if isinstance(cache, PagedKV4):
        f = _nat().kv4_append if _native(k) and "kv4_append" in NATIVE else ref.kv4_append
        return f(k, v, cache, block_table, cu_seqlens, kv_lens, max_new, cos, sin, positions, queries)
    if _native(k) and "kv_append" in NATIVE:
        return _nat().kv_append(k, v, cache, block_table, cu_seqlens, kv_lens, max_new, cos, sin, positions, queries)
    return ref.kv_append(k, v, cache, block_table, cu_seqlens, kv_lens, cos, sin, positions, queries)


def paged_attention(q: torch.Tensor, cache: Union[PagedKV, PagedKV4], block_table: torch.Tensor, cu_seqlens: torch.Tensor,
                    kv_lens: torch.Tensor, max_new: int, q2: Optional[torch.Tensor] = None,
                    lam: Optional[torch.Tensor] = None, window: int = 0, scale: Optional[float] = None) -> torch.Tensor:
    """Causal attention of packed queries (T, H, hd) over the paged cache, H / G query heads per KV head -> (T, H, hd).
    On the GPU the queries are bf16 or f16.

    Arguments as in :func:`kv_append`, called after it: query i of a sequence's n sees slots up to
    kv_lens - n + i, with ``window`` > 0 only the last ``window`` of them; block table entries of pages below that may be
    anything.  With ``q2`` and ``lam`` (H,) fp32, the
    differential form (softmax(q k) v - lam softmax(q2 k) v) / (1 - lam + 1e-8).  A query that sees nothing, and
    rows past cu_seqlens[-1], give 0.  No gradient.

    ``cache`` is a :class:`PagedKV` or a :class:`PagedKV4`.  With ``cache.mass`` of the latter, each slot's mass grows by
    the softmax weights that it receives, summed over the queries, the heads of its group and both maps, in fp32 and in
    the same order every time; its pages must then belong to one sequence each."""
    _no_gradient("paged_attention", q) if q2 is None or lam is None else _no_gradient("paged_attention", q, q2, lam)
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    if isinstance(cache, PagedKV4):
        f = _nat().paged4_attention if _native(q) and "paged4_attention" in NATIVE else ref.paged4_attention
        return f(q, cache, block_table, cu_seqlens, kv_lens, max_new, q2, lam, window, scale)
    if _native(q) and "paged_attention" in NATIVE:
        return _nat().paged_attention(q, cache, block_table, cu_seqlens, kv_lens, max_new, q2, lam, window, scale)
    return ref.paged_attention(q, cache, block_table, cu_seqlens, kv_lens, q2, lam, window, scale)


def kv_read(cache: PagedKV4, block_table: torch.Tensor, cu_seqlens: torch.Tensor, kv_lens: torch.Tensor, tokens: int,
            dtype: torch.dtype = torch.float16) -> Tuple[torch.Tensor, torch.Tensor]:
    """The keys and values that a 4-bit cache holds of each sequence's last tokens, packed: (tokens, G, hd) each.

    Rows cu_seqlens[b] : cu_seqlens[b + 1] are the last of sequence b's kv_lens[b] tokens (zeros in front of a shorter
    one, and in rows of no sequence), as :func:`kv_append` took them, keys rotated.  f16 and fp32 hold them exactly."""
    if not isinstance(cache, PagedKV4):
        raise TypeError(f"kv_read: a PagedKV4, got {type(cache).__name__}")
    if dtype not in (torch.bfloat16, torch.float16, torch.float32):
        raise ValueError(f"kv_read: bf16, f16 or fp32, got {dtype}")
    if tokens < 0:
        raise ValueError(f"kv_read: tokens must not be negative, got {tokens}")
    if _native(cache.blocks) and "kv_read" in NATIVE:
        return _nat().kv_read(cache, block_table, cu_seqlens, kv_lens, tokens, dtype)
    return ref.kv_read(cache, block_table, cu_seqlens, kv_lens, tokens, dtype)


def kv_evict(cache: PagedKV4, block_table: torch.Tensor, kv_lens: torch.Tensor, budget: int, recent: int = 0,
             out_table: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Cut every sequence of a 4-bit cache to ``budget`` tokens, each KV head by itself: the last ``recent`` ones stay, and
    of the others those of the largest ``cache.mass`` (ties to the earlier slot).

    The kept tokens move, in order, with their mass, to slots 0 .. budget - 1; sequences of up to ``budget`` tokens keep
    all of theirs.  Without ``out_table`` that is in place, and a page must belong to one sequence only.  With it
    (B, W') int32 they go to its pages, which must be no page of ``block_table``'s, and what block_table names stays as it
    is: a prompt that other sequences share, for instance.  Returns the kept slots (B, G, budget) int32, -1 past a shorter
    sequence's end, and the new lengths (B,) int32.  Keys stay rotated as they were appended.  Sliding windows count slots, so they do not go with a cache that
    has been evicted from.  On the GPU, a token of a page out of range is not moved, what is in its new slot stays, and
    ``fault.check_device_status`` raises afterwards.  NaN counts as heavier than infinity."""
    if not isinstance(cache, PagedKV4):
        raise TypeError(f"kv_evict: a PagedKV4 (the 8-bit cache's pages share a scale), got {type(cache).__name__}")
    if cache.mass is None:
        raise ValueError("kv_evict: a cache with mass")
    if budget < 1 or not 0 <= recent <= budget:
        raise ValueError(f"kv_evict: 0 <= recent <= budget and budget >= 1, got {recent} and {budget}")
    if _native(cache.blocks) and "kv_evict" in NATIVE:
        return _nat().kv_evict(cache, block_table, kv_lens, budget, recent, out_table)
    return ref.kv_evict(cache, block_table, kv_lens, budget, recent, out_table)


# Register native ops (import has no side effects when the extension is absent).
if has_native():
    from mamformer_b200.ops import native as _native_mod  # noqa: F401

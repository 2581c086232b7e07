"""Paged KV cache of a batch of sequences, in 8 or 4 bits.

The cache a decoding batch keeps instead of growing (B, S, G, hd) tensors with ``torch.cat`` (reference
``layers/attention.py:143-149``, ``kda_diff.py:813-818``): pages of ``page_size`` tokens, e4m3 codes with one
power-of-two scale per page and KV head (:class:`mamformer_b200.ops.PagedKV`), one block table for all layers.

    cache = PagedKVCache(n_layers, n_kv_heads, head_dim, batch, max_len, device=...)
    cache.extend(S)                                  # S new tokens of every sequence (or a list of counts)
    out = cache.layer(i).attend(q, k, v, cos, sin)   # per attention layer: append, then attend

A layer's pages are allocated when it first attends.  Sequences may differ in length and in the number of new
tokens; :meth:`release` gives a finished sequence's pages back; :meth:`check` raises what the kernels recorded.  What
an 8-bit page holds is rounded to 4 significant bits, so decoded logits differ from an unquantised cache's by that rounding.

``bits=4`` takes 9 bytes for 16 dims instead of 16: sixteen even levels for each 32 dims of a token's head
(:class:`mamformer_b200.ops.PagedKV4`).  With ``weights=True`` such a cache adds up the attention weight that each slot
receives, and :meth:`evict` cuts the sequences to a budget by it, every layer and KV head by itself:

    cache = PagedKVCache(..., bits=4, weights=True)
    cache.evict(budget=2048, recent=512)             # between steps: the last 512 tokens and the heaviest others stay

Layers with sliding windows are refused while a sequence is there that was evicted from: windows count slots.
"""

from __future__ import annotations

from typing import List, Optional, Sequence, Union

import torch

from mamformer_b200 import ops
from mamformer_b200.utils.precision import compute_dtype_of

PAGE_SIZES = (16, 32, 64, 128)


class PagedLayer:
    """One attention layer's pages, with the batch's current step."""

    def __init__(self, owner: "PagedKVCache", index: int) -> None:
        self.owner = owner
        self.index = index
        self.kv: Union[ops.PagedKV, ops.PagedKV4, None] = None
        self._skipped: Optional[torch.Tensor] = None             # tokens of each sequence from before the last restart

    def restart(self) -> "PagedLayer":
        """Forget the layer's tokens from before the current step, for a layer that has taken no part in the steps
        before it.  The block table stays: the layer then uses its first pages."""
        self._skipped = self.owner.kv_lens - self.owner._added
        return self

    def attend(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
               q2: Optional[torch.Tensor] = None, lam: Optional[torch.Tensor] = None, window: int = 0,
               scale: Optional[float] = None) -> torch.Tensor:
        """Append the step's k, v and attend with its queries.  q, q2 (B, S, H, hd), k, v (B, S, G, hd), not rotated;
        cos, sin (S, hd / 2): the rotation of the step's S positions.  Or packed (T, H, hd) with a row of cos / sin
        per token, where the step's counts differ.  Returns a tensor like q."""
        o = self.owner
        if window > 0 and o.evicted:
            raise ValueError("paged cache: sliding windows count slots, and evicted tokens' are gone")
        if self.kv is None:
            self.kv = o._allocate(q.device)
        flat = lambda x: x.reshape(-1, *x.shape[-2:])  # noqa: E731
        queries = [flat(q)] if q2 is None else [flat(q), flat(q2)]
        if queries[0].shape[0] != o.tokens:
            raise ValueError(f"paged cache: {queries[0].shape[0]} query rows in a step of {o.tokens} tokens")
        pos = o._positions(cos.shape[0], q.device)
        kf, vf = flat(k), flat(v)
        lens = o.kv_lens if self._skipped is None else o.kv_lens - self._skipped
        queries = ops.kv_append(kf, vf, self.kv, o.block_table, o.cu_seqlens, lens, o.max_new, cos, sin, pos, queries)
        out = ops.paged_attention(queries[0], self.kv, o.block_table, o.cu_seqlens, lens, o.max_new,
                                  q2=queries[1] if q2 is not None else None, lam=lam, window=window, scale=scale)
        return out.view(q.shape)


class PagedKVCache:
    def __init__(self, n_layers: int, n_kv_heads: int, head_dim: int, batch: int, max_len: int, page_size: int = 64,
                 n_pages: Optional[int] = None, device: Union[str, torch.device] = "cuda", bits: int = 8,
                 weights: bool = False) -> None:
        if bits not in (4, 8):
            raise ValueError(f"the paged cache holds 4 or 8 bits, got {bits}")
        if weights and bits != 4:
            raise ValueError("received weights are kept by the 4-bit cache")
        if page_size not in PAGE_SIZES:
            raise ValueError(f"page_size must be one of {PAGE_SIZES}, got {page_size}")
        if head_dim not in (64, 128):
            raise ValueError(f"the paged cache holds heads of 64 or 128 dims, got {head_dim}")
        self.n_kv_heads, self.head_dim, self.page_size = n_kv_heads, head_dim, page_size
        self.bits, self.weights = bits, weights
        self._cut: set = set()                                   # sequences that were evicted from
        self.batch = batch
        self.width = max(1, -(-max_len // page_size))            # pages of a sequence
        self.n_pages = n_pages if n_pages is not None else batch * self.width
        self.layers = [PagedLayer(self, i) for i in range(n_layers)]
        self.lens: List[int] = [0] * batch
        self._free = list(range(self.n_pages - 1, -1, -1))
        self._pages: List[List[int]] = [[] for _ in range(batch)]
        dev = torch.device(device)
        self.block_table = torch.full((batch, self.width), -1, dtype=torch.int32, device=dev)
        self.kv_lens = torch.zeros(batch, dtype=torch.int32, device=dev)
        self.cu_seqlens = torch.zeros(batch + 1, dtype=torch.int32, device=dev)
        self.tokens = self.max_new = 0
        self._counts: Optional[List[int]] = None                 # of the step that cu_seqlens describes
        self._added: Optional[torch.Tensor] = None
        self._pos: dict = {}

    @classmethod
    def for_model(cls, model, batch: int, max_len: int, page_size: int = 64, bits: int = 8,
                  weights: bool = False) -> "PagedKVCache":
        """A cache with a place for every layer of a Mamformer model.  ``weights``: one that is going to be evicted
        from, so without sliding windows."""
        heads = set()                                            # of the modules: a tensor-parallel rank holds its share
        for layer in model.model.layers:
            att = layer.attention
            if att is None:
                continue
            full = getattr(att, "full_attn", att)
            heads.add((full.n_kv_heads, full.head_dim))
            if getattr(full, "sliding_window", 0) > 0 and full.window_mode != "causal":
                raise ValueError("the paged cache attends causally: sliding windows need window_mode='causal' "
                                 "(a field of the config; --window_mode of the scripts)")
            if getattr(full, "sliding_window", 0) > 0 and weights:
                raise ValueError("sliding windows count slots: they do not go with eviction")
        dtype = compute_dtype_of(model)
        if next(model.parameters()).is_cuda and dtype == torch.float32 and not torch.is_autocast_enabled("cuda"):
            raise ValueError("the paged attention kernels take bf16 or f16 queries: convert the model first "
                             "(utils.precision.to_compute_dtype; scripts/generate.py --bf16)")
        if len(heads) != 1:
            raise ValueError(f"the paged cache takes layers of one number and size of KV heads, got {sorted(heads)}")
        return cls(len(model.model.layers), *heads.pop(), batch, max_len, page_size,
                   device=next(model.parameters()).device, bits=bits, weights=weights)

    @property
    def evicted(self) -> bool:
        """Some sequence's slots are no longer its positions: tokens of it were evicted, and it has not been released since."""
        return bool(self._cut)

    def layer(self, i: int) -> PagedLayer:
        return self.layers[i]

    def layer_caches(self) -> List[dict]:
        """The per-layer ``cache`` list that starts a model's decoding on this cache."""
        return [{"attn": {"attn_type": "full", "paged": layer}} for layer in self.layers]

    def extend(self, new: Union[int, Sequence[int]]) -> None:
        """Begin a step of ``new`` tokens per sequence: allocates pages and sets the step's lengths."""
        counts = [new] * self.batch if isinstance(new, int) else list(new)
        if len(counts) != self.batch or min(counts, default=0) < 0:
            raise ValueError(f"extend: a count for each of {self.batch} sequences, got {counts}")
        need = [-(-(n + a) // self.page_size) - len(p) for n, a, p in zip(self.lens, counts, self._pages)]
        for b, (n, a) in enumerate(zip(self.lens, counts)):
            if n + a > self.width * self.page_size:
                raise ValueError(f"extend: sequence {b} would hold {n + a} tokens, the cache has room for {self.width * self.page_size}")
        if sum(max(0, x) for x in need) > len(self._free):
            raise RuntimeError(f"paged cache: {sum(max(0, x) for x in need)} pages needed, {len(self._free)} free")
        rows, cols, pages = [], [], []
        for b, x in enumerate(need):
            for _ in range(x):
                rows.append(b)
                cols.append(len(self._pages[b]))
                pages.append(self._free.pop())
                self._pages[b].append(pages[-1])
        dev = self.block_table.device
        if rows:
            r, c, p = torch.tensor([rows, cols, pages], device=dev).unbind()
            self.block_table[r, c] = p.to(torch.int32)
        if counts != self._counts:
            self._added = torch.tensor(counts, dtype=torch.int32, device=dev)
            self.cu_seqlens = torch.cat([self._added.new_zeros(1), self._added.cumsum(0).to(torch.int32)])
            self._counts = counts
        self.kv_lens = self.kv_lens + self._added
        self.lens = [n + a for n, a in zip(self.lens, counts)]
        self.tokens, self.max_new = sum(counts), max(counts, default=0)

    def release(self, b: int) -> None:
        """Give sequence b's pages back; it is empty afterwards."""
        self._free.extend(reversed(self._pages[b]))
        self._pages[b] = []
        self._cut.discard(b)
        self.lens[b] = 0
        self.block_table[b] = -1
        self.kv_lens = self.kv_lens.clone()
        self.kv_lens[b] = 0
        for layer in self.layers:
            if layer._skipped is not None:
                layer._skipped = layer._skipped.clone()
                layer._skipped[b] = 0

    def evict(self, budget: int, recent: int = 0) -> None:
        """Cut every sequence of more than ``budget`` tokens to that many, between steps: in each layer and KV head by
        itself the last ``recent`` ones stay and, of the others, those that have received the most attention weight.
        What the sequences then no longer need of their pages is given back."""
        if not self.weights:
            raise ValueError("evict: a cache with weights=True")
        if budget < 1 or not 0 <= recent <= budget:
            raise ValueError(f"evict: 0 <= recent <= budget and budget >= 1, got {recent} and {budget}")
        if max(self.lens, default=0) <= budget:
            return
        left = self.kv_lens.clamp(max=budget)
        for layer in self.layers:
            if layer.kv is None:
                continue
            lens = self.kv_lens if layer._skipped is None else self.kv_lens - layer._skipped
            _, lens = ops.kv_evict(layer.kv, self.block_table, lens, budget, recent)
            if layer._skipped is not None:
                layer._skipped = left - lens
        self.kv_lens = left
        self._cut.update(b for b, n in enumerate(self.lens) if n > budget)
        self.lens = [min(n, budget) for n in self.lens]
        rows, cols = [], []
        for b, (n, pages) in enumerate(zip(self.lens, self._pages)):
            need = -(-n // self.page_size)
            while len(pages) > need:
                self._free.append(pages.pop())
                rows.append(b)
                cols.append(len(pages))
        if rows:
            r, c = torch.tensor([rows, cols], device=self.block_table.device).unbind()
            self.block_table[r, c] = -1

    def check(self) -> None:
        """Wait for the steps so far and raise what their kernels recorded: PagedCacheError for a page, length or
        position out of range, KernelTimeoutError.  :meth:`MamformerForCausalLM.generate` does so before it returns."""
        if self.block_table.is_cuda:
            from mamformer_b200.fault import check_paged_status
            with torch.cuda.device(self.block_table.device):
                torch.cuda.current_stream().synchronize()
                check_paged_status()

    def _allocate(self, device) -> Union[ops.PagedKV, ops.PagedKV4]:
        if self.bits == 4:
            blocks = torch.empty(self.n_pages, self.n_kv_heads, self.page_size // 16, 18 * self.head_dim, dtype=torch.uint8, device=device)
            mass = torch.zeros(self.n_pages, self.n_kv_heads, self.page_size, device=device) if self.weights else None
            return ops.PagedKV4(blocks, mass)
        shape = (self.n_pages, self.n_kv_heads, self.page_size, self.head_dim)
        code = lambda: torch.empty(shape, dtype=torch.float8_e4m3fn, device=device)  # noqa: E731
        return ops.PagedKV(code(), code(), torch.ones(shape[:2], device=device), torch.ones(shape[:2], device=device))

    def _positions(self, rows: int, device) -> torch.Tensor:
        """Row of the rotation tables of each packed token."""
        if rows == self.tokens:
            key, make = (rows, 0), lambda: torch.arange(rows, device=device)
        elif self._counts is not None and all(n == rows for n in self._counts):
            key, make = (rows, self.batch), lambda: torch.arange(rows, device=device).repeat(self.batch)
        else:
            raise ValueError(f"paged cache: {rows} rotation rows for a step of {self.tokens} tokens")
        if key not in self._pos:
            self._pos = {key: make()}                            # the last step's only
        return self._pos[key]

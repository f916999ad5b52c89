"""Keys and values of many requests in one pool of pages, per layer of a decoder.

The caches of ``PI05Model`` are ``[B, G, keys, D]``: every request takes the room of the longest and is masked.  Here a request holds
pages for the tokens that it has, whatever the others hold; which page serves whom is planned on the GPU
(``ops.page_plan_``), so a step of a server is three kinds of launches and can be captured into a graph::

    cache = PagedCache(layers=18, requests=16, pages=4096, page_size=16, kv_heads=1, head_dim=256, width=128)
    plan = cache.step(new_lens, tokens=16, finished=left)        # once per step; here of single tokens
    for i, layer in enumerate(decoder):                          # norms, rotation, store, attention
        out, _ = cache.attend(i, layer.qkv(x), cos, sin, heads=8, max_tokens=1)

``width`` (the most pages of one request) and ``max_tokens`` (the most tokens that one request brings to the step) choose between forms of
the attention and change no more than rounding.  Without them the host has to allow for requests as long as the pool and
for a step that is all one request's: single tokens then take the kernels of whole prompts.

The counterpart of the key/value caches that the reference's decoder keeps per request (tybok/policies/pi05/models/gemma.py:61-125).
"""

from __future__ import annotations

import torch

from . import ops
from .ops import DEFAULT_SHIFT, PagePlan


class PagedCache:
    """Pools ``k_pages`` / ``v_pages`` ``[layers, pages, kv_heads, page_size, head_dim]`` and the state of ``requests`` rows: ``key_lens``,
    ``block_table`` (``width`` pages a row, the most that one request may hold; all of them by default, but a width near the truth lets
    short calls take quicker forms), ``free_pages`` and ``free_count``, on ``device``.

    Every request begins with no keys.  All work goes to the current stream of the device; one cache takes one step at a time."""

    def __init__(self, *, layers: int, requests: int, pages: int, page_size: int, kv_heads: int, head_dim: int, width: int | None = None,
                 device: str | torch.device = "cuda"):
        width = pages if width is None else width
        for name, value in dict(layers=layers, requests=requests, pages=pages, kv_heads=kv_heads, width=width).items():
            if value < 1:
                raise ValueError(f"{name} must be positive, not {value}")
        if page_size < 16 or page_size & (page_size - 1):
            raise ValueError(f"page_size must be a power of two, 16 at least, not {page_size}")
        if head_dim not in (128, 256):
            raise ValueError(f"head_dim must be 128 or 256, not {head_dim}")
        if requests > 2048:
            raise ValueError(f"{requests} requests: 2048 at most")
        shape = (layers, pages, kv_heads, page_size, head_dim)
        self.page_size = page_size
        self.k_pages = torch.empty(shape, dtype=torch.bfloat16, device=device)
        self.v_pages = torch.empty(shape, dtype=torch.bfloat16, device=device)
        self.key_lens = torch.zeros(requests, dtype=torch.int32, device=device)
        self.block_table = torch.zeros(requests, width, dtype=torch.int32, device=device)
        self.free_pages = torch.arange(pages, dtype=torch.int32, device=device)
        self.free_count = torch.full((1,), pages, dtype=torch.int32, device=device)
        self.plan: PagePlan | None = None

    def step(self, new_lens: torch.Tensor, *, tokens: int, finished: torch.Tensor | None = None) -> PagePlan:
        """Plans a step in which request ``b`` brings ``new_lens[b]`` tokens; rows that are ``finished`` return their pages first and start anew.
        ``tokens``: token rows of the step, padding behind the last token included.  Where ``plan.missing`` is not 0 (read it when
        the host looks anyway) the state has stayed as it was, and ``attend`` stores nothing and gives zeros."""
        self.plan = ops.page_plan_(self.key_lens, new_lens, self.block_table, self.free_pages, self.free_count, tokens=tokens,
                                   page_size=self.page_size, finished=finished)
        return self.plan

    def attend(self, layer: int, qkv: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, *, heads: int, scale: float | None = None,
               causal: bool = True, norm_q: torch.Tensor | None = None, norm_k: torch.Tensor | None = None, eps: float = 1e-6,
               paired: bool = False, max_tokens: int | None = None, out_bf16: bool = True, out_planes: bool = False,
               out_shift: int = DEFAULT_SHIFT) -> tuple[torch.Tensor, torch.Tensor]:
        """One layer of the planned step: the projection rows ``qkv`` ``[tokens, (heads + 2 * kv_heads) * head_dim]`` are normed, rotated and
        stored, and every request's new tokens attend to all its keys.  Returns ``(out_bf16, out_planes)`` as ``ops.paged_attention``
        does; ``scale`` is ``head_dim ** -0.5`` unless given.  ``max_tokens``: as there, the step's token rows unless given, so a step of single
        tokens is quickest with ``max_tokens=1``."""
        if self.plan is None:
            raise RuntimeError("attend() before the first step()")
        if not 0 <= layer < self.k_pages.shape[0]:
            raise IndexError(f"layer {layer} of {self.k_pages.shape[0]}")
        k, v, plan = self.k_pages[layer], self.v_pages[layer], self.plan
        q = ops.head_norm_rope_store(qkv, plan.pos, plan.slots, cos, sin, k, v, heads=heads, norm_q=norm_q, norm_k=norm_k, eps=eps,
                                     paired=paired)
        return ops.paged_attention(q, k, v, plan.block_table, plan.cu_tokens, plan.key_lens, scale=k.shape[-1] ** -0.5 if scale is None else scale,
                                   causal=causal, max_tokens=max_tokens, out_bf16=out_bf16, out_planes=out_planes, out_shift=out_shift)

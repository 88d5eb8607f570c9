"""Decoder layers with attention over a paged cache.

The reference's decoder layer is RMSNorm -> grouped-query attention -> residual
-> RMSNorm -> MLP -> residual (models/modeling_llama.py:979-1002,
bench/e2e_block.py:264-282).  ``DecoderLayer`` is that layer: the projections on
the library's GEMM, rotary positions and the cache write in one kernel
(attention.rope_cache), prompt or tree attention, and an ``SvdMlpBlock`` with its
RMSNorm and residual fused.  ``PagedDecoder`` is a stack of them with its caches
and block tables: ``prefill`` takes whole prompts, ``step`` the newest tokens of
every request (one each, or a chain or tree of drafted tokens), ``keep`` takes
rejected tokens back.  Inputs and outputs are hidden states; embedding and the
language-model head belong to the caller.
"""
from __future__ import annotations

import itertools
from typing import List, Optional, Sequence

import torch

from ..kernels import attention, ops
from .svd_mlp import SvdMlpBlock

__all__ = ["DecoderLayer", "PagedDecoder"]


class DecoderLayer(torch.nn.Module):
    """x + wo . attention(rope(rmsnorm(x) . [wq|wk|wv])), then the MLP block.

    Weights are natural matmul operands ([in, out]): wq [H, heads * D], wk and
    wv [H, kv_heads * D], wo [heads * D, H]; `inv_freq` and `rope_scale` come
    from attention.rope_frequencies."""

    def __init__(self, wq, wk, wv, wo, attn_norm, mlp: SvdMlpBlock, *, heads: int, kv_heads: int, inv_freq: torch.Tensor,
                 rope_scale: float = 1.0, interleaved: bool = False, eps: float = 1e-5):
        super().__init__()
        hidden = wq.shape[0]
        if heads <= 0 or kv_heads <= 0 or heads % kv_heads or wq.shape[1] % heads:
            raise ValueError("heads must divide wq's columns and be a multiple of kv_heads")
        self.heads, self.kv_heads, self.head_dim = heads, kv_heads, wq.shape[1] // heads
        kv_columns = kv_heads * self.head_dim
        if tuple(wk.shape) != (hidden, kv_columns) or tuple(wv.shape) != (hidden, kv_columns):
            raise ValueError("wk and wv must be [hidden, kv_heads * head_dim]: dimensions do not match")
        if tuple(wo.shape) != (heads * self.head_dim, hidden) or mlp.hidden_size != hidden:
            raise ValueError("wo and the MLP must return to the hidden size: dimensions do not match")
        self.w_qkv = torch.cat((wq, wk, wv), 1).to(torch.bfloat16).contiguous()
        self.wo = wo.to(torch.bfloat16).contiguous()
        self.attn_norm = attn_norm.to(torch.bfloat16).contiguous()
        self.mlp = mlp
        self.inv_freq, self.rope_scale, self.interleaved, self.eps = inv_freq, float(rope_scale), interleaved, float(eps)

    def forward(self, x: torch.Tensor, pages: attention.PageStep, block_table: torch.Tensor, k_cache: torch.Tensor,
                v_cache: torch.Tensor, *, max_tree: Optional[int] = None,
                tree_mask: Optional[torch.Tensor] = None) -> torch.Tensor:
        """x [N, H] bf16, the new tokens `pages` describes.  Without `max_tree`
        they are whole prompts; with it, the newest tokens of requests whose
        earlier ones are in the cache.  Tokens are turned to pages.positions:
        those of drafted trees are attention.tree_positions."""
        h, hk, d = self.heads, self.kv_heads, self.head_dim
        qkv = ops.dense_matmul(ops.rmsnorm(x, self.attn_norm, self.eps), self.w_qkv).unflatten(1, (h + 2 * hk, d))
        v = qkv[:, h + hk:]
        prompt = max_tree is None
        q, k = attention.rope_cache(qkv[:, :h], qkv[:, h:h + hk], v, pages.positions, pages.slots, self.inv_freq, k_cache,
                                    v_cache, interleaved=self.interleaved, scale=self.rope_scale, return_k=prompt)
        if prompt:
            o = attention.prompt_attention(q, k, v, pages.cu_seqlens)
        else:
            o = attention.tree_attention(q, k_cache, v_cache, block_table, pages.seq_lens, pages.cu_seqlens,
                                         max_tree=max_tree, tree_mask=tree_mask)
        x = x + ops.dense_matmul(o.flatten(1), self.wo)
        return self.mlp(x)


class PagedDecoder:
    """A stack of DecoderLayers, its caches and the tables of `batch` requests.

    Lengths, tables and the free list live on the GPU, in tensors that every call
    updates in place; a step's token counts come from the host, so no call waits
    for the device.  A step can therefore be captured in a CUDA graph (one step
    on the capturing stream before it sets up weights and workspaces): each
    replay goes on from where the requests are, for the counts that it was
    captured with."""

    def __init__(self, layers: Sequence[DecoderLayer], batch: int, num_blocks: int, max_length: int, *,
                 block_size: int = 16, device="cuda"):
        self.layers = list(layers)
        if not self.layers:
            raise ValueError("at least one layer is required")
        self.batch, self.block_size = batch, block_size
        first = self.layers[0]
        self.caches = [attention.kv_cache(num_blocks, l.kv_heads, block_size, l.head_dim, device=device)
                       for l in self.layers]
        width = -(-max_length // block_size)
        dev = first.w_qkv.device
        self.block_table = torch.full((batch, width), -1, dtype=torch.int32, device=dev)
        self.seq_lens = torch.zeros(batch, dtype=torch.int32, device=dev)
        # one place more than there are blocks: keep() writes there what it does not free
        self.free_blocks = torch.arange(num_blocks + 1, dtype=torch.int32, device=dev)
        self.free_count = torch.tensor([num_blocks], dtype=torch.int32, device=dev)
        self.num_blocks = num_blocks
        self.missing = torch.zeros(1, dtype=torch.int32, device=dev)
        # the longest that each request has been: page_step drops what lies beyond the table's width
        self.longest = torch.zeros(batch, dtype=torch.int32, device=dev)
        # tokens that a request held when prefill was given more of it
        self.prefilled = torch.zeros(batch, dtype=torch.int32, device=dev)

    def _run(self, x: torch.Tensor, new_lens: Sequence[int], **kw) -> torch.Tensor:
        new_lens = [int(n) for n in new_lens]
        if len(new_lens) != self.batch or min(new_lens) < 0 or sum(new_lens) != x.shape[0]:
            raise ValueError(f"new_lens must give {self.batch} counts that sum to x's {x.shape[0]} rows")
        if not x.shape[0]:
            return x
        counts = self._counts(new_lens)
        pages = attention.page_step(self.block_table, self.seq_lens, counts, self.free_blocks[:self.num_blocks],
                                    self.free_count, self.block_size, sum(new_lens))
        if kw.get("tree_mask") is not None:
            pages = pages._replace(positions=attention.tree_positions(pages, kw["tree_mask"]))
        for layer, (k_cache, v_cache) in zip(self.layers, self.caches):
            x = layer(x, pages, self.block_table, k_cache, v_cache, **kw)
        if "max_tree" not in kw:  # prompt attention sees the call's own tokens only
            torch.maximum(self.prefilled, self.seq_lens * (counts > 0), out=self.prefilled)
        self.seq_lens.copy_(pages.seq_lens)
        self.free_count.copy_(pages.free_count)
        torch.maximum(self.missing, pages.missing, out=self.missing)
        torch.maximum(self.longest, pages.seq_lens, out=self.longest)
        return x

    def _counts(self, new_lens: List[int]) -> torch.Tensor:
        """`new_lens` on the device."""
        device = self.seq_lens.device
        if len(set(new_lens)) == 1:
            return torch.full((self.batch,), new_lens[0], dtype=torch.int32, device=device)
        if not torch.cuda.is_current_stream_capturing():
            return torch.tensor(new_lens, dtype=torch.int32).pin_memory().to(device, non_blocking=True)
        # a captured copy would read host memory at every replay, long after this call: filled in place, run by run
        counts, at = torch.empty(self.batch, dtype=torch.int32, device=device), 0
        for n, run in itertools.groupby(new_lens):
            length = len(list(run))
            counts[at:at + length].fill_(n)
            at += length
        return counts

    def prefill(self, x: torch.Tensor, lens: Sequence[int]) -> torch.Tensor:
        """Whole prompts: x [sum(lens), H] bf16, requests in order; those that get
        tokens are empty before (check() reports one that was not: step takes
        the chunks of a prompt).  Returns the hidden states of every token."""
        return self._run(x, lens)

    def step(self, x: torch.Tensor, new_lens: Optional[Sequence[int]] = None, *,
             tree_mask: Optional[torch.Tensor] = None) -> torch.Tensor:
        """The next tokens of every request: one each by default, a chain of
        new_lens[b], or a tree (tree_mask, attention.tree_attention), whose
        tokens are turned to their depth: each one's hidden state is that of its
        own path.  Their places in the cache are successive; the caller keeps one
        path that is a prefix of them (keep), or takes the tree back and feeds
        the accepted tokens again."""
        new_lens = [1] * self.batch if new_lens is None else list(new_lens)
        if tree_mask is not None and max(new_lens, default=0) > 64:
            raise ValueError(f"a tree has at most 64 tokens, got {max(new_lens)}")
        return self._run(x, new_lens, max_tree=max(1, *new_lens) if new_lens else 1, tree_mask=tree_mask)

    def keep(self, lens: torch.Tensor) -> None:
        """Shortens the requests to `lens` (int32 [batch], at most what they
        hold) and returns the blocks behind them to the free list."""
        lens = torch.minimum(lens.to(torch.int32), self.seq_lens).clamp(min=0)
        block = self.block_size
        column = torch.arange(self.block_table.shape[1], device=lens.device)
        freed = (column >= ((lens + block - 1) // block)[:, None]) & (column < ((self.seq_lens + block - 1) // block)[:, None])
        freed &= self.block_table >= 0
        flat = freed.flatten()
        place = torch.where(flat, self.free_count + flat.cumsum(0) - 1, self.num_blocks)
        self.free_blocks[place] = self.block_table.flatten()
        self.block_table[:] = torch.where(freed, -1, self.block_table)
        self.free_count += flat.sum(dtype=torch.int32)
        self.seq_lens.copy_(lens)

    def check(self) -> None:
        """Waits for the device; raises if, since the decoder was made, the cache ran out of blocks, a request outgrew
        its table or prefill was given one that held tokens, or if a kernel reported an error."""
        short, longest = int(self.missing.item()), int(self.longest.max().item())
        before = int(self.prefilled.max().item())
        ops.check_device_status(self.seq_lens.device)
        places = self.block_table.shape[1] * self.block_size
        if longest > places:
            raise RuntimeError(f"a request of {longest} tokens outgrew its table of {places}: tokens were dropped")
        if before:
            raise RuntimeError(f"prefill was given a request that held {before} tokens: its new ones did not see them")
        if short:
            raise RuntimeError(f"the cache had {short} blocks too few: tokens were dropped")

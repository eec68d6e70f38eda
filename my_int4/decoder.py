"""A decoder layer's step on the quantized operators, and the paged 8-bit cache
it keeps.  The reference has neither: its layers are the W4A4 products alone.

The parts, in the order in which a step runs them:

  norm -> w8a8_linear (query, key and value in one product)
       -> kv8_append (rotation by position, keys and values into the cache)
       -> kv8_attention -> w8a8_linear (output projection) -> add
  norm -> W4A4 step of my_int4.chain (WUSH transform, quantization, product)
       -> activation -> w8a8_linear (down projection) -> add

The same call takes one new token per sequence (decode) or many (prefill, or a
chunk of it): ``cu_q`` says where each sequence's tokens begin.  Nothing in it
synchronizes, so a decode step can be captured with ``my_int4.chain.graphed``
and replayed while ``seq_lens`` and the inputs advance in place.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional, Tuple

import torch

from my_int4 import _C
from my_int4.chain import make_chain


def quant_weight_int8(w: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """(N, K) weights -> int8 codes and one fp32 scale per output channel."""
    wf = w.float()
    s = (wf.abs().amax(1) / 127).clamp_min(2.0 ** -126)
    return (wf / s[:, None]).round().clamp(-127, 127).to(torch.int8), s


def rotation_table(positions: int, channels: int, theta: float = 10000.0, device="cuda") -> torch.Tensor:
    """(positions, channels) fp32: the cosines, then the sines, of position *
    theta^(-2 i / channels)."""
    f = theta ** (-torch.arange(0, channels, 2, dtype=torch.float64, device=device) / channels)
    a = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * f
    return torch.cat((a.cos(), a.sin()), 1).float()


class KV8Cache:
    """Pages of 8-bit keys and values with a scale per (page, head), and the
    list of pages that no sequence holds."""

    def __init__(self, pages: int, heads: int, head_dim: int, page_size: int = 64, device="cuda"):
        self.page_size = page_size
        self.k = torch.zeros(pages, heads, page_size, head_dim, dtype=torch.int8, device=device)
        self.v = torch.zeros(pages, heads, head_dim, page_size, dtype=torch.int8, device=device)
        self.k_scale = torch.zeros(pages, heads, device=device)
        self.v_scale = torch.zeros(pages, heads, device=device)
        self.free = list(range(pages))[::-1]

    def tensors(self):
        return self.k, self.v, self.k_scale, self.v_scale

    def grow(self, table: torch.Tensor, row: int, tokens: int, held: int = 0) -> int:
        """Gives sequence ``row`` of the (host) block table the pages for
        ``tokens`` tokens and returns how many it holds then.  An entry without a page is
        -1; pages that the row has already stay in their places, whatever ``held``, a
        number of first entries that need not be looked at, says."""
        need = -(-tokens // self.page_size)
        if need > table.shape[1]:
            raise ValueError(f"{tokens} tokens need {need} pages, the table has {table.shape[1]}")
        entries = table[row, held:need].tolist()
        kept = [p for p in entries if p >= 0]
        if kept and not set(kept).isdisjoint(self.free):
            raise ValueError(f"row {row} of the table names a page that is free: an entry without a page is -1")
        if len(entries) - len(kept) > len(self.free):
            raise MemoryError(f"{len(entries) - len(kept)} pages needed, {len(self.free)} free")
        for i, p in enumerate(entries, held):
            if p < 0:
                table[row, i] = self.free.pop()
        return max(need, held)

    def release(self, table: torch.Tensor, row: int, held: int) -> None:
        """Takes the row's first ``held`` entries back."""
        self.free.extend(p for p in table[row, :held].tolist() if p >= 0)
        table[row, :held] = -1


def _norm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-5) -> torch.Tensor:
    xf = x.float()
    return (xf * torch.rsqrt(xf.square().mean(-1, keepdim=True) + eps) * weight).to(x.dtype)


@dataclass
class DecoderLayer:
    """Weights of a layer: W8A8 projections as (codes, scales) of
    quant_weight_int8, the up projection as W4A4 codes, scales and transform."""
    q_heads: int
    kv_heads: int
    qkv: Tuple[torch.Tensor, torch.Tensor]
    out: Tuple[torch.Tensor, torch.Tensor]
    up: Tuple[torch.Tensor, torch.Tensor, torch.Tensor]        # (transform, wq, ws)
    down: Tuple[torch.Tensor, torch.Tensor]
    norm1: torch.Tensor
    norm2: torch.Tensor
    window: int = 0
    softcap: float = 0.0

    def attention(self, x, cache: KV8Cache, cos_sin, block_table, seq_lens, cu_q: Optional[torch.Tensor] = None,
                  max_len: int = 0) -> torch.Tensor:
        """The attention half: x (tokens, K) plus what its tokens attend to."""
        D = cache.k.shape[3]
        qkv = _C.w8a8_linear(_norm(x, self.norm1), *self.qkv).view(x.shape[0], -1, D)
        q, k, v = qkv.split([self.q_heads, self.kv_heads, self.kv_heads], 1)
        q = _C.kv8_append(q, k, v, cos_sin, *cache.tensors(), block_table, seq_lens, cu_q=cu_q)
        o = _C.kv8_attention(q, *cache.tensors(), block_table, seq_lens, cu_q=cu_q, window=self.window,
                             softcap=self.softcap, max_len=max_len)
        return x + _C.w8a8_linear(o.view(x.shape[0], -1), *self.out)

    def step(self, x, cache: KV8Cache, cos_sin, block_table, seq_lens, cu_q: Optional[torch.Tensor] = None,
             max_len: int = 0) -> torch.Tensor:
        """x (tokens, K) bf16 -> the layer's output, the new tokens' keys and
        values in the cache.  seq_lens counts them."""
        x = self.attention(x, cache, cos_sin, block_table, seq_lens, cu_q, max_len)
        h = make_chain(_norm(x, self.norm2), *self.up)().view(x.shape[0], -1)     # fp16
        h = torch.nn.functional.gelu(h.float()).to(x.dtype)
        return x + _C.w8a8_linear(h, *self.down)

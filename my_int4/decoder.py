"""A decoder layer's step on the quantized operators, and the paged 8-bit cache
it keeps.  The reference has neither: its layers are the W4A4 products alone.

The parts, in the order in which a step runs them:

  norm -> w8a8_linear (query, key and value in one product)
       -> kv8_append (rotation by position, keys and values into the cache)
       -> kv8_attention -> w8a8_linear (output projection) -> add
  norm -> W4A4 step of my_int4.chain (WUSH transform, quantization, product)
       -> activation -> w8a8_linear (down projection) -> add

or, in a layer of experts, for the second line:

  norm -> router -> moe_route -> fp8_experts (beside fp8_linear for a shared expert) -> add

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


def quant_weight_fp8(w: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """(..., N, K) weights -> e4m3 codes and an fp32 scale per block of 128 x 128, (..., N / 128, K / 128)."""
    N, K = w.shape[-2:]
    b = torch.nn.functional.pad(w.float(), (0, -K % 128, 0, -N % 128)).unflatten(-1, (-1, 128)).unflatten(-3, (-1, 128))
    s = (b.abs().amax((-3, -1)) / 448).clamp_min(2.0 ** -126)                # b: (..., N / 128, 128, K / 128, 128)
    q = (b / s[..., :, None, :, None]).flatten(-2).flatten(-3, -2)[..., :N, :K]
    return q.contiguous().to(torch.float8_e4m3fn), s


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
class ExpertLayer:
    """A router and its gated experts, weights as (codes, scales) of quant_weight_fp8: ``up`` (experts, 2 I, K), each
    gate's rows before its up projection's, ``down`` (experts, K, I); ``shared`` the same two of an expert that
    every token takes.  A process that holds some of the experts only (expert parallelism) has their
    weights here, all experts' router, and the first one's number in ``first``: the others' choices add nothing.
    The processes' outputs are then added up, so that only one of them has ``shared``: each that has it adds it."""
    router: torch.Tensor                                       # (all experts, K) fp32
    k: int
    up: Tuple[torch.Tensor, torch.Tensor]
    down: Tuple[torch.Tensor, torch.Tensor]
    bias: Optional[torch.Tensor] = None
    sigmoid: bool = False
    groups: int = 1
    keep_groups: int = 1
    group_best: int = 1
    renorm: bool = True
    scale: float = 1.0
    shared: Optional[Tuple[Tuple[torch.Tensor, torch.Tensor], Tuple[torch.Tensor, torch.Tensor]]] = None
    first: int = 0

    def __call__(self, x: torch.Tensor) -> torch.Tensor:
        """x (tokens, K) bf16 or fp16 -> the weighted sum of its experts."""
        logits = torch.nn.functional.linear(x.float(), self.router)
        weights, ids = _C.moe_route(logits, self.k, bias=self.bias, sigmoid=self.sigmoid, groups=self.groups,
                                    keep_groups=self.keep_groups, group_best=self.group_best, renorm=self.renorm, scale=self.scale)
        y = _C.fp8_experts(x, weights, ids - self.first if self.first else ids, *self.up, *self.down)
        if self.shared is not None:
            # gate, up and h are rounded to x's type between the two products, as between any two layers: 1.5e-2 of this expert's
            # exact output in bf16 and 5e-3 in fp16, where e4m3 weights and activations themselves are 6.39e-2 from unquantized ones
            # (6.39e-2 with these roundings too).  fp8_experts with one expert keeps them in fp32 (1.7e-3, 2e-4), but has tiles for
            # few CUs and does not split K: 4096 x 4096, bf16, 16 tokens 77 us for 42, 128 tokens 111 for 53, 4096 tokens 356 for 309.
            gate, up = _C.fp8_linear(x, *self.shared[0]).float().chunk(2, -1)
            y = y + _C.fp8_linear((torch.nn.functional.silu(gate) * up).to(x.dtype), *self.shared[1])
        return y


@dataclass
class DecoderLayer:
    """Weights of a layer: W8A8 projections as (codes, scales) of
    quant_weight_int8, the up projection as W4A4 codes, scales and transform; with ``experts``, those instead of
    ``up`` and ``down``."""
    q_heads: int
    kv_heads: int
    qkv: Tuple[torch.Tensor, torch.Tensor]
    out: Tuple[torch.Tensor, torch.Tensor]
    up: Optional[Tuple[torch.Tensor, torch.Tensor, torch.Tensor]]        # (transform, wq, ws)
    down: Optional[Tuple[torch.Tensor, torch.Tensor]]
    norm1: torch.Tensor
    norm2: torch.Tensor
    window: int = 0
    softcap: float = 0.0
    experts: Optional[ExpertLayer] = None

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
        if self.experts is not None:
            return x + self.experts(_norm(x, self.norm2))
        h = make_chain(_norm(x, self.norm2), *self.up)().view(x.shape[0], -1)     # fp16
        h = torch.nn.functional.gelu(h.float()).to(x.dtype)
        return x + _C.w8a8_linear(h, *self.down)

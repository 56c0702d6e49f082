"""GPT-2-shaped decoder used by the data-parallel gradient benchmark.

GPT-2 medium: 24 layers, d_model 1024, 16 heads, MLP 4096, vocab 50257,
context 1024, learned positions, pre-LayerNorm blocks, GELU MLP, tied
embedding / LM head.  Weights are random-initialised (std 0.02, residual
projections scaled by 1/sqrt(2 * layers)); the benchmark feeds synthetic
token ids.  Attention runs through torch's scaled_dot_product_attention.

Options beyond the benchmark's model, on CUDA through cail_b200.ops: a sliding
window with sinks (``window``, ``sinks``), rotary positions in place of the
learned ones (``rotary``), padded batches (``lengths``), training against a
teacher's top logits (``teacher``), and a key/value cache with single-token
decoding (``new_cache``, ``prefill``, ``decode``).
"""
from __future__ import annotations

import math
from dataclasses import dataclass
from typing import List, Optional, Tuple

import torch
import torch.nn as nn
import torch.nn.functional as F

from .. import ops


@dataclass
class GPT2Config:
    n_layer: int = 24
    d_model: int = 1024
    n_head: int = 16
    d_mlp: int = 4096
    vocab: int = 50257
    n_ctx: int = 1024
    window: int = 0  # keys that a token sees behind itself, itself included; 0: all
    sinks: int = 0  # first tokens that stay visible beyond the window
    rotary: int = 0  # elements of a head that rotate with the position; 0: learned positions
    rotary_base: float = 10000.0
    rotary_interleaved: bool = False
    rotary_scaling: Optional[str] = None  # "linear", "ntk" or "parts" (cail_b200.ops.Rotary), by rotary_factor
    rotary_factor: float = 1.0

    @staticmethod
    def medium() -> "GPT2Config":
        return GPT2Config()

    @staticmethod
    def tiny() -> "GPT2Config":
        return GPT2Config(n_layer=2, d_model=64, n_head=4, d_mlp=256, vocab=512, n_ctx=64)


class KVCache:
    """The keys and values of a batch of sequences, [B, length, heads, D] per
    layer, and how many tokens each sequence holds (int32, on the device).
    ``filled`` is the most that any of them can hold, known on the host."""

    def __init__(self, c: GPT2Config, batch: int, length: int, device, dtype):
        shape = (batch, length, c.n_head, c.d_model // c.n_head)
        with torch.inference_mode(False):  # so that what fills it may run in inference mode or outside
            self.k = [torch.zeros(shape, device=device, dtype=dtype) for _ in range(c.n_layer)]
            self.v = [torch.zeros(shape, device=device, dtype=dtype) for _ in range(c.n_layer)]
            self.lengths = torch.zeros(batch, device=device, dtype=torch.int32)
        self.length = length
        self.filled = 0


class Block(nn.Module):
    def __init__(self, c: GPT2Config):
        super().__init__()
        self.n_head = c.n_head
        self.window, self.sinks = c.window, c.sinks
        self.ln1 = nn.LayerNorm(c.d_model)
        self.qkv = nn.Linear(c.d_model, 3 * c.d_model)
        self.proj = nn.Linear(c.d_model, c.d_model)
        self.ln2 = nn.LayerNorm(c.d_model)
        self.fc = nn.Linear(c.d_model, c.d_mlp)
        self.out = nn.Linear(c.d_mlp, c.d_model)

    def _rest(self, x: torch.Tensor, a: torch.Tensor) -> torch.Tensor:
        x = x + self.proj(a)
        return x + self.out(F.gelu(self.fc(self.ln2(x)), approximate="tanh"))

    def forward(self, x: torch.Tensor, plan: Optional[ops.Rotary] = None, lengths: Optional[torch.Tensor] = None,
                keep: Optional[Tuple[torch.Tensor, torch.Tensor]] = None) -> torch.Tensor:
        b, t, d = x.shape
        q, k, v = self.qkv(self.ln1(x)).split(d, dim=2)
        shape = (b, t, self.n_head, d // self.n_head)
        if self.window == 0 and plan is None and lengths is None and keep is None:
            q, k, v = (z.view(shape).transpose(1, 2) for z in (q, k, v))
            a = F.scaled_dot_product_attention(q, k, v, is_causal=True)
            return self._rest(x, a.transpose(1, 2).reshape(b, t, d))
        q, k, v = (z.view(shape) for z in (q, k, v))
        if plan is not None:
            q, k = ops.rotary(q, k, plan)
        if keep is not None:
            keep[0][:, :t], keep[1][:, :t] = k, v
        a = ops.window_attention(q, k, v, self.window or max(t, 1), self.sinks, lengths=lengths)
        return self._rest(x, a.reshape(b, t, d))

    def decode(self, x: torch.Tensor, plan: Optional[ops.Rotary], k_cache: torch.Tensor, v_cache: torch.Tensor, at: torch.Tensor,
               lengths: torch.Tensor) -> torch.Tensor:
        """One token per sequence: x [B, d]; ``at`` is where each goes, ``lengths`` what each sequence then holds."""
        b, d = x.shape
        q, k, v = (z.view(b, self.n_head, d // self.n_head) for z in self.qkv(self.ln1(x)).split(d, dim=1))
        if plan is not None:
            q, k = (z[:, 0] for z in ops.rotary(q[:, None], k[:, None], plan, at[:, None]))
        row = torch.arange(b, device=x.device)
        k_cache[row, at] = k.to(k_cache.dtype)
        v_cache[row, at] = v.to(v_cache.dtype)
        a = ops.window_attention_decode(q.to(k_cache.dtype), k_cache, v_cache, lengths, self.window or k_cache.size(1), self.sinks)
        return self._rest(x, a.reshape(b, d))


class GPT2(nn.Module):
    def __init__(self, c: GPT2Config):
        super().__init__()
        self.c = c
        self.wte = nn.Embedding(c.vocab, c.d_model)
        if c.rotary == 0:
            self.wpe = nn.Embedding(c.n_ctx, c.d_model)
        self.blocks = nn.ModuleList(Block(c) for _ in range(c.n_layer))
        self.ln_f = nn.LayerNorm(c.d_model)
        self.apply(self._init)
        for blk in self.blocks:
            for lin in (blk.proj, blk.out):
                nn.init.normal_(lin.weight, std=0.02 / math.sqrt(2 * c.n_layer))
        self._plan(self.wte.weight.device)

    def _apply(self, fn, *args, **kwargs):
        super()._apply(fn, *args, **kwargs)
        self._plan(self.wte.weight.device)  # here, as a first call may be under capture, where nothing is copied from the host
        return self

    @staticmethod
    def _init(m: nn.Module) -> None:
        if isinstance(m, nn.Linear):
            nn.init.normal_(m.weight, std=0.02)
            nn.init.zeros_(m.bias)
        elif isinstance(m, nn.Embedding):
            nn.init.normal_(m.weight, std=0.02)

    def _plan(self, device: torch.device) -> Optional[ops.Rotary]:
        """The rotary frequencies on ``device``, made once per device: when the model is built or moved."""
        c = self.c
        if c.rotary == 0:
            return None
        plans = self.__dict__.setdefault("_plans", {})
        if device not in plans:
            plans[device] = ops.Rotary(c.rotary, c.rotary_base, c.rotary_interleaved, c.rotary_scaling, c.rotary_factor,
                                       c.n_ctx, device=device)
        return plans[device]

    def _trunk(self, idx: torch.Tensor, lengths: Optional[torch.Tensor], cache: Optional[KVCache]) -> torch.Tensor:
        b, t = idx.shape
        x = self.wte(idx)
        if self.c.rotary == 0:
            x = x + self.wpe(torch.arange(t, device=idx.device))
        plan = self._plan(idx.device)
        for i, blk in enumerate(self.blocks):
            x = blk(x, plan, lengths, None if cache is None else (cache.k[i], cache.v[i]))
        return x

    def forward(self, idx: torch.Tensor, targets: Optional[torch.Tensor] = None,
                teacher: Optional[Tuple[torch.Tensor, torch.Tensor]] = None, temperature: float = 1.0,
                hard_weight: float = 0.5, lengths: Optional[torch.Tensor] = None):
        """Logits [B, T, vocab]; with ``targets`` [B, T] the cross entropy; with
        ``teacher`` (ids and logits, [B, T, K]) the distillation loss, in which the
        cross entropy against ``targets`` has the weight ``hard_weight``
        (cail_b200.ops.distill_loss).  ``lengths`` (int32 [B]) are the sequences'
        lengths in a padded batch: pad ``targets`` with -100.  With a teacher and
        no targets, the positions behind a length are left out of the loss."""
        logits = F.linear(self.ln_f(self._trunk(idx, lengths, None)), self.wte.weight)
        if teacher is not None:
            ids, top = (z.reshape(-1, z.size(-1)) for z in teacher)
            if targets is None:
                hard_weight = 0.0  # targets then only say which positions count
                if lengths is not None:
                    targets = torch.where(torch.arange(idx.size(1), device=idx.device) < lengths[:, None], 0, -100)
            return ops.distill_loss(logits.view(-1, logits.size(-1)), ids, top, None if targets is None else targets.reshape(-1),
                                    temperature=temperature, hard_weight=hard_weight)
        if targets is None:
            return logits
        return F.cross_entropy(logits.view(-1, logits.size(-1)), targets.view(-1))

    def new_cache(self, batch: int, length: Optional[int] = None) -> KVCache:
        """An empty cache for ``length`` tokens per sequence (n_ctx if not given)."""
        length = self.c.n_ctx if length is None else length
        if length < 1 or (self.c.rotary == 0 and length > self.c.n_ctx):
            raise ValueError(f"a cache of {length} tokens; learned positions reach {self.c.n_ctx}")
        return KVCache(self.c, batch, length, self.wte.weight.device, self.wte.weight.dtype)

    @torch.no_grad()
    def prefill(self, idx: torch.Tensor, cache: KVCache, lengths: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Puts the prompts idx [B, T] into an empty cache; the logits that
        follow each prompt, [B, vocab].  ``lengths`` (int32 [B], at least 1 each)
        when they are of unequal length."""
        b, t = idx.shape
        if cache.filled:
            raise ValueError("prefill needs an empty cache")
        if not 1 <= t <= cache.length or b != cache.lengths.numel():
            raise ValueError(f"prompts {tuple(idx.shape)} do not fit a cache of {cache.lengths.numel()} x {cache.length}")
        x = self._trunk(idx, lengths, cache)
        if lengths is None:
            cache.lengths.fill_(t)
        else:
            cache.lengths.copy_(lengths)
            cache.lengths.clamp_(0, t)
        cache.filled = t
        last = (cache.lengths.long() - 1).clamp_(min=0)
        return F.linear(self.ln_f(x[torch.arange(b, device=x.device), last]), self.wte.weight)

    @torch.no_grad()
    def decode(self, idx: torch.Tensor, cache: KVCache) -> torch.Tensor:
        """Appends one token per sequence, idx [B], and gives the logits that
        follow, [B, vocab].  Captured into a CUDA graph, each replay appends a
        token; the caller counts them: past the cache's length they overwrite
        its last place."""
        if idx.shape != cache.lengths.shape:
            raise ValueError(f"one token for each of {cache.lengths.numel()} sequences, got {tuple(idx.shape)}")
        if cache.filled >= cache.length:
            raise ValueError(f"the cache is full ({cache.length} tokens)")
        at = cache.lengths.clamp(max=cache.length - 1).long()
        x = self.wte(idx)
        if self.c.rotary == 0:
            x = x + self.wpe(at)
        cache.lengths += 1
        cache.filled += 1
        plan = self._plan(idx.device)
        for blk, k, v in zip(self.blocks, cache.k, cache.v):
            x = blk.decode(x, plan, k, v, at, cache.lengths)
        return F.linear(self.ln_f(x), self.wte.weight)

    def num_params(self) -> int:
        return sum(p.numel() for p in self.parameters())

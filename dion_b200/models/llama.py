"""Llama-3-shaped decoder (grouped-query attention, SwiGLU feed-forward, RMSNorm with
learnable gains, rotary embedding, untied embedding / lm_head) on the kernels of
:mod:`dion_b200.ops.nn`.  The reference ships no Llama model; this one exists so that the
optimizers can be exercised and benchmarked at the 8B shape (4096 x 4096, 1024 x 4096,
14336 x 4096 and 4096 x 14336 matrices) under FSDP2.

All 2-D block weights go to Dion / Muon; the 1-D norm gains, the embedding and the lm_head
go to the scalar optimizer, as `make_llama_param_groups` arranges.
"""

from __future__ import annotations

import math
from dataclasses import dataclass
from typing import List, Optional

import torch
import torch.nn as nn
from torch.distributed.device_mesh import DeviceMesh
from torch.distributed.tensor import Shard

from ..ops import nn as K
from .generation import CacheStep, PagedCache, generate_cached, generate_drafted
from .gpt import _refuse_drafts_of_shards


@dataclass
class LlamaConfig:
    sequence_len: int = 4096
    vocab_size: int = 128256
    n_layer: int = 32
    n_head: int = 32
    n_kv_head: int = 8
    n_embd: int = 4096
    ffn_dim: int = 14336
    rope_theta: float = 500000.0
    norm_eps: float = 1e-5

    @staticmethod
    def llama3_8b(**overrides) -> "LlamaConfig":
        return LlamaConfig(**overrides)


class RMSNormGain(nn.Module):
    def __init__(self, dim: int, eps: float):
        super().__init__()
        self.weight = nn.Parameter(torch.ones(dim))
        self.eps = eps

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return K.rms_norm_gain(x, self.weight, self.eps)


class LlamaAttention(nn.Module):
    def __init__(self, cfg: LlamaConfig):
        super().__init__()
        self.n_head, self.n_kv_head = cfg.n_head, cfg.n_kv_head
        self.head_dim = cfg.n_embd // cfg.n_head
        self.wq = nn.Linear(cfg.n_embd, cfg.n_head * self.head_dim, bias=False)
        self.wk = nn.Linear(cfg.n_embd, cfg.n_kv_head * self.head_dim, bias=False)
        self.wv = nn.Linear(cfg.n_embd, cfg.n_kv_head * self.head_dim, bias=False)
        self.wo = nn.Linear(cfg.n_head * self.head_dim, cfg.n_embd, bias=False)
        self.rope_theta = cfg.rope_theta
        self._tables = None

    def _rope(self, T: int, device):
        if self._tables is None or self._tables[0].shape[0] != T or self._tables[0].device != torch.device(device):
            self._tables = K.rotary_tables(T, self.head_dim, device, self.rope_theta)
        return self._tables

    def forward(self, h: torch.Tensor, residual: torch.Tensor) -> torch.Tensor:
        B, T, _ = h.shape
        q = K.linear(h, self.wq.weight).view(B, T, self.n_head, self.head_dim)
        k = K.linear(h, self.wk.weight).view(B, T, self.n_kv_head, self.head_dim)
        v = K.linear(h, self.wv.weight).view(B, T, self.n_kv_head, self.head_dim)
        cos, sin = self._rope(T, h.device)
        q = K.rope(q, cos, sin)
        k = K.rope(k, cos, sin)
        y = K.causal_attention(q, k, v)
        return K.linear(y, self.wo.weight, residual=residual)

    def forward_cached(self, h: torch.Tensor, residual: torch.Tensor, step: CacheStep, layer: int) -> torch.Tensor:
        """The same for the new tokens of a cache's sequences, [1, tokens, C]."""
        q, k, v = (K.linear(h, w.weight).view(h.shape[1], -1, self.head_dim) for w in (self.wq, self.wk, self.wv))
        y = step.attend(layer, q, k, v, *step.cache.rotary(self.rope_theta))
        return K.linear(y.view(1, h.shape[1], -1), self.wo.weight, residual=residual)


class LlamaMLP(nn.Module):
    def __init__(self, cfg: LlamaConfig):
        super().__init__()
        self.w_gate = nn.Linear(cfg.n_embd, cfg.ffn_dim, bias=False)
        self.w_up = nn.Linear(cfg.n_embd, cfg.ffn_dim, bias=False)
        self.w_down = nn.Linear(cfg.ffn_dim, cfg.n_embd, bias=False)

    def forward(self, h: torch.Tensor, residual: torch.Tensor) -> torch.Tensor:
        g = K.linear(h, self.w_gate.weight)
        u = K.linear(h, self.w_up.weight)
        return K.linear(K.swiglu(g, u), self.w_down.weight, residual=residual)


class LlamaBlock(nn.Module):
    def __init__(self, cfg: LlamaConfig):
        super().__init__()
        self.attention_norm = RMSNormGain(cfg.n_embd, cfg.norm_eps)
        self.attention = LlamaAttention(cfg)
        self.ffn_norm = RMSNormGain(cfg.n_embd, cfg.norm_eps)
        self.feed_forward = LlamaMLP(cfg)

    def forward(self, x: torch.Tensor, step: Optional[CacheStep] = None, layer: int = 0) -> torch.Tensor:
        if step is not None:
            x = self.attention.forward_cached(self.attention_norm(x), x, step, layer)
        else:
            x = self.attention(self.attention_norm(x), x)
        x = self.feed_forward(self.ffn_norm(x), x)
        return x


class Llama(nn.Module):
    def __init__(self, cfg: LlamaConfig):
        super().__init__()
        self.config = cfg
        self.tok_embeddings = nn.Embedding(cfg.vocab_size, cfg.n_embd)
        self.layers = nn.ModuleList([LlamaBlock(cfg) for _ in range(cfg.n_layer)])
        self.norm = RMSNormGain(cfg.n_embd, cfg.norm_eps)
        self.output = nn.Linear(cfg.n_embd, cfg.vocab_size, bias=False)

    def init_weights(self, std: float = 0.02) -> None:
        for m in self.modules():
            if isinstance(m, nn.Linear):
                nn.init.normal_(m.weight, mean=0.0, std=std)
            elif isinstance(m, nn.Embedding):
                nn.init.normal_(m.weight, mean=0.0, std=1.0)
            elif isinstance(m, RMSNormGain):
                nn.init.ones_(m.weight)

    def forward(self, idx: torch.Tensor, targets: Optional[torch.Tensor] = None, return_logits: bool = False,
                cache: Optional[CacheStep] = None):
        if cache is not None:
            with cache.passing(idx, targets):
                return self._forward_cached(idx, cache)
        dtype = torch.bfloat16 if idx.is_cuda else self.output.weight.dtype
        x = K.embedding(idx, self.tok_embeddings.weight, dtype)
        for layer in self.layers:
            x = layer(x)
        x = self.norm(x)
        if targets is not None and not return_logits:
            return K.linear_cross_entropy(x, self.output.weight, targets, ignore_index=-1)
        if targets is None:
            if not return_logits:
                return None
            x = x[:, [-1], :]
        return K.linear(x, self.output.weight).float()

    def _forward_cached(self, tokens: torch.Tensor, step: CacheStep) -> torch.Tensor:
        """fp32 logits [rows that the step wants, vocabulary] of the new tokens of a cache's sequences."""
        dtype = torch.bfloat16 if tokens.is_cuda else self.output.weight.dtype
        x = K.embedding(tokens, self.tok_embeddings.weight, dtype)[None]
        for i, layer in enumerate(self.layers):
            x = layer(x, step=step, layer=i)
        return K.linear(self.norm(step.wanted(x[0])[None]), self.output.weight)[0].float()

    def new_cache(self, sequences: int, max_len: Optional[int] = None, page_size: int = 64, pages: Optional[int] = None) -> PagedCache:
        """An empty cache for `sequences` texts of up to `max_len` tokens (the model's by default)."""
        c, w = self.config, self.output.weight
        max_len = c.sequence_len if max_len is None else max_len
        if max_len > c.sequence_len:
            raise ValueError(f"a cache for {max_len} tokens, the model takes {c.sequence_len}")
        dtype = torch.bfloat16 if w.is_cuda else w.dtype
        return PagedCache(c.n_layer, c.n_kv_head, c.n_embd // c.n_head, sequences, max_len, page_size, pages, dtype, w.device)

    @torch.no_grad()
    def generate(self, input_ids: torch.LongTensor, max_new_tokens: int, temperature: float = 1.0, top_k: Optional[int] = None,
                 draft_model: Optional["Llama"] = None, draft_tokens: int = 4) -> torch.LongTensor:
        """Sample `max_new_tokens` tokens over a paged cache; prompt and new tokens have to fit `sequence_len`.  `draft_model`
        and `draft_tokens` as for ``GPT.generate``."""
        if draft_model is not None:
            _refuse_drafts_of_shards(self, draft_model)
            return generate_drafted(self, self.config.sequence_len, draft_model, draft_model.config.sequence_len, draft_tokens,
                                    input_ids, max_new_tokens, temperature, top_k)
        return generate_cached(self, self.config.sequence_len, input_ids, max_new_tokens, temperature, top_k)


def make_llama_param_groups(model: Llama, scalar_opt: str = "adamw", lr: float = 0.01) -> List[dict]:
    """Matrices of the blocks -> default (Dion / Muon) group; gains, embedding, lm_head ->
    the scalar optimizer, no weight decay."""
    matrices = [p for layer in model.layers for p in layer.parameters() if p.ndim == 2]
    gains = [p for p in model.parameters() if p.ndim == 1]
    return [
        dict(params=matrices),
        dict(params=gains, algorithm=scalar_opt, lr=lr, weight_decay=0),
        dict(params=list(model.tok_embeddings.parameters()), algorithm=scalar_opt, lr=lr, weight_decay=0),
        dict(params=list(model.output.parameters()), algorithm=scalar_opt,
             lr=lr / math.sqrt(model.config.n_embd), weight_decay=0),
    ]


def parallelize_llama_model(model: Llama, fsdp_mesh: DeviceMesh, reshard_after_forward: bool = True) -> None:
    """FSDP2 per block with bf16 parameters / fp32 reduction.  Every matrix is sharded along
    its *long* dimension (rows of gate/up, columns of down), so that Dion's P factor - the
    thing that is reduced, orthonormalised and gathered - spans the short dimension."""
    from torch.distributed.fsdp import MixedPrecisionPolicy, fully_shard

    mp = MixedPrecisionPolicy(param_dtype=torch.bfloat16, reduce_dtype=torch.float32)
    for layer in model.layers:
        ff, at = layer.feed_forward, layer.attention
        shard = {ff.w_gate.weight: Shard(0), ff.w_up.weight: Shard(0), ff.w_down.weight: Shard(1),
                 at.wq.weight: Shard(1), at.wk.weight: Shard(1), at.wv.weight: Shard(1), at.wo.weight: Shard(0)}
        fully_shard(layer, mesh=fsdp_mesh, mp_policy=mp, reshard_after_forward=reshard_after_forward,
                    shard_placement_fn=lambda p, m=shard: m.get(p))
    top = {model.tok_embeddings.weight: Shard(1), model.output.weight: Shard(1)}
    fully_shard(model, mesh=fsdp_mesh, mp_policy=mp, reshard_after_forward=False,
                shard_placement_fn=lambda p, m=top: m.get(p))
    from ..parallel import fsdp_comm

    fsdp_comm.install(model)

"""Sampling from a decoder with a paged cache of keys and values, with or without a smaller model that drafts.

A model that can be sampled this way has ``new_cache(sequences, max_len, pages)`` and takes ``model(tokens, cache=step)``:
`tokens` are the new tokens of all sequences in one row, `step` a :class:`CacheStep`; it returns the fp32 logits of the rows that
the step asks for.  Both models of this package do.
"""

from __future__ import annotations

from contextlib import contextmanager
from dataclasses import dataclass
from typing import Dict, Iterator, List, Optional, Sequence, Tuple

import torch
import torch.nn.functional as F

from ..ops import paged_append, paged_attention, verify_drafts
from ..ops.nn import rotary_tables


class PagedCache:
    """Keys and values of a batch of sequences, a pool of pages per layer shared by all of them.  ``lengths`` says how many tokens
    of each sequence are cached; pages are taken from the pool as sequences grow and given back by ``cut``."""

    def __init__(self, layers: int, kv_heads: int, head_dim: int, sequences: int, max_len: int, page_size: int = 64,
                 pages: Optional[int] = None, dtype: torch.dtype = torch.bfloat16, device="cuda"):
        if page_size < 16 or page_size & (page_size - 1):
            raise ValueError(f"the size of a page is a power of two from 16 on, not {page_size}")
        if min(layers, kv_heads, head_dim, sequences, max_len) < 1:
            raise ValueError("layers, heads, head dimension, sequences and their length are positive")
        each = -(-max_len // page_size)
        pages = sequences * each if pages is None else pages
        self.page_size, self.max_len = page_size, max_len
        pool = torch.empty(layers, 2, max(pages, 1), page_size, kv_heads, head_dim, dtype=dtype, device=device)
        self.k, self.v = [p[0] for p in pool], [p[1] for p in pool]
        self.lengths: List[int] = [0] * sequences
        self._free = list(range(pages - 1, -1, -1))
        self._pages: List[List[int]] = [[] for _ in range(sequences)]
        self._table = torch.zeros(sequences, each, dtype=torch.int32)
        self._on_device: Optional[torch.Tensor] = None
        self._changes = 0  # of the lengths so far
        self._rotary: Dict[float, Tuple[torch.Tensor, torch.Tensor]] = {}

    @property
    def device(self) -> torch.device:
        return self.k[0].device

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def rotary(self, base: float) -> Tuple[torch.Tensor, torch.Tensor]:
        """cos and sin of every position, for all layers.  The layers' own tables are left alone: a captured graph of theirs may
        go on reading them."""
        if base not in self._rotary:
            self._rotary[base] = rotary_tables(self.max_len, self.k[0].shape[-1], self.device, base)
        return self._rotary[base]

    def step(self, counts: Sequence[int], all_rows: bool = False) -> "CacheStep":
        """Room for ``counts[b]`` new tokens of each sequence (none is allowed, not of all), which count as cached from now on, unless
        the model's pass over the step fails."""
        if len(counts) != len(self.lengths) or any(n < 0 for n in counts) or not any(counts):
            raise ValueError(f"{len(self.lengths)} sequences need as many counts, none below zero, one above, not {list(counts)}")
        ends = [p + n for p, n in zip(self.lengths, counts)]
        if max(ends) > self.max_len:
            raise ValueError(f"a sequence of {max(ends)} tokens in a cache for {self.max_len}")
        need = [max(-(-e // self.page_size) - len(p), 0) if n else 0 for e, n, p in zip(ends, counts, self._pages)]
        if sum(need) > len(self._free):
            raise RuntimeError(f"the cache has {len(self._free)} free pages of {self.page_size} tokens, {sum(need)} are needed")
        for b, n in enumerate(need):
            for _ in range(n):
                self._table[b, len(self._pages[b])] = self._free[-1]
                self._pages[b].append(self._free.pop())
                self._on_device = None
        if self._on_device is None:
            self._on_device = self._table.to(self.device, copy=True)
        offsets = [0]
        for n in counts:
            offsets.append(offsets[-1] + n)
        small = torch.tensor([offsets, self.lengths + [0]], dtype=torch.int32).to(self.device)
        past, self.lengths = self.lengths, ends
        self._changes += 1
        return CacheStep(self, self._on_device, small[0], small[1, :-1], offsets[-1], max(counts),
                         None if all_rows else [e - 1 for e, n in zip(offsets[1:], counts) if n], list(counts), past, self._changes)

    def cut(self, lengths: Sequence[int]) -> None:
        """Shortens the sequences to `lengths`; pages that hold nothing any more go back to the pool."""
        if len(lengths) != len(self.lengths) or any(not 0 <= n <= p for n, p in zip(lengths, self.lengths)):
            raise ValueError(f"sequences of {self.lengths} tokens cannot be cut to {list(lengths)}")
        self.lengths = list(lengths)
        self._changes += 1
        for pages, n in zip(self._pages, lengths):
            while len(pages) > -(-n // self.page_size):
                self._free.append(pages.pop())


@dataclass
class CacheStep:
    """One forward pass over a cache: whose tokens are new, how many in all and of a sequence at most, and of which rows the
    logits are wanted (None: of all)."""

    cache: PagedCache
    page_table: torch.Tensor
    offsets: torch.Tensor
    lengths: torch.Tensor
    tokens: int
    max_new: int
    rows: Optional[List[int]]
    counts: Sequence[int] = ()  # of each sequence: its new tokens, and those that were cached before
    past: Sequence[int] = ()
    change: int = -1  # which of the cache's changes this step was
    state: str = "taken"  # or "passed", or "back" where the cache has taken the tokens back

    @contextmanager
    def passing(self, tokens: torch.Tensor, targets: Optional[torch.Tensor]) -> Iterator[None]:
        """Around a model's pass over this step.  Where the pass fails, the pages may hold anything in place of its tokens: if nothing
        has changed the lengths since, the cache is then as it was before the step, which can be passed again or dropped."""
        try:
            self.check(tokens, targets)
            if self.state == "back":
                if self.cache.lengths != list(self.past):
                    raise ValueError("a pass over this step has failed and the cache has changed since: take another step")
                again = self.cache.step(self.counts)
                self.page_table, self.offsets, self.lengths, self.change = again.page_table, again.offsets, again.lengths, again.change
            self.state = "taken"
            yield
            self.state = "passed"
        except BaseException:
            ends = [p + n for p, n in zip(self.past, self.counts)]
            if self.state == "taken" and self.cache._changes == self.change and self.cache.lengths == ends:
                self.cache.cut(self.past)
                self.state = "back"
            raise

    def check(self, tokens: torch.Tensor, targets: Optional[torch.Tensor]) -> None:
        """Refuses what a model's pass over this step cannot take."""
        if targets is not None:
            raise ValueError("a pass over a cache has no loss: targets go without")
        if list(tokens.shape) != [self.tokens]:
            raise ValueError(f"the step has room for {self.tokens} new tokens in one row, not for {list(tokens.shape)}")

    def attend(self, layer: int, q, k, v, cos, sin, norm_eps: Optional[float] = None) -> torch.Tensor:
        """Rotates, caches and attends: q, k, v of the new tokens, [tokens, heads, head_dim], to the attention's result."""
        where = (self.cache.k[layer], self.cache.v[layer], self.page_table, self.offsets, self.lengths)
        q = paged_append(q, k, v, cos, sin, *where, norm_eps=norm_eps)
        return paged_attention(q, *where, max_new=self.max_new)

    def wanted(self, x: torch.Tensor) -> torch.Tensor:
        """Of x [tokens, features] the rows whose logits are wanted."""
        return x if self.rows is None else x[torch.tensor(self.rows, device=x.device)]


def probabilities(logits: torch.Tensor, temperature: float, top_k: Optional[int]) -> torch.Tensor:
    """What the next token is drawn from."""
    logits = logits / temperature
    if top_k is not None:
        v, _ = torch.topk(logits, min(top_k, logits.size(-1)))
        logits[logits < v[..., [-1]]] = -float("Inf")
    return F.softmax(logits, dim=-1)


def _fits(input_ids: torch.Tensor, max_new_tokens: int, limit: int) -> Tuple[int, int]:
    if input_ids.dim() != 2 or input_ids.shape[0] < 1 or input_ids.shape[1] < 1:
        raise ValueError(f"prompts are [sequences, tokens], at least one of either, not {list(input_ids.shape)}")
    B, T = input_ids.shape
    if T + max_new_tokens - 1 > limit:
        raise ValueError(f"{T} tokens and {max_new_tokens} new ones do not fit the model's {limit}: a cache does not slide")
    return B, T


@torch.no_grad()
def generate_cached(model, limit: int, input_ids: torch.Tensor, max_new_tokens: int, temperature: float = 1.0,
                    top_k: Optional[int] = None, page_size: int = 64) -> torch.Tensor:
    """Samples `max_new_tokens` tokens per sequence; each pass sees the new tokens alone."""
    B, T = _fits(input_ids, max_new_tokens, limit)
    if max_new_tokens < 1:
        return input_ids
    cache = model.new_cache(B, T + max_new_tokens - 1, page_size)
    idx, new = input_ids, input_ids
    for _ in range(max_new_tokens):
        logits = model(new.reshape(-1), cache=cache.step([new.shape[1]] * B))
        new = torch.multinomial(probabilities(logits, temperature, top_k), num_samples=1)
        idx = torch.cat([idx, new], dim=1)
    return idx


@torch.no_grad()
def generate_drafted(model, limit: int, draft_model, draft_limit: int, draft_tokens: int, input_ids: torch.Tensor,
                     max_new_tokens: int, temperature: float = 1.0, top_k: Optional[int] = None, page_size: int = 64) -> torch.Tensor:
    """The same with `draft_model` proposing up to `draft_tokens` tokens at a time, which `model` checks in one pass.  The tokens
    are distributed as without it; with a draft that is often right there are fewer passes of the large model."""
    if draft_tokens < 1:
        raise ValueError(f"at least one drafted token at a time, not {draft_tokens}")
    limit = min(limit, draft_limit)
    B, T = _fits(input_ids, max_new_tokens, limit)
    if max_new_tokens < 1:
        return input_ids
    total, device = T + max_new_tokens, input_ids.device
    room = min(limit, total - 1 + draft_tokens)
    cache, drafts = (m.new_cache(B, room, page_size) for m in (model, draft_model))
    idx = torch.zeros(B, total + draft_tokens, dtype=input_ids.dtype, device=device)
    idx[:, :T] = input_ids
    if T > 1:
        for m, c in ((model, cache), (draft_model, drafts)):
            m(input_ids[:, :-1].reshape(-1), cache=c.step([T - 1] * B))
    have = [T] * B  # tokens of each sequence; all but the last are in the model's cache
    while min(have) < total:
        active = [b for b in range(B) if have[b] < total]
        at = torch.tensor(active, device=device)
        k = min(draft_tokens, max(total - have[b] for b in active) - 1, room - max(have[b] for b in active))

        def counts(n):
            out = [0] * B
            for b in active:
                out[b] = n(b)
            return out

        q, proposed = [], []
        for i in range(k):
            # what the draft's cache lacks first: the last token, and the one before where all drafts of the round before stood
            feed = torch.cat([idx[b, drafts.lengths[b]:have[b]] for b in active]) if i == 0 else proposed[-1].reshape(-1)
            step = drafts.step(counts(lambda b: have[b] - drafts.lengths[b]) if i == 0 else counts(lambda b: 1))
            q.append(probabilities(draft_model(feed, cache=step), temperature, top_k))
            proposed.append(torch.multinomial(q[-1], num_samples=1))
        tokens = torch.cat(proposed, 1) if k else torch.zeros(len(active), 0, dtype=torch.int64, device=device)
        last = idx[at, torch.tensor([have[b] - 1 for b in active], device=device)]
        logits = model(torch.cat([last[:, None], tokens], 1).reshape(-1), cache=cache.step(counts(lambda b: k + 1), all_rows=True))
        p = probabilities(logits, temperature, top_k).view(len(active), k + 1, -1)
        accepted, token = verify_drafts(p, torch.stack(q, 1) if k else p[:, :0], tokens, torch.rand(len(active), k + 1, device=device))
        place = torch.arange(k + 1, device=device)
        row = torch.where(place < accepted[:, None], F.pad(tokens, (0, 1)), token[:, None])  # the drafts that stand and the next
        for j, (b, a) in enumerate(zip(active, accepted.tolist())):
            idx[b, have[b]:have[b] + a + 1] = row[j, :a + 1]
            have[b] += a + 1
        cache.cut([min(have[b] - 1, cache.lengths[b]) for b in range(B)])
        drafts.cut([min(have[b] - 1, drafts.lengths[b]) for b in range(B)])
    return idx[:, :total]

"""A paged cache of keys and values, and the operators that sampling from a decoder needs around it.

``paged_append`` rotates the queries and keys of new tokens (and normalises them, as the GPT model does), writes keys and
values into the pages and hands the queries on; ``paged_attention`` is causal attention of those tokens over the pages;
``verify_drafts`` decides which tokens of a cheaper model stand.

Pages are ``[pages, page_size, kv heads, head_dim]`` in any memory order with the head dimension contiguous; the size of a page
is a power of two from 16 on.  ``page_table: [sequences, most pages]`` names the pages of each sequence in order; what lies behind
its last page is not looked at.  The new tokens of all sequences follow one another in one tensor: those of sequence b are rows
``new_offsets[b]`` to ``new_offsets[b + 1]`` (the first offset is zero), and ``lengths[b]`` tokens of it are in the cache already,
so that its row i stands at position ``lengths[b] + i``.  Sequences may have no new token.  Rows behind the last sequence belong to
nobody: their results are zero, nothing of theirs is written to the pages.  Table, offsets and lengths are int32.

As for the other model ops, bf16 tensors on a GPU (head dimension 64 or 128) run the kernels, anything else plain PyTorch of the
same semantics.  The kernels never wait for the host and can be captured: what the host cannot see (a position beyond the page table
or the rotation tables, a page that does not exist, offsets that run backwards) sets the device's status word, which
``check_status`` raises, and reaches no memory outside the tensors; the results of such a call are not to be used.  The plain path
raises ``ValueError``.  None of the three has a gradient: inputs that
ask for one are refused, and the kernels refuse forward-mode tangents, which the plain path carries.
"""

from __future__ import annotations

import math
from typing import Optional, Tuple

import torch

from . import runtime


def _no_gradients(name: str, *tensors: Optional[torch.Tensor]) -> None:
    for t in tensors:
        if t is not None and t.requires_grad and torch.is_grad_enabled():
            raise RuntimeError(f"{name} has no gradient: call it under torch.no_grad() or with detached inputs")


_kernels = None  # the operators of the library, from the first call with CUDA tensors on


def _load(t: torch.Tensor):
    global _kernels
    runtime.use_cuda_kernels(t)
    lib = torch.ops.dion_b200
    _kernels = (lib.paged_append.default, lib.paged_attention.default, lib.verify_drafts.default)
    return _kernels


# --------------------------------------------------------------------------- plain path

def _plain_layout(name, q, others, k_pages, v_pages, page_table, new_offsets, lengths):
    """The checks that the kernels' bindings make, and (tokens cached, first row, rows) of every sequence."""
    def need(ok, what):
        if not ok:
            raise ValueError(f"{name}: {what}")

    need(q.dim() == 3 and all(t.dim() == 3 for t in others), "queries, keys and values are [tokens, heads, head_dim]")
    need(k_pages.dim() == 4 and v_pages.shape == k_pages.shape, "key and value pages are [pages, page_size, kv heads, head_dim], both of one shape")
    for t in (*others, k_pages, v_pages):
        need(t.dtype == q.dtype and t.device == q.device, f"tensors of one type on one device, not {t.dtype} on {t.device} beside {q.dtype} on {q.device}")
    size, heads, dim = k_pages.shape[1:]
    need(size >= 16 and size & (size - 1) == 0, f"the size of a page is a power of two from 16 on, not {size}")
    need(q.shape[2] == dim and q.shape[1] > 0 and heads > 0 and q.shape[1] % heads == 0,
         f"{q.shape[1]} query heads of {q.shape[2]} do not go with {heads} cached heads of {dim}")
    for t in others:
        need(t.shape == (q.shape[0], heads, dim), f"keys and values are [{q.shape[0]}, {heads}, {dim}], not {list(t.shape)}")
    for t, d in ((page_table, 2), (new_offsets, 1), (lengths, 1)):
        need(t.dtype == torch.int32 and t.device == q.device and t.dim() == d, "page table, offsets and lengths are int32, on the device of the queries")
    n = lengths.shape[0]
    need(page_table.shape[0] == n and new_offsets.shape[0] == n + 1, f"{n} lengths need as many rows of the page table and {n + 1} offsets")
    at, past = new_offsets.tolist(), lengths.tolist()
    need(at[0] == 0 and all(a <= b for a, b in zip(at, at[1:])) and at[-1] <= q.shape[0], "offsets start at zero, never fall and end within the tokens")
    out = []
    for b, (a, e, p) in enumerate(zip(at, at[1:], past)):
        if e > a:
            used = -(-(p + e - a) // size)
            need(p >= 0 and used <= page_table.shape[1], f"sequence {b}: {p} + {e - a} tokens do not fit {page_table.shape[1]} pages of {size}")
            pages = page_table[b, :used]
            need(int(pages.min()) >= 0 and int(pages.max()) < k_pages.shape[0], f"sequence {b}: a page that does not exist")
        out.append((p, a, e - a))
    return out


def _wide(t: torch.Tensor) -> torch.Tensor:
    return t if t.dtype == torch.float64 else t.float()


def _rotated(x, cos, sin, eps):
    d = x.shape[-1] // 2
    x1, x2 = _wide(x[..., :d]), _wide(x[..., d:])
    y = torch.cat([x1 * cos + x2 * sin, x2 * cos - x1 * sin], dim=-1)
    if eps is not None:
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + eps)
    return y.to(x.dtype)


def _append_plain(q, k, v, cos, sin, k_pages, v_pages, page_table, new_offsets, lengths, eps):
    layout = _plain_layout("paged_append", q, (k, v), k_pages, v_pages, page_table, new_offsets, lengths)
    half = q.shape[2] // 2
    if q.shape[2] % 2 or cos.dim() != 2 or cos.shape[1] != half or sin.shape != cos.shape or sin.dtype != cos.dtype:
        raise ValueError(f"paged_append: cos and sin are two tables [positions, {half}] of one type")
    if cos.shape[0] >= 2 ** 31:
        raise ValueError("paged_append: more than 2^31 - 1 rows of the rotation tables")
    if any(n and p + n > cos.shape[0] for p, _, n in layout):
        raise ValueError(f"paged_append: a position beyond the {cos.shape[0]} rows of the rotation tables")
    out = torch.zeros(q.shape, dtype=q.dtype, device=q.device)
    size = k_pages.shape[1]
    for b, (p, a, n) in enumerate(layout):
        if n == 0:
            continue
        c, s = _wide(cos[p:p + n])[:, None], _wide(sin[p:p + n])[:, None]
        at = torch.arange(p, p + n, device=q.device)
        page, row = page_table[b].long()[at // size], at % size
        out[a:a + n] = _rotated(q[a:a + n], c, s, eps)
        k_pages[page, row] = _rotated(k[a:a + n], c, s, eps)
        v_pages[page, row] = v[a:a + n]
    return out


def _attention_plain(q, k_pages, v_pages, page_table, new_offsets, lengths, scale, max_new):
    layout = _plain_layout("paged_attention", q, (), k_pages, v_pages, page_table, new_offsets, lengths)
    size, heads, dim = k_pages.shape[1:]
    out = torch.zeros(q.shape, dtype=q.dtype, device=q.device)
    for b, (p, a, n) in enumerate(layout):
        if n > max_new:
            raise ValueError(f"paged_attention: sequence {b} has {n} new tokens, more than max_new = {max_new}")
        if n == 0:
            continue
        pages = page_table[b, :-(-(p + n) // size)].long()
        k, v = (_wide(t[pages].reshape(-1, heads, dim)[:p + n]) for t in (k_pages, v_pages))
        x = torch.einsum("tgrd,sgd->grts", _wide(q[a:a + n]).view(n, heads, -1, dim), k) * scale
        later = torch.arange(p + n, device=q.device)[None] > p + torch.arange(n, device=q.device)[:, None]
        y = torch.einsum("grts,sgd->tgrd", torch.softmax(x.masked_fill(later, -math.inf), -1), v)
        out[a:a + n] = y.reshape(n, -1, dim).to(q.dtype)
    return out


def _verify_plain(p, q, tokens, u):
    n, k = tokens.shape
    if tokens.numel() and (int(tokens.min()) < 0 or int(tokens.max()) >= p.shape[2]):
        raise ValueError("verify_drafts: a drafted token outside the vocabulary")
    every = torch.arange(n, device=p.device)
    u = u.double()
    p_of = p[:, :k].gather(-1, tokens[..., None])[..., 0].double()
    q_of = torch.ones_like(p_of) if q is None else q.gather(-1, tokens[..., None])[..., 0].double()
    accepted = (u[:, :k] * q_of < p_of).long().cumprod(-1).sum(-1)
    row = p[every, accepted].double()
    rest = row
    if k:
        last = accepted.clamp_max(k - 1)
        minus = torch.zeros_like(row).scatter_(-1, tokens[every, last][:, None], 1.0) if q is None else q[every, last].double()
        rest = torch.where((accepted < k)[:, None], row - minus, row)
    rest, row = (torch.where((t > 0) & (t < math.inf), t, 0.0) for t in (rest, row))
    rest = torch.where((rest.sum(-1) > 0)[:, None], rest, row)
    upto = rest.cumsum(-1)
    token = (upto <= u[:, k:] * upto[:, -1:]).sum(-1).clamp_max(p.shape[2] - 1)
    return accepted, torch.where(upto[:, -1] > 0, token, 0)


# --------------------------------------------------------------------------- public functions

def paged_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, k_pages: torch.Tensor,
                 v_pages: torch.Tensor, page_table: torch.Tensor, new_offsets: torch.Tensor, lengths: torch.Tensor,
                 norm_eps: Optional[float] = None) -> torch.Tensor:
    """Rotates ``q: [tokens, heads, head_dim]`` and ``k: [tokens, kv heads, head_dim]`` to their positions, writes k and v into the
    pages in place and returns the rotated q.  ``cos`` / ``sin``: ``[positions, head_dim / 2]``, bf16 or fp32, as
    ``rotary_tables`` makes them.  With `norm_eps` every head of q and k goes through an RMS norm after the rotation, as
    ``rope_qknorm`` does; without, this is ``rope``.  fp32 arithmetic, rounded once."""
    if norm_eps is not None and not norm_eps >= 0.0:
        raise ValueError(f"paged_append: norm_eps is None or not negative, not {norm_eps}")
    if q.is_cuda:
        out = (_kernels or _load(q))[0](q, k, v, cos, sin, k_pages, v_pages, page_table, new_offsets, lengths,
                                        -1.0 if norm_eps is None else norm_eps, runtime.status_tensor(q.device))
        if out is not None:
            return out
    _no_gradients("paged_append", q, k, v, cos, sin, k_pages, v_pages)
    return _append_plain(q, k, v, cos, sin, k_pages, v_pages, page_table, new_offsets, lengths, norm_eps)


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
                    new_offsets: torch.Tensor, lengths: torch.Tensor, scale: Optional[float] = None,
                    max_new: Optional[int] = None) -> torch.Tensor:
    """Causal attention of the new tokens, whose keys and values ``paged_append`` has put into the pages, over everything up to
    themselves: ``softmax(scale q K^T) V`` per head, ``[tokens, heads, head_dim]``.  `lengths` is what it was for ``paged_append``:
    without the new tokens.  Grouped heads: the kv heads divide the heads.  `scale` defaults to ``1 / sqrt(head_dim)``.  What lies in the
    pages behind a sequence's last token has no influence; the values of its own tokens meet every row of their chunk, those of later
    ones with weight zero, and have to be finite.  The kernels round the softmax's weights to bf16 before they meet the values, their sum is
    that of the unrounded ones in fp32: an output is off by at most a half step of bf16 of ``sum p |v|`` beside its own rounding.  The
    plain path keeps fp32 weights.

    `max_new`: the most new tokens of a sequence, where the host knows it; a longer sequence is an error.  It goes into the choice
    of the kernel, as does the width of the page table, which says how long a sequence can be; any choice gives the result, to its
    roundings."""
    scale = 1.0 / math.sqrt(q.size(-1)) if scale is None else float(scale)
    if not 2.0 ** -100 <= scale <= 2.0 ** 100:
        raise ValueError(f"paged_attention: the scale is positive, from 2^-100 to 2^100, not {scale}")
    if max_new is None:
        max_new = q.size(0)
    elif max_new < 1:
        raise ValueError(f"paged_attention: max_new is at least 1, not {max_new}")
    if q.is_cuda:
        out = (_kernels or _load(q))[1](q, k_pages, v_pages, page_table, new_offsets, lengths, scale, max_new, runtime.status_tensor(q.device))
        if out is not None:
            return out
    _no_gradients("paged_attention", q, k_pages, v_pages)
    return _attention_plain(q, k_pages, v_pages, page_table, new_offsets, lengths, scale, max_new)


def verify_drafts(target_probs: torch.Tensor, draft_probs: Optional[torch.Tensor], draft_tokens: torch.Tensor,
                  uniforms: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """Which drafted tokens stand, and the token after them, so that the outcome is distributed as if the target had sampled.

    ``target_probs: [sequences, drafts + 1, vocabulary]`` (the target's distribution at each draft and behind the last),
    ``draft_probs: [sequences, drafts, vocabulary]`` (what the drafts were drawn from; None: they were certain), both fp32;
    ``draft_tokens: [sequences, drafts]`` (int64); ``uniforms: [sequences, drafts + 1]`` (fp32 in [0, 1)).  Draft i is accepted
    while ``u_i q_i(x_i) < p_i(x_i)``.  The next token is drawn with the last uniform from ``max(p - q, 0)`` at the first draft
    that fell, or from the target's row behind the last: the lowest token whose running sum exceeds u times the whole.  Sums are in
    64 bits.  Where p - q leaves nothing, p itself stands in; differences and probabilities that are negative, infinite or no
    numbers count as zero there, and a row of zeros gives token 0.  Returns ``(accepted, token)``, int64 per sequence."""
    if target_probs.is_cuda:
        return (_kernels or _load(target_probs))[2](target_probs, draft_probs, draft_tokens, uniforms, runtime.status_tensor(target_probs.device))
    _no_gradients("verify_drafts", target_probs, draft_probs, uniforms)
    p, q = target_probs, draft_probs

    def need(ok, what):
        if not ok:
            raise ValueError(f"verify_drafts: {what}")

    need(p.dim() == 3 and p.shape[1] >= 1 and p.shape[2] >= 1 and p.dtype == torch.float32, "the target's probabilities are fp32 [sequences, drafts + 1, vocabulary]")
    shape = (p.shape[0], p.shape[1] - 1)
    need(draft_tokens.shape == shape and draft_tokens.dtype == torch.int64, f"drafted tokens are int64 {list(shape)}")
    need(q is None or (q.shape == (*shape, p.shape[2]) and q.dtype == torch.float32), f"the draft's probabilities are fp32 {[*shape, p.shape[2]]}")
    need(uniforms.shape == p.shape[:2] and uniforms.dtype == torch.float32, f"uniforms are fp32 {list(p.shape[:2])}")
    need(all(t is None or t.device == p.device for t in (q, draft_tokens, uniforms)), "tensors on one device")
    return _verify_plain(p, q, draft_tokens, uniforms)

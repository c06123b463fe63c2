"""The operators of cached generation, as they are measured: appending keys and values to a paged cache with the rotation on
the way, attention of new tokens over such a cache, and the check of drafted tokens against the target's probabilities.

``listed()`` names the fixed cases, ``draw(rng)`` gives one more of the same ranges; ``prepare`` makes what a program has in
hand before the call, ``run`` is one call, ``work`` what the call cannot do without, ``exact`` what it should give, in 64 bits.
"""

from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False  # False: `run` computes the plain form; True: it calls the framework's operators

EPS = 1.1920929e-07  # of the norm over a head, as in the GPT model


# ----------------------------------------------------------------------------------------------- the cases

def _append(batch, past, new, ragged, heads, kv_heads, dim, page, norm, mix):
    return dict(op="append", batch=batch, past=past, new=new, ragged=ragged, heads=heads, kv_heads=kv_heads, dim=dim, page=page,
                norm=norm, mix=mix)


def _attend(batch, past, new, ragged, heads, kv_heads, dim, page, mix):
    return dict(op="attend", batch=batch, past=past, new=new, ragged=ragged, heads=heads, kv_heads=kv_heads, dim=dim, page=page,
                mix=mix)


def _verify(batch, drafts, vocab, certain):
    return dict(op="verify", batch=batch, drafts=drafts, vocab=vocab, certain=certain)


def listed():
    return [
        # one token of one text, GPT-160M with 6 heads of 128: what every layer of every sampled token pays
        dict(_append(1, 500, 1, False, 6, 6, 128, 64, True, 1), name="append_one_token"),
        # ragged prompts of a batch, 12 heads of 64 with the norm, small pages
        dict(_append(33, 300, 900, True, 12, 12, 64, 16, True, 2), name="append_ragged_norm"),
        # prompts of the 8B shape written at once, grouped heads
        dict(_append(8, 0, 2048, False, 32, 8, 128, 64, False, 3), name="append_prompt_8b_shape"),
        # one token of one text over a short cache: latency
        dict(_attend(1, 777, 1, False, 6, 6, 128, 16, 4), name="attend_one_token"),
        # a batch of texts of all lengths, one token each, 8B shape: the bandwidth of the cache
        dict(_attend(64, 8000, 1, True, 32, 8, 128, 64, 5), name="attend_batch_8b_shape"),
        # few sequences with a long cache: the cache has to be split over the GPU
        dict(_attend(2, 120000, 1, False, 32, 8, 128, 128, 6), name="attend_long_cache"),
        # five drafted tokens each of a ragged batch, GPT-160M with 12 heads of 64
        dict(_attend(16, 1000, 5, True, 12, 12, 64, 32, 7), name="attend_drafts"),
        # prompts of all lengths from nothing in the cache, 12 heads of 64
        dict(_attend(48, 0, 1024, True, 12, 12, 64, 64, 8), name="attend_ragged_prompts"),
        # a long chunk on top of a cached prefix, 8B shape: the rate of the tensor cores
        dict(_attend(2, 6000, 2048, False, 32, 8, 128, 64, 9), name="attend_chunk_8b_shape"),
        # four drafted tokens of one text, the GPT-2 vocabulary
        dict(_verify(1, 4, 50304, False), name="verify_one"),
        # a batch, 8B-shaped vocabulary
        dict(_verify(64, 7, 128256, False), name="verify_batch"),
        # drafts that were looked up rather than sampled
        dict(_verify(24, 5, 50304, True), name="verify_certain"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


_LIMIT = {"append": "append_prompt_8b_shape", "attend": "attend_chunk_8b_shape", "verify": "verify_batch"}


def draw(rng):
    limits = {c["name"]: work(c) for c in listed()}
    op = rng.choice(["append", "attend", "attend", "verify"])
    most = limits[_LIMIT[op]]
    # a cache of long texts reads more and computes less than a chunk does
    most_bytes = max(most["bytes"], limits["attend_batch_8b_shape"]["bytes"]) if op == "attend" else most["bytes"]
    while True:
        if op == "verify":
            case = _verify(_log(rng, 1, 64), rng.randint(1, 8), rng.choice([50304, 128256, _log(rng, 500, 130000)]), rng.random() < 0.25)
        else:
            heads, kv_heads, dim = rng.choice([(6, 6, 128), (12, 12, 64), (32, 8, 128), (16, 2, 64), (8, 1, 128), (12, 4, 64)])
            new = rng.choice([1, 1, rng.randint(2, 9), _log(rng, 10, 2048)])
            past = rng.choice([0, _log(rng, 1, 8000), _log(rng, 1000, 120000)])
            if past == 0 and new == 1:
                continue
            batch, page, ragged = _log(rng, 1, 64), rng.choice([16, 32, 64, 128]), rng.random() < 0.7
            mix = rng.randint(0, 1 << 20)
            if op == "append":
                past = min(past, 8000)  # what is cached already is not touched
                case = _append(batch, past, new, ragged, heads, kv_heads, dim, page, rng.random() < 0.5, mix)
            else:
                case = _attend(batch, past, new, ragged, heads, kv_heads, dim, page, mix)
        w = work(case)
        if w["bytes"] <= most_bytes and w["flops"] <= most["flops"] and _cache_values(case) <= 2 ** 29:
            return case


# ----------------------------------------------------------------------------------------------- sizes

def _sizes(case):
    """(cached tokens, new tokens) of each sequence; the first has the most of both."""
    b, past, new = case["batch"], case["past"], case["new"]
    if not case["ragged"]:
        return [(past, new)] * b
    rng = random.Random(case["mix"])
    out = [(past, new)]
    for _ in range(b - 1):
        # mostly anything up to the longest, some that have just begun
        out.append((_log(rng, 1, past + 1) - 1 if rng.random() < 0.25 else rng.randint(0, past), rng.randint(1, new)))
    return out


def _pages(case):
    return [-(-(p + n) // case["page"]) for p, n in _sizes(case)]


def _cache_values(case):
    """Values in the pages of the keys (those of the values are as many)."""
    if case["op"] == "verify":
        return 0
    return (sum(_pages(case)) + 3) * case["page"] * case["kv_heads"] * case["dim"]


def work(case):
    if case["op"] == "verify":
        # the scattered values that decide, and one row of the target (and of the draft) to draw from
        rows = 1 if case["certain"] else 2
        return {"bytes": case["batch"] * (4 * rows * case["vocab"] + case["drafts"] * 20 + 16), "flops": case["batch"] * case["vocab"] * 3}
    h, hkv, d = case["heads"], case["kv_heads"], case["dim"]
    sizes = _sizes(case)
    n = sum(s[1] for s in sizes)
    if case["op"] == "append":
        tables = max(s[1] for s in sizes) * d * 2
        return {"bytes": 2 * 2 * n * (h + 2 * hkv) * d + tables, "flops": n * (h + hkv) * d * (6 if case["norm"] else 3)}
    seen = sum(c * p + c * (c + 1) // 2 for p, c in sizes)
    return {"bytes": 2 * 2 * hkv * d * sum(p + c for p, c in sizes) + 2 * 2 * n * h * d, "flops": 4 * h * d * seen}


# ----------------------------------------------------------------------------------------------- inputs

class _Cache:
    """Pages of keys and values in random order, what a program keeps between its calls."""

    def __init__(self, case, gen, dev):
        self.sizes, pages = _sizes(case), _pages(case)
        hkv, d, page = case["kv_heads"], case["dim"], case["page"]
        total = sum(pages) + 3
        shape = (total, page, hkv, d)
        # pages hold what earlier texts left there until they are written
        self.k = torch.randn(shape, generator=gen, device=dev, dtype=torch.bfloat16)
        self.v = torch.randn(shape, generator=gen, device=dev, dtype=torch.bfloat16)
        order = torch.randperm(total, generator=gen, device=dev).to(torch.int32)
        self.table = torch.full((len(pages), max(pages)), -1, dtype=torch.int32, device=dev)
        at = 0
        for b, n in enumerate(pages):
            self.table[b, :n] = order[at:at + n]
            at += n
        offsets = [0]
        for _, n in self.sizes:
            offsets.append(offsets[-1] + n)
        self.offsets = torch.tensor(offsets, dtype=torch.int32, device=dev)
        self.lengths = torch.tensor([p for p, _ in self.sizes], dtype=torch.int32, device=dev)
        self.tokens = offsets[-1]
        self.most_new = max(n for _, n in self.sizes)


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    if case["op"] == "verify":
        b, k, v = case["batch"], case["drafts"], case["vocab"]
        target = torch.randn(b, k + 1, v, generator=gen, device=dev) * 2
        if case["certain"]:
            draft = None
            tokens = target[:, :k].argmax(-1)
        else:
            # a smaller model's opinion: the target's with noise
            draft = torch.softmax(target[:, :k] + torch.randn(b, k, v, generator=gen, device=dev) * 0.7, -1)
            tokens = torch.multinomial(draft.reshape(b * k, v), 1, generator=gen).reshape(b, k)
        target = torch.softmax(target, -1)
        return dict(case=case, target=target, draft=draft, tokens=tokens, uniforms=torch.rand(b, k + 1, generator=gen, device=dev))
    cache = _Cache(case, gen, dev)
    h, hkv, d, n = case["heads"], case["kv_heads"], case["dim"], cache.tokens
    state = dict(case=case, cache=cache)
    if case["op"] == "append":
        # the projections' output of one layer, and the tables of the model
        qkv = torch.randn(n, h + 2 * hkv, d, generator=gen, device=dev, dtype=torch.bfloat16)
        state["q"], state["k"], state["v"] = (t.contiguous() for t in qkv.split([h, hkv, hkv], dim=1))
        positions = torch.arange(max(p + c for p, c in cache.sizes), device=dev, dtype=torch.float64)
        inv = 10000.0 ** (-torch.arange(0, d, 2, device=dev, dtype=torch.float64) / d)
        angle = positions[:, None] * inv
        state["cos"], state["sin"] = angle.cos().bfloat16(), angle.sin().bfloat16()
    else:
        # queries on the scale of normalised ones that have learnt to look somewhere
        state["q"] = torch.randn(n, h, d, generator=gen, device=dev, dtype=torch.bfloat16) * 1.5
    return state


# ----------------------------------------------------------------------------------------------- plain forms

def _rotate(x, cos, sin, eps):
    d = x.shape[-1] // 2
    x1, x2 = x[..., :d].float(), x[..., d:].float()
    y = torch.cat([x1 * cos + x2 * sin, x2 * cos - x1 * sin], dim=-1)
    if eps is not None:
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + eps)
    return y.bfloat16()


def _plain_append(s, eps):
    c, page = s["cache"], s["case"]["page"]
    lengths, counts = c.lengths.long(), (c.offsets[1:] - c.offsets[:-1]).long()
    seq = torch.repeat_interleave(torch.arange(len(c.sizes), device=lengths.device), counts, output_size=c.tokens)
    pos = lengths[seq] + torch.arange(c.tokens, device=lengths.device) - c.offsets.long()[seq]
    cos, sin = s["cos"].float()[pos][:, None], s["sin"].float()[pos][:, None]
    to, row = c.table[seq, pos // page].long(), pos % page
    c.k[to, row] = _rotate(s["k"], cos, sin, eps)
    c.v[to, row] = s["v"]
    return _rotate(s["q"], cos, sin, eps)


def _plain_attend(s):
    c, case = s["cache"], s["case"]
    h, hkv, d, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    new, keys, n = c.most_new, max(p + n for p, n in c.sizes), len(c.sizes)
    # all sequences at once, padded to the longest, as far as 2 GB of scores (and of keys in 32 bits) go
    some = max(1, min(n, 2 ** 29 // (keys * max(h * new, hkv * d))))
    place, key = torch.arange(new, device=c.k.device), torch.arange(keys, device=c.k.device)
    out = []
    for b in range(0, n, some):
        first, count, past = c.offsets[b:b + some + 1].long(), c.offsets[b:b + some + 1].diff().long(), c.lengths[b:b + some].long()
        rows = (first[:-1, None] + place).clamp_max(c.tokens - 1)
        q = s["q"][rows].float().reshape(-1, new, hkv, h // hkv, d)
        pages = c.table[b:b + some, :-(-keys // page)].long().clamp_min(0)
        k = c.k[pages].reshape(len(past), -1, hkv, d)[:, :keys].float()
        v = c.v[pages].reshape(len(past), -1, hkv, d)[:, :keys].float()
        scores = torch.einsum("btgrd,bsgd->bgrts", q, k) * (1.0 / math.sqrt(d))
        scores.masked_fill_((key > past[:, None, None] + place[:, None])[:, None, None], -math.inf)
        scores -= scores.amax(-1, keepdim=True)
        scores.exp_()
        total = scores.sum(-1)
        o = torch.einsum("bgrts,bsgd->btgrd", scores, v) / total.permute(0, 3, 1, 2)[..., None]
        tokens = sum(m for _, m in c.sizes[b:b + some])
        seq = torch.repeat_interleave(torch.arange(len(past), device=first.device), count, output_size=tokens)
        i = torch.arange(tokens, device=first.device) - (first[:-1] - first[0])[seq]
        out.append(o[seq, i].reshape(tokens, h, d).bfloat16())
    return torch.cat(out)


def _plain_verify(s):
    p, q, tokens, u = s["target"], s["draft"], s["tokens"], s["uniforms"].double()
    b, k = tokens.shape
    every = torch.arange(b, device=p.device)
    p_of = p[:, :k].gather(-1, tokens[..., None])[..., 0].double()
    q_of = torch.ones_like(p_of) if q is None else q.gather(-1, tokens[..., None])[..., 0].double()
    accepted = (u[:, :k] * q_of < p_of).long().cumprod(-1).sum(-1)
    last = accepted.clamp_max(k - 1)
    row = p[every, accepted].double()
    if q is None:
        minus = torch.zeros_like(row).scatter_(-1, tokens[every, last][:, None], 1.0)
    else:
        minus = q[every, last].double()
    rest = (row - minus).clamp_min(0)
    rest = torch.where(((accepted == k) | (rest.sum(-1) == 0))[:, None], row, rest)
    upto = rest.cumsum(-1)
    token = (upto <= u[:, k:] * upto[:, -1:]).sum(-1)
    return accepted, torch.where(upto[:, -1] > 0, token, 0)


def run(state):
    case = state["case"]
    if case["op"] == "verify":
        if own:
            from dion_b200 import ops

            accepted, token = ops.verify_drafts(state["target"], state["draft"], state["tokens"], state["uniforms"])
        else:
            accepted, token = _plain_verify(state)
        return {"accepted": accepted, "token": token}
    c = state["cache"]
    if case["op"] == "append":
        eps = EPS if case["norm"] else None
        if own:
            from dion_b200 import ops

            q = ops.paged_append(state["q"], state["k"], state["v"], state["cos"], state["sin"], c.k, c.v, c.table, c.offsets,
                                 c.lengths, norm_eps=eps)
        else:
            q = _plain_append(state, eps)
        return {"q": q, "k_pages": c.k, "v_pages": c.v}
    if own:
        from dion_b200 import ops

        out = ops.paged_attention(state["q"], c.k, c.v, c.table, c.offsets, c.lengths, max_new=c.most_new)
    else:
        out = _plain_attend(state)
    return {"out": out}


# ----------------------------------------------------------------------------------------------- 64 bits

def _exact_append(case, s):
    c, d, page = s["cache"], case["dim"], case["page"]
    half = d // 2

    def turned(x, cos, sin):  # complex numbers whose real parts are the first half of the head
        z = torch.complex(x[..., :half].double(), x[..., half:].double()) * torch.complex(cos.double(), -sin.double())[:, None]
        y = torch.cat([z.real, z.imag], -1)
        return y / (y.pow(2).sum(-1, keepdim=True) / d + EPS).sqrt() if case["norm"] else y

    k, v, q = c.k.double(), c.v.double(), torch.empty(s["q"].shape, dtype=torch.float64, device=c.k.device)
    at = 0
    for b, (past, new) in enumerate(c.sizes):
        here = slice(at, at + new)
        cos, sin = s["cos"][past:past + new], s["sin"][past:past + new]
        q[here] = turned(s["q"][here], cos, sin)
        keys = turned(s["k"][here], cos, sin)
        first = past // page
        for i in range(first, (past + new - 1) // page + 1):
            lo, hi = max(past, i * page), min(past + new, (i + 1) * page)
            p = int(c.table[b, i])
            k[p, lo - i * page:hi - i * page] = keys[lo - past:hi - past]
            v[p, lo - i * page:hi - i * page] = s["v"][at + lo - past:at + hi - past].double()
        at += new
    return {"q": q, "k_pages": k, "v_pages": v}


def _exact_attend(case, s):
    c, d, page = s["cache"], case["dim"], case["page"]
    group = case["heads"] // case["kv_heads"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=c.k.device)
    at = 0
    for b, (past, new) in enumerate(c.sizes):
        n = past + new
        rows = (c.table[b].long().clamp_min(0)[:, None] * page + torch.arange(page, device=c.k.device)).reshape(-1)[:n]
        for g in range(case["kv_heads"]):
            k = c.k[:, :, g].reshape(-1, d)[rows].double()
            v = c.v[:, :, g].reshape(-1, d)[rows].double()
            for h in range(g * group, (g + 1) * group):
                x = s["q"][at:at + new, h].double() @ k.T / math.sqrt(d)
                if new > 1:
                    x = x + torch.full((new, n), -math.inf, device=x.device, dtype=x.dtype).triu_(past + 1)
                out[at:at + new, h] = torch.softmax(x, -1) @ v
        at += new
    return {"out": out}


def _exact_verify(case, s):
    p, u = s["target"].cpu().numpy(), s["uniforms"].cpu().numpy().astype(np.float64)
    q = None if s["draft"] is None else s["draft"].cpu().numpy()
    tokens = s["tokens"].cpu().numpy()
    b, k = tokens.shape
    accepted, out = [], []
    for i in range(b):
        a = 0
        while a < k and u[i, a] * (1.0 if q is None else np.float64(q[i, a, tokens[i, a]])) < np.float64(p[i, a, tokens[i, a]]):
            a += 1
        w = p[i, a].astype(np.float64)
        if a < k:
            r = w.copy()
            if q is None:
                r[tokens[i, a]] -= 1.0
            else:
                r -= q[i, a]
            r = np.maximum(r, 0.0)
            w = r if r.any() else w
        upto = np.cumsum(w)
        accepted.append(a)
        out.append(int(np.searchsorted(upto, u[i, k] * upto[-1], side="right")) if w.any() else 0)
    return {"accepted": torch.tensor(accepted), "token": torch.tensor(out)}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "append":
        return _exact_append(case, s)
    return _exact_attend(case, s) if case["op"] == "attend" else _exact_verify(case, s)

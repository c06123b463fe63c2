"""Sampling over a paged cache: the cache's bookkeeping, cached passes against whole ones, and drafts."""
import pytest
import torch

from dion_b200 import ops
from dion_b200.models import GPT, GPTConfig, Llama, LlamaConfig, PagedCache
from dion_b200.ops import nn as N

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def _gpt(layers=2, width=64, heads=4, seq=64, vocab=97, device="cpu"):
    m = GPT(GPTConfig(sequence_len=seq, vocab_size=vocab, n_layer=layers, n_head=heads, n_embd=width)).to(device)
    m.init_weights()
    return m


def _llama(layers=2, width=64, heads=4, kv_heads=2, seq=64, vocab=97, device="cpu"):
    m = Llama(LlamaConfig(sequence_len=seq, vocab_size=vocab, n_layer=layers, n_head=heads, n_kv_head=kv_heads, n_embd=width, ffn_dim=2 * width)).to(device)
    m.init_weights(std=0.2)
    return m


def _whole_logits(m, idx):
    """Logits of every position by the pass that training makes."""
    return m(idx, idx, return_logits=True)


# --------------------------------------------------------------------------- the cache

def test_cache_takes_pages_as_sequences_grow_and_gives_them_back():
    c = PagedCache(2, 3, 8, sequences=3, max_len=100, page_size=16, pages=9, dtype=torch.float32, device="cpu")
    s = c.step([20, 0, 16])
    assert c.lengths == [20, 0, 16] and c.free_pages == 6
    assert s.offsets.tolist() == [0, 20, 20, 36] and s.lengths.tolist() == [0, 0, 0] and s.max_new == 20 and s.rows == [19, 35]
    s = c.step([1, 5, 1], all_rows=True)
    assert s.lengths.tolist() == [20, 0, 16] and s.rows is None and c.free_pages == 4
    used = [c._table[b, :n].tolist() for b, n in enumerate((2, 1, 2))]
    assert len({p for u in used for p in u}) == 5
    with pytest.raises(RuntimeError, match="free pages"):
        c.step([60, 60, 0])
    with pytest.raises(ValueError):
        c.step([80, 0, 0])
    with pytest.raises(ValueError):
        c.step([1, 1])
    with pytest.raises(ValueError):
        c.step([1, -1, 0])
    assert c.lengths == [21, 5, 17] and c.free_pages == 4  # a refused step changes nothing
    with pytest.raises(ValueError):
        c.cut([22, 0, 0])
    c.cut([16, 0, 17])
    assert c.free_pages == 6 and c.lengths == [16, 0, 17]
    s = c.step([1, 33, 0])
    assert c.free_pages == 2 and len({p for b, n in enumerate((2, 3, 2)) for p in s.page_table[b, :n].tolist()}) == 7
    for bad in (dict(page_size=24), dict(page_size=8), dict(max_len=0), dict(sequences=0)):
        with pytest.raises(ValueError):
            PagedCache(**{**dict(layers=1, kv_heads=1, head_dim=8, sequences=1, max_len=10, device="cpu"), **bad})


def test_a_step_taken_before_keeps_its_table():
    c = PagedCache(1, 1, 8, sequences=2, max_len=64, page_size=16, dtype=torch.float32, device="cpu")
    s = c.step([16, 16])
    before = s.page_table.clone()
    c.step([16, 16])
    assert torch.equal(s.page_table, before) and s.lengths.tolist() == [0, 0]


# --------------------------------------------------------------------------- passes over the cache

@pytest.mark.parametrize("make", [_gpt, _llama])
def test_cached_passes_give_the_logits_of_whole_ones(make):
    """Chunk by chunk with ragged counts, in 64 bits but for the norms and the rotation of whole passes, which take 32: at most ten
    roundings a layer, 21 with the head, each by at most a half step, on either side, as norms."""
    torch.manual_seed(3)
    m = make().double()
    with torch.no_grad():
        idx = torch.randint(0, 97, (3, 40))
        want = _whole_logits(m, idx).double()
        cache = m.new_cache(3, page_size=16)
        done = [0, 0, 0]
        for counts in ([5, 1, 0], [1, 0, 17], [20, 30, 1], [0, 1, 1], [14, 8, 21]):
            tokens = torch.cat([idx[b, done[b]:done[b] + n] for b, n in enumerate(counts)])
            got = m(tokens, cache=cache.step(counts, all_rows=True)).double()
            at = 0
            for b, n in enumerate(counts):
                w = want[b, done[b]:done[b] + n]
                assert (got[at:at + n] - w).norm() <= 2 * 21 * 2.0 ** -24 * w.norm()
                at += n
                done[b] += n
        assert done == cache.lengths == [40, 40, 40]


@pytest.mark.gpu
@pytest.mark.parametrize("make,kw", [(_gpt, dict(width=256, heads=4)), (_gpt, dict(width=256, heads=2)), (_gpt, dict(width=256, heads=8)), (_llama, dict(width=256, heads=4, kv_heads=2))])
def test_cached_passes_on_the_kernels(make, kw):
    """bf16 activations are rounded some ten times a layer on either way, each time by at most a half step: two layers and
    the head are within 21 half steps of the exact, and of one another within twice that, as norms."""
    torch.manual_seed(4)
    m = make(seq=512, device="cuda", **kw)
    with torch.no_grad():
        idx = torch.randint(0, 97, (3, 400), device="cuda")
        want = _whole_logits(m, idx)
        cache = m.new_cache(3)
        done = [0, 0, 0]
        launches = ops.launch_count()
        for counts in ([300, 1, 64], [1, 1, 0], [5, 300, 5], [1, 0, 200], [93, 98, 131]):
            tokens = torch.cat([idx[b, done[b]:done[b] + n] for b, n in enumerate(counts)])
            got = m(tokens, cache=cache.step(counts, all_rows=True))
            at = 0
            for b, n in enumerate(counts):
                if n:
                    w = want[b, done[b]:done[b] + n]
                    assert (got[at:at + n] - w).norm() <= 2 * 21 * 2.0 ** -8 * w.norm()
                at += n
                done[b] += n
        ops.check_status()
        assert ops.launch_count() > launches and done == [400, 400, 400]


@pytest.mark.parametrize("make,tables", [(_gpt, lambda m: [x for b in m.transformer.h for x in (b.attn.rotary.cos_cached, b.attn.rotary.sin_cached)]),
                                         (_llama, lambda m: [x for b in m.layers for x in b.attention._tables])])
def test_the_layers_keep_their_rotation_tables(make, tables):
    """What a captured pass of the model reads is still there after a cache has been used."""
    m = make()
    with torch.no_grad():
        _whole_logits(m, torch.randint(0, 97, (2, 24)))
        before = tables(m)
        m(torch.randint(0, 97, (9,)), cache=m.new_cache(2).step([4, 5]))
    assert all(a is b for a, b in zip(before, tables(m)))


@pytest.mark.parametrize("make", [_gpt, _llama])
def test_a_pass_over_a_cache_refuses_what_its_step_has_no_room_for(make):
    m = make()
    cache = m.new_cache(2)
    with pytest.raises(ValueError, match="counts"):
        cache.step([0, 0])
    with torch.no_grad():
        step = cache.step([3, 1])
        for tokens in (torch.zeros(3, dtype=torch.long), torch.zeros(2, 2, dtype=torch.long)):
            with pytest.raises(ValueError, match="room for 4"):
                m(tokens, cache=step)
        with pytest.raises(ValueError, match="targets"):
            m(torch.zeros(4, dtype=torch.long), torch.zeros(4, dtype=torch.long), cache=step)
    with pytest.raises(RuntimeError, match="no gradient"):
        m(torch.zeros(4, dtype=torch.long), cache=step)


@pytest.mark.parametrize("make", [_gpt, _llama])
def test_a_pass_that_fails_leaves_the_cache_as_it_was(make):
    """Wrong tokens, gradients left on, a layer that raises half way: the tokens count as cached no longer, and another step, or the
    same one again, gives the logits of a cache that has seen no failure."""
    torch.manual_seed(11)
    m = make()
    tokens = torch.randint(0, 97, (22,))
    first, then = tokens[:20], torch.cat([tokens[20:], tokens[:1]])
    with torch.no_grad():
        good = m.new_cache(2, page_size=16)
        m(first, cache=good.step([14, 6]))
        want = m(then, cache=good.step([3, 0], all_rows=True))

    def broken(*_):
        raise KeyError("half way")

    layers = m.transformer.h if make is _gpt else m.layers
    for again in (False, True):
        cache = m.new_cache(2, page_size=16)
        with torch.no_grad():
            m(first, cache=cache.step([14, 6]))
        free = cache.free_pages
        step = cache.step([3, 0], all_rows=True)
        assert cache.lengths == [17, 6] and cache.free_pages == free - 1
        with pytest.raises(RuntimeError, match="no gradient"):
            m(then, cache=step)
        assert cache.lengths == [14, 6] and cache.free_pages == free
        with torch.no_grad():
            with pytest.raises(ValueError, match="room for"):
                m(then[:2], cache=step if again else cache.step([3, 0], all_rows=True))
            assert cache.lengths == [14, 6] and cache.free_pages == free
            hook = layers[1].register_forward_pre_hook(broken)
            with pytest.raises(KeyError):
                m(tokens[:3], cache=step if again else cache.step([3, 0]))
            hook.remove()
            assert cache.lengths == [14, 6] and cache.free_pages == free
            got = m(then, cache=step if again else cache.step([3, 0], all_rows=True))
            assert cache.lengths == [17, 6] and torch.equal(got, want)
            with pytest.raises(ValueError, match="room for"):  # what a pass has cached stays
                m(then[:2], cache=step)
            assert cache.lengths == [17, 6]


@pytest.mark.parametrize("make", [_gpt, _llama])
def test_a_failed_step_does_not_take_back_what_came_after(make):
    m = make()
    cache = m.new_cache(2, page_size=16)
    with torch.no_grad():
        one = cache.step([3, 1])
        m(torch.zeros(5, dtype=torch.long), cache=cache.step([0, 5]))
        with pytest.raises(ValueError, match="room for"):
            m(torch.zeros(5, dtype=torch.long), cache=one)
        assert cache.lengths == [3, 6]
        cache.cut([0, 0])
        one = cache.step([3, 1])
        with pytest.raises(ValueError, match="room for"):
            m(torch.zeros(5, dtype=torch.long), cache=one)
        m(torch.zeros(5, dtype=torch.long), cache=cache.step([0, 5]))
        with pytest.raises(ValueError, match="take another step"):
            m(torch.zeros(4, dtype=torch.long), cache=one)
        assert cache.lengths == [0, 5]


@pytest.mark.parametrize("new", [1, 2, 6])
def test_prompts_of_32_bits_draw_the_same_tokens(new):
    torch.manual_seed(10)
    m = _gpt()
    idx = torch.randint(0, 97, (3, 5))
    want = m.generate(idx, new, top_k=1, use_cache=True)
    assert torch.equal(m.generate(idx.int(), new, top_k=1, use_cache=True), want)
    assert torch.equal(m.generate(idx.int(), new, top_k=1, draft_model=m, draft_tokens=2), want.int())


# --------------------------------------------------------------------------- sampling

def test_cached_sampling_draws_the_same_tokens():
    torch.manual_seed(5)
    m = _gpt()
    idx = torch.randint(0, 97, (3, 7))
    for kw in (dict(), dict(top_k=5), dict(temperature=0.5, top_k=1000)):
        torch.manual_seed(9)
        want = m.generate(idx, 20, **kw)
        torch.manual_seed(9)
        assert torch.equal(m.generate(idx, 20, use_cache=True, **kw), want)
    assert torch.equal(m.generate(idx, 58, top_k=1, use_cache=True), m.generate(idx, 58, top_k=1))  # to the last position
    assert torch.equal(m.generate(idx, 0, use_cache=True), idx)
    with pytest.raises(ValueError, match="do not fit"):
        m.generate(idx, 59, use_cache=True)
    with pytest.raises(ValueError):
        m.generate(idx[:, :0], 3, use_cache=True)


def _greedy(m, idx, n):
    for _ in range(n):
        idx = torch.cat([idx, m(idx, return_logits=True)[:, -1].argmax(-1, keepdim=True)], 1)
    return idx


@pytest.mark.parametrize("make", [_gpt, _llama])
@pytest.mark.parametrize("prompt", [1, 6])
def test_greedy_tokens_do_not_depend_on_the_draft(make, prompt):
    """The most likely token every time, whatever a draft proposes: itself (always right), a smaller model (mostly wrong)."""
    torch.manual_seed(6)
    m, small = make(), make(layers=1, width=32, heads=2, **(dict(kv_heads=1) if make is _llama else {}))
    idx = torch.randint(0, 97, (4, prompt))
    want = _greedy(m, idx, 25)
    assert torch.equal(m.generate(idx, 25, top_k=1, **({} if make is _llama else dict(use_cache=True))), want)
    for draft in (m, small):
        for k in (1, 3, 40):
            assert torch.equal(m.generate(idx, 25, top_k=1, draft_model=draft, draft_tokens=k), want)
    full = m.config.sequence_len - prompt + 1
    assert torch.equal(m.generate(idx, full, top_k=1, draft_model=m), _greedy(m, idx, full))


def test_drafted_sampling_runs_on_its_own_draws():
    torch.manual_seed(7)
    m, small = _gpt(), _gpt(layers=1)
    idx = torch.randint(0, 97, (5, 4))
    out = m.generate(idx, 30, temperature=0.8, top_k=20, draft_model=small)
    assert out.shape == (5, 34) and torch.equal(out[:, :4], idx) and 0 <= int(out.min()) and int(out.max()) < 97
    with pytest.raises(ValueError, match="vocabulary"):
        m.generate(idx, 3, draft_model=_gpt(vocab=98))
    with pytest.raises(ValueError):
        m.generate(idx, 3, draft_model=small, draft_tokens=0)
    with pytest.raises(ValueError, match="do not fit"):
        m.generate(idx, 30, draft_model=_gpt(seq=32))


@pytest.mark.parametrize("make,top_k", [(_gpt, None), (_llama, 3)])
def test_drafted_sampling_is_distributed_as_without_a_draft(make, top_k):
    """Three tokens of a vocabulary of five, temperature 0.7, from a draft of another opinion.  The counts of the 125 outcomes against the
    products of the model's probabilities: the chi-square sum has its degrees of freedom as mean and twice these as variance, of
    which four standard deviations are allowed.  Sequences finish after different numbers of passes.  What the draft, or the model at
    another temperature, would say is far outside."""
    torch.manual_seed(12)
    m, small = make(vocab=5, seq=16), make(layers=1, width=32, heads=2, vocab=5, seq=16, **(dict(kv_heads=1) if make is _llama else {}))
    with torch.no_grad():
        for w in (*m.parameters(), *small.parameters()):
            if w.dim() == 2:
                w.normal_(std=2 * w.shape[1] ** -0.5)
    n, new = 2000, 3
    prompt = torch.tensor([[1, 4, 2]])
    out = m.generate(prompt.expand(n, -1), new, temperature=0.7, top_k=top_k, draft_model=small, draft_tokens=2)
    counts = torch.bincount(out[:, 3] * 25 + out[:, 4] * 5 + out[:, 5], minlength=125).double()

    def outcomes(model, temperature=0.7):
        every = torch.cartesian_prod(*[torch.arange(5)] * new)
        with torch.no_grad():
            logits = model(torch.cat([prompt.expand(125, -1), every], 1), torch.zeros(125, 3 + new, dtype=torch.long), return_logits=True).double()
        logits = logits[:, 2:2 + new] / temperature
        if top_k is not None:
            logits = logits.masked_fill(logits < logits.topk(top_k).values[..., -1:], -torch.inf)
        return torch.softmax(logits, -1).gather(-1, every[..., None]).prod(1)[:, 0]

    def far(p):  # outcomes that are expected fewer than five times count as one
        often = p * n >= 5
        e, c = (torch.cat([t[often], t[~often].sum()[None]]) for t in (p * n, counts))
        e, c = e[e > 0], c[e > 0]
        return ((c - e).square() / e).sum().item() / (len(e) - 1 + 4 * (2 * (len(e) - 1)) ** 0.5)

    p = outcomes(m)
    assert abs(p.sum().item() - 1) < 1e-6 and (counts[p == 0] == 0).all()
    assert far(p) <= 1 and far(outcomes(small).clamp_min(1e-9)) > 2 and far(outcomes(m, 1.0)) > 2


@pytest.mark.gpu
def test_generation_on_the_kernels():
    """Cached and drafted sampling through all operators.  With a draft that is the model itself nearly everything is accepted: fewer
    passes, hence fewer kernels, than tokens one by one."""
    torch.manual_seed(8)
    m = _gpt(width=256, heads=2, seq=256, vocab=512, device="cuda")
    idx = torch.randint(0, 512, (4, 30), device="cuda")
    out = m.generate(idx, 40, top_k=50, use_cache=True)
    assert out.shape == (4, 70) and torch.equal(out[:, :30], idx)
    seen = []

    class Counting(GPT):
        def forward(self, tokens, *a, **kw):
            seen.append(tokens.numel())
            return super().forward(tokens, *a, **kw)

    c = Counting(m.config).cuda()
    c.load_state_dict(m.state_dict())
    out = c.generate(idx, 40, top_k=50, draft_model=m, draft_tokens=4)
    ops.check_status()
    assert out.shape == (4, 70) and 0 <= int(out.min()) and int(out.max()) < 512
    assert 9 <= len(seen) <= 25  # the prompt, and at least a fifth of 40 tokens
    big = _llama(width=256, heads=4, kv_heads=2, seq=256, vocab=512, device="cuda")
    out = big.generate(idx, 20, temperature=0.7, draft_model=_llama(layers=1, width=128, heads=2, kv_heads=1, seq=256, vocab=512, device="cuda"))
    ops.check_status()
    assert out.shape == (4, 50)

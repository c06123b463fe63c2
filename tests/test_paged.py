"""The paged cache: appending with rotation, attention over the pages and the check of drafted tokens, against their definitions
in 64 bits."""
import math

import pytest
import torch
import torch.autograd.forward_ad as fwd

from dion_b200 import ops
from dion_b200.ops import nn as N

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
HALF_STEP = torch.finfo(torch.bfloat16).eps / 2  # a rounding to bf16 is off by at most this, relative to the value
U32 = torch.finfo(torch.float32).eps / 2


class Paged:
    """Pages in random order, filled with garbage where nothing has been written; sizes = [(cached, new), ...]."""

    def __init__(self, sizes, heads, kv_heads, dim, page, device, dtype=torch.bfloat16, order="rows", tail=0, garbage=math.nan,
                 spare=2, wide=3):
        self.sizes, self.page, self.kv_heads, self.dim = sizes, page, kv_heads, dim
        need = [-(-(p + n) // page) for p, n in sizes]
        total = sum(need) + spare
        if order == "rows":      # [pages, page_size, kv heads, dim] as it lies
            shape, perm = (total, page, kv_heads, dim), (0, 1, 2, 3)
        elif order == "heads":   # each head's part of a page contiguous
            shape, perm = (total, kv_heads, page, dim), (0, 2, 1, 3)
        self.both = torch.full((total, 2, *shape[1:]) if order == "rows" else (2, *shape), garbage, dtype=dtype, device=device)
        self.k, self.v = (self.both[:, i] if order == "rows" else self.both[i] for i in (0, 1))
        self.k, self.v = self.k.permute(perm), self.v.permute(perm)
        ids = torch.randperm(total)[:sum(need)].to(torch.int32)
        table = torch.full((len(sizes), max(need, default=0) + wide), -7, dtype=torch.int32)  # nobody looks behind the last page
        at = 0
        for b, n in enumerate(need):
            table[b, :n] = ids[at:at + n]
            at += n
        starts = [0]
        for _, n in sizes:
            starts.append(starts[-1] + n)
        self.tokens = starts[-1] + tail
        self.starts = starts
        self.table, self.offsets = table.to(device), torch.tensor(starts, dtype=torch.int32, device=device)
        self.lengths = torch.tensor([p for p, _ in sizes], dtype=torch.int32, device=device)

    def slots(self, b, lo, hi):
        at = torch.arange(lo, hi, device=self.table.device)
        return self.table[b].long()[at // self.page], at % self.page

    def fill(self, upto_new=True):
        for b, (p, n) in enumerate(self.sizes):
            page, row = self.slots(b, 0, p + (n if upto_new else 0))
            for t in (self.k, self.v):
                t[page, row] = torch.randn(len(row), self.kv_heads, self.dim, device=t.device).to(t.dtype)
        return self

    def where(self):
        return self.k, self.v, self.table, self.offsets, self.lengths


def same(a, b):
    return torch.equal(torch.nan_to_num(a.double(), nan=1e30), torch.nan_to_num(b.double(), nan=1e30))


SIZES = {
    "one": [(0, 1)],
    "one_later": [(777, 1)],
    "decode": [(0, 1), (15, 1), (16, 1), (300, 1), (1023, 1), (64, 1)],
    "drafts": [(31, 5), (0, 5), (200, 5), (511, 4)],
    "ragged": [(0, 70), (3, 0), (130, 200), (0, 0), (0, 1), (500, 33)],
    "prompt": [(0, 300), (0, 129), (0, 256)],
    "none_new": [(5, 0), (0, 0)],
}


# --------------------------------------------------------------------------- append

def _turned(x, cos, sin, eps):
    """In 64 bits, with the largest a rounded intermediate may be: |x1 c| + |x2 s|, scaled as the result is."""
    d = x.shape[-1] // 2
    x1, x2, c, s = x[..., :d].double(), x[..., d:].double(), cos.double()[:, None], sin.double()[:, None]
    y = torch.cat([x1 * c + x2 * s, x2 * c - x1 * s], -1)
    m = torch.cat([(x1 * c).abs() + (x2 * s).abs(), (x2 * c).abs() + (x1 * s).abs()], -1)
    f = 1.0 if eps is None else torch.rsqrt(y.square().mean(-1, keepdim=True) + eps)
    return y * f, m * f


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("sizes", list(SIZES))
@pytest.mark.parametrize("heads,kv_heads,dim,page,order,eps,wide", [
    (6, 6, 128, 64, "rows", 1e-6, False), (12, 4, 64, 16, "heads", None, False), (5, 1, 128, 32, "heads", 1e-6, True), (3, 3, 64, 128, "rows", None, True)])
def test_append(device, sizes, heads, kv_heads, dim, page, order, eps, wide):
    c = Paged(SIZES[sizes], heads, kv_heads, dim, page, device, order=order, tail=3).fill(upto_new=False)
    fused = torch.randn(c.tokens, heads + 2 * kv_heads, dim, device=device).bfloat16()  # the rows of one projection
    q, k, v = fused.split([heads, kv_heads, kv_heads], 1)
    cos, sin = N.rotary_tables(1100, dim, device)
    if wide:
        cos, sin = cos.float() * 1.0078, sin.float() * 0.9921
    want_k, want_v = c.k.clone().double(), c.v.clone()
    out = ops.paged_append(q, k, v, cos, sin, *c.where(), norm_eps=eps)
    if device == "cuda":
        ops.check_status()
    assert out.shape == q.shape and out.dtype == q.dtype and out.is_contiguous()
    touched = torch.zeros(c.k.shape[:2], dtype=torch.bool, device=device)
    # four fp32 roundings of a pair, those of a sum of `dim` squares and the root's few, times what they apply to
    slack = U32 * (8 + dim)
    for b, (p, n) in enumerate(c.sizes):
        a = c.starts[b]
        rows = slice(a, a + n)
        page_, row = c.slots(b, p, p + n)
        touched[page_, row] = True
        for got, x in ((out[rows], q[rows]), (c.k[page_, row], k[rows])):
            want, most = _turned(x, cos[p:p + n], sin[p:p + n], eps)
            assert ((got.double() - want).abs() <= HALF_STEP * want.abs() + 2 * slack * most + 1e-38).all()
        assert torch.equal(c.v[page_, row], v[rows])
    assert (out[c.starts[-1]:] == 0).all()
    assert same(c.k[~touched], want_k[~touched]) and same(c.v[~touched], want_v[~touched])


@pytest.mark.gpu
def test_append_gives_the_bits_of_the_training_kernels():
    """Chunk by chunk into the cache, the same queries and keys as from the kernels of a whole sequence."""
    T, H, D = 200, 4, 64
    cos, sin = N.rotary_tables(T, D, "cuda")
    q, k, v = (torch.randn(1, T, H, D, device="cuda").bfloat16() for _ in range(3))
    for eps in (None, N.RMS_EPS):
        if eps is None:
            qr, kr = N.rope(q, cos, sin), N.rope(k, cos, sin)
        else:
            qr, kr = N.rope_qknorm(q, k, cos, sin, eps)
        c = Paged([(0, T)], H, H, D, 16, "cuda")
        at, parts = 0, []
        for n in (1, 63, 100, 36):
            c.lengths.fill_(at)
            c.offsets[1] = n
            parts.append(ops.paged_append(q[0, at:at + n], k[0, at:at + n], v[0, at:at + n], cos, sin, *c.where(), norm_eps=eps))
            at += n
        assert torch.equal(torch.cat(parts), qr[0])
        page, row = c.slots(0, 0, T)
        assert torch.equal(c.k[page, row], kr[0]) and torch.equal(c.v[page, row], v[0])


# --------------------------------------------------------------------------- attention

def _attend(q, c, scale=None):
    """(out, sum of p |v|, the largest sum of |q k|) in 64 bits: what the bounds of the kernels' roundings are made of."""
    out, weight, big = (torch.zeros(q.shape, dtype=torch.float64, device=q.device) for _ in range(3))
    scale = 1.0 / math.sqrt(c.dim) if scale is None else scale
    for b, (p, n) in enumerate(c.sizes):
        if n == 0:
            continue
        page, row = c.slots(b, 0, p + n)
        rows = slice(c.starts[b], c.starts[b] + n)
        group = q.shape[1] // c.kv_heads
        k, v = (t[page, row].double().repeat_interleave(group, 1) for t in (c.k, c.v))
        x = q[rows].double()
        s = torch.einsum("thd,shd->hts", x, k) * scale
        s = s.masked_fill(torch.arange(p + n, device=q.device)[None] > p + torch.arange(n, device=q.device)[:, None], -math.inf)
        w = torch.softmax(s, -1)
        out[rows] = torch.einsum("hts,shd->thd", w, v)
        weight[rows] = torch.einsum("hts,shd->thd", w, v.abs())
        big[rows] = (torch.einsum("thd,shd->hts", x.abs(), k.abs()) * scale).amax(-1).T[..., None]
    return out, weight, big


def _check_attention(got, q, c, scale=None):
    want, weight, big = _attend(q, c, scale)
    # Weights are rounded to bf16 before they meet the values (a half step of each, so of sum p |v|) and the result once.  A score
    # is off by the roundings of `dim` products and sums, twice 2^-24 each as the tensor core cuts off, and a weight by twice
    # that relative to itself (its own and the sum's); the exponential, the rescaling and the sums in fp32 add 2^-16.
    bound = HALF_STEP * (weight + want.abs()) + weight * (4 * c.dim * 2 * U32 * big + 2.0 ** -16)
    off = (got.double() - want).abs()
    assert torch.isfinite(got).all()
    assert (off <= bound * (1 + 2 ** -6) + 1e-38).all(), (off / bound.clamp_min(1e-38)).max().item()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("sizes", list(SIZES))
@pytest.mark.parametrize("heads,kv_heads,dim,page,order", [
    (6, 6, 128, 64, "rows"), (12, 12, 64, 16, "heads"), (32, 8, 128, 16, "heads"), (6, 2, 64, 32, "rows"), (8, 1, 128, 256, "heads"), (5, 1, 64, 16, "rows")])
@pytest.mark.parametrize("wide", [3, 5000])  # columns of the page table that no sequence reaches
def test_attention(device, sizes, heads, kv_heads, dim, page, order, wide):
    c = Paged(SIZES[sizes], heads, kv_heads, dim, page, device, order=order, tail=2, wide=wide).fill()
    q = torch.randn(c.tokens, heads, dim, device=device).bfloat16() * 1.5
    for most in (None, max(n for _, n in c.sizes) or 1):
        got = ops.paged_attention(q, *c.where(), max_new=most)
        if device == "cuda":
            ops.check_status()
        assert got.shape == q.shape and got.is_contiguous()
        _check_attention(got, q, c)
        assert (got[c.starts[-1]:] == 0).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (17, 1), (64, 1), (71, 1), (130, 1), (40, 20), (9, 3)])
@pytest.mark.parametrize("new", [1, 3, 40])
@pytest.mark.parametrize("wide", [3, 5000])
def test_attention_of_any_group(device, heads, kv_heads, new, wide):
    """Groups of heads that fill no tile, and ones larger than one."""
    c = Paged([(100, new), (0, new), (37, 1)], heads, kv_heads, 64, 16, device, order="heads", wide=wide).fill()
    q = torch.randn(c.tokens, heads, 64, device=device).bfloat16()
    got = ops.paged_attention(q, *c.where(), max_new=new)
    if device == "cuda":
        ops.check_status()
    _check_attention(got, q, c)


@pytest.mark.gpu
@pytest.mark.parametrize("sizes,heads,kv_heads,dim,page", [
    ([(30000, 1), (5, 1), (2000, 3)], 32, 8, 128, 64),        # one long cache among short ones
    ([(20000, 1)], 12, 12, 64, 16),
    ([(5000, 600), (0, 1), (100, 1), (7000, 7)], 8, 2, 128, 32),  # a chunk beside single tokens
    ([(1, 1500), (2500, 1100)], 6, 6, 64, 64),
    ([(i * 7 % 900, 1 + (i % 5 == 0) * 2) for i in range(200)], 12, 4, 64, 16),
    ([(0, 1)] * 1500, 2, 2, 64, 16),                          # more sequences than threads of a block
])
@pytest.mark.parametrize("wide", [0, 5000])
def test_attention_split_over_the_gpu(sizes, heads, kv_heads, dim, page, wide):
    c = Paged(sizes, heads, kv_heads, dim, page, "cuda", order="heads", wide=wide).fill()
    q = torch.randn(c.tokens, heads, dim, device="cuda").bfloat16()
    first = ops.paged_attention(q, *c.where())
    _check_attention(first, q, c)
    assert torch.equal(first, ops.paged_attention(q, *c.where()))  # the split goes by the sizes alone
    ops.check_status()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("new", [1, 90])
@pytest.mark.parametrize("wide", [3, 5000])
def test_attention_of_large_and_small_scores(device, new, wide):
    """Scores that grow along the sequence, so that the running maximum moves at every step, far from zero on either side, and all
    equal: the weights are exact multiples then."""
    c = Paged([(700, new)], 4, 2, 64, 16, device, wide=wide).fill()
    page, row = c.slots(0, 0, 700 + new)
    ramp = torch.linspace(-6, 6, 700 + new, device=device)[:, None, None].expand(-1, 2, 64)
    q = torch.ones(new, 4, 64, device=device).bfloat16() * 5
    for keys in (ramp, -ramp, ramp - 60, ramp * 0):
        c.k[page, row] = keys.bfloat16()
        got = ops.paged_attention(q, *c.where())
        _check_attention(got, q, c)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("new", [1, 90])
@pytest.mark.parametrize("wide", [3, 5000])
def test_attention_of_no_numbers(device, new, wide):
    """A query that is no number, and keys whose scores are all minus infinity, have no result that is a number, and the rows beside
    them theirs."""
    c = Paged([(700, new), (30, new)], 4, 2, 64, 16, device, wide=wide).fill()
    q = torch.randn(c.tokens, 4, 64, device=device).bfloat16()
    page, row = c.slots(0, 0, 700 + new)
    c.k[page, row, 0, 3] = -math.inf
    q[:new, :2, 3] = 1.0
    q[new - 1, 3, 7] = math.nan
    q[new, 1, 60] = math.nan
    want, weight, big = _attend(q, c)
    assert want[:new, :2].isnan().all() and want[new - 1, 3].isnan().all() and int(want.isnan().sum()) == (2 * new + 2) * 64
    got = ops.paged_attention(q, *c.where())
    if device == "cuda":
        ops.check_status()
    assert torch.equal(got.isnan(), want.isnan())
    there = ~want.isnan()
    bound = HALF_STEP * (weight + want.abs()) + weight * (4 * c.dim * 2 * U32 * big + 2.0 ** -16)  # as in _check_attention
    assert ((got.double() - want).abs()[there] <= (bound * (1 + 2 ** -6) + 1e-38)[there]).all()


@pytest.mark.parametrize("device", DEVICES)
def test_attention_takes_scale_and_strided_queries(device):
    c = Paged([(50, 3), (0, 200)], 4, 4, 64, 16, device).fill()
    wide = torch.randn(c.tokens, 8, 64, device=device).bfloat16()
    for q in (wide[:, ::2], wide[:, 4:], wide[:, :1].expand(-1, 4, -1), wide[:1, :4].expand(c.tokens, -1, -1), wide.transpose(0, 1).contiguous().transpose(0, 1)[:, :4], wide.repeat(1, 1, 2)[:, 1:5, 1:65]):
        _check_attention(ops.paged_attention(q, *c.where(), scale=0.3), q, c, 0.3)


def test_plain_path_of_other_types():
    c = Paged([(20, 3), (0, 7)], 4, 2, 16, 16, "cpu", dtype=torch.float64).fill()
    q = torch.randn(c.tokens, 4, 16, dtype=torch.float64)
    torch.testing.assert_close(ops.paged_attention(q, *c.where()), _attend(q, c)[0], rtol=1e-12, atol=1e-12)


@pytest.mark.gpu
def test_other_types_run_plainly_on_the_gpu():
    c = Paged([(20, 3), (0, 7)], 4, 2, 80, 16, "cuda", dtype=torch.float32).fill()
    q = torch.randn(c.tokens, 4, 80, device="cuda")
    torch.testing.assert_close(ops.paged_attention(q, *c.where()).double(), _attend(q, c)[0], rtol=1e-4, atol=1e-5)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("new,wide", [(1, 3), (1, 5000), (90, 5000)])
def test_sequences_that_share_pages(device, new, wide):
    """The pages of a common beginning stand in both sequences' tables; each goes on in pages of its own."""
    c = Paged([(70, new), (64, new), (48, 0)], 4, 2, 64, 16, device, wide=wide).fill()
    c.table[1, :3] = c.table[0, :3]
    q = torch.randn(c.tokens, 4, 64, device=device).bfloat16()
    _check_attention(ops.paged_attention(q, *c.where()), q, c)


@pytest.mark.gpu
def test_pages_beyond_32_bits():
    """Pages of 2.6e9 values each: offsets that pass 2^31 values and 2^32 bytes, in both kernels and the append."""
    pages, size, heads, dim = 40000, 64, 8, 128
    c = Paged([(100, 1), (300, 40), (0, 200)], heads, heads, dim, size, "cpu")
    c.k = c.v = None
    c.k, c.v = (torch.empty(pages, size, heads, dim, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    c.table[c.table >= 0] += pages - 1 - int(c.table.max())
    c.table, c.offsets, c.lengths = c.table.cuda(), c.offsets.cuda(), c.lengths.cuda()
    c.fill(upto_new=False)
    q, k, v = (torch.randn(c.tokens, heads, dim, device="cuda").bfloat16() for _ in range(3))
    cos, sin = N.rotary_tables(512, dim, "cuda")
    turned = ops.paged_append(q, k, v, cos, sin, *c.where())
    ops.check_status()
    for b, (p, n) in enumerate(c.sizes):
        page, row = c.slots(b, p, p + n)
        rows = slice(c.starts[b], c.starts[b] + n)
        assert torch.equal(c.v[page, row], v[rows])
        want, most = _turned(k[rows], cos[p:p + n], sin[p:p + n], None)
        assert ((c.k[page, row].double() - want).abs() <= HALF_STEP * want.abs() + 16 * U32 * most).all()
    for most in (None, 200):
        _check_attention(ops.paged_attention(turned, *c.where(), max_new=most), turned, c)
    c.table = torch.cat([c.table, torch.zeros(3, 5000, dtype=torch.int32, device="cuda")], 1)
    _check_attention(ops.paged_attention(turned, *c.where()), turned, c)
    ops.check_status()


@pytest.mark.gpu
@pytest.mark.parametrize("new,wide", [(2, 8), (2, 5000), (90, 5000)])
def test_append_and_attention_in_a_graph_and_on_another_stream(new, wide):
    """Captured once and replayed with other lengths, tables and inputs; two graphs in turn, on a stream of their own."""
    sizes = [(40, new), (300, new), (0, new)]
    cos, sin = N.rotary_tables(512, 64, "cuda")
    side = torch.cuda.Stream()
    graphs = []
    for k in range(2):
        c = Paged([(p + 20 * k, n) for p, n in sizes], 8, 4, 64, 16, "cuda", wide=wide).fill(upto_new=False)
        qkv = torch.randn(c.tokens, 16, 64, device="cuda").bfloat16()

        def call(c=c, qkv=qkv):
            q, k_, v = qkv.split([8, 4, 4], 1)
            return ops.paged_attention(ops.paged_append(q, k_, v, cos, sin, *c.where(), norm_eps=1e-6), *c.where(), max_new=new)

        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            call()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                out = call()
        graphs.append((c, qkv, call, g, out))
    torch.cuda.synchronize()
    for step in range(3):
        for c, qkv, call, g, out in graphs:
            qkv.copy_(torch.randn(qkv.shape, device="cuda"))
            c.lengths.sub_(1).clamp_(min=0)
            with torch.cuda.stream(side):
                side.wait_stream(torch.cuda.default_stream())
                g.replay()
        torch.cuda.synchronize()
        for c, qkv, call, g, out in graphs:
            assert torch.equal(out, call())
    ops.check_status()


@pytest.mark.gpu
@pytest.mark.parametrize("new,wide", [(1, 8), (2, 5000), (90, 5000)])
def test_a_graph_follows_the_pages_as_they_move(new, wide):
    """Captured once; between replays the pages go to other places, the table is changed in place to match, sequences grow and the
    inputs change.  Results and pages against the definitions, and rows that are nobody's as they were."""
    c = Paged([(40, new), (300, new), (0, new)], 8, 4, 64, 16, "cuda", wide=wide, garbage=3.0, spare=9).fill(upto_new=False)
    room = [int((row >= 0).sum()) * 16 for row in c.table]  # of each sequence's pages
    cos, sin = N.rotary_tables(512, 64, "cuda")
    qkv = torch.randn(c.tokens, 16, 64, device="cuda").bfloat16()

    def call():
        q, k, v = qkv.split([8, 4, 4], 1)
        turned = ops.paged_append(q, k, v, cos, sin, *c.where(), norm_eps=1e-6)
        return turned, ops.paged_attention(turned, *c.where(), max_new=new)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            turned, out = call()
    torch.cuda.synchronize()
    for step in range(4):
        to = torch.randperm(c.k.shape[0], device="cuda")  # page i goes to to[i]
        for t in (c.k, c.v):
            moved = torch.empty_like(t)
            moved[to] = t
            t.copy_(moved)
        c.table.copy_(torch.where(c.table >= 0, to[c.table.clamp_min(0).long()].int(), c.table))
        c.sizes = [(max(0, min(p + (3 if step % 2 else -5), r - n)), n) for (p, n), r in zip(c.sizes, room)]
        c.lengths.copy_(torch.tensor([p for p, _ in c.sizes], dtype=torch.int32))
        qkv.copy_(torch.randn(qkv.shape, device="cuda"))
        q, k, v = qkv.split([8, 4, 4], 1)
        was_k, was_v = c.k.clone(), c.v.clone()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            g.replay()
        torch.cuda.current_stream().wait_stream(side)
        ops.check_status()
        touched = torch.zeros(c.k.shape[:2], dtype=torch.bool, device="cuda")
        for b, (p, n) in enumerate(c.sizes):
            rows = slice(c.starts[b], c.starts[b] + n)
            at = c.slots(b, p, p + n)
            touched[at] = True
            for got, x in ((turned[rows], q[rows]), (c.k[at], k[rows])):
                want, most = _turned(x, cos[p:p + n], sin[p:p + n], 1e-6)
                assert ((got.double() - want).abs() <= HALF_STEP * want.abs() + 2 * U32 * (8 + 64) * most + 1e-38).all()  # as in test_append
            assert torch.equal(c.v[at], v[rows])
        assert torch.equal(c.k[~touched], was_k[~touched]) and torch.equal(c.v[~touched], was_v[~touched])
        _check_attention(out, turned, c)


# --------------------------------------------------------------------------- check of drafts

def _verify(p, q, tokens, u):
    accepted, out = [], []
    for b in range(tokens.shape[0]):
        a, k = 0, tokens.shape[1]
        while a < k and u[b, a].item() * (1.0 if q is None else q[b, a, tokens[b, a]].item()) < p[b, a, tokens[b, a]].item():
            a += 1
        w = p[b, a].double()
        if a < k:
            r = w.clone()
            if q is None:
                r[tokens[b, a]] -= 1.0
            else:
                r -= q[b, a].double()
            w = r.clamp_min(0) if (r > 0).any() else w
        upto = w.cumsum(0)
        accepted.append(a)
        out.append(int((upto <= u[b, k].item() * upto[-1]).sum()) if upto[-1] > 0 else 0)
    return torch.tensor(accepted), torch.tensor(out)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("seqs,drafts,vocab", [(1, 4, 50304), (5, 1, 1), (7, 3, 33), (3, 0, 1000), (64, 8, 4097), (2, 2, 128256), (40, 5, 1031)])
@pytest.mark.parametrize("certain", [False, True])
def test_verify(device, seqs, drafts, vocab, certain):
    p = torch.softmax(torch.randn(seqs, drafts + 1, vocab) * 2, -1)
    q = None if certain else torch.softmax(p[:, :drafts].log() + torch.randn(seqs, drafts, vocab), -1)
    tokens = p[:, :drafts].argmax(-1) if certain else torch.multinomial(q.reshape(-1, vocab), 1).view(seqs, drafts) if drafts else torch.zeros(seqs, 0, dtype=torch.long)
    u = torch.rand(seqs, drafts + 1)
    u[0, -1] = 0.0
    u[-1, -1] = 1 - 2.0 ** -24
    want = _verify(p, q, tokens, u)
    dev = [None if t is None else t.to(device) for t in (p, q, tokens, u)]
    got = ops.verify_drafts(*dev)
    if device == "cuda":
        ops.check_status()
    assert all(g.dtype == torch.int64 and torch.equal(g.cpu(), w) for g, w in zip(got, want))


@pytest.mark.parametrize("device", DEVICES)
def test_verify_at_the_borders(device):
    """Equal distributions are always accepted, impossible drafts never; what is left over decides, zeros are not drawn."""
    p = torch.zeros(5, 2, 8)
    q = torch.zeros(5, 1, 8)
    tokens = torch.tensor([[3], [3], [2], [5], [1]])
    u = torch.tensor([[1 - 2.0 ** -24, 0.5], [0.0, 0.0], [0.5, 0.999], [0.25, 0.5], [0.9, 0.0]])
    p[0, :, 3] = q[0, :, 3] = 1.0                        # sure of the same token
    p[1, 0, 6], q[1, 0, 3] = 1.0, 1.0                    # u q = 0 is not below p = 0
    p[2, 0, 2:4], q[2, 0, 2] = 0.5, 1.0                  # u q = 0.5 is not below p = 0.5; the rest is token 3
    p[3, 0], q[3, 0, 5] = torch.full((8,), math.nan), 1.0  # no numbers: refused, nothing to draw from
    p[4, 0, 1], p[4, 0, 4], q[4, 0, 1], q[4, 0, 4] = 0.25, 0.25, 0.5, 0.5  # nothing is left over: the target's row itself
    got = ops.verify_drafts(*(t.to(device) for t in (p, q, tokens, u)))
    assert got[0].tolist() == [1, 0, 0, 0, 0] and got[1].tolist() == [3, 6, 3, 0, 1]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("seqs,drafts,vocab,top_k", [(16, 4, 50304, 50), (24, 7, 128256, 50), (9, 3, 50304, 1), (5, 2, 128256, 3), (12, 5, 40001, 7)])
@pytest.mark.parametrize("certain", [False, True])
def test_verify_of_rows_that_are_mostly_zeros(device, seqs, drafts, vocab, top_k, certain):
    """What sampling from the most likely tokens hands over: the distributions' few tokens anywhere, and partly the same ones."""
    if device == "cpu":
        seqs = min(seqs, 4)
    logits = torch.randn(seqs, drafts + 1, vocab) * 2

    def top(x):
        return torch.softmax(x.masked_fill(x < x.topk(top_k).values[..., -1:], -math.inf), -1)

    p, q = top(logits), None if certain else top(logits[:, :drafts] + torch.randn(seqs, drafts, vocab) * 0.1)
    tokens = torch.multinomial((p[:, :drafts] if certain else q).reshape(-1, vocab), 1).view(seqs, drafts)
    u = torch.rand(seqs, drafts + 1)
    u[0], u[-1, -1] = 0.0, 1 - 2.0 ** -24
    want = _verify(p, q, tokens, u)
    got = ops.verify_drafts(*[None if t is None else t.to(device) for t in (p, q, tokens, u)])
    if device == "cuda":
        ops.check_status()
    assert all(torch.equal(g.cpu(), w) for g, w in zip(got, want))
    assert (p[torch.arange(seqs), want[0], want[1]] > 0).all()


@pytest.mark.parametrize("device", DEVICES)
def test_verify_takes_strided_rows(device):
    p = torch.softmax(torch.randn(4, 6, 300, device=device), -1)
    q = torch.softmax(torch.randn(4, 6, 300, device=device), -1)
    tokens, u = torch.randint(0, 300, (4, 6), device=device), torch.rand(4, 6, device=device)
    want = ops.verify_drafts(p[:, ::2].contiguous(), q[:, 1::3].contiguous(), tokens[:, 1::3].contiguous(), u[:, :3].contiguous())
    got = ops.verify_drafts(p[:, ::2], q[:, 1::3], tokens[:, 1::3], u[:, :3])
    again = ops.verify_drafts(p.transpose(1, 2).contiguous().transpose(1, 2)[:, ::2], q[:, 1::3], tokens[:, 1::3], u[:, :3])
    assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(want, got, again))


def test_verified_tokens_follow_the_target():
    """Over every cell of a fine grid of uniforms, drafts weighted by their probability: the token that comes out is
    distributed as the target's row, to the width of the grid's cells."""
    p, q = torch.tensor([0.1, 0.5, 0.25, 0.15]), torch.tensor([0.4, 0.3, 0.0, 0.3])
    g = 128
    mid = (torch.arange(g) + 0.5) / g
    u = torch.stack(torch.meshgrid(mid, mid, indexing="ij"), -1).reshape(-1, 2)
    share = torch.zeros(4, dtype=torch.float64)
    for x in range(4):
        n = u.shape[0]
        a, t = ops.verify_drafts(p.expand(n, 2, 4), q.expand(n, 1, 4), torch.full((n, 1), x), u)
        first = torch.where(a == 1, torch.full_like(t, x), t)
        share += q[x].double() * torch.bincount(first, minlength=4) / n
    assert (share - p.double()).abs().max() <= 4 * 2 / g


# --------------------------------------------------------------------------- refusals

def _call(c, query, **changes):
    a = dict(q=query, k_pages=c.k, v_pages=c.v, page_table=c.table, new_offsets=c.offsets, lengths=c.lengths)
    a.update(changes)
    return ops.paged_attention(**a)


@pytest.mark.parametrize("device", DEVICES)
def test_refusals_of_shapes_and_types(device):
    c = Paged([(20, 2), (3, 1)], 4, 2, 64, 16, device).fill()
    q = torch.randn(3, 4, 64, device=device).bfloat16()
    odd = torch.zeros(4, 24, 2, 64, dtype=torch.bfloat16, device=device)
    small = torch.zeros(4, 8, 2, 64, dtype=torch.bfloat16, device=device)
    for changes in (dict(q=q[0]), dict(k_pages=c.k[0]), dict(k_pages=c.k[:2]), dict(k_pages=odd, v_pages=odd), dict(k_pages=small, v_pages=small),
                    dict(q=q[:, :3]), dict(q=torch.cat([q, q], -1)), dict(k_pages=c.k.half(), v_pages=c.v.half()),
                    dict(page_table=c.table.long()), dict(page_table=c.table[:1]), dict(new_offsets=c.offsets[:2]),
                    dict(lengths=c.lengths.float()), dict(lengths=c.lengths[None]), dict(new_offsets=c.offsets.long())):
        with pytest.raises(ValueError):
            _call(c, q, **changes)
    for changes in (dict(scale=0.0), dict(scale=-1.0), dict(scale=math.nan), dict(scale=math.inf), dict(scale=1e-40), dict(scale=1e40), dict(max_new=0)):
        with pytest.raises(ValueError):
            ops.paged_attention(q, *c.where(), **changes)
    k = v = q[:, :2]
    cos, sin = N.rotary_tables(64, 64, device)
    for args in ((q, k[:2], v, cos, sin), (q, k, v[:, :1], cos, sin), (q, k, v.float(), cos, sin), (q, k, v, cos[:, :16], sin),
                 (q, k, v, cos, sin.float()), (q, k, v, cos[0], sin[0])):
        with pytest.raises(ValueError):
            ops.paged_append(*args, *c.where())
    for eps in (-1.0, math.nan):
        with pytest.raises(ValueError):
            ops.paged_append(q, k, v, cos, sin, *c.where(), norm_eps=eps)
    p, d = torch.rand(2, 4, 9, device=device), torch.rand(2, 3, 9, device=device)
    t, u = torch.zeros(2, 3, dtype=torch.long, device=device), torch.rand(2, 4, device=device)
    for args in ((p[0], d, t, u), (p.double(), d, t, u), (p, d[:, :2], t, u), (p, d, t[:1], u), (p, d, t.int(), u), (p, d, t, u[:, :3]),
                 (p, d.bfloat16(), t, u), (p, d[..., :8], t, u), (p[..., :0], d[..., :0], t, u), (p[:, :0], None, t[:, :0], u[:, :0])):
        with pytest.raises(ValueError):
            ops.verify_drafts(*args)


@pytest.mark.parametrize("device", DEVICES)
def test_rotation_tables_beyond_32_bits_are_refused(device):
    """Positions are 32-bit numbers in the kernel.  One row of either table, which stands for all of them, in no memory."""
    c = Paged([(20, 2)], 2, 2, 64, 16, device).fill()
    q = torch.randn(2, 2, 64, device=device).bfloat16()
    cos, sin = (t[:1] for t in N.rotary_tables(1, 64, device))
    for rows, good in ((2 ** 31 - 1, True), (2 ** 31, False)):
        tables = cos.expand(rows, -1), sin.expand(rows, -1)
        if good:
            ops.paged_append(q, q, q, *tables, *c.where())
        else:
            with pytest.raises(ValueError, match="2\\^31"):
                ops.paged_append(q, q, q, *tables, *c.where())


@pytest.mark.parametrize("device", DEVICES)
def test_gradients_are_refused(device):
    c = Paged([(20, 2)], 2, 2, 64, 16, device).fill()
    q = torch.randn(2, 2, 64, device=device).bfloat16().requires_grad_()
    cos, sin = N.rotary_tables(64, 64, device)
    p = torch.rand(1, 2, 9, device=device, requires_grad=True)
    t, u = torch.zeros(1, 1, dtype=torch.long, device=device), torch.rand(1, 2, device=device)
    for call in (lambda: ops.paged_attention(q, *c.where()), lambda: ops.paged_append(q, q.detach(), q.detach(), cos, sin, *c.where()),
                 lambda: ops.verify_drafts(p, None, t, u)):
        with pytest.raises(RuntimeError, match="gradient"):
            call()
        with torch.no_grad():
            call()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("which", ["cos", "sin"])
def test_gradients_of_the_rotation_tables_are_refused(device, which):
    c = Paged([(20, 2)], 2, 2, 64, 16, device, garbage=7.0).fill()
    q = torch.randn(2, 2, 64, device=device).bfloat16()
    tables = dict(zip(("cos", "sin"), N.rotary_tables(64, 64, device)))
    tables[which] = tables[which].clone().requires_grad_()
    was = c.both.clone()
    with pytest.raises(RuntimeError, match="gradient"):
        ops.paged_append(q, q, q, *tables.values(), *c.where())
    assert torch.equal(c.both, was)
    with torch.no_grad():
        assert not ops.paged_append(q, q, q, *tables.values(), *c.where()).requires_grad


@pytest.mark.gpu
def test_tangents_are_refused_by_the_kernels():
    """A forward-mode derivative would be lost there, whichever input it comes with, and under no_grad too."""
    c = Paged([(20, 2)], 2, 2, 64, 16, "cuda", garbage=7.0).fill()
    q = torch.randn(2, 2, 64, device="cuda").bfloat16()
    p, d = torch.rand(1, 2, 9, device="cuda"), torch.rand(1, 1, 9, device="cuda")
    t, u = torch.zeros(1, 1, dtype=torch.long, device="cuda"), torch.rand(1, 2, device="cuda")
    calls = [(lambda q, k, v, cos, sin, k_pages, v_pages: ops.paged_append(q, k, v, cos, sin, k_pages, v_pages, *c.where()[2:]),
              (q, q, q, *N.rotary_tables(64, 64, "cuda"), c.k, c.v)),
             (lambda q, k_pages, v_pages: ops.paged_attention(q, k_pages, v_pages, *c.where()[2:]), (q, c.k, c.v)),
             (lambda p, d, u: ops.verify_drafts(p, d, t, u), (p, d, u))]
    was = c.both.clone()
    for call, args in calls:
        for i, x in enumerate(args):
            with fwd.dual_level():
                dual = list(args)
                dual[i] = fwd.make_dual(x, torch.ones_like(x))
                for grad in (True, False):
                    with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="forward-mode"):
                        call(*dual)
    assert torch.equal(c.both, was)
    for call, args in calls:
        call(*args)
    ops.check_status()


def test_the_plain_path_carries_tangents():
    c = Paged([(20, 2)], 2, 2, 16, 16, "cpu", dtype=torch.float64).fill()
    q, t = torch.randn(2, 2, 2, 16, dtype=torch.float64)
    with fwd.dual_level():
        got = fwd.unpack_dual(ops.paged_attention(fwd.make_dual(q, t), *c.where())).tangent
    h = 1e-6  # the difference is off by h^2 / 6 of a third derivative, at most some tens here, and by roundings over 2 h
    want = (ops.paged_attention(q + h * t, *c.where()) - ops.paged_attention(q - h * t, *c.where())) / (2 * h)
    torch.testing.assert_close(got, want, rtol=0, atol=1e-7)


def _bad(device):
    """(what, changed tensors) that only the values tell from good ones."""
    def table(c, b, i, to):
        t = c.table.clone()
        t[b, i] = to
        return dict(page_table=t)

    def ints(*v):
        return torch.tensor(v, dtype=torch.int32, device=device)

    return [("a page below", lambda c: table(c, 1, 1, -1)), ("a page beyond", lambda c: table(c, 0, 1, c.k.shape[0])),
            ("a page far beyond", lambda c: table(c, 1, 1, 2 ** 31 - 1)),
            ("a length below zero", lambda c: dict(lengths=ints(20, -1))), ("a length beyond the table", lambda c: dict(lengths=ints(20, 16 * c.table.shape[1] - 1))),
            ("the largest length", lambda c: dict(lengths=ints(2 ** 31 - 1, 17))),
            ("offsets that fall", lambda c: dict(new_offsets=ints(0, 3, 2))), ("offsets beyond the tokens", lambda c: dict(new_offsets=ints(0, 2, 2 ** 31 - 1))),
            ("offsets below zero", lambda c: dict(new_offsets=ints(-4, 2, 4))), ("offsets that start late", lambda c: dict(new_offsets=ints(1, 2, 4)))]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("what", range(10))
@pytest.mark.parametrize("most", [None, 2])
@pytest.mark.parametrize("wide", [3, 5000])
def test_bad_values_are_reported_and_touch_nothing(device, what, most, wide):
    c = Paged([(20, 2), (17, 2)], 2, 2, 64, 16, device, garbage=7.0, wide=wide).fill()
    change = _bad(device)[what][1](c)
    a = dict(k_pages=c.k, v_pages=c.v, page_table=c.table, new_offsets=c.offsets, lengths=c.lengths)
    a.update(change)
    q = torch.randn(4, 2, 64, device=device).bfloat16()
    cos, sin = N.rotary_tables(64, 64, device)
    before = c.both.clone()
    own = torch.zeros(c.k.shape[:2], dtype=torch.bool, device=device)  # rows that good values may reach
    for b, (p, n) in enumerate(c.sizes):
        own[c.slots(b, 0, p + n)] = True
    calls = (lambda: ops.paged_attention(q, **a, max_new=most), lambda: ops.paged_append(q, q, q, cos, sin, **a))
    for call in calls:
        if device == "cpu":
            with pytest.raises(ValueError):
                call()
        else:
            call()
            with pytest.raises(ops.DionKernelError, match="bad kernel argument"):
                ops.check_status()
    if what not in (6, 7, 8, 9):  # where offsets are wrong, rows of other sequences are written where these may write
        now = c.both.clone()
        c.both.copy_(before)
        was_k, was_v = c.k[~own].clone(), c.v[~own].clone()
        c.both.copy_(now)
        assert torch.equal(c.k[~own], was_k) and torch.equal(c.v[~own], was_v)


@pytest.mark.parametrize("device", DEVICES)
def test_positions_beyond_the_rotation_tables_are_reported(device):
    c = Paged([(20, 2)], 2, 2, 64, 16, device, garbage=7.0).fill()
    q = torch.randn(2, 2, 64, device=device).bfloat16()
    cos, sin = N.rotary_tables(21, 64, device)
    if device == "cpu":
        with pytest.raises(ValueError):
            ops.paged_append(q, q, q, cos, sin, *c.where())
        return
    out = ops.paged_append(q, q, q, cos, sin, *c.where())
    with pytest.raises(ops.DionKernelError):
        ops.check_status()
    assert (out[0] != 0).any() and (out[1] == 0).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dim,eps,wide", [(64, None, False), (64, 1e-6, True), (128, 1e-6, False), (128, None, True)])
@pytest.mark.parametrize("new,tail", [(2, 0), (0, 3), (700, 5)])
def test_rotation_tables_without_a_row(device, dim, eps, wide, new, tail):
    """Every position lies beyond them, and rows that are nobody's need none: nothing is read from them and nothing is written
    to the pages."""
    c = Paged([(20, new), (5, 0)], 2, 2, dim, 16, device, garbage=7.0, tail=tail).fill()
    q = torch.randn(c.tokens, 2, dim, device=device).bfloat16()
    cos, sin = (t[:0].float() if wide else t[:0] for t in N.rotary_tables(8, dim, device))
    was_k, was_v = c.k.clone(), c.v.clone()
    if device == "cpu" and new:
        with pytest.raises(ValueError, match="rotation tables"):
            ops.paged_append(q, q, q, cos, sin, *c.where(), norm_eps=eps)
        return
    out = ops.paged_append(q, q, q, cos, sin, *c.where(), norm_eps=eps)
    if new:
        with pytest.raises(ops.DionKernelError, match="bad kernel argument"):
            ops.check_status()
    elif device == "cuda":
        ops.check_status()
    assert (out == 0).all() and torch.equal(c.k, was_k) and torch.equal(c.v, was_v)


@pytest.mark.parametrize("device", DEVICES)
def test_more_new_tokens_than_announced(device):
    c = Paged([(20, 1), (5, 100)], 2, 2, 64, 16, device).fill()
    q = torch.randn(101, 2, 64, device=device).bfloat16()
    if device == "cpu":
        with pytest.raises(ValueError):
            ops.paged_attention(q, *c.where(), max_new=1)
        return
    ops.paged_attention(q, *c.where(), max_new=1)
    with pytest.raises(ops.DionKernelError):
        ops.check_status()


@pytest.mark.parametrize("device", DEVICES)
def test_drafts_outside_the_vocabulary_are_reported(device):
    p, d = torch.rand(2, 3, 9, device=device), torch.rand(2, 2, 9, device=device)
    u = torch.zeros(2, 3, device=device)
    for bad in (-1, 9, 2 ** 62):
        t = torch.tensor([[1, 2], [bad, 3]], device=device)
        if device == "cpu":
            with pytest.raises(ValueError):
                ops.verify_drafts(p, d, t, u)
            continue
        accepted, token = ops.verify_drafts(p, d, t, u)
        with pytest.raises(ops.DionKernelError):
            ops.check_status()
        assert accepted.tolist() == [2, 0] and 0 <= token[1] < 9


@pytest.mark.gpu
def test_pages_that_the_kernels_cannot_address_are_refused():
    c = Paged([(20, 2)], 2, 2, 64, 16, "cuda").fill()
    q = torch.randn(2, 2, 64, device="cuda").bfloat16()
    n = c.k.numel()
    late = torch.zeros(n + 4, device="cuda").bfloat16()[4:].view(c.k.shape)
    odd = torch.zeros(*c.k.shape[:3], 68, device="cuda").bfloat16()[..., :64]
    apart = torch.zeros(*c.k.shape, 2, device="cuda").bfloat16()[..., 0]
    one = torch.zeros(1, *c.k.shape[1:], device="cuda").bfloat16().expand(c.k.shape)
    for pages in (late, odd, apart, one):
        with pytest.raises(ValueError):
            _call(c, q, k_pages=pages)
    with pytest.raises(ValueError):
        _call(c, q, lengths=c.lengths.cpu())
    with pytest.raises(ValueError):
        _call(c, q, v_pages=c.v.cpu())


@pytest.mark.parametrize("device", DEVICES)
def test_nothing_to_do(device):
    pages = torch.zeros(0, 16, 2, 64, device=device).bfloat16()
    ints = [torch.zeros(s, dtype=torch.int32, device=device) for s in ((0, 4), (1,), (0,))]
    cos, sin = N.rotary_tables(8, 64, device)
    for n in (0, 3):
        q = torch.randn(n, 4, 64, device=device).bfloat16()
        out = ops.paged_attention(q, pages, pages.clone(), *ints)
        assert out.shape == q.shape and (out == 0).all()
        out = ops.paged_append(q, q[:, :2], q[:, :2], cos, sin, pages, pages.clone(), *ints)
        assert out.shape == q.shape and (out == 0).all()
    got = ops.verify_drafts(torch.zeros(0, 3, 7, device=device), None, torch.zeros(0, 2, dtype=torch.long, device=device), torch.zeros(0, 3, device=device))
    assert [t.shape for t in got] == [(0,), (0,)]

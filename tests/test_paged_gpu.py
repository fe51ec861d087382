"""qk_norm_rope, paged_append and paged_attention against their definitions in 64 bits.

Tolerances, derived: u = eps / 2 is a rounding to the type, e = 2^-24 one to fp32.
  rows     the norm's sum (at most 16 additions one behind the other, halved by the root), root, division, two products, sine and cosine
           (1e-7 < 2 e each), two products and a sum: under 24 e of |a| + |b| (the pair before it turns), and u of the result.
  attention  a probability is rounded to the type (u) and the sum takes it as rounded, so a weight w_j is off by u w_j against
           the others: u (sum w |v| + |o|). A score is off by at most (dim + 8) e scale sum |q| |k|, twice (numerator, sum), exp2 and the
           joining of parts by 16 e. fp16 probabilities below 2^-14 of a row's largest are off by 2^-25 of it each. The result: u |o|.
"""
import math
import random
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def rows64(x, weight, inv_freq, positions, eps, pairs):
    """(result, |a| + |b|) of the rows [tokens, heads, dim] in 64 bits on the CPU."""
    x = x.cpu().double()
    if weight is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * weight.cpu().double()
    size = x.abs()
    if inv_freq is None:
        return x, size
    angle = (positions.cpu().double()[:, None] * inv_freq.cpu())[:, None]
    c, s, n = angle.cos(), angle.sin(), inv_freq.numel()
    first = torch.arange(n) * 2 if pairs == "adjacent" else torch.arange(n)
    second = first + 1 if pairs == "adjacent" else first + n
    out, a, b = x.clone(), x[..., first], x[..., second]
    out[..., first], out[..., second] = a * c - b * s, b * c + a * s
    size[..., first] = size[..., second] = a.abs() + b.abs()
    return out, size


def check_rows(got, want, what=""):
    out, size = want
    assert got.shape == out.shape
    off = (got.cpu().double() - out).abs()
    # below the least normal number a rounding is half of a subnormal step, whatever the value
    bound = half_step(got.dtype) * out.abs() + 24 * E * size + torch.finfo(got.dtype).tiny * half_step(got.dtype)
    bad = ~(off <= bound)
    assert not bad.any(), (what, bad.sum().item(), off[bad].max().item(), bound[bad].min().item())


ROWS = [
    # tokens, heads, kv heads (0: no k), dim, rotated columns, dtype, pairs, norms (q, k), positions up to
    (1, 1, 0, 2, 2, "f32", "adjacent", (False, False), 9), (1, 32, 8, 128, 128, "bf16", "halves", (True, True), 1 << 20),
    (3, 5, 1, 64, 32, "f16", "halves", (True, False), 100), (257, 12, 12, 64, 64, "f16", "adjacent", (False, False), 4096),
    (33, 4, 2, 80, 40, "bf16", "halves", (False, True), 5000), (7, 3, 3, 96, 48, "f16", "halves", (True, True), 70000),
    (5, 2, 1, 256, 256, "f16", "halves", (True, True), 1000), (9, 7, 2, 256, 100, "bf16", "adjacent", (True, True), 1000),
    (4, 3, 1, 20, 10, "f32", "halves", (True, True), 1000), (6, 2, 2, 66, 6, "f16", "adjacent", (True, True), 1000),
    (2, 3, 1, 512, 512, "f32", "halves", (True, True), 1 << 30), (130, 8, 2, 128, 64, "f32", "adjacent", (True, False), 1 << 20),
    (21, 2, 2, 7, 0, "f16", "adjacent", (True, True), 5), (1000, 2, 1, 128, 128, "bf16", "halves", (True, True), 131072),
    (64, 1, 1, 8, 8, "bf16", "halves", (True, True), 100), (40, 6, 2, 16, 16, "f32", "halves", (True, True), 100),
    (12, 10, 2, 104, 104, "f16", "adjacent", (True, True), 100), (11, 64, 64, 128, 128, "f16", "halves", (False, False), 100),
]


@pytest.mark.parametrize("case", ROWS, ids=str)
@pytest.mark.parametrize("form", ["slices", "whole", "in_place"])
def test_rows_against_the_definition(hexmi, case, form):
    T, H, K, D, R, dt, pairs, (nq, nk), far = case
    g, dtype = _gen(T * 1000 + D), DTYPES[dt]
    wide = (torch.randn(T, (H + K + 1) * D, generator=g) * 2).to(dtype).cuda()
    q, k = wide[:, :H * D].unflatten(1, (H, D)), wide[:, H * D:(H + K) * D].unflatten(1, (K, D)) if K else None
    if form == "whole":
        q, k = q.contiguous(), k.contiguous() if K else None
    qw = (1 + 0.2 * torch.randn(D, generator=g)).to(dtype).cuda() if nq else None
    kw = (1 + 0.2 * torch.randn(D, generator=g)).to(dtype).cuda() if nk and K else None
    freq = hexmi.rope_frequencies(R, 10000.0) if R else None
    pos = torch.randint(0, far, (T,), generator=g, dtype=torch.int64 if T % 2 else torch.int32).cuda()
    want = [rows64(x, w, freq, pos, 1e-5, pairs) if x is not None else None for x, w in ((q, qw), (k, kw))]
    before = wide.clone()
    outs = {"q_out": q, "k_out": k} if form == "in_place" else {}
    got = hexmi.qk_norm_rope(q, k, qw, kw, freq, pos, 1e-5, pairs, **outs)
    got = got if K else (got,)
    check_rows(got[0], want[0], "q")
    if K:
        check_rows(got[1], want[1], "k")
    if form == "in_place":
        assert got[0].data_ptr() == q.data_ptr()
        assert torch.equal(wide[:, (H + K) * D:], before[:, (H + K) * D:])           # what stands beside the rows
    else:
        assert torch.equal(wide, before)
        ptrs = [t.data_ptr() for t in got]
        again = hexmi.qk_norm_rope(q, k, qw, kw, freq, pos, 1e-5, pairs, q_out=torch.empty_like(got[0]))   # the route through ctypes
        again = again if K else (again,)
        assert all(torch.equal(a, b) for a, b in zip(got, again)) and ptrs != [t.data_ptr() for t in again]


def test_rows_off_the_boundaries_and_far_and_negative_positions(hexmi):
    g = _gen(3)
    base = torch.randn(1 + 50 * 3 * 64, generator=g).half().cuda()
    q = base[1:].view(50, 3, 64)                                  # two bytes off
    pos = torch.randint(-(1 << 31), (1 << 31) - 1, (50,), generator=g).cuda()
    freq = hexmi.rope_frequencies(64, 500000.0)
    for pairs in ("adjacent", "halves"):
        # positions of 2^31 times frequencies of 1 are whole in 53 bits; the product's own rounding is 2^-53 of 2^31 turns
        out, size = rows64(q, None, freq, pos, 1e-5, pairs)
        check_rows(hexmi.qk_norm_rope(q, None, None, None, freq, pos, pairs=pairs), (out, size * 2), pairs)


def test_rows_take_host_tensors_and_other_streams(hexmi):
    g = _gen(4)
    q, k, w = torch.randn(9, 4, 64, generator=g).half(), torch.randn(9, 2, 64, generator=g).half(), torch.ones(64).half()
    freq, pos = hexmi.rope_frequencies(64), torch.arange(9)
    qo, ko = torch.zeros_like(q), torch.zeros_like(k)
    got = hexmi.qk_norm_rope(q, k, w, w, freq, pos, q_out=qo, k_out=ko)
    assert got[0] is qo and got[1] is ko and not qo.is_cuda
    check_rows(qo, rows64(q, w, freq, pos, 1e-5, "adjacent"))
    check_rows(ko, rows64(k, w, freq, pos, 1e-5, "adjacent"))
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        qd, kd, wd, pd = q.cuda(), k.cuda(), w.cuda(), pos.cuda()
        a, b = hexmi.qk_norm_rope(qd, kd, wd, wd, freq, pd)
    stream.synchronize()
    assert torch.equal(a.cpu(), qo) and torch.equal(b.cpu(), ko)


def test_rows_with_infinities_beside_what_turns(hexmi):
    q = torch.ones(1, 1, 64, dtype=torch.float16, device="cuda")
    q[..., 40], q[..., 41] = math.inf, -math.inf
    got = hexmi.qk_norm_rope(q, None, None, None, hexmi.rope_frequencies(36), torch.tensor([5], device="cuda"))
    assert got[0, 0, 40].item() == math.inf and got[0, 0, 41].item() == -math.inf and torch.isfinite(got[0, 0, :40]).all()


class Cache:
    """A cache and a batch: pages in random order, everything that no token owns NaN, and the tokens in 64 bits beside it."""

    def __init__(self, new, context, heads, kv_heads, dim, page, dtype, order="head", seed=0, padding=0, spare=3, ragged=None, shared=0,
                 scale=1.0):
        g = _gen(seed)
        self.new, self.lengths = list(new), [c + n for c, n in zip(context, new)]
        self.heads, self.kv_heads, self.dim, self.page, self.dtype = heads, kv_heads, dim, page, dtype
        self.ragged = any(n != 1 for n in new) or padding > 0 if ragged is None else ragged
        B, T = len(new), sum(new) + padding
        columns = [-(-n // page) for n in self.lengths]
        first = shared // page
        pool = first + sum(max(0, c - first) for c in columns) + spare
        order_of = torch.randperm(pool, generator=g, dtype=torch.int32)
        self.table = torch.full((B, max(columns + [1]) + 1), -1, dtype=torch.int32)
        self.shared_pages = order_of[:first].clone().cuda() if first else None
        used = first
        for b, c in enumerate(columns):
            self.table[b, :min(first, c)] = order_of[:min(first, c)]
            if c > first:
                self.table[b, first:c] = order_of[used:used + c - first]
                used += c - first
        shape = (pool, kv_heads, page, dim) if order == "head" else (pool, page, kv_heads, dim)
        self.k_pages, self.v_pages = (torch.full(shape, math.nan, dtype=dtype, device="cuda") for _ in range(2))
        if order != "head":
            self.k_pages, self.v_pages = self.k_pages.transpose(1, 2), self.v_pages.transpose(1, 2)
        self.q = (torch.randn(T, heads, dim, generator=g) * scale).to(dtype).cuda()
        # every token's key and value in 64 bits, [length, kv heads, dim], the shared ones the same for all
        common = [torch.randn(shared, kv_heads, dim, generator=g).to(dtype) for _ in range(2)]
        self.k64, self.v64 = [], []
        for b, n in enumerate(self.lengths):
            kv = [torch.cat((c, torch.randn(max(0, n - shared), kv_heads, dim, generator=g).to(dtype)))[:n] for c in common]
            at = torch.arange(n)
            for pages, t in zip((self.k_pages, self.v_pages), kv):
                if n:
                    pages[self.table[b][at // page].long().cuda(), :, (at % page).cuda()] = t.cuda()
            self.k64.append(kv[0].double())
            self.v64.append(kv[1].double())
        self.page_table = self.table.cuda()
        self.lengths_d = torch.tensor(self.lengths, dtype=torch.int32, device="cuda")
        starts = [sum(self.new[:i]) for i in range(B + 1)]
        self.starts = torch.tensor(starts, dtype=torch.int32, device="cuda") if self.ragged else None

    def batch(self):
        return self.k_pages, self.v_pages, self.page_table, self.lengths_d, self.starts

    def attention64(self, sm_scale=None):
        """(result, bound) on the CPU."""
        scale = 1.0 / math.sqrt(self.dim) if sm_scale is None else sm_scale
        G, u = self.heads // self.kv_heads, half_step(self.dtype)
        q = self.q.cpu().double()
        out, bound = torch.zeros_like(q), torch.zeros_like(q)
        t = 0
        for n, L, k, v in zip(self.new, self.lengths, self.k64, self.v64):
            for h in range(self.heads if n and L else 0):
                kh, vh, qh = k[:, h // G], v[:, h // G], q[t:t + n, h]
                hidden = torch.arange(L)[None] > torch.arange(L - n, L)[:, None]
                s = (qh @ kh.T * scale).masked_fill(hidden, -math.inf)
                w = torch.softmax(s, 1).nan_to_num(0.0)                     # a row without a key: zeros
                size = (qh.abs() @ kh.abs().T * scale).masked_fill(hidden, 0).amax(1, keepdim=True)
                o, a = w @ vh, w @ vh.abs()
                out[t:t + n, h] = o
                b = u * (a + o.abs()) + (2 * (self.dim + 8) * E * size + 16 * E) * (a + o.abs()) + u * o.abs()
                if self.dtype == torch.float16:
                    b = b + L * 2.0 ** -25 * vh.abs().amax(0) + 2.0 ** -25
                bound[t:t + n, h] = b
            t += n
        return out, bound

    def check(self, got, sm_scale=None, what=""):
        out, bound = self.attention64(sm_scale)
        assert got.shape == out.shape and got.dtype == self.dtype
        off = (got.cpu().double() - out).abs()
        bad = ~(off <= bound)
        assert not bad.any(), (what, bad.sum().item(), (off / bound.clamp_min(1e-30))[bad].max().item(), bad.nonzero()[:3].tolist())


DECODE = [
    # contexts, heads, kv heads, dim, page, dtype, order
    ([0], 1, 1, 64, 16, "f16", "head"), ([0, 0, 3], 4, 2, 128, 16, "bf16", "token"), ([999], 32, 8, 128, 16, "f16", "head"),
    ([15, 16, 17, 31, 32, 33, 62, 63, 64, 65], 8, 2, 128, 16, "f16", "head"), ([127, 128, 255, 256, 257], 12, 12, 64, 64, "bf16", "token"),
    ([500, 3, 77], 16, 1, 128, 1, "f16", "head"), ([500, 0, 300], 20, 1, 128, 3, "bf16", "token"), ([100] * 70, 4, 4, 64, 100, "f16", "head"),
    ([40, 2000, 1, 700], 64, 4, 128, 32, "bf16", "head"), ([300, 10], 40, 1, 64, 16, "f16", "token"), ([333, 21], 4, 2, 80, 16, "f16", "head"),
    ([333, 21], 6, 2, 96, 8, "bf16", "token"), ([333, 21], 4, 1, 256, 16, "f16", "head"), ([90, 200, 1], 5, 1, 8, 7, "f16", "head"),
    ([90, 200], 3, 3, 72, 16, "bf16", "head"), ([90, 200], 4, 2, 136, 16, "f16", "token"), ([6000, 10], 8, 1, 128, 256, "f16", "head"),
    ([5, 4000], 2, 2, 200, 64, "bf16", "head"), ([30] * 300, 2, 1, 64, 16, "bf16", "token"),
]


@pytest.mark.parametrize("case", DECODE, ids=lambda c: "x".join(map(str, (len(c[0]), max(c[0])) + c[1:])))
def test_decode_against_the_definition(hexmi, case):
    context, heads, kv, dim, page, dt, order = case
    c = Cache([1] * len(context), context, heads, kv, dim, page, DTYPES[dt], order, seed=dim + len(context))
    got = hexmi.paged_attention(c.q, *c.batch())
    c.check(got)
    out = torch.full_like(got, 7.0)
    assert hexmi.paged_attention(c.q, *c.batch(), sm_scale=1 / math.sqrt(dim), out=out) is out      # the route through ctypes
    assert torch.equal(out, got)


RAGGED = [
    # new tokens, contexts, heads, kv heads, dim, page, dtype, order, rows behind the last sequence
    ([1, 5, 0, 3], [0, 2, 9, 60], 4, 2, 64, 16, "f16", "head", 0), ([200], [0], 8, 2, 128, 16, "bf16", "token", 0),
    ([130, 1, 1, 64], [300, 777, 0, 5], 16, 4, 128, 64, "f16", "head", 9), ([63, 64, 65], [1, 0, 64], 3, 3, 128, 32, "bf16", "head", 1),
    ([31, 33], [500, 0], 5, 1, 80, 16, "f16", "token", 0), ([70], [70], 6, 2, 96, 7, "bf16", "head", 2), ([40, 2], [0, 100], 4, 1, 256, 16, "f16", "head", 0),
    ([129], [1000], 2, 1, 64, 1, "bf16", "head", 0), ([3] * 70, [10] * 70, 8, 8, 64, 16, "f16", "head", 5), ([0, 0], [5, 0], 2, 1, 64, 16, "f16", "head", 4),
    ([509, 1], [2046, 900], 8, 2, 128, 16, "f16", "head", 0), ([12], [7], 4, 2, 24, 16, "f16", "head", 0), ([300], [0], 4, 4, 160, 64, "bf16", "token", 0),
    ([17, 260], [3, 0], 40, 1, 64, 16, "bf16", "head", 0), ([1000, 900], [0, 0], 4, 1, 128, 64, "f16", "head", 0), ([2], [4090], 8, 1, 128, 64, "f16", "head", 0),
]


@pytest.mark.parametrize("case", RAGGED, ids=lambda c: "x".join(map(str, (len(c[0]), max(c[0]), max(c[1])) + c[2:])))
def test_ragged_against_the_definition(hexmi, case):
    new, context, heads, kv, dim, page, dt, order, padding = case
    c = Cache(new, context, heads, kv, dim, page, DTYPES[dt], order, seed=dim + len(new), padding=padding, ragged=True)
    got = hexmi.paged_attention(c.q, *c.batch())
    c.check(got)
    out = torch.full_like(got, 7.0)
    assert hexmi.paged_attention(c.q, *c.batch(), out=out) is out
    assert torch.equal(out, got)


SHARED = [
    # new tokens, contexts behind the prefix, shared tokens, heads, kv heads, dim, page, dtype
    ([1] * 5, [0, 3, 40, 200, 1], 64, 8, 2, 128, 16, "f16"), ([1] * 33, list(range(33)), 1024, 32, 8, 128, 64, "bf16"),
    ([1], [10], 2000, 4, 4, 64, 16, "f16"), ([30, 1, 0, 90], [1, 1, 1, 1], 400, 16, 4, 64, 16, "f16"), ([1] * 3, [5, 6, 7], 96, 40, 1, 128, 3, "bf16"),
    ([200, 7], [0, 300], 333, 6, 2, 80, 9, "bf16"), ([1] * 4, [0, 1, 2, 3], 128, 4, 2, 256, 16, "f16"), ([5, 260], [0, 3], 640, 4, 1, 256, 64, "bf16"),
    ([1] * 200, [2] * 200, 256, 4, 1, 64, 16, "f16"),
]


@pytest.mark.parametrize("case", SHARED, ids=lambda c: "x".join(map(str, (len(c[0]), max(c[0]), max(c[1])) + c[2:])))
def test_shared_prefix_against_the_definition(hexmi, case):
    new, context, shared, heads, kv, dim, page, dt = case
    c = Cache(new, [shared + x for x in context], heads, kv, dim, page, DTYPES[dt], seed=dim + len(new), shared=shared)
    c.check(hexmi.paged_attention(c.q, *c.batch()), what="each for itself")
    k_pages, v_pages, table, lengths, starts = c.batch()
    blind = table.clone()
    blind[:, :shared // page] = -7                           # not read
    c.check(hexmi.paged_attention(c.q, k_pages, v_pages, blind, lengths, starts, shared_pages=c.shared_pages), what="shared")


def test_shared_prefix_with_sequences_that_have_no_part_of_it(hexmi):
    # sequences shorter than the prefix see as much of it as they are long; an empty one is zeros
    c = Cache([1] * 6, [63, 0, 199, 127, 30, 64], 8, 2, 64, 16, torch.float16, seed=9, shared=128)
    c.lengths_d = torch.tensor([64, 0, 200, 128, 31, -5], dtype=torch.int32, device="cuda")
    c.lengths = [64, 0, 200, 128, 31, 0]
    c.k64, c.v64 = [[x[:n] for x, n in zip(t, c.lengths)] for t in (c.k64, c.v64)]
    c.check(hexmi.paged_attention(c.q, *c.batch(), shared_pages=c.shared_pages))


def test_pages_that_are_none_and_lengths_that_are_too_long(hexmi):
    c = Cache([1, 1, 2], [70, 40, 30], 4, 2, 64, 16, torch.float16, seed=5)
    # sequence 0 loses its second and last page, sequence 1 all of them; sequence 2 claims more than the table has columns for
    columns = c.table.shape[1]
    c.table[0, 1], c.table[0, 4] = -1, c.k_pages.shape[0]
    c.table[1] = 1 << 30
    c.page_table = c.table.cuda()
    c.lengths_d = torch.tensor([71, 41, 5 + columns * 16], dtype=torch.int32, device="cuda")
    got = hexmi.paged_attention(c.q, *c.batch()).cpu().double()
    kept = torch.cat((torch.arange(16), torch.arange(32, 64)))
    for h in range(4):
        w = torch.softmax(c.q[0, h].cpu().double() @ c.k64[0][kept, h // 2].T / 8, 0)
        want = w @ c.v64[0][kept, h // 2]
        assert (got[0, h] - want).abs().max() <= 4 * half_step(torch.float16) * c.v64[0].abs().max()
    assert (got[1] == 0).all()
    # sequence 2: its tokens stand at positions past the table, so they see all of it: two whole pages
    for i in (2, 3):
        for h in range(4):
            w = torch.softmax(c.q[i, h].cpu().double() @ c.k64[2][:, h // 2].T / 8, 0)
            assert (got[i, h] - w @ c.v64[2][:, h // 2]).abs().max() <= 4 * half_step(torch.float16) * c.v64[2].abs().max()


@pytest.mark.parametrize("ragged", [False, True])
def test_index_tensors_that_make_no_sense_touch_nothing_outside(hexmi, ragged):
    g = _gen(11)
    pages = [torch.randn(5, 2, 16, 64, generator=g).half().cuda() for _ in range(2)]
    q = torch.randn(6, 4, 64, generator=g).half().cuda()
    k = torch.randn(6, 2, 64, generator=g).half().cuda()
    B = 4 if ragged else 6
    lengths = torch.tensor([-(1 << 31), (1 << 31) - 1, 3, 0, 40, 41][:B], dtype=torch.int32, device="cuda")
    table = torch.tensor([[-(1 << 31), (1 << 31) - 1, 5]] * B, dtype=torch.int32, device="cuda")
    starts = torch.tensor([3, -9, 1 << 30, 2, 70], dtype=torch.int32, device="cuda") if ragged else None
    before = [p.clone() for p in pages]
    around = torch.full((18, 4, 64), 7.0, dtype=torch.float16, device="cuda")
    out = around[6:12]
    hexmi.paged_attention(q, *pages, table, lengths, starts, out=out)
    assert (around[:6] == 7).all() and (around[12:] == 7).all()
    # no page is one: zeros, but in rows that starts which fall give to nobody
    assert ((out == 0) | (out == 7 if ragged else False)).all()
    assert hexmi.paged_append(k, k, *pages, table, lengths, starts) is None
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(pages, before))
    shared = torch.tensor([-1, 99], dtype=torch.int32, device="cuda")
    hexmi.paged_attention(q, *pages, table, lengths, starts, shared_pages=shared, out=out)
    torch.cuda.synchronize()
    assert (around[:6] == 7).all() and (around[12:] == 7).all() and (ragged or (out == 0).all())


@pytest.mark.parametrize("dt", ["f16", "bf16"])
def test_large_scores_and_one_key_far_above_the_others(hexmi, dt):
    c = Cache([1, 20], [600, 500], 8, 2, 128, 16, DTYPES[dt], seed=21, scale=6.0)
    c.check(hexmi.paged_attention(c.q, *c.batch(), sm_scale=1.0), sm_scale=1.0)


def test_cache_past_32_bits(hexmi):
    # pages of 2^20 elements, the used ones beyond 2^31 elements of the pool
    page, kv, dim = 1024, 8, 128
    pool = 2060
    pages = [torch.empty(pool, kv, page, dim, dtype=torch.float16, device="cuda") for _ in range(2)]
    small = Cache([1, 1], [1500, 20], 16, kv, dim, page, torch.float16, seed=2)
    big = small.page_table.clone()
    for i, p in enumerate(small.page_table.flatten().tolist()):
        if p >= 0:
            at = pool - 1 - p
            pages[0][at], pages[1][at] = small.k_pages[p], small.v_pages[p]
            big.view(-1)[i] = at
    small.check(hexmi.paged_attention(small.q, *pages, big, small.lengths_d))
    k = torch.randn(2, kv, dim, device="cuda").half()
    hexmi.paged_append(k, k, *pages, big, small.lengths_d)
    torch.cuda.synchronize()
    assert torch.equal(pages[0][big[0, 1].item(), :, 1500 % page], k[0]) and torch.equal(pages[1][big[1, 0].item(), :, 20], k[1])


APPEND = [
    # new tokens, contexts, heads (0: no q), kv heads, dim, page, dtype, order, rotated columns, pairs, norm, rows behind the last sequence
    ([1], [0], 4, 1, 64, 16, "f16", "head", 64, "adjacent", False, 0), ([1] * 9, [0, 15, 16, 17, 5, 100, 31, 32, 33], 8, 2, 128, 16, "bf16", "token", 128, "halves", True, 0),
    ([3, 0, 70, 1], [0, 4, 10, 63], 4, 4, 80, 7, "f16", "head", 40, "halves", True, 3), ([5, 6], [1000, 0], 0, 2, 128, 64, "f16", "token", 0, "adjacent", False, 0),
    ([2] * 80, [3] * 80, 6, 3, 64, 1, "bf16", "head", 32, "adjacent", True, 7), ([1] * 3, [8, 9, 10], 0, 1, 256, 16, "bf16", "head", 256, "halves", True, 0),
    ([33], [5], 5, 1, 12, 16, "f16", "head", 12, "halves", True, 0), ([400, 3], [0, 50], 32, 8, 128, 64, "bf16", "token", 128, "halves", True, 0),
]


@pytest.mark.parametrize("case", APPEND, ids=lambda c: "x".join(map(str, (len(c[0]), max(c[0]), max(c[1])) + c[2:])))
@pytest.mark.parametrize("in_place", [False, True])
def test_append_against_the_definition(hexmi, case, in_place):
    new, context, heads, kv, dim, page, dt, order, R, pairs, norm, padding = case
    dtype, g = DTYPES[dt], _gen(dim + len(new))
    c = Cache(new, context, max(heads, kv), kv, dim, page, dtype, order, seed=dim, padding=padding)
    T = sum(new) + padding
    wide = torch.randn(T, (heads + 2 * kv) * dim, generator=g).to(dtype).cuda()
    q, k, v = (t.unflatten(1, (-1, dim)) if t.shape[1] else None for t in wide.split((heads * dim, kv * dim, kv * dim), 1))
    qw, kw = ((1 + 0.2 * torch.randn(dim, generator=g)).to(dtype).cuda() for _ in range(2)) if norm else (None, None)
    freq = hexmi.rope_frequencies(R) if R else None
    position = torch.cat([torch.arange(L - n, L) for n, L in zip(new, c.lengths)] + [torch.zeros(padding, dtype=torch.long)])
    want_k, want_q = rows64(k, kw, freq, position, 1e-5, pairs), rows64(q, qw, freq, position, 1e-5, pairs) if heads else None
    k_before, v_before = c.k_pages.clone(), c.v_pages.clone()
    got = hexmi.paged_append(k, v, *c.batch(), kw, freq, 1e-5, pairs, q, qw if heads else None, q_out=q if in_place and heads else None)
    rows = sum(new)
    if heads:
        check_rows(got[:rows], tuple(t[:rows] for t in want_q), "q")
        assert (got[rows:] == 0).all() and (got.data_ptr() == q.data_ptr()) == in_place
    else:
        assert got is None
    t, k_want, v_want = 0, k_before, v_before
    for b, (n, L) in enumerate(zip(new, c.lengths)):
        at = torch.arange(L - n, L)
        where = c.table[b][at // page].long().cuda(), slice(None), (at % page).cuda()
        check_rows(c.k_pages[where], tuple(x[t:t + n] for x in want_k), "k")
        k_want[where], v_want[where] = c.k_pages[where], v[t:t + n]
        t += n
    same = torch.int16
    assert torch.equal(c.k_pages.contiguous().view(same), k_want.contiguous().view(same))            # nothing else has changed
    assert torch.equal(c.v_pages.contiguous().view(same), v_want.contiguous().view(same))


def test_append_leaves_out_tokens_without_a_place(hexmi):
    pages = [torch.zeros(4, 1, 16, 64, dtype=torch.float16, device="cuda") for _ in range(2)]
    k = torch.ones(4, 1, 64, dtype=torch.float16, device="cuda")
    table = torch.tensor([[0, -1], [1, 9], [2, 3], [3, 2]], dtype=torch.int32, device="cuda")
    hexmi.paged_append(k, k, *pages, table, torch.tensor([17, 32, 33, 0], dtype=torch.int32, device="cuda"))
    assert all((p == 0).all() for p in pages)
    hexmi.paged_append(k, k, *pages, table, torch.tensor([16, 16, 17, 32], dtype=torch.int32, device="cuda"))
    assert all(p.sum().item() == 4 * 64 for p in pages) and pages[0][3, 0, 0, 0] == 1 and pages[1][2, 0, 15, 0] == 1


def test_results_do_not_change_from_call_to_call(hexmi):
    c = Cache([1] * 24, [37 * i % 3000 for i in range(24)], 16, 2, 128, 16, torch.bfloat16, seed=8)
    first = hexmi.paged_attention(c.q, *c.batch())
    junk = torch.full((64 << 20,), math.nan, device="cuda")              # what a freed workspace holds next
    del junk
    for _ in range(3):
        assert torch.equal(hexmi.paged_attention(c.q, *c.batch()), first)
    assert not torch.isnan(first).any()


@pytest.mark.parametrize("shared", [False, True])
@pytest.mark.parametrize("ragged", [False, True])
def test_two_graphs_replayed_as_their_batches_change(hexmi, ragged, shared):
    """Append and attention captured twice, replayed in turn with other lengths and pages and eager work between."""
    prefix = 64 if shared else 0
    states, graphs = [], []
    for i in range(2):
        new = [1, 20, 3, 1] if ragged else [1] * 6
        c = Cache(new, [prefix + 400 + 10 * i] * len(new), 8, 2, 64, 16, torch.float16, seed=30 + i, shared=prefix, ragged=ragged)
        T = sum(new)
        k, v = (torch.randn(T, 2, 64, device="cuda").half() for _ in range(2))
        freq = hexmi.rope_frequencies(64)

        def step(c=c, k=k, v=v, freq=freq):
            q = hexmi.paged_append(k, v, *c.batch(), inv_freq=freq, q=c.q)
            return hexmi.paged_attention(q, *c.batch(), shared_pages=c.shared_pages)
        step()
        torch.cuda.synchronize()
        graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        with torch.cuda.stream(stream):
            with torch.cuda.graph(graph, stream=stream):
                out = step()
        states.append((c, k, v, step, out))
        graphs.append(graph)
    full = [c.lengths_d.clone() for c, *_ in states]
    for replay in range(4):
        for (c, k, v, step, out), graph, lengths in zip(states, graphs, full):
            k.normal_()
            v.normal_()
            c.lengths_d.copy_((lengths - 23 * replay).clamp_(min=prefix + 21))
            c.page_table[0, prefix // 16 + 1:prefix // 16 + 3] = c.page_table[0, prefix // 16 + 1:prefix // 16 + 3].flip(0).clone()
            want = step()
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want), replay


def test_other_stream_and_two_calls_at_once(hexmi):
    caches = [Cache([1] * 8, [300 * (i + 1)] * 8, 8, 2, 128, 16, torch.float16, seed=40 + i) for i in range(2)]
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in caches], []
    for _ in range(4):
        for s, c in zip(streams, caches):
            with torch.cuda.stream(s):
                outs.append(hexmi.paged_attention(c.q, *c.batch()))
    torch.cuda.synchronize()
    for i, o in enumerate(outs):
        caches[i % 2].check(o, what=i)


def test_out_over_the_queries(hexmi):
    c = Cache([1] * 5, [100, 2000, 3, 50, 700], 8, 2, 64, 16, torch.float16, seed=50)
    want = hexmi.paged_attention(c.q, *c.batch())
    q = c.q.clone()
    assert torch.equal(hexmi.paged_attention(q, *c.batch(), out=q), want) and torch.equal(q, want)
    wide = torch.zeros(5, 2, 8, 64, dtype=torch.float16, device="cuda")
    out = hexmi.paged_attention(c.q, *c.batch(), out=wide[:, 1])
    assert torch.equal(wide[:, 1], want) and (wide[:, 0] == 0).all() and out.data_ptr() == wide[:, 1].data_ptr()
    odd = torch.zeros(1 + c.q.numel(), dtype=torch.float16, device="cuda")[1:].view_as(c.q).copy_(c.q)      # off the boundaries
    assert torch.equal(hexmi.paged_attention(odd, *c.batch()), want)


def test_through_the_dispatcher(hexmi):
    c = Cache([2, 5], [40, 0], 4, 2, 64, 16, torch.float16, seed=60)
    freq, k = hexmi.rope_frequencies(64), torch.randn(7, 2, 64, device="cuda").half()
    results = []
    for on in (False, True):
        pages = c.k_pages.clone(), c.v_pages.clone()
        previous = hexmi.through_dispatcher(on)
        try:
            q = hexmi.paged_append(k, k, *pages, *c.batch()[2:], inv_freq=freq, q=c.q)
            a, b = hexmi.qk_norm_rope(c.q, k, None, None, freq, torch.arange(7, device="cuda"))
            o = hexmi.paged_attention(q, *pages, *c.batch()[2:])
        finally:
            hexmi.through_dispatcher(previous)
        results.append((q, a, b, o) + tuple(p.view(torch.int16) for p in pages))
    assert all(torch.equal(x, y) for x, y in zip(*results))


def test_a_layer_over_the_cache(hexmi):
    """A layer with shared key heads and norms of its heads: two prompts in pieces, then tokens one at a time, against the same layer in
    64 bits over the whole sequences at once. Every operator rounds its result, so the bound is not of one rounding: six results one
    behind the other (norm, projection, rows, attention, product, sum), each u of its size, doubled by the sums they go into."""
    E_, H, KV, D, page, dtype = 512, 8, 2, 64, 16, torch.float16
    g = _gen(70)

    def made(*shape, std):
        return (torch.randn(*shape, generator=g) * std).to(dtype).cuda()
    norm, qw, kw = (1 + made(E_, std=0.1)), 1 + made(D, std=0.1), 1 + made(D, std=0.1)
    wqkv, wo = made(E_, (H + 2 * KV) * D, std=E_ ** -0.5), made(H * D, E_, std=(H * D) ** -0.5)
    freq = hexmi.rope_frequencies(D)
    lengths = [45, 90]
    xs = [made(n, E_, std=1.0) for n in lengths]
    pages = [torch.full((12, page, KV, D), math.nan, dtype=dtype, device="cuda").transpose(1, 2) for _ in range(2)]
    table = torch.full((2, 7), -1, dtype=torch.int32)
    order = torch.randperm(12, generator=g, dtype=torch.int32)
    table[0, :3], table[1, :6] = order[:3], order[3:9]
    table = table.cuda()

    def layer(x, lengths, starts):
        h = hexmi.rms_norm(x, norm, 1e-5)
        q, k, v = (t.unflatten(1, (-1, D)) for t in hexmi.matmul(h, wqkv).split((H * D, KV * D, KV * D), 1))
        q = hexmi.paged_append(k, v, *pages, table, lengths, starts, kw, freq, 1e-5, "halves", q, qw)
        return hexmi.matmul(hexmi.paged_attention(q, *pages, table, lengths, starts).flatten(1), wo, residual=x)

    done, results = [0, 0], [[], []]
    for piece in ([32, 70], [5, 0], [0, 12], [1, 1], [1, 1], [1, 1], [1, 1], [1, 1], [1, 1], [1, 1], [1, 1]):
        piece = [min(p, n - d) for p, n, d in zip(piece, lengths, done)]
        x = torch.cat([t[d:d + p] for t, d, p in zip(xs, done, piece)])
        done = [d + p for d, p in zip(done, piece)]
        starts = None if piece == [1, 1] else torch.tensor([0, piece[0], sum(piece)], dtype=torch.int32, device="cuda")
        y = layer(x, torch.tensor(done, dtype=torch.int32, device="cuda"), starts)
        for r, t in zip(results, y.split(piece)):
            r.append(t)
    for x, n, d, r in zip(xs, lengths, done, results):
        x64 = x.cpu().double()[:d]
        h = x64 / (x64.square().mean(-1, keepdim=True) + 1e-5).sqrt() * norm.cpu().double()
        q, k, v = (t.unflatten(1, (-1, D)) for t in (h @ wqkv.cpu().double()).split((H * D, KV * D, KV * D), 1))
        at = torch.arange(d)
        q, k = rows64(q, qw, freq, at, 1e-5, "halves")[0], rows64(k, kw, freq, at, 1e-5, "halves")[0]
        s = torch.einsum("thd,shd->hts", q, k.repeat_interleave(H // KV, 1)) / math.sqrt(D)
        w = torch.softmax(s.masked_fill(at[None] > at[:, None], -math.inf), -1)
        want = x64 + torch.einsum("hts,shd->thd", w, v.repeat_interleave(H // KV, 1)).flatten(1) @ wo.cpu().double()
        got = torch.cat(r).cpu().double()
        assert got.shape == want.shape and d == n
        rel = (got - want).norm() / want.norm()
        assert rel <= 12 * half_step(dtype), rel


@pytest.mark.parametrize("dim", [8, 24])
def test_joins_read_no_sums_that_nobody_left(hexmi, dim):
    """More parts than a narrow head has columns, in a workspace full of large numbers: sequences of one token, whose keys several workers
    share, leave word that the parts of longer runs are empty."""
    c = Cache([3, 1, 1, 2], [6000, 5000, 4001, 9000], 2, 1, dim, 16, torch.float16, seed=71, shared=4000)
    ops, lib = sys.modules["hexmi.ops"], sys.modules["hexmi._lib"].lib()
    batch = ops._paged_batch(c.q.shape[0], c.k_pages, c.v_pages, c.page_table, c.lengths_d, c.starts)
    need, out = lib.hexmi_paged_attention_workspace(batch, 2, c.shared_pages.numel()), torch.empty_like(c.q)
    junk = torch.full((need // 4 + 4,), 1e30, device="cuda")
    assert need > 0
    assert lib.hexmi_paged_attention(ops._head_rows(c.q, out), batch, c.shared_pages.data_ptr(), c.shared_pages.numel(), 1 / math.sqrt(dim),
                                     sys.modules["hexmi._lib"].F16, junk.data_ptr(), need, None) == 0
    torch.cuda.synchronize()
    c.check(out)


@pytest.mark.parametrize("new, context, heads, kv, dim, shared", [
    ([1], [9000], 8, 2, 128, 0), ([1] * 3, [200, 40, 700], 8, 2, 64, 0), ([1, 1], [5000, 4300], 8, 2, 128, 4096), ([1, 1], [100, 20], 4, 4, 256, 0),
    ([6, 1, 1], [3000, 5000, 80], 8, 2, 128, 0), ([6, 1, 1], [7000, 5000, 4100], 8, 2, 64, 4096), ([300, 40], [0, 700], 16, 2, 128, 0),
    ([700, 900], [0, 700], 32, 32, 64, 0), ([70, 200], [500, 0], 4, 1, 256, 0),
])
def test_nan_among_a_sequence_s_keys_shows(hexmi, new, context, heads, kv, dim, shared):
    """A NaN in a key of the first sequence makes NaN of its rows, however its keys are cut up, and of no other sequence's; in a value, of
    that column."""
    for where in ("k", "v"):
        c = Cache(new, context, heads, kv, dim, 16, torch.float16, seed=72, shared=shared)
        at = c.lengths[0] - new[0] if shared else (c.lengths[0] - new[0]) // 2     # seen by all its new tokens, behind the prefix
        pages = c.k_pages if where == "k" else c.v_pages
        pages[c.table[0][at // 16].item(), kv - 1, at % 16, 3] = math.nan
        got = hexmi.paged_attention(c.q, *c.batch(), shared_pages=c.shared_pages)
        mine = got[:new[0], heads - heads // kv:]                                 # the heads of the last key head
        assert torch.isnan(mine if where == "k" else mine[..., 3]).all(), where
        got[:new[0], heads - heads // kv:] = 0
        out, bound = c.attention64()
        out[:new[0], heads - heads // kv:] = 0
        assert ((got.cpu().double() - out).abs() <= bound).all(), where


@pytest.mark.parametrize("dim, offset", [(64, 0), (128, 0), (64, 1)])
def test_rows_whose_squares_are_subnormal(hexmi, dim, offset):
    """eps 0 and squares of 1e-40: a square is off by 2^-150 at most, the mean's product by as much, and the root halves that."""
    g = _gen(73)
    x = ((1 + torch.rand(1 + 9 * 3 * dim, generator=g)) * 1e-20)[offset:][:9 * 3 * dim].view(9, 3, dim).cuda()
    w = torch.ones(dim, device="cuda")
    want, size = rows64(x, w, None, None, 0.0, "adjacent")
    got = hexmi.qk_norm_rope(x, None, w, eps=0.0).cpu().double()
    least = x.cpu().double().square().mean(-1).min().item()
    assert ((got - want).abs() <= (24 * E + 2.0 ** -150 / least) * size).all()


def test_append_of_rows_that_stand_in_the_pages(hexmi):
    """One sequence's keys and values go to another's pages, in the same call as others to theirs; queries land outside the pages."""
    g = _gen(74)
    pages = [torch.randn(6, 16, 2, 64, generator=g).half().cuda().transpose(1, 2) for _ in range(2)]
    before = [p.clone() for p in pages]
    table = torch.tensor([[1], [2], [3]], dtype=torch.int32, device="cuda")
    lengths, starts = (torch.tensor(t, dtype=torch.int32, device="cuda") for t in ([16, 16, 16], [0, 16, 32, 48]))
    rows = [p.transpose(1, 2).flatten(0, 1)[:48] for p in pages]                  # pages 0, 1, 2: every one but the first read and written
    assert rows[0].data_ptr() == pages[0].data_ptr()
    hexmi.paged_append(*rows, *pages, table, lengths, starts)
    for p, b in zip(pages, before):
        assert torch.equal(p[1:4], b[:3]) and torch.equal(p[0], b[0]) and torch.equal(p[4:], b[4:])
    q_out = pages[0].transpose(1, 2).flatten(0, 1)[80:]                           # the last page: kept until the keys are in
    q = torch.randn(16, 2, 64, generator=g).half().cuda()
    got = hexmi.paged_append(q, q, *pages, torch.tensor([[4]], dtype=torch.int32, device="cuda"), lengths[:1], starts[:2], q=q, q_out=q_out)
    assert torch.equal(got, q) and torch.equal(pages[0][4].transpose(0, 1), q) and torch.equal(q_out, q)
    with pytest.raises(ValueError, match="pages of their own"):
        hexmi.paged_append(q, q, pages[0], pages[0], table[:1], lengths[:1], starts[:2])


@pytest.mark.parametrize("seed", range(40))
def test_batches_of_any_kind(hexmi, seed):
    """Sizes, orders and kinds of batch drawn together."""
    r = random.Random(seed)
    kind = ("decode", "mixed", "mixed", "prompts", "singles")[seed % 5]
    dim, kv, group = r.choice([8, 24, 64, 64, 80, 96, 128, 128, 136, 200, 256]), r.choice([1, 2, 3, 8]), r.choice([1, 2, 4, 5, 7, 16, 17, 33])
    page, B = r.choice([1, 3, 8, 16, 16, 24, 64, 100, 256]), r.choice([1, 2, 3, 9, 20, 70])
    shared = r.choice([0, page * r.randint(1, 1 + 600 // page), page * r.randint(1, 1 + 4000 // page)])
    new = [1 if kind in ("decode", "singles") else r.choice([0, 1, 1, r.randint(1, 90)]) for _ in range(B)] if kind != "prompts" else [
        r.randint(1, 600 // B + 2) for _ in range(B)]
    context = [shared] + [shared + r.randint(0, 300) if r.random() < 0.9 else r.randint(0, shared) for _ in range(B - 1)]
    c = Cache(new, context, kv * group, kv, dim, page, r.choice([torch.float16, torch.bfloat16]), r.choice(["head", "token"]), seed=seed,
              padding=0 if kind == "decode" else r.choice([0, 3]), ragged=kind != "decode", shared=shared)
    c.check(hexmi.paged_attention(c.q, *c.batch(), shared_pages=c.shared_pages), what=(kind, new, context, shared, page, c.heads, kv, dim))


@pytest.mark.parametrize("seed", range(40))
def test_rows_of_any_kind(hexmi, seed):
    r, g = random.Random(seed), _gen(seed)
    D, H, K, T = r.choice([1, 2, 8, 30, 64, 72, 128, 130, 256, 320, 512]), r.randint(1, 40), r.randint(1, 9), r.choice([1, 2, 17, 300])
    dtype, pairs, R = r.choice(list(DTYPES.values())), r.choice(["adjacent", "halves"]), 2 * r.randint(0, D // 2)
    wide = torch.randn(T, (H + K) * D + r.choice([0, 1, 8]), generator=g).to(dtype).cuda()[:, :(H + K) * D].unflatten(1, (H + K, D))
    q, k = wide[:, :H], wide[:, H:]
    qw, kw = (torch.randn(D, generator=g).to(dtype).cuda() if r.random() < 0.7 else None for _ in range(2))
    freq = hexmi.rope_frequencies(R, r.choice([1e4, 5e5])) if R else None
    pos = torch.randint(0, 1 << 17, (T,), generator=g).cuda()
    got = hexmi.qk_norm_rope(q, k, qw, kw, freq, pos, 1e-6, pairs)
    for x, w, y in ((q, qw, got[0]), (k, kw, got[1])):
        check_rows(y, rows64(x, w, freq, pos, 1e-6, pairs), (D, H, K, T, R, pairs))


def test_a_step_without_new_tokens(hexmi):
    """Sequences, and no new token of any: nothing is computed, through the operator and through the registered one."""
    c = Cache([0, 0, 0], [70, 0, 5], 4, 2, 64, 16, torch.float16, seed=75, ragged=True, shared=0)
    before, k = c.k_pages.clone(), torch.empty(0, 2, 64, dtype=torch.float16, device="cuda")
    out = torch.empty_like(c.q)
    assert c.q.shape[0] == 0 and hexmi.paged_attention(c.q, *c.batch()).shape == c.q.shape
    torch.ops.hexmi.paged_attention(c.q, *c.batch(), 0.125, None, out)
    hexmi.paged_append(k, k, *c.batch())
    torch.cuda.synchronize()
    assert torch.equal(c.k_pages.view(torch.int16), before.view(torch.int16))


@pytest.mark.parametrize("new", [[3, 9], [3, 8, 1], [2] * 70])
def test_starts_past_the_rows_there_are(hexmi, new):
    """starts that begin below the first row and end behind the last: a sequence's new tokens are those of its rows that there are, at
    its last positions, for what is appended, behind a prefix and without one alike."""
    prefix, T = 64, sum(new)
    c = Cache(new, [prefix + 1] * len(new), 4, 2, 64, 16, torch.float16, seed=76, ragged=True, shared=prefix)
    whole = c.starts
    beyond = whole.clone()
    beyond[0], beyond[-1] = -4, T + 30
    k, freq = torch.randn(T, 2, 64, generator=_gen(77)).half().cuda(), hexmi.rope_frequencies(64)
    results = []
    for starts in (whole, beyond):
        pages = c.k_pages.clone(), c.v_pages.clone()
        q = hexmi.paged_append(k, k, *pages, c.page_table, c.lengths_d, starts, inv_freq=freq, q=c.q)
        results.append([q] + [p.view(torch.int16) for p in pages])
    assert all(torch.equal(a, b) for a, b in zip(*results))
    c.starts = beyond
    c.check(hexmi.paged_attention(c.q, *c.batch()), what="each for itself")
    c.check(hexmi.paged_attention(c.q, *c.batch(), shared_pages=c.shared_pages), what="shared")


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("new, shared", [(2048, 0), (1, 0), (20, 1 << 16)])
def test_many_keys_far_below_one(hexmi, dt, new, shared):
    """A key that all rows see first and 2^17 others of 2^-26 of its weight each: together they have 2^-9 of it. Column 0 is what comes of them
    alone (their values are 1 there, the first's is 0), column 1 the first key's.
    fp16 weights have steps of 2^-24 where the largest is 2^7 and more, so each is off by at most 2^-32 of it, and all by 2^17 times that. The
    weights are powers of two, and sums of 8 and more of them whole steps of the sum that they are added to; beyond that the result's
    rounding, and for the quotient and the order of sums in parts (2 u + 2^17 E) of what the others come to, 2^-9."""
    dtype, L, dim, page, heads = DTYPES[dt], 1 << 17, 64, 256, 64
    k, v = (torch.zeros(L // page, 1, page, dim, dtype=dtype, device="cuda") for _ in range(2))
    q = torch.zeros(new, heads, dim, dtype=dtype, device="cuda")
    q[..., 0], k[0, 0, 0, 0] = 2.0, 13.0                             # 26 in log2 with this scale; the others' scores are 0
    v[..., 0], v[0, 0, 0, 0], v[0, 0, 0, 1] = 1.0, 0.0, 1.0
    table = torch.arange(L // page, dtype=torch.int32, device="cuda")[None]
    starts = None if new == 1 else torch.tensor([0, new], dtype=torch.int32, device="cuda")
    got = hexmi.paged_attention(q, k, v, table, torch.tensor([L], dtype=torch.int32, device="cuda"), starts, sm_scale=math.log(2.0),
                                shared_pages=table[0, :shared // page] if shared else None).cpu().double()
    others = torch.arange(L - new, L, dtype=torch.float64)[:, None] * 2.0 ** -26
    u = half_step(dtype)
    bound = L * 2.0 ** -32 + (2 * u + L * E) * 2.0 ** -9
    assert (got[..., 0] - others / (1 + others)).abs().max() <= bound
    assert (got[..., 1] - 1 / (1 + others)).abs().max() <= bound + u and (got[..., 2:] == 0).all()


@pytest.mark.parametrize("new, shared", [([1, 1], 0), ([5, 30], 0), ([1, 1], 64), ([5, 1], 64)])
def test_pages_that_are_only_read_stay_shared(hexmi, new, shared):
    """Copy-on-write pages are not copied for attention over them; an append makes them the caller's own."""
    c = Cache(new, [70 + shared, 90 + shared], 4, 2, 64, 16, torch.float16, seed=78, shared=shared)
    want = hexmi.paged_attention(c.q, *c.batch(), shared_pages=c.shared_pages)
    plain = c.k_pages, c.v_pages
    c.k_pages, c.v_pages = (torch._lazy_clone(p) for p in plain)
    assert torch.equal(hexmi.paged_attention(c.q, *c.batch(), shared_pages=c.shared_pages), want)
    assert all(torch._C._is_cow_tensor(p) for p in (c.k_pages, c.v_pages))
    before = [p.clone().view(torch.int16) for p in plain]
    k = torch.zeros(sum(new), 2, 64, dtype=torch.float16, device="cuda")
    hexmi.paged_append(k, k, *c.batch())
    assert not any(torch._C._is_cow_tensor(p) for p in (c.k_pages, c.v_pages))
    assert all(torch.equal(p.view(torch.int16), b) for p, b in zip(plain, before))
    assert not any(torch.equal(p.view(torch.int16), b) for p, b in zip((c.k_pages, c.v_pages), before))


@pytest.mark.parametrize("name, shared", [("page_table", 0), ("lengths_d", 0), ("starts", 0), ("page_table", 64), ("lengths_d", 64), ("starts", 64),
                                          ("shared_pages", 64)])
def test_out_over_an_index_tensor(hexmi, name, shared):
    """A result that lands where an index tensor stood is complete before it is written there. Tiles of the last rows, where it stands, are
    done before those of the first are begun."""
    c = Cache([2100, 1, 1900, 700], [shared] * 4, 32, 8, 128, 16, torch.float16, seed=79, shared=shared)
    want = hexmi.paged_attention(c.q, *c.batch(), shared_pages=c.shared_pages)
    out = torch.empty_like(c.q)
    index = getattr(c, name)
    setattr(c, name, out.view(torch.int32).flatten()[-index.numel():].view(index.shape).copy_(index))
    assert hexmi.paged_attention(c.q, *c.batch(), shared_pages=c.shared_pages, out=out) is out
    assert torch.equal(out, want)

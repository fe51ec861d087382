"""A paged cache in 8 bits, attention within a window, forks and compaction of pages, against their definitions in 64 bits.

Tolerances, derived: u = eps / 2 is a rounding to the type, e = 2^-24 one to fp32.
  append     a row is off by 24 e of |a| + |b| before it is rounded (test_paged_gpu.py), to e4m3 by half a step: 2^-4 of the value, half of
             2^-9 times the scale below the normal numbers. A block's exponent is exact but where the largest value is within 24 e of it of a border;
             what may come out of either is taken. Older numbers, of four significant bits, are rounded to half a step again. At the type's
             largest scale numbers end at 240: what is above is off by at most (65504 - 61440) / 65504 < 2^-4 in fp16.
  attention  numbers times their scales are the type's, so the bound is that of a cache in 16 bits: u (sum w |v| + |o|) for the
             probabilities' rounding, (dim + 8) e scale sum |q| |k| twice for the scores, 16 e, 2^-25 of a row's largest a key in fp16, u |o|.
  fork, compact  copies: equal.
"""
import math
import random

import pytest
import torch

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
E4M3 = torch.float8_e4m3fn
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
RANGE = {torch.float16: (-15, 8), torch.bfloat16: (-117, 120)}


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def values(codes, scales):
    """Numbers of e4m3 [pages, heads, slots, dim] times their scales, in 64 bits on the CPU."""
    e = scales.cpu().double() - 127
    return codes.cpu().double() * torch.exp2(e).repeat_interleave(codes.shape[2] // scales.shape[2], 2)[..., None]


def in_order(t, order):
    """The same tensor with the heads of a token side by side in memory."""
    return t if order == "head" else t.transpose(1, 2).contiguous().transpose(1, 2)


class Long:
    """A cache and a batch: pages in random order; whatever no new token sees is NaN or has no page, now the one, now the other."""

    def __init__(self, new, context, heads, kv_heads, dim, page, block, dtype, order="head", window=None, sinks=0, seed=0, padding=0, ragged=None,
                 shared=0):
        g = _gen(seed)
        self.new, self.lengths = list(new), [c + n for c, n in zip(context, new)]
        self.heads, self.kv_heads, self.dim, self.page, self.block, self.dtype = heads, kv_heads, dim, page, block, dtype
        self.window, self.sinks = window, sinks
        self.ragged = any(n != 1 for n in new) or padding > 0 if ragged is None else ragged
        B, T = len(new), sum(new) + padding
        columns = [-(-n // page) for n in self.lengths]
        first = shared // page
        pool = first + sum(max(0, c - first) for c in columns) + 3
        names = torch.randperm(pool, generator=g)
        junk = names[-1].item()                                       # a page that is all NaN
        table = torch.full((B, max(columns + [1]) + 1), -1)
        self.shared_pages = names[:first].int().cuda() if first else None
        x = [torch.randn(pool, kv_heads, page, dim, generator=g) for _ in range(2)]
        if block:
            blocks = page // block
            self.scales = [torch.randint(118, 122, (pool, kv_heads, blocks), generator=g, dtype=torch.uint8) for _ in range(2)]
            x = [(t * 100).clamp(-448, 448).to(E4M3) for t in x]
            held = [values(t.double(), s) for t, s in zip(x, self.scales)]
            for t, s in zip(held, self.scales):
                assert torch.equal(t, t.to(dtype).double())
        else:
            self.scales = [None, None]
            x = [t.to(dtype) for t in x]
            held = [t.double() for t in x]
        seen = torch.zeros(pool, page, dtype=torch.bool)
        used = first
        self.k64, self.v64 = [], []
        for b, (n, L) in enumerate(zip(self.new, self.lengths)):
            table[b, :min(first, columns[b])] = names[:min(first, columns[b])]
            if columns[b] > first:
                table[b, first:columns[b]] = names[used:used + columns[b] - first]
                used += columns[b] - first
            at = torch.arange(L)
            mine = (at < sinks) | (at > L - max(n, 1) - window) if window else at >= 0
            pages = table[b, at // page]
            seen[pages[mine], at[mine] % page] = True
            self.k64.append(held[0][pages, :, at % page])
            self.v64.append(held[1][pages, :, at % page])
            for c in range(columns[b]):                               # pages that nobody sees
                if window and not mine[c * page:(c + 1) * page].any():
                    table[b, c] = (-1, junk, pool, 1 << 30)[(b + c) % 4]
        if first:
            seen[names[:first]] = True
        for t, s in zip(x, self.scales):
            unseen = ~seen[:, None, :, None].expand(t.shape)
            if block:
                t.view(torch.uint8)[unseen] = 0x7f
            else:
                t[unseen] = math.nan
        self.k_pages, self.v_pages = (in_order(t.cuda(), order) for t in x)
        self.k_scales, self.v_scales = (None if s is None else in_order(s.cuda(), order) for s in self.scales)
        self.table, self.page_table = table, table.int().cuda()
        self.lengths_d = torch.tensor(self.lengths, dtype=torch.int32, device="cuda")
        self.starts = torch.tensor([sum(self.new[:i]) for i in range(B + 1)], dtype=torch.int32, device="cuda") if self.ragged else None
        self.q = torch.randn(T, heads, dim, generator=g).to(dtype).cuda()

    def kw(self):
        kw = {"k_scales": self.k_scales, "v_scales": self.v_scales} if self.block else {}
        return {**kw, "window": self.window, "sinks": self.sinks} if self.window else kw

    def run(self, hexmi, **kw):
        return hexmi.paged_attention(self.q, self.k_pages, self.v_pages, self.page_table, self.lengths_d, self.starts, **{**self.kw(), **kw})

    def check(self, got, what=""):
        scale, G, u = 1.0 / math.sqrt(self.dim), self.heads // self.kv_heads, half_step(self.dtype)
        q = self.q.cpu().double()
        out, bound = torch.zeros_like(q), torch.zeros_like(q)
        t = 0
        for n, L, k, v in zip(self.new, self.lengths, self.k64, self.v64):
            at, p = torch.arange(L)[None], torch.arange(L - n, L)[:, None]
            hidden = at > p
            if self.window:
                hidden = hidden | (at <= p - self.window) & (at >= self.sinks)
            for h in range(self.heads if n and L else 0):
                kh, vh, qh = k[:, h // G], v[:, h // G], q[t:t + n, h]
                w = torch.softmax((qh @ kh.T * scale).masked_fill(hidden, -math.inf), 1)
                size = (qh.abs() @ kh.abs().T * scale).masked_fill(hidden, 0).amax(1, keepdim=True)
                o, a = w @ vh, w @ vh.abs()
                out[t:t + n, h] = o
                b = u * (a + o.abs()) + (2 * (self.dim + 8) * E * size + 16 * E) * (a + o.abs()) + u * o.abs()
                if self.dtype == torch.float16:
                    b = b + L * 2.0 ** -25 * vh.abs().amax(0) + 2.0 ** -25
                bound[t:t + n, h] = b
            t += n
        assert got.shape == out.shape and got.dtype == self.dtype
        off = (got.cpu().double() - out).abs()
        bad = ~(off <= bound)
        assert not bad.any(), (what, bad.sum().item(), (off / bound.clamp_min(1e-30))[bad].max().item(), bad.nonzero()[:3].tolist())


ATTEND = [
    # new tokens, contexts, heads, kv heads, dim, page, slots a block (0: 16 bits), dtype, order, window, sinks, rows behind the last sequence
    ([1], [0], 1, 1, 64, 16, 16, "f16", "head", None, 0, 0), ([1, 1, 1], [0, 15, 16], 4, 2, 128, 16, 1, "bf16", "token", None, 0, 0),
    ([1], [999], 32, 8, 128, 16, 16, "f16", "head", None, 0, 0), ([1] * 10, [15, 16, 17, 31, 32, 33, 62, 63, 64, 65], 8, 2, 128, 32, 8, "bf16", "head", None, 0, 0),
    ([1] * 5, [127, 128, 255, 256, 257], 12, 12, 64, 64, 64, "bf16", "token", None, 0, 0), ([1] * 3, [500, 3, 77], 20, 1, 128, 3, 3, "f16", "head", None, 0, 0),
    ([1] * 70, [100] * 70, 4, 4, 64, 100, 50, "f16", "head", None, 0, 0), ([1, 1], [333, 21], 4, 2, 80, 16, 4, "f16", "head", None, 0, 0),
    ([1, 1], [333, 21], 6, 2, 96, 8, 8, "bf16", "token", None, 0, 0), ([1, 1], [333, 4021], 4, 1, 256, 16, 2, "f16", "head", None, 0, 0),
    ([1, 1], [90, 200], 5, 1, 8, 7, 7, "f16", "head", None, 0, 0), ([1, 1], [90, 200], 3, 3, 72, 16, 16, "bf16", "head", None, 0, 0),
    ([1, 1], [90, 700], 4, 2, 136, 16, 16, "f16", "token", None, 0, 0), ([1, 1], [5, 4000], 2, 2, 200, 64, 32, "bf16", "head", None, 0, 0),
    ([1] * 300, [30] * 300, 2, 1, 64, 16, 16, "bf16", "token", None, 0, 0),
    ([1, 5, 0, 3], [0, 2, 9, 60], 4, 2, 64, 16, 16, "f16", "head", None, 0, 0), ([200], [0], 8, 2, 128, 16, 8, "bf16", "token", None, 0, 0),
    ([130, 1, 1, 64], [300, 777, 0, 5], 16, 4, 128, 64, 16, "f16", "head", None, 0, 9), ([63, 64, 65], [1, 0, 64], 3, 3, 128, 32, 32, "bf16", "head", None, 0, 1),
    ([31, 33], [500, 0], 5, 1, 80, 16, 1, "f16", "token", None, 0, 0), ([70], [70], 6, 2, 96, 7, 7, "bf16", "head", None, 0, 2),
    ([40, 2], [0, 100], 4, 1, 256, 16, 16, "f16", "head", None, 0, 0), ([129], [1000], 2, 1, 64, 1, 1, "bf16", "head", None, 0, 0),
    ([12], [7], 4, 2, 24, 16, 16, "f16", "head", None, 0, 0), ([1000, 900], [0, 0], 4, 1, 128, 64, 64, "f16", "head", None, 0, 0),
    ([300], [0], 4, 4, 160, 64, 16, "bf16", "token", None, 0, 0), ([2], [4090], 8, 1, 128, 64, 32, "f16", "head", None, 0, 0),
    ([509, 1], [2046, 900], 8, 2, 128, 16, 16, "f16", "head", None, 0, 0),
    # windows, 16 bits
    ([1], [0], 2, 1, 64, 16, 0, "f16", "head", 1, 0, 0), ([1] * 4, [0, 1, 2, 700], 4, 2, 128, 16, 0, "bf16", "token", 1, 1, 0),
    ([1] * 6, [5, 30, 31, 32, 100, 5000], 8, 2, 128, 16, 0, "f16", "head", 32, 0, 0), ([1] * 3, [4000, 70, 300], 32, 8, 128, 64, 0, "bf16", "head", 500, 4, 0),
    ([1] * 3, [4000, 70, 300], 4, 1, 80, 5, 0, "f16", "token", 129, 7, 0), ([1, 1], [900, 3000], 4, 2, 256, 16, 0, "bf16", "head", 700, 100, 0),
    ([1] * 70, list(range(0, 700, 10)), 2, 2, 64, 8, 0, "f16", "head", 100, 3, 0), ([1] * 2, [2000, 20000], 2, 1, 96, 256, 0, "f16", "head", 1500, 1, 0),
    ([200], [0], 8, 2, 128, 16, 0, "bf16", "token", 1, 0, 0), ([300], [0], 4, 1, 64, 16, 0, "f16", "head", 64, 4, 0), ([257], [1000], 4, 2, 128, 16, 0, "f16", "head", 33, 70, 3),
    ([130, 1, 1, 64], [300, 777, 0, 5], 16, 4, 128, 64, 0, "f16", "head", 100, 10, 9), ([1, 5, 0, 3], [0, 2, 9, 60], 4, 2, 64, 16, 0, "f16", "head", 2, 1, 0),
    ([1500], [0], 2, 1, 128, 64, 0, "bf16", "head", 200, 4, 0), ([40, 2], [0, 900], 4, 1, 256, 16, 0, "f16", "head", 30, 20, 0),
    ([60, 70], [3000, 1], 6, 2, 96, 7, 0, "bf16", "token", 1000, 3, 0), ([509, 1], [2046, 900], 8, 2, 128, 16, 0, "f16", "head", 1000, 0, 0),
    ([3] * 70, [200] * 70, 8, 8, 64, 16, 0, "f16", "head", 50, 5, 5),
    # windows, 8 bits
    ([1] * 6, [5, 30, 31, 32, 100, 5000], 8, 2, 128, 16, 16, "f16", "head", 32, 5, 0), ([1] * 3, [4000, 70, 300], 32, 8, 128, 64, 16, "bf16", "token", 500, 4, 0),
    ([1, 1], [900, 3000], 4, 2, 72, 6, 3, "bf16", "head", 700, 100, 0), ([257], [1000], 4, 2, 128, 16, 4, "f16", "head", 33, 70, 3),
    ([130, 1, 1, 64], [300, 777, 0, 5], 16, 4, 64, 64, 32, "f16", "head", 100, 10, 9), ([1500], [0], 2, 1, 128, 64, 64, "bf16", "token", 200, 4, 0),
    ([40, 2], [0, 900], 4, 1, 256, 16, 16, "f16", "head", 30, 20, 0), ([509, 1], [2046, 900], 8, 2, 128, 16, 16, "f16", "head", 1000, 0, 0),
]


@pytest.mark.parametrize("case", ATTEND, ids=lambda c: "x".join(map(str, (len(c[0]), max(c[0]), max(c[1])) + c[2:])))
def test_attention_against_the_definition(hexmi, case):
    new, context, heads, kv, dim, page, block, dt, order, window, sinks, padding = case
    c = Long(new, context, heads, kv, dim, page, block, DTYPES[dt], order, window, sinks, seed=dim + len(new), padding=padding)
    got = c.run(hexmi)
    c.check(got)
    out = torch.full_like(got, 7.0)
    assert c.run(hexmi, out=out) is out and torch.equal(out, got)


@pytest.mark.parametrize("new, context, shared, heads, kv, dim, page, block, dt", [
    ([1] * 5, [0, 3, 40, 200, 1], 64, 8, 2, 128, 16, 16, "f16"), ([1] * 33, list(range(33)), 1024, 32, 8, 128, 64, 16, "bf16"),
    ([30, 1, 0, 90], [1, 1, 1, 1], 400, 16, 4, 64, 16, 8, "f16"), ([200, 7], [0, 300], 333, 6, 2, 80, 9, 9, "bf16"),
    ([1] * 4, [0, 1, 2, 3], 128, 4, 2, 256, 16, 16, "f16"),
], ids=str)
def test_shared_prefix_in_8_bits(hexmi, new, context, shared, heads, kv, dim, page, block, dt):
    c = Long(new, [shared + x for x in context], heads, kv, dim, page, block, DTYPES[dt], seed=dim + len(new), shared=shared)
    c.check(c.run(hexmi), "each for itself")
    c.page_table[:, :shared // page] = -7                             # not read
    c.check(c.run(hexmi, shared_pages=c.shared_pages), "shared")


@pytest.mark.parametrize("seed", range(24))
def test_drawn_batches(hexmi, seed):
    rng = random.Random(seed)
    B, page = rng.randint(1, 6), rng.choice((1, 5, 8, 16, 16, 64, 128))
    kv = rng.choice((1, 2, 3))
    block = 0 if rng.random() < 0.3 else rng.choice([b for b in range(1, 65) if page % b == 0])
    window = rng.choice((1, 3, 17, 64, 100, 333, 2000)) if block == 0 or rng.random() < 0.5 else None
    new = [rng.choice((1, 1, 0, 2, 33, 150, 300)) for _ in range(B)] if rng.random() < 0.6 else [1] * B
    c = Long(new, [rng.choice((0, 1, 50, 700, 2500)) for _ in range(B)], kv * rng.choice((1, 2, 5, 17)), kv, rng.choice((16, 64, 64, 128, 104, 192, 256)), page,
             block, DTYPES[rng.choice(("f16", "bf16"))], rng.choice(("head", "token")), window, rng.choice((0, 1, 4, 90)) if window else 0, seed=seed,
             padding=rng.choice((0, 0, 3)))
    c.check(c.run(hexmi))


def test_windows_that_hide_nothing_are_none(hexmi):
    c = Long([40, 1], [300, 777], 8, 2, 128, 16, 0, torch.float16)
    whole = c.run(hexmi)
    for window, sinks in ((1 << 70, 0), (1 << 70, 1 << 70), (2000, 0), (1, 2000), (1, 1 << 70)):
        assert torch.equal(c.run(hexmi, window=window, sinks=sinks), whole), (window, sinks)


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("new", [[1, 1, 1], [70, 1, 40]])
def test_scales_at_the_ends_of_their_range(hexmi, dt, new):
    """Values with the least exponent (in fp16 subnormal numbers among them), keys with a large one beside small queries."""
    dtype = DTYPES[dt]
    c = Long(new, [300, 20, 77], 4, 2, 64, 16, 8, dtype, seed=6)
    least, large = RANGE[dtype][0], 7
    for i, (name, e) in enumerate((("k", large), ("v", least))):
        old = c.scales[i].double() - 127
        whole = []
        for b, t in enumerate(getattr(c, name + "64")):
            at = torch.arange(t.shape[0])
            whole.append(t * torch.exp2(e - old[c.table[b, at // 16], :, at % 16 // 8])[..., None])
            assert torch.equal(whole[-1], whole[-1].to(dtype).double())
        setattr(c, name + "64", whole)
        getattr(c, name + "_scales").fill_(e + 127)
    c.q.mul_(2.0 ** -12)
    c.check(c.run(hexmi))


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 72, 128, 256])
def test_queries_of_very_different_sizes(hexmi, dt, dim):
    """Columns of a query from 2^-20 to 1 of its largest, over keys in 8 bits. A bf16 query is multiplied as the sum of two numbers of e4m3: a
    value x of a row whose largest is m is off by half of the second one's last step, 2^-10 / 16 of the row's scale, which is at least m / 448
    and at most m / 224: by 2^-14 / 224 m < 2^-21 m, so a score by scale 2^-21 m sum |k|, and the weights by twice that."""
    c = Long([90, 1, 1], [40, 300, 9], 4, 2, dim, 16, 8, DTYPES[dt], seed=12)
    g = _gen(13)
    c.q = (c.q.cpu().double() * torch.exp2(torch.randint(-20, 1, c.q.shape, generator=g).double())).to(c.dtype).cuda()
    got = c.run(hexmi).cpu().double()
    t, G, scale, u = 0, 2, 1 / math.sqrt(dim), half_step(c.dtype)
    for n, L, k, v in zip(c.new, c.lengths, c.k64, c.v64):
        hidden = torch.arange(L)[None] > torch.arange(L - n, L)[:, None]
        for h in range(4):
            q, kh, vh = c.q[t:t + n, h].cpu().double(), k[:, h // G], v[:, h // G]
            w = torch.softmax((q @ kh.T * scale).masked_fill(hidden, -math.inf), 1)
            o, a = w @ vh, w @ vh.abs()
            size = (q.abs() @ kh.abs().T * scale).amax(1, keepdim=True)
            off = scale * 2.0 ** -21 * q.abs().amax(1, keepdim=True) * kh.abs().sum(1).amax()
            bound = u * (a + o.abs()) + (2 * (dim + 8) * E * size + 2 * off + 16 * E) * (a + o.abs()) + u * o.abs()
            if dt == "f16":
                bound = bound + L * 2.0 ** -25 * vh.abs().amax(0) + 2.0 ** -25
            assert ((got[t:t + n, h] - o).abs() <= bound).all(), (n, h)
        t += n


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("block, window", [(8, None), (8, 50), (0, 50)])
def test_queries_that_are_not_finite_stay_in_their_rows(hexmi, dt, block, window):
    c = Long([90, 1, 1], [40, 300, 9], 4, 2, 64, 16, block, DTYPES[dt], seed=14, window=window, sinks=2 if window else 0)
    want = c.run(hexmi)
    rows = [(3, 1, math.nan), (70, 0, math.inf), (90, 2, -math.inf), (91, 3, math.nan)]
    for t, h, x in rows:
        c.q[t, h, 5] = x
    got = c.run(hexmi)
    hit = torch.zeros(92, 4, dtype=torch.bool, device="cuda")
    for t, h, _ in rows:
        hit[t, h] = True
    assert torch.isnan(got[hit].float()).all() and torch.equal(got[~hit], want[~hit])


@pytest.mark.parametrize("scaled", [False, True])
@pytest.mark.parametrize("ragged", [False, True])
def test_index_tensors_that_make_no_sense_touch_nothing_outside(hexmi, scaled, ragged):
    g = _gen(11)
    pages = [torch.randn(5, 2, 16, 64, generator=g).to(E4M3 if scaled else torch.float16).cuda() for _ in range(2)]
    kw = {n: torch.full((5, 2, 2), 120, dtype=torch.uint8, device="cuda") for n in ("k_scales", "v_scales")} if scaled else {}
    q = torch.randn(6, 4, 64, generator=g).half().cuda()
    B = 4 if ragged else 6
    lengths = torch.tensor([-(1 << 31), (1 << 31) - 1, 3, 0, 40, 41][:B], dtype=torch.int32, device="cuda")
    table = torch.tensor([[-(1 << 31), (1 << 31) - 1, 5]] * B, dtype=torch.int32, device="cuda")
    starts = torch.tensor([3, -9, 1 << 30, 2, 70], dtype=torch.int32, device="cuda") if ragged else None
    around = torch.full((18, 4, 64), 7.0, dtype=torch.float16, device="cuda")
    out = around[6:12]
    for window, sinks in ((5, 2), (30, 1 << 50), (None, 0)):
        hexmi.paged_attention(q, *pages, table, lengths, starts, out=out, window=window, sinks=sinks, **kw)
        assert (around[:6] == 7).all() and (around[12:] == 7).all()
        assert ((out == 0) | (out == 7 if ragged else False)).all()
    if scaled:
        before = [t.clone() for t in (*pages, *kw.values())]
        rows = torch.randn(6, 2, 64, generator=g).half().cuda()
        hexmi.paged_append(rows, rows.clone(), *pages, table, lengths, starts, q=q, inv_freq=hexmi.rope_frequencies(64), **kw)
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(before, (*pages, *kw.values())))
    before = [t.clone() for t in pages]
    index = torch.tensor([-1, 3, 1 << 30, -(1 << 31), 2, 0, 1], dtype=torch.int32, device="cuda")
    new_table, new_lengths = hexmi.paged_fork(*pages, table, lengths, index, torch.full_like(index, 1 << 30), **kw)
    for i, parent in enumerate(index.tolist()):
        known = 0 <= parent < B
        assert new_lengths[i].item() == (lengths[parent].item() if known else 0)
        assert torch.equal(new_table[i], table[parent] if known else torch.full_like(table[0], -1))
    new_table, count = hexmi.paged_compact(*pages, table, lengths, **kw)
    assert count.item() == 0 and (new_table == -1).all()
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(before, pages))


# ---- appends
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


def least_exponent(most, lo, hi):
    """The least e of lo .. hi with most <= 448 * 2^e."""
    e = lo
    while e < hi and most > 448 * 2.0 ** e:
        e += 1
    return e


def half_steps(value, e):
    """Half a step of e4m3 times 2^e at a value."""
    return torch.maximum(value.abs() * 2.0 ** -4, torch.full_like(value, 2.0 ** (e - 10)))


def check_appended(pages, scales, before, scales_before, rows, size, new, lengths, table, dtype, ragged):
    """pages, scales: after a call that put rows [tokens, heads, dim] there; before, scales_before: what stood there."""
    lo, hi = RANGE[dtype]
    page = pages.shape[2]
    block = page // scales.shape[2]
    now, then = pages.cpu().double(), before.cpu().double()
    s_now, s_then = scales.cpu().int() - 127, scales_before.cpu().int() - 127
    touched = torch.zeros(pages.shape[:3], dtype=torch.bool)
    t = 0
    for b, (n, L) in enumerate(zip(new, lengths)):
        for start in range((L - n) // block * block, L, block) if n else ():
            p = table[b, start // page].item()
            at = start % page
            old, end = max(0, L - n - start), min(block, L - start)
            mine = slice(t + start + old - (L - n), t + start + end - (L - n))
            touched[p, :, at:at + end] = True
            for h in range(pages.shape[1]):
                y, off = rows[mine, h], 24 * E * size[mine, h]
                most = y.abs().max().item()
                e = s_now[p, h, at // block].item()
                could = {least_exponent(m, lo, hi) for m in (most, most - off.max().item(), most + off.max().item())}
                was = s_then[p, h, at // block].item()
                if old:
                    could = {max(x, was) for x in could}
                assert e in could, (b, start, h, e, could)
                got = now[p, h, at + old:at + end] * 2.0 ** e
                wrong = ~((got - y).abs() <= half_steps(y, e) + off)
                assert not wrong.any(), (b, start, h, (got - y)[wrong][:4], y[wrong][:4])
                if old:
                    a, o = then[p, h, at:at + old] * 2.0 ** was, now[p, h, at:at + old] * 2.0 ** e
                    assert ((a - o).abs() <= (half_steps(a, e) if e > was else torch.zeros(()))).all(), (b, start, h)
        t += n
    same = ~touched[..., None].expand(pages.shape)
    assert torch.equal(pages.cpu().view(torch.uint8)[same], before.cpu().view(torch.uint8)[same])


APPEND = [
    # new tokens, contexts, heads (0: no q), kv heads, dim, rotated columns, page, block, dtype, order, pairs, norms, rows behind the last
    ([1], [0], 0, 1, 64, 0, 16, 16, "f16", "head", "adjacent", False, 0), ([1] * 5, [0, 15, 16, 17, 100], 4, 2, 128, 128, 16, 16, "f16", "head", "adjacent", False, 0),
    ([1] * 70, list(range(70)), 32, 8, 128, 128, 16, 8, "bf16", "token", "halves", True, 0), ([1] * 3, [5, 6, 7], 3, 3, 80, 40, 8, 1, "bf16", "head", "halves", True, 0),
    ([1, 1], [63, 64], 2, 2, 256, 256, 64, 64, "f16", "head", "halves", True, 0), ([1, 1], [63, 9], 5, 5, 8, 8, 32, 32, "f16", "token", "adjacent", True, 0),
    ([700], [0], 4, 2, 128, 128, 64, 16, "bf16", "token", "halves", True, 0), ([33, 1, 0, 17], [3, 15, 8, 0], 8, 2, 64, 32, 16, 16, "f16", "head", "adjacent", True, 5),
    ([2, 3, 4, 5] * 9, [14] * 36, 4, 4, 96, 96, 16, 4, "bf16", "head", "halves", False, 1), ([130, 70], [1, 63], 2, 1, 256, 256, 128, 64, "bf16", "head", "halves", True, 0),
    ([100], [7], 0, 3, 72, 72, 5, 5, "f16", "head", "adjacent", True, 2), ([50, 60], [11, 0], 6, 6, 104, 52, 48, 48, "f16", "token", "halves", True, 0),
    ([40], [1], 2, 2, 200, 200, 32, 32, "bf16", "head", "adjacent", False, 0), ([5] * 40, [2] * 40, 12, 12, 64, 64, 32, 32, "f16", "head", "halves", False, 3),
    ([64] * 3, [0, 32, 16], 16, 1, 128, 64, 16, 16, "f16", "head", "halves", True, 0),
]


@pytest.mark.parametrize("case", APPEND, ids=lambda c: "x".join(map(str, (len(c[0]), max(c[0]), max(c[1])) + c[2:])))
@pytest.mark.parametrize("form", ["slices", "odd"])
def test_append_against_the_definition(hexmi, case, form):
    new, context, heads, kv, dim, R, page, block, dt, order, pairs, norms, padding = case
    g, dtype = _gen(dim + sum(new)), DTYPES[dt]
    c = Long(new, context, max(heads, kv) // kv * kv, kv, dim, page, block, dtype, order, seed=dim + len(new), padding=padding)
    T = sum(new) + padding
    # rows of very different sizes, so that scales rise
    wide = torch.randn(T + 1, (heads + 2 * kv) * dim + 8, generator=g) * torch.exp2(torch.randint(-6, 5, (T + 1, 1), generator=g).float())
    wide = wide.to(dtype).cuda()
    wide = wide.view(-1)[1:1 + T * wide.shape[1]].view(T, -1) if form == "odd" else wide[:T]            # two bytes off the boundaries
    q, k, v = (wide[:, a:a + n * dim].unflatten(1, (n, dim)) if n else None for a, n in ((0, heads), (heads * dim, kv), ((heads + kv) * dim, kv)))
    weight = lambda: (1 + 0.2 * torch.randn(dim, generator=g)).to(dtype).cuda() if norms else None
    kw, qw = weight(), weight() if heads else None
    freq = hexmi.rope_frequencies(R) if R else None
    before = [t.clone() for t in (c.k_pages, c.v_pages, c.k_scales, c.v_scales)]
    got = hexmi.paged_append(k, v, c.k_pages, c.v_pages, c.page_table, c.lengths_d, c.starts, kw, freq, 1e-5, pairs, q, qw, k_scales=c.k_scales,
                             v_scales=c.v_scales)
    at = torch.cat([torch.arange(L - n, L) for n, L in zip(new, c.lengths)] + [torch.zeros(padding, dtype=torch.long)])
    ragged = c.starts is not None
    check_appended(c.k_pages, c.k_scales, before[0], before[2], *rows64(k, kw, freq, at, 1e-5, pairs), new, c.lengths, c.table, dtype, ragged)
    check_appended(c.v_pages, c.v_scales, before[1], before[3], v.cpu().double(), torch.zeros(v.shape, dtype=torch.float64), new, c.lengths, c.table,
                   dtype, ragged)
    if heads:
        want, size = rows64(q, qw, freq, at, 1e-5, pairs)
        want[T - padding:], size[T - padding:] = 0, 0
        bound = half_step(dtype) * want.abs() + 24 * E * size + torch.finfo(dtype).tiny * half_step(dtype)
        assert ((got.cpu().double() - want).abs() <= bound).all()
    else:
        assert got is None


MANY = [61, 62, 63, 64, 65, 127, 300, 4100]


@pytest.mark.parametrize("sequences", MANY)
@pytest.mark.parametrize("block", [2, 16])
def test_append_of_many_sequences(hexmi, sequences, block):
    """Which sequence a block of new tokens belongs to is looked up 64 starts at a time: ragged batches around that and far beyond, sequences without
    new tokens and rows behind the last among them."""
    new = [(1, 0, 3, 17, 0, 1)[(5 * i + i // 7) % 6] for i in range(sequences)]
    context = [(0, 3, 15, 30, 7)[i % 5] for i in range(sequences)]
    case = (new, context, 2, 1, 64, 64, 16, block, "f16", "head", "adjacent", False, 5)
    test_append_against_the_definition(hexmi, case, "slices")


@pytest.mark.parametrize("sequences", MANY)
def test_all_sequences_but_one_without_new_tokens(hexmi, sequences):
    for at in (0, sequences // 2, sequences - 1):
        new = [40 if i == at else 0 for i in range(sequences)]
        test_append_against_the_definition(hexmi, (new, [5] * sequences, 0, 1, 64, 0, 16, 16, "bf16", "head", "adjacent", False, 0), "slices")


def one_block(hexmi, rows, contexts, dtype, block=16, **kw):
    """Values put one call after the other into a cache of one head of 64; (numbers, exponents)."""
    pages = [torch.full((2, 1, 16, 64), 0x7f, dtype=torch.uint8, device="cuda").view(E4M3) for _ in range(2)]
    scales = [torch.full((2, 1, 16 // block), 255, dtype=torch.uint8, device="cuda") for _ in range(2)]      # what was there before is nothing
    table = torch.tensor([[1]], dtype=torch.int32, device="cuda")
    for x, n in zip(rows, contexts):
        x = x.to(dtype).cuda().view(1, 1, 64)
        hexmi.paged_append(x, x.clone(), *pages, table, torch.tensor([n + 1], dtype=torch.int32, device="cuda"), k_scales=scales[0], v_scales=scales[1], **kw)
    for t, s in zip(pages, scales):
        assert torch.equal(t.view(torch.uint8), pages[0].view(torch.uint8)) and torch.equal(s, scales[0])
        assert (t[0].view(torch.uint8) == 0x7f).all() and (s[0] == 255).all()
    return pages[0][1, 0].cpu(), scales[0][1, 0].cpu().int() - 127


def test_scales_rise_and_do_not_fall_within_a_block(hexmi):
    one, two = torch.full((64,), 1.75), torch.full((64,), 0.875)
    codes, e = one_block(hexmi, [two, one, two, one * 2 ** 6, two], range(5), torch.float16)
    assert e.item() == -2                                             # 112 = 448 / 4
    assert torch.equal(codes[:5].float() * 0.25, torch.stack((two, one, two, one * 64, two)))
    codes, e = one_block(hexmi, [one * 64, two, two], (14, 15, 0), torch.float16)        # the block's first slot again: a new sequence's
    assert e.item() == -9 and torch.equal(codes[0].float() * 2.0 ** -9, two)
    # blocks of four: the second one's scale is its own (the first slots are written before, as a sequence's older tokens are)
    codes, e = one_block(hexmi, [two, two, two, one, one * 4, one], range(6), torch.bfloat16, block=4)
    assert e[:2].tolist() == [-8, -6]
    assert torch.equal(codes[3:6].float() * torch.exp2(e[:2].float()).repeat_interleave(4)[3:6, None], torch.stack((one, one * 4, one)))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_values_at_the_ends(hexmi, dtype):
    lo, hi = RANGE[dtype]
    most = torch.finfo(dtype).max
    row = torch.zeros(64)
    codes, e = one_block(hexmi, [row], [0], dtype)
    assert e.item() == lo and (codes[0].float() == 0).all()
    row[:6] = torch.tensor([most, -most, most * 0.75, 1.0, -0.0, most * 0.9375])
    codes, e = one_block(hexmi, [row], [0], dtype)
    got = codes[0].double() * 2.0 ** e.item()
    assert e.item() == hi and torch.equal(got.to(dtype).double(), got)          # numbers of the type, none of them infinite
    assert ((got - row.to(dtype).double()).abs() <= row.to(dtype).double().abs() * 2.0 ** -4 + 2.0 ** (hi - 10)).all()
    row = torch.full((64,), 1.0)
    row[3], row[4], row[5] = math.inf, -math.inf, math.nan
    codes, e = one_block(hexmi, [row], [0], dtype)
    assert e.item() == -8 and torch.isnan(codes[0, 3:6].float()).all() and (codes[0, 6:].float() == 256).all() and (codes[0, :3].float() == 256).all()
    codes, e = one_block(hexmi, [row, torch.full((64,), 8.0)], [0, 1], dtype)     # NaN stays one as the scale rises
    assert e.item() == -5 and torch.isnan(codes[0, 3:6].float()).all() and (codes[0, 6:].float() == 32).all()
    tiny = torch.full((64,), 2.0 ** (lo - 9))
    codes, e = one_block(hexmi, [tiny], [0], dtype)
    assert e.item() == lo and (codes[0].float() == 2.0 ** -9).all()
    # every border between two exponents: 448 * 2^e and the next number
    for x in (1.75, 1.0, 1.5, 0.4375):
        above = torch.nextafter(torch.tensor(x, dtype=torch.float32), torch.tensor(9.0)) if dtype == torch.float32 else torch.tensor(x) * (1 + torch.finfo(dtype).eps)
        for y in (torch.tensor(x), above):
            y = y.to(dtype).float()
            _, e = one_block(hexmi, [torch.full((64,), y.item())], [0], dtype)
            assert e.item() == least_exponent(y.item(), lo, hi), (x, y.item())


@pytest.mark.parametrize("dt, befores", [("f16", (7, 8, 9, 10, 13, 20, 21, 22, 25, 60, 127)), ("bf16", (119, 120, 121, 124, 127))])
@pytest.mark.parametrize("new", [1, 3, 9])
def test_older_exponents_above_the_range_stay(hexmi, dt, befores, new):
    """A block that another type filled, with an exponent that this one's appends do not reach: it does not fall, the older numbers stay as they
    are, and the new ones are numbers of the type. Rounding is e4m3's own, so all of it is exact."""
    dtype, g = DTYPES[dt], _gen(21)
    hi = RANGE[dtype][1]
    for before in befores:
        old, kv, dim = 5, 3, 64
        codes = torch.randint(0, 0x7f, (2, kv, 16, dim), generator=g, dtype=torch.uint8)
        k_pages, v_pages = codes.view(E4M3).cuda(), codes.view(E4M3).cuda()
        scales = [torch.full((2, kv, 1), before + 127, dtype=torch.uint8, device="cuda") for _ in range(2)]
        largest = torch.finfo(dtype).max
        y = (torch.randn(new, kv, dim, generator=g) * torch.exp2(torch.randint(-20, 2, (new, kv, 1), generator=g).float()) * (largest / 16)).clamp(-largest, largest)
        y[0, 0, 0], y[0, 0, 1] = largest, -largest
        y = y.to(dtype)
        starts = None if new == 1 else torch.tensor([0, new], dtype=torch.int32, device="cuda")
        hexmi.paged_append(y.cuda(), y.cuda(), k_pages, v_pages, torch.tensor([[1]], dtype=torch.int32, device="cuda"),
                           torch.tensor([old + new], dtype=torch.int32, device="cuda"), starts, k_scales=scales[0], v_scales=scales[1])
        e = max(before, hi)                                           # the largest value asks for the type's largest exponent
        limit = 448.0 if e < hi else math.floor(240 * 512 * 2.0 ** (hi - e)) / 512
        for pages, s in zip((k_pages, v_pages), scales):
            got = pages.cpu().view(torch.uint8)
            at = s.cpu().int()[1, :, 0] - 127
            want_e = [max(before, least_exponent(y[:, h].abs().max().item(), *RANGE[dtype])) for h in range(kv)]
            assert at.tolist() == want_e and (s[0] == before + 127).all(), (before, at)
            for h in range(kv):
                if want_e[h] == before:
                    assert torch.equal(got[1, h, :old], codes[1, h, :old]), before
                if want_e[h] < hi:
                    continue
                x = (y[:, h].double() * 2.0 ** -want_e[h]).clamp(-limit, limit)
                put = got[1, h, old:old + new].view(E4M3)
                assert torch.equal(put.float(), x.float().to(E4M3).float()), (before, h)
                back = put.double() * 2.0 ** want_e[h]
                assert torch.equal(back.to(dtype).double(), back) and torch.isfinite(back.to(dtype)).all(), before
            assert torch.equal(got[:, :, old + new:], codes[:, :, old + new:]) and torch.equal(got[0], codes[0])


def test_an_older_exponent_of_255_is_none(hexmi):
    """What it scales is NaN and becomes so; the new numbers are as in a fresh block."""
    codes = torch.randint(0, 0x7f, (1, 1, 16, 64), generator=_gen(22), dtype=torch.uint8)
    pages = [codes.view(E4M3).cuda() for _ in range(2)]
    scales = [torch.full((1, 1, 1), 255, dtype=torch.uint8, device="cuda") for _ in range(2)]
    x = torch.full((1, 1, 64), 1.75, dtype=torch.float16, device="cuda")
    hexmi.paged_append(x, x.clone(), *pages, torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.tensor([4], dtype=torch.int32, device="cuda"),
                       k_scales=scales[0], v_scales=scales[1])
    for t, s in zip(pages, scales):
        assert s.item() == 127 - 8 and torch.isnan(t[0, 0, :3].float()).all() and (t[0, 0, 3].float() == 448).all()
        assert torch.equal(t.cpu().view(torch.uint8)[0, 0, 4:], codes[0, 0, 4:])


def test_every_number_of_e4m3_is_rounded_to_even(hexmi):
    """All numbers and the middles between neighbours, at a scale of 1 (the largest is 448)."""
    numbers = torch.arange(127, dtype=torch.uint8).view(E4M3).double()
    middles = (numbers[1:] + numbers[:-1]) / 2
    all_of = torch.cat((numbers, middles, -numbers, -middles))
    for i in range(0, all_of.numel(), 60):
        row = torch.zeros(64, dtype=torch.float64)
        row[:min(60, all_of.numel() - i)] = all_of[i:i + 60]
        row[63] = 448
        x = row.to(torch.float16)
        assert torch.equal(x.double(), row)
        codes, e = one_block(hexmi, [x], [0], torch.float16)
        assert e.item() == 0 and torch.equal(codes[0].view(torch.uint8), row.float().to(E4M3).view(torch.uint8))


# ---- forks and compaction
def fork_reference(c, parents, pages):
    """(table, lengths, copies (from, to, slots))."""
    table, lengths, copies = [], [], []
    for parent, page in zip(parents, pages):
        if not 0 <= parent < len(c.lengths):
            table.append([-1] * c.table.shape[1])
            lengths.append(0)
            continue
        row, L = c.table[parent].tolist(), c.lengths[parent]
        column, filled = min(L, len(row) * c.page) // c.page, min(L, len(row) * c.page) % c.page
        if 0 <= page < c.k_pages.shape[0] and column < len(row) and (filled == 0 or 0 <= row[column] < c.k_pages.shape[0]):
            if filled:
                copies.append((row[column], page, filled))
            row[column] = page
        table.append(row)
        lengths.append(L)
    return torch.tensor(table, dtype=torch.int32), torch.tensor(lengths, dtype=torch.int32), copies


def raw(t):
    return t.contiguous().view(torch.uint8) if t.dtype == E4M3 else t.contiguous().view(torch.int16) if t.dtype != torch.uint8 else t


FORK = [
    # contexts, rows, kv heads, dim, page, block (0: 16 bits), dtype, order
    ([0], 1, 1, 64, 16, 0, "f16", "head"), ([600, 601, 615, 15], 4, 8, 128, 16, 0, "f16", "head"), ([599, 31, 32, 33, 0], 200, 2, 80, 16, 0, "bf16", "token"),
    ([100, 2000, 255, 256], 50, 8, 128, 256, 32, "bf16", "token"), ([100, 2000, 255], 7, 3, 96, 128, 16, "f16", "head"), ([9, 5, 3], 30, 1, 8, 5, 5, "f16", "head"),
    ([40] * 70, 70, 2, 72, 7, 1, "bf16", "head"), ([40, 3], 5, 2, 36, 16, 0, "f16", "head"), ([40, 3], 5, 2, 20, 16, 2, "f16", "token"), ([40, 3], 5, 3, 7, 16, 16, "f16", "head"),
]


@pytest.mark.parametrize("case", FORK, ids=lambda c: "x".join(map(str, (len(c[0]), max(c[0])) + c[1:])))
def test_fork_against_the_definition(hexmi, case):
    context, rows, kv, dim, page, block, dt, order = case
    rng = random.Random(rows)
    c = Long([1] * len(context), context, kv, kv, dim, page, block, DTYPES[dt], order, seed=rows)
    pool = c.k_pages.shape[0]
    tensors = [t for t in (c.k_pages, c.v_pages, c.k_scales, c.v_scales) if t is not None]
    grown = [in_order(torch.cat((t.contiguous(), t[:1].expand(rows, *t.shape[1:]))), order) for t in tensors]      # fresh pages behind
    c.k_pages, c.v_pages = grown[:2]
    scales = dict(zip(("k_scales", "v_scales"), grown[2:]))
    parents = [rng.randrange(len(context)) if rng.random() < 0.9 else rng.choice((-1, len(context), 1 << 30)) for _ in range(rows)]
    pages = [pool + i if rng.random() < 0.85 else rng.choice((-1, pool + rows, 1 << 30)) for i in range(rows)]
    table, lengths, copies = fork_reference(c, parents, pages)
    want = [t.clone() for t in grown]
    for a, b, filled in copies:
        for t in want[:2]:
            raw_t = t.view(torch.uint8) if block else t
            raw_t[b, :, :filled] = raw_t[a, :, :filled]
        for t in want[2:]:
            t[b, :, :-(-filled // block)] = t[a, :, :-(-filled // block)]
    index = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    got = hexmi.paged_fork(c.k_pages, c.v_pages, c.page_table, c.lengths_d, index(parents), index(pages), **scales)
    assert torch.equal(got[0].cpu(), table) and torch.equal(got[1].cpu(), lengths)
    for a, b in zip(grown, want):
        assert torch.equal(raw(a), raw(b))
    # into tensors of the caller's, one of them the table itself
    outs = torch.full_like(got[0], 9), torch.full_like(got[1], 9)
    again = hexmi.paged_fork(c.k_pages, c.v_pages, c.page_table, c.lengths_d, index(parents), index(pages), table_out=outs[0], lengths_out=outs[1], **scales)
    assert again[0] is outs[0] and again[1] is outs[1] and torch.equal(outs[0], got[0]) and torch.equal(outs[1], got[1])
    if rows == len(context):
        hexmi.paged_fork(c.k_pages, c.v_pages, c.page_table, c.lengths_d, index(parents), index(pages), table_out=c.page_table, lengths_out=c.lengths_d, **scales)
        assert torch.equal(c.page_table, got[0]) and torch.equal(c.lengths_d, got[1])


def compact_reference(table, lengths, pool, page, window, sinks):
    used = [[0 <= c < pool and i * page < min(L, len(row) * page) and (not window or i * page < sinks or (i + 1) * page > min(L, len(row) * page) - window)
             for i, c in enumerate(row)] for row, L in zip(table, lengths)]
    marked = {c for row, u in zip(table, used) for c, x in zip(row, u) if x}
    n = len(marked)
    moves = dict(zip(sorted(p for p in marked if p >= n), sorted(set(range(n)) - marked)))
    return [[moves.get(c, c) if x else -1 for c, x in zip(row, u)] for row, u in zip(table, used)], n, moves


COMPACT = [
    # lengths, pool, columns, kv heads, dim, page, block, dtype, order, window, sinks
    ([], 5, 3, 1, 64, 16, 0, "f16", "head", None, 0), ([0, 0], 5, 3, 1, 64, 16, 0, "f16", "head", None, 0), ([40, 16, 17, 0, 48], 20, 3, 2, 128, 16, 0, "f16", "head", None, 0),
    ([100, 90, 7], 64, 8, 2, 80, 16, 16, "bf16", "token", None, 0), ([100, 90, 7], 32, 8, 2, 80, 16, 4, "bf16", "head", None, 0), ([1000] * 30, 2000, 64, 2, 64, 16, 0, "bf16", "head", None, 0),
    ([1000, 77, 3000], 700, 200, 3, 20, 16, 2, "f16", "head", 100, 20), ([1000, 77, 3000], 33333, 200, 1, 8, 16, 16, "f16", "token", 1, 0), ([128], 8, 8, 1, 64, 16, 0, "f16", "head", None, 0),
    ([64 * 16], 64, 64, 1, 64, 16, 0, "f16", "head", None, 0), ([500, 400], 200, 500, 2, 7, 1, 1, "f16", "head", 50, 3), ([9] * 100, 100, 1, 1, 16, 9, 0, "f16", "head", None, 0),
]


@pytest.mark.parametrize("case", COMPACT, ids=lambda c: "x".join(map(str, (len(c[0]), sum(c[0])) + c[1:])))
def test_compact_against_the_definition(hexmi, case):
    lengths, pool, columns, kv, dim, page, block, dt, order, window, sinks = case
    g, rng = _gen(pool), random.Random(pool)
    shape = (pool, kv, page, dim)
    pages = [in_order((torch.randint(0, 256, shape, generator=g, dtype=torch.uint8).view(E4M3) if block else torch.randn(shape, generator=g).to(DTYPES[dt])).cuda(), order)
             for _ in range(2)]
    scales = {n: torch.randint(0, 256, (pool, kv, page // block), generator=g, dtype=torch.uint8).cuda() for n in ("k_scales", "v_scales")} if block else {}
    # some pages are several sequences', some none, some no page's number; entries past a length are whatever
    names = torch.randperm(pool, generator=g).tolist()
    table = [[rng.choice((names[(b * columns + i) % pool], names[(b * columns + i) % pool], names[i % pool], names[(b * columns + i) % pool], -1 if rng.random() < 0.2 else names[0]))
              if rng.random() < 0.97 else rng.choice((-1, pool, 1 << 30)) for i in range(columns)] for b in range(len(lengths))]
    if len(lengths) == 1 or len(lengths) == 100:
        table = [[names[(b * columns + i) % pool] for i in range(columns)] for b in range(len(lengths))]        # every page in use
    want, n, moves = compact_reference(table, lengths, pool, page, window, sinks)
    held = [t.clone() for t in (*pages, *scales.values())]
    for t in held:
        flat = t.view(torch.uint8) if t.dtype == E4M3 else t
        source = flat.clone()
        for a, b in moves.items():
            flat[b] = source[a]
    page_table = torch.tensor(table, dtype=torch.int32, device="cuda").view(len(lengths), columns)
    lens = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    kw = {**scales, "window": window, "sinks": sinks}
    got, count = hexmi.paged_compact(*pages, page_table, lens, **kw)
    assert count.tolist() == [n] and got.tolist() == want
    for a, b in zip((*pages, *scales.values()), held):
        assert torch.equal(raw(a), raw(b))
    # nothing is left to move, and the table may be its own result
    kept = got.clone()
    result, count = hexmi.paged_compact(*pages, got, lens, table_out=got, **kw)
    assert result is got and count.tolist() == [n] and torch.equal(got, kept)
    for a, b in zip((*pages, *scales.values()), held):
        assert torch.equal(raw(a), raw(b))


def kept_reference(table, lengths, pool, page, window, sinks, ahead):
    """compact_reference where `ahead` positions past a length count too."""
    positions = [min(max(L, 0), len(row) * page) for row, L in zip(table, lengths)]
    used = [[0 <= c < pool and i * page < n + ahead and (not window or i * page < sinks or (i + 1) * page > n - window) for i, c in enumerate(row)]
            for row, n in zip(table, positions)]
    marked = {c for row, u in zip(table, used) for c, x in zip(row, u) if x}
    n = len(marked)
    moves = dict(zip(sorted(p for p in marked if p >= n), sorted(set(range(n)) - marked)))
    return [[moves.get(c, c) if x else -1 for c, x in zip(row, u)] for row, u in zip(table, used)], n, moves


@pytest.mark.parametrize("ahead", [1, 2, 16, 17, 40, 1 << 50])
@pytest.mark.parametrize("window, sinks", [(None, 0), (20, 3)])
def test_compact_keeps_pages_ahead(hexmi, ahead, window, sinks):
    rng, pool, page = random.Random(ahead), 60, 16
    lengths = [0, 15, 16, 17, 32, 47, 96, 200, -5]                    # the table ends at 96
    table = [rng.sample(range(pool), 6) for _ in lengths]
    table[2][1], table[3][2] = -1, pool                               # no page there yet
    x = [torch.randn(pool, 2, page, 64, generator=_gen(1)).half().cuda() for _ in range(2)]
    before = [t.clone() for t in x]
    want, n, moves = kept_reference(table, lengths, pool, page, window, sinks, ahead)
    index = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    got, count = hexmi.paged_compact(*x, index(table), index(lengths), window=window, sinks=sinks, ahead=ahead)
    assert got.tolist() == want and count.tolist() == [n]
    for now, then in zip(x, before):
        held = then.clone()
        for a, b in moves.items():
            held[b] = then[a]
        assert torch.equal(now, held)
    previous = hexmi.through_dispatcher(True)
    try:
        again, _ = hexmi.paged_compact(*before, index(table), index(lengths), window=window, sinks=sinks, ahead=ahead)
    finally:
        hexmi.through_dispatcher(previous)
    assert torch.equal(again, got)


LARGE = [
    # sequences, columns, pool, page, window, sinks, shared pages: one workgroup marks up to 8192 entries and 262144 pages, shared ones among them
    (1, 8192, 9000, 1, None, 0, 0), (1, 8193, 9000, 1, None, 0, 0), (64, 128, 5000, 4, None, 0, 0), (64, 129, 20000, 4, 70, 9, 0), (300, 40, 7001, 2, None, 0, 0),
    (2, 4096, 9000, 1, None, 0, 1), (3, 50, 262144, 1, None, 0, 0), (3, 50, 262145, 1, None, 0, 2), (700, 300, 262175, 1, 100, 0, 0), (1, 8193, 33, 1, None, 0, 0),
    (9000, 1, 9000, 1, None, 0, 0), (0, 8193, 40, 1, None, 0, 8193),
]


@pytest.mark.parametrize("case", LARGE, ids=lambda c: "x".join(map(str, c)))
def test_compact_of_many_entries_and_pages(hexmi, case):
    """Around the sizes from which marks are made by many workgroups, in a workspace that held ones."""
    from hexmi import _lib, ops
    B, columns, pool, page, window, sinks, shared = case
    rng, g = random.Random(B + pool), _gen(pool)
    lengths = [rng.choice((0, rng.randint(0, columns * page), columns * page)) for _ in range(B)] or []
    if B in (1, 9000):
        lengths = [columns * page] * B
    # the upper half of the pool is named more often, some pages by several rows
    table = [[rng.randrange(pool // 2, pool) if rng.random() < 0.8 else rng.choice((-1, pool, rng.randrange(pool))) for _ in range(columns)] for _ in range(B)]
    prefix = [rng.randrange(pool) for _ in range(shared)]
    want, n, moves = kept_reference([prefix + row[shared:] for row in table] + [prefix], lengths + [shared * page], pool, page, window, sinks, 0)
    index = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    x = [torch.randint(-(1 << 15), 1 << 15, (pool, 1, page, 8), generator=g, dtype=torch.int16).view(torch.float16).cuda() for _ in range(2)]
    held = [t.clone() for t in x]
    if moves:
        source, target = (torch.tensor(list(v), device="cuda") for v in (moves.keys(), moves.values()))
        for t in held:
            t[target] = t[source]
    page_table, lens, prefix_d = index(table).view(B, columns), index(lengths), index(prefix)
    out, names, count = torch.full_like(page_table, 9), torch.full_like(prefix_d, 9), torch.full((1,), 9, dtype=torch.int32, device="cuda")
    batch = ops._paged_batch(B, *x, page_table, lens, None)
    ws = torch.full((_lib.lib().hexmi_paged_compact_workspace(batch),), 255, dtype=torch.uint8, device="cuda")
    _lib.check(_lib.lib().hexmi_paged_compact_ex(batch, None, prefix_d.data_ptr() if shared else None, shared, window or 0, sinks, 0, out.data_ptr(), columns,
                                                 names.data_ptr() if shared else None, count.data_ptr(), _lib.F16, ws.data_ptr(), ws.numel(),
                                                 torch.cuda.current_stream().cuda_stream), "hexmi_paged_compact_ex")
    assert count.item() == n and out.tolist() == want[:-1] and names.tolist() == want[-1]
    assert all(torch.equal(a.view(torch.int16), b.view(torch.int16)) for a, b in zip(x, held))


@pytest.mark.parametrize("ahead", [0, 1])
@pytest.mark.parametrize("columns", ["none", "stale", "named"])
@pytest.mark.parametrize("shared", [[], [40, 3], [57, 41, 41, -1, 60, 2]], ids=len)
def test_compact_of_a_shared_prefix_against_the_definition(hexmi, shared, columns, ahead):
    """The prefix's pages are in use whatever the lengths, and what the table says in their columns does not count."""
    rng, pool, page = random.Random(len(shared)), 60, 16
    lengths = [0, 31, 32, 97, 128, 1, -5]
    others = [p for p in range(pool) if p not in shared]
    table = [rng.sample(others, 8) for _ in lengths]
    for row in table:
        row[:len(shared)] = {"none": [-7] * len(shared), "stale": rng.sample(others, len(shared)), "named": shared}[columns]
    x = [torch.randn(pool, 1, page, 64, generator=_gen(1)).half().cuda() for _ in range(2)]
    before = [t.clone() for t in x]
    # the same as a table that names them, with a row of their own
    want, n, moves = kept_reference([shared + row[len(shared):] for row in table] + [shared], lengths + [len(shared) * page], pool, page, None, 0, ahead)
    index = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    got, count, names = hexmi.paged_compact(*x, index(table), index(lengths), shared_pages=index(shared), ahead=ahead)
    assert got.tolist() == want[:-1] and count.tolist() == [n] and names.tolist() == want[-1]
    for now, then in zip(x, before):
        held = then.clone()
        for a, b in moves.items():
            held[b] = then[a]
        assert torch.equal(now, held)
    # into the table itself, through the dispatcher, and with the prefix on the host
    previous = hexmi.through_dispatcher(True)
    try:
        t = index(table)
        again = hexmi.paged_compact(*before, t, index(lengths), shared_pages=torch.tensor(shared, dtype=torch.int32), ahead=ahead, table_out=t)
    finally:
        hexmi.through_dispatcher(previous)
    assert again[0] is t and all(torch.equal(a, b) for a, b in zip(again, (got, count, names)))
    assert all(torch.equal(a, b) for a, b in zip(x, before))


def test_compact_of_a_shared_prefix_and_no_sequence(hexmi):
    x = [torch.randn(9, 1, 4, 8, generator=_gen(1)).half().cuda() for _ in range(2)]
    before = [t.clone() for t in x]
    table = torch.zeros(0, 5, dtype=torch.int32, device="cuda")
    got, count, names = hexmi.paged_compact(*x, table, torch.zeros(0, dtype=torch.int32, device="cuda"),
                                            shared_pages=torch.tensor([8, 1], dtype=torch.int32, device="cuda"))
    assert got.shape == (0, 5) and count.item() == 2 and names.tolist() == [0, 1]
    assert all(torch.equal(a[0], b[8]) and torch.equal(a[1:], b[1:]) for a, b in zip(x, before))


# ---- a run of them
def step(hexmi, state, x, freq, graph=False):
    q = hexmi.paged_append(x[:, 4:6], x[:, 6:], state["k"], state["v"], state["table"], state["lengths"], inv_freq=freq, q=x[:, :4], k_scales=state["ks"],
                           v_scales=state["vs"])
    return hexmi.paged_attention(q, state["k"], state["v"], state["table"], state["lengths"], window=40, sinks=4, k_scales=state["ks"], v_scales=state["vs"])


def small_state(seed, rows=3):
    g = _gen(seed)
    state = {"k": (torch.randn(40, 2, 16, 64, generator=g) * 50).to(E4M3).cuda(), "v": (torch.randn(40, 2, 16, 64, generator=g) * 50).to(E4M3).cuda(),
             "ks": torch.full((40, 2, 2), 121, dtype=torch.uint8, device="cuda"), "vs": torch.full((40, 2, 2), 122, dtype=torch.uint8, device="cuda"),
             "lengths": torch.tensor([30, 47, 80][:rows], dtype=torch.int32, device="cuda"),
             "table": torch.randperm(40, generator=g)[:rows * 8].view(rows, 8).int().cuda()}
    return state


def test_beams_that_fork_and_compact_go_on_as_without(hexmi):
    """Decode steps of three rows; every row forked into two, the pages compacted, and on: the same as rows that kept pages of their own."""
    freq = hexmi.rope_frequencies(64)
    g = _gen(1)
    xs = [torch.randn(3, 8, 64, generator=g).half().cuda() for _ in range(40)]
    a = small_state(5)
    apart = {n: t.clone() for n, t in a.items()}
    for x in xs[:5]:
        for s in (a, apart):
            s["lengths"] += 1
        assert torch.equal(step(hexmi, a, x, freq), step(hexmi, apart, x, freq))
    fresh = torch.tensor([p for p in range(40) if p not in set(a["table"].flatten().tolist())][:6], dtype=torch.int32, device="cuda")
    parents = torch.tensor([2, 0, 1, 1, 0, 2], dtype=torch.int32, device="cuda")
    table, lengths = hexmi.paged_fork(a["k"], a["v"], a["table"], a["lengths"], parents, fresh, k_scales=a["ks"], v_scales=a["vs"])
    a["table"], a["lengths"] = table, lengths
    for i, x in enumerate(xs[5:12]):
        both = torch.randn(6, 8, 64, generator=g).half().cuda()
        a["lengths"] += 1
        apart["lengths"] += 1
        got = step(hexmi, a, both, freq)
        if i == 3:                                                    # in the middle: the table renamed, pages moved
            a["table"], count = hexmi.paged_compact(a["k"], a["v"], a["table"], a["lengths"], k_scales=a["ks"], v_scales=a["vs"], window=40, sinks=4)
            assert 0 < count.item() <= 40
            again = hexmi.paged_attention(torch.ones(6, 4, 64, device="cuda").half(), a["k"], a["v"], a["table"], a["lengths"], window=40, sinks=4,
                                          k_scales=a["ks"], v_scales=a["vs"])
            assert torch.isfinite(again).all()
            free = iter(range(count.item(), 40))                      # every row's next pages
            for r in range(6):
                for col in range((a["lengths"][r].item() + 15) // 16, 8):
                    a["table"][r, col] = next(free, -1)
        if i == 0:
            # rows 1, 2 and 0 of the fork go on as rows 0, 1 and 2 of the batch apart
            first = step(hexmi, apart, both[[1, 2, 0]], freq)
            assert torch.equal(got[[1, 2, 0]], first)
        else:
            assert torch.equal(got[[1, 2, 0]], step(hexmi, apart, both[[1, 2, 0]], freq)), i


def test_a_fork_at_the_end_of_a_page_keeps_its_page_through_a_compaction(hexmi):
    """Rows whose next token begins the page that the fork gave them: appends and attention go on as without the compaction."""
    freq, g = hexmi.rope_frequencies(64), _gen(3)
    a = small_state(7)
    a["lengths"].copy_(torch.tensor([48, 33, 64], dtype=torch.int32))
    for r in range(3):                                                # no page is named past a length
        a["table"][r, (a["lengths"][r].item() + 15) // 16:] = -1
    used = set(a["table"].flatten().tolist())
    fresh = torch.tensor([p for p in range(39, -1, -1) if p not in used][:5], dtype=torch.int32, device="cuda")
    parents = torch.tensor([0, 2, 0, 1, 2], dtype=torch.int32, device="cuda")
    a["table"], a["lengths"] = hexmi.paged_fork(a["k"], a["v"], a["table"], a["lengths"], parents, fresh, k_scales=a["ks"], v_scales=a["vs"])
    apart = {n: t.clone() for n, t in a.items()}
    a["table"], count = hexmi.paged_compact(a["k"], a["v"], a["table"], a["lengths"], k_scales=a["ks"], v_scales=a["vs"], window=40, sinks=4, ahead=1)
    assert not torch.equal(a["k"].view(torch.uint8), apart["k"].view(torch.uint8)) and a["table"].max().item() < count.item()
    for i in range(16):                                               # the tokens of the new page
        x = torch.randn(5, 8, 64, generator=g).half().cuda()
        for s in (a, apart):
            s["lengths"] += 1
        assert torch.equal(step(hexmi, a, x, freq), step(hexmi, apart, x, freq)), i
        if a["lengths"][3].item() == 48:
            break


@pytest.mark.parametrize("new, context, shared, dim, page, block, dt", [
    ([1] * 5, [0, 3, 40, 200, 1], 64, 128, 16, 16, "f16"), ([30, 1, 0, 90], [1, 1, 1, 1], 400, 64, 16, 8, "bf16"), ([1] * 3, [5, 90, 20], 96, 64, 32, 0, "f16"),
], ids=str)
@pytest.mark.parametrize("named", [False, True])
def test_a_shared_prefix_through_a_compaction(hexmi, new, context, shared, dim, page, block, dt, named):
    """A cache of which the first pages are nobody's: the prefix moves with the rest, and attention is the same behind it."""
    c = Long(new, [shared + x for x in context], 4, 2, dim, page, block, DTYPES[dt], seed=dim, shared=shared)
    tensors = [t for t in (c.k_pages, c.v_pages, c.k_scales, c.v_scales) if t is not None]
    grown = [torch.cat((t[:1].expand(7, *t.shape[1:]), t)) for t in tensors]
    c.k_pages, c.v_pages = grown[:2]
    if block:
        c.k_scales, c.v_scales = grown[2:]
    c.page_table, c.shared_pages = torch.where(c.page_table >= 0, c.page_table + 7, c.page_table), c.shared_pages + 7
    want = c.run(hexmi, shared_pages=c.shared_pages)
    c.check(want)
    if not named:
        c.page_table[:, :shared // page] = -7
    scales = {"k_scales": c.k_scales, "v_scales": c.v_scales} if block else {}
    old = c.shared_pages
    c.page_table, count, c.shared_pages = hexmi.paged_compact(c.k_pages, c.v_pages, c.page_table, c.lengths_d, shared_pages=old, **scales)
    assert not torch.equal(c.shared_pages, old) and c.page_table.max().item() < count.item() and c.shared_pages.max().item() < count.item()
    for t in (c.k_pages, c.v_pages):                                  # what is free now may be anything
        t[count.item():].view(torch.uint8 if block else torch.int16).fill_(0x7f if block else 0x7fff)
    assert torch.equal(c.run(hexmi, shared_pages=c.shared_pages), want)
    c.check(c.run(hexmi), "each for itself")                          # the table names them now


def test_a_captured_step_is_replayed(hexmi):
    """Append, attention within a window, fork and compaction in one graph, replayed as lengths and tables change, with eager work between."""
    freq = hexmi.rope_frequencies(64)
    g = _gen(2)
    state, x = small_state(6), torch.zeros(3, 8, 64, dtype=torch.float16, device="cuda")
    parents, pages = torch.zeros(3, dtype=torch.int32, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")

    def all_of(s):
        out = step(hexmi, s, x, freq)
        table, lengths = hexmi.paged_fork(s["k"], s["v"], s["table"], s["lengths"], parents, pages, k_scales=s["ks"], v_scales=s["vs"])
        packed, count = hexmi.paged_compact(s["k"], s["v"], table, lengths, k_scales=s["ks"], v_scales=s["vs"], window=40, sinks=4)
        return out, table, lengths, packed, count

    warm = {n: t.clone() for n, t in state.items()}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        all_of(warm)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        results = all_of(state)
    fresh = small_state(6)
    for name in state:
        state[name].copy_(fresh[name])
    eager = {n: t.clone() for n, t in state.items()}
    free = [p for p in range(40) if p not in set(fresh["table"].flatten().tolist())]
    for i in range(5):
        x.copy_(torch.randn(3, 8, 64, generator=g).half())
        parents.copy_(torch.tensor([i % 3, 2, 0], dtype=torch.int32))
        pages.copy_(torch.tensor(free[3 * i % 12:3 * i % 12 + 3], dtype=torch.int32))
        for s in (state, eager):
            s["lengths"] += 1
        graph.replay()
        want = all_of(eager)
        torch.cuda.synchronize()
        for a, b in zip(results, want):
            assert torch.equal(a, b), i
        for name in state:
            assert torch.equal(raw(state[name]) if name in "kv" else state[name], raw(eager[name]) if name in "kv" else eager[name]), (i, name)


def test_calls_on_two_streams(hexmi):
    c = [Long([1] * 4, [700, 33, 2000, 90], 8, 2, 128, 16, 16, torch.float16, seed=s, window=300, sinks=4) for s in (1, 2)]
    want = [x.run(hexmi) for x in c]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(c[i].run(hexmi))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])


def test_through_the_dispatcher_and_host_index_tensors(hexmi):
    c = Long([3, 1], [40, 90], 4, 2, 64, 16, 8, torch.float16, window=30, sinks=2, seed=3)
    got = c.run(hexmi)
    c.page_table, c.lengths_d, c.starts = c.page_table.cpu(), c.lengths_d.cpu(), c.starts.cpu()
    assert torch.equal(c.run(hexmi), got)
    previous = hexmi.through_dispatcher(True)
    try:
        assert torch.equal(c.run(hexmi), got)
        index = torch.tensor([1, 0], dtype=torch.int32, device="cuda")
        a = hexmi.paged_fork(c.k_pages, c.v_pages, c.page_table, c.lengths_d, index, torch.full_like(index, -1), c.k_scales, c.v_scales)
        b = hexmi.paged_compact(c.k_pages, c.v_pages, c.page_table, c.lengths_d, c.k_scales, c.v_scales)
    finally:
        hexmi.through_dispatcher(previous)
    assert torch.equal(a[0].cpu(), c.page_table[[1, 0]]) and b[0].shape == c.page_table.shape


def test_caches_past_32_bits(hexmi):
    """Pages that stand past 4 GiB of their tensors: append, attention, fork and compaction as over a small cache."""
    g = _gen(9)
    size, dim, rows = 128, 256, 4
    far = (1 << 32) // (size * dim) + 100
    big = {n: torch.zeros(far, 1, size, dim, dtype=torch.uint8, device="cuda").view(E4M3) for n in ("k", "v")}
    small = {n: torch.zeros(40, 1, size, dim, dtype=torch.uint8, device="cuda").view(E4M3) for n in ("k", "v")}
    scales = {c: {n: torch.full((pool, 1, 4), 121, dtype=torch.uint8, device="cuda") for n in ("k_scales", "v_scales")} for c, pool in (("big", far), ("small", 40))}
    at = far - 40                                                     # page p of the small cache is page at + p of the large one
    assert at * size * dim > 1 << 32
    for n in ("k", "v"):
        x = torch.randint(0, 0x70, (40, 1, size, dim), generator=g, dtype=torch.uint8).cuda()
        small[n].view(torch.uint8).copy_(x)
        big[n].view(torch.uint8)[at:].copy_(x)
    table = torch.randperm(40, generator=g)[:rows * 5].view(rows, 5).int().cuda()
    lengths = torch.tensor([300, 640, 1, 511], dtype=torch.int32, device="cuda")
    free = torch.tensor([p for p in range(40) if p not in set(table.flatten().tolist())][:rows], dtype=torch.int32, device="cuda")
    x = torch.randn(rows, 4, dim, generator=g).half().cuda()
    freq = hexmi.rope_frequencies(dim)
    results = []
    for pages, kw, add in ((small, scales["small"], 0), (big, scales["big"], at)):
        q = hexmi.paged_append(x[:, 2:3], x[:, 3:], pages["k"], pages["v"], table + add, lengths, inv_freq=freq, q=x[:, :2], **kw)
        out = [hexmi.paged_attention(q, pages["k"], pages["v"], table + add, lengths, **kw)]
        starts = torch.tensor([0, 1, 4, 4, 4], dtype=torch.int32, device="cuda")
        out.append(hexmi.paged_attention(q, pages["k"], pages["v"], table + add, lengths, starts, window=200, sinks=3, **kw))
        new_table, new_lengths = hexmi.paged_fork(pages["k"], pages["v"], table + add, lengths, torch.tensor([3, 0, 1, 1], dtype=torch.int32, device="cuda"), free + add, **kw)
        out += [new_table - add, new_lengths, raw(pages["k"][add:add + 40]).clone(), raw(pages["v"][add:add + 40]).clone(), kw["k_scales"][add:add + 40].clone()]
        packed, count = hexmi.paged_compact(pages["k"], pages["v"], new_table, new_lengths, **kw)
        out += [count, hexmi.paged_attention(q, pages["k"], pages["v"], packed, new_lengths, **kw)]
        results.append(out)
    for i, (a, b) in enumerate(zip(*results)):
        assert torch.equal(torch.where(a < 0, torch.full_like(a, -1), a) if i == 2 else a, torch.where(b < 0, torch.full_like(b, -1), b) if i == 2 else b), i


def test_lengths_past_the_table_end_with_it(hexmi):
    c = Long([3, 1], [60, 77], 4, 2, 64, 16, 0, torch.float16, window=20, sinks=5, seed=8, ragged=True)
    table = c.page_table[:, :5].contiguous()                          # 80 positions
    at_end = torch.tensor([80, 80], dtype=torch.int32, device="cuda")
    pages = torch.randn(2, *c.k_pages.shape, generator=_gen(1)).half().cuda()
    one = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    q = c.q[:2].contiguous()
    want = hexmi.paged_attention(q, pages[0], pages[1], table.clamp(0, 3), at_end, one, window=20, sinks=5)
    got = hexmi.paged_attention(q, pages[0], pages[1], table.clamp(0, 3), at_end + 1000, one, window=20, sinks=5)
    assert torch.equal(got, want)
    assert torch.equal(hexmi.paged_attention(q, pages[0], pages[1], table.clamp(0, 3), at_end + 1000, window=20, sinks=5),
                       hexmi.paged_attention(q, pages[0], pages[1], table.clamp(0, 3), at_end, window=20, sinks=5))


def test_pages_with_room_between_them(hexmi):
    """Strides of pages, heads, slots and scales that are not the tensors' own."""
    c = Long([40, 1, 1], [100, 300, 9], 4, 2, 64, 16, 8, torch.bfloat16, seed=4, window=90, sinks=2)
    want = c.run(hexmi)
    for name in ("k_pages", "v_pages"):
        t = getattr(c, name)
        wide = torch.full((t.shape[0], t.shape[1] + 1, 2 * t.shape[2], t.shape[3] + 16), 0x7f, dtype=torch.uint8, device="cuda").view(E4M3)
        view = wide[:, 1:, ::2, 16:]
        view.view(torch.uint8).copy_(t.view(torch.uint8))
        setattr(c, name, view)
    for name in ("k_scales", "v_scales"):
        t = getattr(c, name)
        wide = torch.full((2 * t.shape[0], t.shape[1], t.shape[2], 3), 255, dtype=torch.uint8, device="cuda")
        view = wide[1::2, :, :, 1]
        view.copy_(t)
        setattr(c, name, view)
    assert torch.equal(c.run(hexmi), want)
    rows = torch.randn(3, 2, 64, generator=_gen(3)).bfloat16().cuda()
    close = Long([1] * 3, [100, 300, 9], 4, 2, 64, 16, 8, torch.bfloat16, seed=4)
    apart = Long([1] * 3, [100, 300, 9], 4, 2, 64, 16, 8, torch.bfloat16, seed=4)
    wide = torch.zeros(apart.k_pages.shape[0], 2, 32, 80, dtype=torch.uint8, device="cuda").view(E4M3)
    wide[:, :, ::2, 16:].view(torch.uint8).copy_(apart.k_pages.view(torch.uint8))
    apart.k_pages = wide[:, :, ::2, 16:]
    for x in (close, apart):
        hexmi.paged_append(rows, rows.clone(), x.k_pages, x.v_pages, x.page_table, x.lengths_d, k_scales=x.k_scales, v_scales=x.v_scales)
    assert torch.equal(raw(close.k_pages), raw(apart.k_pages)) and torch.equal(close.k_scales, apart.k_scales)
    assert (wide[:, :, 1::2].float() == 0).all() and (wide[..., :16].float() == 0).all()
    index = torch.tensor([2, 0, 1], dtype=torch.int32, device="cuda")
    got = [hexmi.paged_fork(x.k_pages, x.v_pages, x.page_table, x.lengths_d, index, torch.full_like(index, -1), x.k_scales, x.v_scales) for x in (close, apart)]
    packed = [hexmi.paged_compact(x.k_pages, x.v_pages, *t, x.k_scales, x.v_scales) for x, t in zip((close, apart), got)]
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1]) and torch.equal(packed[0][0], packed[1][0]) and torch.equal(raw(close.k_pages), raw(apart.k_pages))


def test_a_table_of_one_row_of_any_stride(hexmi):
    """A column turned into a row is contiguous, whatever its row stride says: read, written in place and as the result."""
    c = Long([1], [100], 2, 2, 64, 16, 8, torch.float16, seed=5)
    want_attention = c.run(hexmi)
    kw = {"k_scales": c.k_scales, "v_scales": c.v_scales}
    plain = [t.clone() for t in (c.k_pages, c.v_pages)]
    parents, pages = torch.zeros(1, dtype=torch.int32, device="cuda"), torch.full((1,), -1, dtype=torch.int32, device="cuda")
    fork = hexmi.paged_fork(*plain, c.page_table, c.lengths_d, parents, pages, **kw)
    compact = hexmi.paged_compact(*plain, c.page_table, c.lengths_d, k_scales=c.k_scales.clone(), v_scales=c.v_scales.clone())
    row = c.page_table.clone().view(-1, 1).T
    assert row.stride() == (1, 1) and row.is_contiguous()
    c.page_table = row
    assert torch.equal(c.run(hexmi), want_attention)
    out = torch.zeros_like(row).view(-1, 1).T
    table, lengths = hexmi.paged_fork(c.k_pages, c.v_pages, row, c.lengths_d, parents, pages, table_out=out, **kw)
    assert table is out and torch.equal(out, fork[0]) and torch.equal(lengths, fork[1])
    table, count = hexmi.paged_compact(c.k_pages, c.v_pages, row, c.lengths_d, table_out=row, **kw)
    assert table is row and torch.equal(row, compact[0]) and torch.equal(count, compact[1])


@pytest.mark.parametrize("new", [[1] * 4, [5, 0, 40, 1]])
def test_append_in_8_bits_into_rows_of_the_callers(hexmi, new):
    """q's rows into q itself, into rows off the boundaries, into the keys' rows (read by others), and through the dispatcher: all the same."""
    g, freq = _gen(15), hexmi.rope_frequencies(64)
    T = sum(new)
    rows = torch.randn(T, 6, 64, generator=g).half().cuda()

    def call(q_out=None, x=None):
        c = Long(new, [30, 3, 9, 100], 2, 2, 64, 16, 8, torch.float16, seed=3, ragged=len(set(new)) > 1)
        x = rows.clone() if x is None else x
        q_out = q_out(x) if callable(q_out) else q_out
        y = hexmi.paged_append(x[:, 2:4], x[:, 4:], c.k_pages, c.v_pages, c.page_table, c.lengths_d, c.starts, inv_freq=freq, q=x[:, :2], q_out=q_out,
                               k_scales=c.k_scales, v_scales=c.v_scales)
        assert q_out is None or y is q_out
        return [y.clone(), raw(c.k_pages), raw(c.v_pages), c.k_scales, c.v_scales]

    want = call()
    odd = torch.zeros(T * 2 * 64 + 1, dtype=torch.float16, device="cuda")[1:].view(T, 2, 64)
    for q_out in (lambda x: x[:, :2], odd, lambda x: x[:, 2:4], lambda x: x[:, 1:3], torch.zeros(T, 2, 64, dtype=torch.float16)):
        got = call(q_out)
        assert all(torch.equal(a.cpu(), b.cpu()) for a, b in zip(got, want))
    previous = hexmi.through_dispatcher(True)
    try:
        got = call()
    finally:
        hexmi.through_dispatcher(previous)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_what_is_only_read_stays_shared(hexmi):
    """Attention over copy-on-write pages and scales in 8 bits, and within a window, copies neither; a fork, which writes, has its own."""
    c = Long([1] * 3, [40, 90, 7], 4, 2, 64, 16, 8, torch.float16, seed=4, window=30, sinks=2)
    want = c.run(hexmi)
    plain = {n: getattr(c, n) for n in ("k_pages", "v_pages", "k_scales", "v_scales")}
    for n, t in plain.items():
        setattr(c, n, torch._lazy_clone(t))
    assert torch.equal(c.run(hexmi), want)
    assert all(torch._C._is_cow_tensor(getattr(c, n)) for n in plain)
    before = {n: (raw(t) if n in ("k_pages", "v_pages") else t).clone() for n, t in plain.items()}
    parents, pages = torch.tensor([1], dtype=torch.int32, device="cuda"), torch.tensor([c.k_pages.shape[0] - 1], dtype=torch.int32, device="cuda")
    hexmi.paged_fork(c.k_pages, c.v_pages, c.page_table, c.lengths_d, parents, pages, c.k_scales, c.v_scales)
    for n, t in before.items():
        assert torch.equal(raw(plain[n]) if n in ("k_pages", "v_pages") else plain[n], t), n


@pytest.mark.parametrize("block", [2, 8])
def test_tokens_before_the_first_position_are_left_out(hexmi, block):
    """More new tokens than a length has positions: those below 0 leave nothing and see nothing, the others are as alone."""
    g = _gen(6)
    rows = torch.randn(25, 6, 64, generator=g).half().cuda()
    results = []
    for first, n in ((0, 25), (18, 7)):
        c = Long([7], [0], 2, 2, 64, 16, block, torch.float16, seed=3, ragged=True)
        starts = torch.tensor([0, n], dtype=torch.int32, device="cuda")
        x = rows[first:]
        hexmi.paged_append(x[:, 2:4], x[:, 4:], c.k_pages, c.v_pages, c.page_table, c.lengths_d, starts, k_scales=c.k_scales, v_scales=c.v_scales)
        kw = {"k_scales": c.k_scales, "v_scales": c.v_scales}
        out = hexmi.paged_attention(x[:, :2], c.k_pages, c.v_pages, c.page_table, c.lengths_d, starts, window=5, sinks=1, **kw)
        results.append([out[18 - first:], raw(c.k_pages), raw(c.v_pages), c.k_scales, c.v_scales])
        assert (out[:18 - first] == 0).all()
    assert all(torch.equal(a, b) for a, b in zip(*results))


def test_a_captured_compaction_behind_a_prefix_is_replayed(hexmi):
    """A fork and a compaction that keeps its pages and a shared prefix, in one graph, replayed as tables, lengths and prefix change."""
    g = _gen(8)
    pool, page, cols = 50, 8, 6
    pages = [torch.randn(pool, 2, page, 64, generator=g).half().cuda() for _ in range(2)]
    table, lengths = torch.zeros(4, cols, dtype=torch.int32, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda")
    prefix, parents, fresh = (torch.zeros(n, dtype=torch.int32, device="cuda") for n in (2, 5, 5))

    def both(x, t, n, shared):
        t, n = hexmi.paged_fork(*x, t, n, parents, fresh)
        return (t, n, *hexmi.paged_compact(*x, t, n, ahead=1, shared_pages=shared))

    warm = [t.clone() for t in pages]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both(warm, table, lengths, prefix)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        results = both(pages, table, lengths, prefix)
    for i in range(5):
        order = torch.randperm(pool, generator=g).int()
        prefix.copy_(order[:2])
        fresh.copy_(order[2:7])
        parents.copy_(torch.randint(-1, 5, (5,), generator=g).int())
        table.copy_(order[7:7 + 4 * cols].view(4, cols))
        lengths.copy_(torch.randint(2, cols + 1, (4,), generator=g).int() * page - (torch.arange(4) % 2 * 3).int())
        for t in pages:
            t.copy_(torch.randn(t.shape, generator=g).half())
        eager = [t.clone() for t in pages]
        graph.replay()
        want = both(eager, table, lengths, prefix)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(results, want)), i
        assert all(torch.equal(a, b) for a, b in zip(pages, eager)), i


def test_the_registered_compaction_takes_its_former_arguments(hexmi):
    x = [torch.randn(6, 1, 4, 8, generator=_gen(1)).half().cuda() for _ in range(2)]
    table, lengths = torch.tensor([[5, 1]], dtype=torch.int32, device="cuda"), torch.tensor([8], dtype=torch.int32, device="cuda")
    out, count = torch.empty_like(table), torch.empty(1, dtype=torch.int32, device="cuda")
    torch.ops.hexmi.paged_compact(*x, None, None, table, lengths, None, 0, out, count)
    assert count.item() == 2 and out.tolist() == [[0, 1]]

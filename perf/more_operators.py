"""What long contexts add to a paged cache of keys and values, as measurable cases.

  append   keys (normed, rotated) and values of new tokens into pages held in 8 bits (e4m3) with one power-of-two scale, as a biased
           exponent, for each block of tokens and head; the queries beside them
  attend   attention of the new tokens over the pages in 8 bits
  window   attention within a sliding window and over a few first tokens (sinks), over pages in 16 or 8 bits; pages that no token sees
           any more are gone from the table
  fork     rows that go on from others' (a step of a beam search): a new table, and the part-filled last pages copied
  compact  the pages in use moved to the front of the cache, and the table renamed

A case is a dict of plain values. Lengths are spread evenly over their logarithm between the two ends a case gives, pages are dealt in
random order. With `own` false, run() is the mathematics in elementary torch operations; with `own` true, the package's operators.
"""
import math
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.getcwd(), "hexagon-mlir_amd"))

own = False

_DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
_EPS, _THETA = 1e-5, 10000.0
# exponents of scales, so that every code times its scale is a number of the 16-bit type
_LEAST, _MOST = {"f16": -15, "bf16": -117}, {"f16": 8, "bf16": 120}


def listed():
    return [
        # A decode step of 64 sequences: one key and value of each into its last block, whose scale may grow; the query beside them.
        {"name": "append_f16_64x1_32+8x128", "op": "append", "sequences": 64, "new": 1, "new_to": 1, "context": 30, "context_to": 1000, "page": 16,
         "block": 16, "q_heads": 32, "kv_heads": 8, "dim": 128, "rotary": 128, "dtype": "f16", "pairs": "adjacent", "norm": False, "order": "head"},
        # Prompts of a batch, ragged, with norms of the heads, into pages that hold all heads of a token side by side.
        {"name": "append_bf16_6x700..2000_32+8x128", "op": "append", "sequences": 6, "new": 700, "new_to": 2000, "context": 1, "context_to": 500, "page": 64,
         "block": 16, "q_heads": 32, "kv_heads": 8, "dim": 128, "rotary": 128, "dtype": "bf16", "pairs": "halves", "norm": True, "order": "token"},
        # Decode of 16 sequences with 2048 tokens behind them, a key head to each query head.
        {"name": "decode8_f16_16x2048_32x128", "op": "attend", "sequences": 16, "new": 1, "new_to": 1, "context": 2047, "context_to": 2047,
         "page": 64, "block": 64, "bits": 8, "q_heads": 32, "kv_heads": 32, "dim": 128, "dtype": "f16", "order": "head"},
        # Decode of 64 sequences of very different lengths, shared key heads.
        {"name": "decode8_bf16_64x100..16384_32/8x128", "op": "attend", "sequences": 64, "new": 1, "new_to": 1, "context": 99, "context_to": 16383,
         "page": 16, "block": 16, "bits": 8, "q_heads": 32, "kv_heads": 8, "dim": 128, "dtype": "bf16", "order": "token"},
        # Four whole prompts of about 4096 tokens.
        {"name": "prompt8_bf16_4x4096_32/8x128", "op": "attend", "sequences": 4, "new": 4033, "new_to": 4096, "context": 0, "context_to": 0,
         "page": 64, "block": 16, "bits": 8, "q_heads": 32, "kv_heads": 8, "dim": 128, "dtype": "bf16", "order": "head"},
        # Decode of 32 long sequences, of which a window is left, in 16 bits.
        {"name": "window_bf16_32x5000..60000_w4096+4_32/8x128", "op": "window", "sequences": 32, "new": 1, "new_to": 1, "context": 4999, "context_to": 59999,
         "page": 16, "block": 16, "bits": 16, "window": 4096, "sinks": 4, "q_heads": 32, "kv_heads": 8, "dim": 128, "dtype": "bf16", "order": "head"},
        # One long prompt within a window of 1024.
        {"name": "window_f16_1x16001_w1024+4_32/8x128", "op": "window", "sequences": 1, "new": 16001, "new_to": 16001, "context": 0, "context_to": 0,
         "page": 64, "block": 16, "bits": 16, "window": 1024, "sinks": 4, "q_heads": 32, "kv_heads": 8, "dim": 128, "dtype": "f16", "order": "token"},
        # The next 300 tokens of one prompt beside seven sequences that decode, heads of 64, in 8 bits.
        {"name": "window8_f16_8x1..300_w500+16_12/12x64", "op": "window", "sequences": 8, "new": 1, "new_to": 300, "context": 700, "context_to": 9000,
         "page": 32, "block": 32, "bits": 8, "window": 500, "sinks": 16, "q_heads": 12, "kv_heads": 12, "dim": 64, "dtype": "f16", "order": "head",
         "one_long": True},
        # Four beams of one answer: the smallest call, a launch and the host's time.
        {"name": "fork_f16_4of4x600_8x128", "op": "fork", "rows": 4, "sequences": 4, "context": 600, "context_to": 620, "page": 16, "block": 16, "bits": 16,
         "kv_heads": 8, "dim": 128, "dtype": "f16", "order": "head"},
        # 256 rows from 64 parents, large pages in 8 bits.
        {"name": "fork_bf16_256of64x100..5000_8x128_8", "op": "fork", "rows": 256, "sequences": 64, "context": 100, "context_to": 5000, "page": 256,
         "block": 32, "bits": 8, "kv_heads": 8, "dim": 128, "dtype": "bf16", "order": "token"},
        # A small cache, half full.
        {"name": "compact_f16_8x200..900_4x64_8", "op": "compact", "sequences": 8, "context": 200, "context_to": 900, "page": 16, "block": 16, "bits": 8,
         "free": 0.5, "kv_heads": 4, "dim": 64, "dtype": "f16", "order": "head"},
        # The cache of 64 sequences after others have gone.
        {"name": "compact_bf16_64x100..16384_8x128", "op": "compact", "sequences": 64, "context": 100, "context_to": 16384, "page": 16, "block": 16,
         "bits": 16, "free": 0.4, "kv_heads": 8, "dim": 128, "dtype": "bf16", "order": "head"},
    ]


def _log(rng, lo, hi):
    """A whole number of [lo, hi], even over the logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    while True:
        case = _draw(rng)
        w = work(case)
        if case["op"] in ("attend", "window"):
            new, length = _tokens(case)
            seen = max(_seen(case, n, L) for n, L in zip(new, length))
            if w["flops"] <= 2.7e11 and w["bytes"] <= 4e8 and case["sequences"] * seen * case["kv_heads"] <= 8.4e6:
                return case
        elif w["bytes"] <= (1.2e8 if case["op"] == "append" else 1e9) and _pool(case) * case["page"] * case["kv_heads"] * case["dim"] <= 3.4e8:
            return case


def _draw(rng):
    op = rng.choice(("append", "attend", "attend", "window", "window", "fork", "compact"))
    kv_heads, group = rng.choice((1, 2, 4, 8, 8, 12, 32)), rng.choice((1, 1, 2, 4, 4, 5, 8, 16))
    while kv_heads * group > 64:
        group = rng.choice((1, 1, 2, 4, 4, 5, 8, 16))
    page = rng.choice((8, 16, 16, 32, 64, 64, 128, 256))
    block = page // rng.choice((1, 1, 2, 4))
    case = {"op": op, "kv_heads": kv_heads, "dim": rng.choice((64, 128, 128, 128, 80, 96, 256)), "dtype": rng.choice(("f16", "bf16")), "page": page,
            "block": min(block, 64), "order": rng.choice(("head", "token"))}
    if op in ("fork", "compact"):
        hi = _log(rng, 2, 8000)
        case |= {"sequences": _log(rng, 1, 128), "bits": rng.choice((8, 16)), "context": _log(rng, 1, hi), "context_to": hi}
        return {**case, "rows": _log(rng, 1, 256)} if op == "fork" else {**case, "free": rng.choice((0.1, 0.3, 0.6, 0.9))}
    case["q_heads"] = kv_heads * group
    decode = rng.random() < 0.5
    case["sequences"] = _log(rng, 1, 128) if decode else _log(rng, 1, 32)
    hi = 1 if decode else _log(rng, 2, 4096)
    case["new"], case["new_to"] = 1 if decode else _log(rng, 1, hi), hi
    if op == "append":
        hi = _log(rng, 1, 2000)
        return {**case, "rotary": case["dim"] // rng.choice((1, 1, 1, 2)), "pairs": rng.choice(("adjacent", "halves")), "norm": rng.random() < 0.5,
                "context": _log(rng, 1, hi), "context_to": hi}
    hi = _log(rng, 1, 16384 if op == "attend" else 60000)
    case |= {"context": _log(rng, 1, hi), "context_to": hi, "bits": 8 if op == "attend" else rng.choice((8, 16))}
    return case if op == "attend" else {**case, "window": _log(rng, 1, 8192), "sinks": rng.choice((0, 1, 4, 4, 16, 100))}


def _spread(lo, hi, n):
    """n whole numbers from lo to hi, even over the logarithm, in no order; both ends are among them where n allows."""
    if lo == hi:
        return [lo] * n
    steps = [hi if n == 1 else round(math.exp(math.log(lo) + (math.log(hi) - math.log(lo)) * i / (n - 1))) for i in range(n)]
    step = next(s for s in range(n * 5 // 8 or 1, n * 2 + 2) if math.gcd(s, n) == 1)
    return [steps[i * step % n] for i in range(n)]


def _tokens(case):
    """New tokens and whole length of each sequence."""
    n = case["sequences"]
    if "new" not in case:
        return [1] * n, _spread(case["context"], case["context_to"], n)
    new = [case["new_to"]] + [case["new"]] * (n - 1) if case.get("one_long") else _spread(case["new"], case["new_to"], n)
    return new, [a + b for a, b in zip(_spread(case["context"], case["context_to"], n), new)]


def _seen(case, new, length):
    """Keys of a sequence that any of its new tokens sees."""
    return min(length, case["sinks"] + case["window"] + new - 1) if case["op"] == "window" else length


def _held(case, new, length):
    """Columns of a sequence's row of the table that are pages."""
    first = max(0, length - new + 1 - case["window"]) if case["op"] == "window" else 0
    return [c for c in range(-(-length // case["page"])) if c * case["page"] < case.get("sinks", 0) or (c + 1) * case["page"] > first]


def _pool(case):
    used = sum(len(_held(case, n, L)) for n, L in zip(*_tokens(case)))
    return used + (case["rows"] if case["op"] == "fork" else 0) if case["op"] != "compact" else max(used + 1, round(used / (1 - case["free"])))


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = _DTYPES[case["dtype"]]
    D, Hkv, size = case["dim"], case["kv_heads"], case["page"]

    def normal(*shape, dtype=dt, std=1.0, mean=0.0):
        return torch.randn(*shape, generator=g, device="cuda").mul_(std).add_(mean).to(dtype)

    def whole(values):
        return torch.tensor(values, device="cuda", dtype=torch.int32)

    new, length = _tokens(case)
    s = {"op": case["op"], "dtype": case["dtype"], "new": new, "length": length, "window": case.get("window"), "sinks": case.get("sinks", 0)}
    s["lengths"] = whole(length)
    # every sequence's pages in random order over the pool
    held = [_held(case, n, L) for n, L in zip(new, length)]
    pool = _pool(case)
    order = torch.randperm(pool, generator=g, device="cuda", dtype=torch.int32)
    at = [(b, c) for b, cs in enumerate(held) for c in cs]
    table = torch.full((len(new), max(-(-n // size) for n in length) + (case["op"] == "fork")), -1, device="cuda", dtype=torch.int32)
    rows, columns = torch.tensor(at, device="cuda").unbind(1)
    table[rows, columns] = order[:len(at)]
    s["page_table"] = table
    shape = (pool, Hkv, size, D) if case["order"] == "head" else (pool, size, Hkv, D)
    bits = case.get("bits", 8)
    for name in ("k", "v"):
        if bits == 16:
            pages = normal(*shape)
            s[name + "_pages"], s[name + "_scales"] = pages if case["order"] == "head" else pages.transpose(1, 2), None
        else:
            # every block's values of a size of its own
            x = normal(pool, Hkv, size // case["block"], case["block"], D, dtype=torch.float32)
            x *= torch.exp(0.5 * normal(pool, Hkv, size // case["block"], 1, 1, dtype=torch.float32))
            e = _exponent(x.abs().amax((3, 4)), case["dtype"])
            codes = (x * torch.exp2(-e.float())[..., None, None]).view(pool, Hkv, size, D)
            if case["order"] == "token":
                codes = codes.transpose(1, 2).contiguous().to(torch.float8_e4m3fn).transpose(1, 2)
            s[name + "_pages"] = codes.to(torch.float8_e4m3fn)
            s[name + "_scales"] = (e + 127).to(torch.uint8)
            del x, codes
    if case["op"] == "fork":
        s["parents"] = torch.randint(0, len(new), (case["rows"],), generator=g, device="cuda", dtype=torch.int32)
        s["pages"] = order[len(at):].clone()
    if case["op"] in ("fork", "compact"):
        return s
    T, Hq = sum(new), case["q_heads"]
    s["starts"] = None if max(new) == 1 else whole([sum(new[:i]) for i in range(len(new) + 1)])
    qkv = normal(T, (Hq + 2 * Hkv) * D)
    # slices of one projection's result
    s["q"], s["k"], s["v"] = (t.unflatten(1, (-1, D)) for t in qkv.split((Hq * D, Hkv * D, Hkv * D), dim=1))
    if case["op"] != "append":
        s["q"] = s["q"].contiguous()                # it comes rotated from the step before
        del s["k"], s["v"]
        return s
    s["block"], s["pairs"] = case["block"], case["pairs"]
    s["inv_freq"] = _THETA ** (-torch.arange(0, case["rotary"], 2, device="cuda", dtype=torch.float64) / case["rotary"])
    s["q_weight"], s["k_weight"] = (normal(D, std=0.1, mean=1.0), normal(D, std=0.1, mean=1.0)) if case["norm"] else (None, None)
    return s


def run(s):
    if own:
        return _own(s)
    return {"append": _append, "attend": _attend, "window": _attend, "fork": _fork, "compact": _compact}[s["op"]](s)


def _cache(s):
    out = {"k_pages": s["k_pages"], "v_pages": s["v_pages"]}
    return out if s["k_scales"] is None else {**out, "k_scales": s["k_scales"], "v_scales": s["v_scales"]}


def _own(s):
    import hexmi
    k_pages, v_pages, scales = s["k_pages"], s["v_pages"], {"k_scales": s["k_scales"], "v_scales": s["v_scales"]}
    if s["op"] == "append":
        q = hexmi.paged_append(s["k"], s["v"], k_pages, v_pages, s["page_table"], s["lengths"], s["starts"], k_weight=s["k_weight"],
                               inv_freq=s["inv_freq"], eps=_EPS, pairs=s["pairs"], q=s["q"], q_weight=s["q_weight"], **scales)
        return {"q": q, **_cache(s)}
    if s["op"] == "fork":
        table, lengths = hexmi.paged_fork(k_pages, v_pages, s["page_table"], s["lengths"], s["parents"], s["pages"], **scales)
        return {"page_table": table, "lengths": lengths, **_cache(s)}
    if s["op"] == "compact":
        table, count = hexmi.paged_compact(k_pages, v_pages, s["page_table"], s["lengths"], **scales)
        return {"page_table": table, "count": count, **_cache(s)}
    return hexmi.paged_attention(s["q"], k_pages, v_pages, s["page_table"], s["lengths"], s["starts"], window=s["window"], sinks=s["sinks"], **scales)


def _exponent(most, dtype):
    """The least e with most <= 448 * 2^e."""
    m, x = torch.frexp(most)
    return (x - 9 + (m > 0.875)).clamp(_LEAST[dtype], _MOST[dtype]).masked_fill(most == 0, _LEAST[dtype])


def _coded(y, e, dtype):
    """y / 2^e where e4m3 has it, not yet rounded; the largest scale's codes end where their values are still numbers of the type."""
    e = e.double() if y.dtype == torch.float64 else e.float()
    return torch.where(e == _MOST[dtype], (y * torch.exp2(-e)).clamp(-240, 240), (y * torch.exp2(-e)).clamp(-448, 448))


def _turned(x, weight, inv_freq, positions, pairs):
    """The rows of [tokens, heads, D], normed and rotated, in 32 bits and angles in 64."""
    y = x.float()
    if weight is not None:
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + _EPS) * weight.float()
    angle = (positions.double()[:, None] * inv_freq)[:, None, :]
    cos, sin = angle.cos().float(), angle.sin().float()
    R = 2 * inv_freq.numel()
    turned, rest = y[..., :R], y[..., R:]
    if pairs == "adjacent":
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = turned[..., :R // 2], turned[..., R // 2:]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, rest), -1)


def _where(s):
    """Sequence and position of each new token."""
    B, T = s["lengths"].numel(), s["q"].shape[0]
    starts = s["starts"].long() if s["starts"] is not None else torch.arange(B + 1, device="cuda")
    row = torch.arange(T, device="cuda")
    seq = torch.searchsorted(starts[1:].contiguous(), row, right=True)
    return seq, s["lengths"].long()[seq] - starts[seq + 1] + row, s["lengths"].long()[seq] - starts[seq + 1] + starts[seq]


def _append(s):
    seq, position, first = _where(s)
    size, block = s["k_pages"].shape[2], s["block"]
    page, slot = s["page_table"].long()[seq, position // size], position % size
    for name, y in (("k", _turned(s["k"], s["k_weight"], s["inv_freq"], position, s["pairs"])), ("v", s["v"].float())):
        codes, scales = s[name + "_pages"].view(torch.uint8), s[name + "_scales"]
        # the blocks that get rows, and the largest value of each block's new rows and head
        number, of_row = torch.unique(page * (size // block) + slot // block, return_inverse=True)
        most = torch.zeros(number.numel(), y.shape[1], device="cuda")
        most = most.scatter_reduce_(0, of_row[:, None].expand(-1, y.shape[1]), y.abs().amax(-1), "amax")
        e = _exponent(most, s["dtype"])
        at_page, at_block = number // (size // block), number % (size // block)
        # older rows of a block: those before the first new position
        start = torch.full_like(number, -1)
        start[of_row] = (first - (position - slot % block)).clamp(min=0)                # per block: slots of it that are older
        before = scales[at_page, :, at_block].int() - 127
        e = torch.where(start[:, None] > 0, torch.maximum(e, before), e)
        slots = at_block[:, None] * block + torch.arange(block, device="cuda")
        old = codes[at_page[:, None], :, slots].view(torch.float8_e4m3fn).float()        # [blocks, block, heads, D]
        again = (old * torch.exp2((before - e).float())[:, None, :, None]).to(torch.float8_e4m3fn).view(torch.uint8)
        older = (torch.arange(block, device="cuda") < start[:, None])[:, :, None, None]
        codes[at_page[:, None], :, slots] = torch.where(older, again, codes[at_page[:, None], :, slots])
        codes[page, :, slot] = _coded(y, e[of_row][..., None], s["dtype"]).to(torch.float8_e4m3fn).view(torch.uint8)
        scales[at_page, :, at_block] = (e + 127).to(torch.uint8)
    q = _turned(s["q"], s["q_weight"], s["inv_freq"], position, s["pairs"]).to(s["q"].dtype)
    return {"q": q, **_cache(s)}


def _rows(s, name, b, positions, dtype=torch.float32):
    """Keys or values [..., heads, D] of sequences b at positions."""
    pages, scales = s[name + "_pages"], s[name + "_scales"]
    size = pages.shape[2]
    page, slot = s["page_table"].long()[b, positions // size].clamp_(min=0), positions % size
    if scales is None:
        return pages[page, :, slot].to(dtype)
    e = scales[page, :, slot // (size // scales.shape[2])].to(dtype) - 127
    return pages.view(torch.uint8)[page, :, slot].view(torch.float8_e4m3fn).to(dtype) * torch.exp2(e)[..., None]


def _softmax_sums(scores, hidden, v):
    scores = scores.masked_fill_(hidden, -math.inf)
    scores = scores.sub_(scores.amax(-1, keepdim=True)).exp_()
    return torch.matmul(scores, v) / scores.sum(-1, keepdim=True)


def _attend(s):
    q = s["q"].float() / math.sqrt(s["q"].shape[2])
    T, Hq, D = q.shape
    Hkv, window, sinks = s["k_pages"].shape[1], s["window"], s["sinks"]
    if s["starts"] is None:                         # one token each: every sequence's keys side by side
        length, n = s["lengths"].long()[:, None], max(s["length"])
        if window is not None:
            n = min(n, sinks + window)
        at = torch.arange(n, device="cuda").expand(T, n)
        if window is not None:
            at = torch.where(at < sinks, at, at + (length - sinks - window).clamp(min=0))
        hidden, at = at >= length, torch.minimum(at, length - 1)
        b = torch.arange(T, device="cuda")[:, None]
        k, v = (_rows(s, name, b, at).transpose(1, 2) for name in ("k", "v"))            # [B, Hkv, n, D]
        scores = torch.matmul(q.unflatten(1, (Hkv, -1)), k.transpose(2, 3))
        return _softmax_sums(scores, hidden[:, None, None, :], v).flatten(1, 2).to(s["q"].dtype)
    out, row = torch.empty_like(s["q"]), 0
    for b, (n, L) in enumerate(zip(s["new"], s["length"])):
        for i in range(0, n, 1024):                 # runs of its tokens, over the keys that any of a run sees
            m = min(1024, n - i)
            p0 = L - n + i
            lo = 0 if window is None else max(0, p0 - window + 1)
            first = min(sinks, lo)
            at = torch.cat((torch.arange(first, device="cuda"), torch.arange(lo, p0 + m, device="cuda")))
            k, v = (_rows(s, name, b, at).transpose(0, 1) for name in ("k", "v"))        # [Hkv, keys, D]
            p = torch.arange(p0, p0 + m, device="cuda")[:, None]
            hidden = at > p
            if window is not None:
                hidden |= (at <= p - window) & (at >= sinks)
            rows = q[row + i:row + i + m].unflatten(1, (Hkv, -1)).permute(1, 2, 0, 3)    # [Hkv, G, m, D]
            scores = torch.matmul(rows.flatten(1, 2), k.transpose(1, 2)).unflatten(1, (-1, m))
            sums = _softmax_sums(scores.flatten(1, 2), hidden.repeat(Hq // Hkv, 1), v).unflatten(1, (-1, m))
            out[row + i:row + i + m] = sums.permute(2, 0, 1, 3).flatten(1, 2)
        row += n
    return out


def _fork(s):
    size = s["k_pages"].shape[2]
    parents, pages = s["parents"].long(), s["pages"]
    table, lengths = s["page_table"][parents], s["lengths"][parents]
    column, filled = lengths.long() // size, lengths.long() % size
    row = torch.arange(parents.numel(), device="cuda")
    last = table[row, column].long()
    table[row, column] = pages
    row, slot = ((torch.arange(size, device="cuda") < filled[:, None])).nonzero().unbind(1)
    for name in ("k", "v"):
        held, scales = s[name + "_pages"], s[name + "_scales"]
        held = held if scales is None else held.view(torch.uint8)
        held[pages.long()[row], :, slot] = held[last[row], :, slot]
        if scales is not None:
            block = size // scales.shape[2]
            r, j = (torch.arange(scales.shape[2], device="cuda") * block < filled[:, None]).nonzero().unbind(1)
            scales[pages.long()[r], :, j] = scales[last[r], :, j]
    return {"page_table": table, "lengths": lengths, **_cache(s)}


def _compact(s):
    pool, _, size, _ = s["k_pages"].shape
    table = s["page_table"].long()
    used = (torch.arange(table.shape[1], device="cuda") * size < s["lengths"][:, None]) & (table >= 0)
    mark = torch.zeros(pool + 1, device="cuda", dtype=torch.bool)
    mark[torch.where(used, table, pool)] = True
    mark = mark[:pool]
    count = mark.sum()
    front = torch.arange(pool, device="cuda") < count
    source, target = (mark & ~front).nonzero().flatten(), (~mark & front).nonzero().flatten()
    name_of = torch.arange(pool, device="cuda")
    name_of[source] = target
    for name in ("k", "v"):
        held, scales = s[name + "_pages"], s[name + "_scales"]
        held = held if scales is None else held.view(torch.uint8)
        held[target] = held[source]
        if scales is not None:
            scales[target] = scales[source]
    return {"page_table": torch.where(used, name_of[table.clamp(min=0)], -1).int(), "count": count.int().view(1), **_cache(s)}


def exact(case, seed):
    """run()'s outputs in 64 bits, from the definitions; copies have no such value."""
    if case["op"] in ("fork", "compact"):
        return None
    s = prepare(case, seed)
    new, length = _tokens(case)
    Hkv, size = case["kv_heads"], case["page"]
    at = torch.cat([torch.arange(L - n, L, device="cuda") for n, L in zip(new, length)])
    if case["op"] == "append":
        k, done = _exact_rows(s["k"], s["k_weight"], s["inv_freq"], at, case), 0
        out = {"q": _exact_rows(s["q"], s["q_weight"], s["inv_freq"], at, case)}
        for name, x in (("k", k), ("v", s["v"].double())):
            pages, scales, done = s[name + "_pages"].double(), s[name + "_scales"].clone(), 0
            for b, (n, L) in enumerate(zip(new, length)):
                for first in range((L - n) // case["block"] * case["block"], L, case["block"]):         # a block at a time
                    page, j = s["page_table"][b, first // size].long(), first % size // case["block"]
                    old, end = max(0, L - n - first), min(L, first + case["block"])
                    rows = x[done + first + old - (L - n):done + end - (L - n)]
                    _, up = torch.frexp(rows.abs().amax((0, 2)) / 448)
                    up = up - (torch.ldexp(torch.ones_like(up, dtype=torch.float64), up - 1) * 448 == rows.abs().amax((0, 2))).int()
                    e = up.clamp(_LEAST[case["dtype"]], _MOST[case["dtype"]])
                    was = scales[page, :, j].int() - 127
                    if old:
                        e = torch.maximum(e, was)
                        pages[page, :, first % size:first % size + old] *= torch.exp2((was - e).double())[:, None, None]
                    pages[page, :, first % size + old:first % size + end - first] = _coded(rows, e[:, None], case["dtype"]).transpose(0, 1)
                    scales[page, :, j] = (e + 127).to(torch.uint8)
                done += n
            out[name + "_pages"], out[name + "_scales"] = pages, scales
        return {n: out[n] for n in ("q", "k_pages", "v_pages", "k_scales", "v_scales")}
    if work(case)["flops"] > 6e11:
        return None
    G, D, window, sinks = case["q_heads"] // Hkv, case["dim"], case.get("window", max(length)), case.get("sinks", 0)
    out, done = torch.empty(*s["q"].shape, device="cuda", dtype=torch.float64), 0
    for b, (n, L) in enumerate(zip(new, length)):
        for i in range(0, n, 4096):
            p = torch.arange(L - n + i, min(L - n + i + 4096, L), device="cuda")[:, None]
            keys = torch.arange(L, device="cuda")
            keys = keys[(keys < sinks) | (keys > L - n + i - window)]
            seen = (keys <= p) & ((keys > p - window) | (keys < sinks))
            k, v = (_rows(s, name, b, keys, torch.float64) for name in ("k", "v"))
            for j in range(Hkv * G):
                x = s["q"][done + i:done + i + p.numel(), j].double() @ k[:, j // G].T / math.sqrt(D)
                out[done + i:done + i + p.numel(), j] = torch.softmax(x.masked_fill(~seen, -math.inf), dim=1) @ v[:, j // G]
        done += n
    return out


def _exact_rows(x, weight, inv_freq, positions, case):
    x = x.double()
    if weight is not None:
        x = x / (x.square().mean(-1, keepdim=True) + _EPS).sqrt() * weight.double()
    turn = torch.polar(torch.ones((), device="cuda", dtype=torch.float64), positions.double()[:, None] * inv_freq)[:, None]
    R = case["rotary"]
    out = x.clone()
    if case["pairs"] == "adjacent":
        out[..., :R] = torch.view_as_real(torch.complex(x[..., 0:R:2], x[..., 1:R:2]) * turn).flatten(-2)
    else:
        z = torch.complex(x[..., :R // 2], x[..., R // 2:R]) * turn
        out[..., :R // 2], out[..., R // 2:R] = z.real, z.imag
    return out


def work(case):
    D, Hkv, page = case["dim"], case["kv_heads"], case["page"]
    bits = case.get("bits", 8)
    a_key = 2 * Hkv * (D * bits // 8 + (1 / case["block"] if bits == 8 else 0))          # a key and its value, all heads
    new, length = _tokens(case)
    T, B = sum(new), len(new)
    if case["op"] == "fork":
        filled, columns = sum(L % page for L in length) / B, max(length) // page + 2
        return {"bytes": int(2 * case["rows"] * (filled * a_key + 4 * columns + 8)), "flops": 0}
    if case["op"] == "compact":
        used, pool = sum(len(_held(case, n, L)) for n, L in zip(new, length)), _pool(case)
        return {"bytes": int(2 * (used * (pool - used) / pool * page * a_key + 4 * used)), "flops": 0}
    Hq = case["q_heads"]
    if case["op"] == "append":
        return {"bytes": int(T * (4 * Hq + 4 * Hkv) * D + T * a_key + 8 * B + 4 * case["rotary"] + (4 * D if case["norm"] else 0)),
                "flops": T * (Hq + Hkv) * D * (7 if case["norm"] else 3)}
    keys = sum(_seen(case, n, L) for n, L in zip(new, length))
    view = case["window"] + case["sinks"] if case["op"] == "window" else max(length)
    pairs = 0
    for n, L in zip(new, length):                   # tokens at positions L - n .. L - 1 see position + 1 keys, at most `view`
        few = max(0, min(L, view) - (L - n))        # of them see all
        pairs += few * (L - n) + few * (few + 1) // 2 + (n - few) * view
    return {"bytes": int(keys * a_key + 4 * T * Hq * D + 4 * (B + keys // page)), "flops": 4 * pairs * Hq * D}

"""The steps between a decoder layer's projections and its output product, over a paged cache of keys and values, as measurable cases.

  heads   norms of the query and key heads and their rotation by position, in one pass, read where the projection left them
  append  keys (normed, rotated) and values of new tokens into the pages of their sequences; the queries beside them
  attend  attention of the new tokens over the pages: one token a sequence (decode) or runs of several (prompts, pieces of
          them), with or without a long prefix that all sequences share

A case is a dict of plain values. Lengths are spread evenly over their logarithm between the two ends a case gives, pages are dealt in
random order. With `own` false, run() is the mathematics in elementary torch operations; with `own` true, the package's operators.
"""
import math
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.getcwd(), "hexagon-mlir_amd"))

own = False

_DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
_EPS, _THETA = 1e-5, 10000.0


def listed():
    return [
        # One new token of each of four sequences: the smallest call, a launch and the host's time.
        {"name": "heads_bf16_4x32+8x128", "op": "heads", "tokens": 4, "q_heads": 32, "kv_heads": 8, "dim": 128, "rotary": 128,
         "dtype": "bf16", "pairs": "halves", "norm": True, "far": 8192},
        # A long prompt's queries and keys.
        {"name": "heads_bf16_8192x32+8x128", "op": "heads", "tokens": 8192, "q_heads": 32, "kv_heads": 8, "dim": 128, "rotary": 128,
         "dtype": "bf16", "pairs": "halves", "norm": True, "far": 131072},
        # fp32, adjacent pairs, a part of a head's columns rotated, a ragged number of tokens.
        {"name": "heads_f32_1021x12+12x64", "op": "heads", "tokens": 1021, "q_heads": 12, "kv_heads": 12, "dim": 64, "rotary": 32,
         "dtype": "f32", "pairs": "adjacent", "norm": False, "far": 4096},
        # A decode step of 64 sequences: one key and value of each into its last page, its query rotated beside them.
        {"name": "append_f16_64x1_32+8x128", "op": "append", "sequences": 64, "new": 1, "new_to": 1, "context": 30, "context_to": 1000, "page": 16,
         "q_heads": 32, "kv_heads": 8, "dim": 128, "rotary": 128, "dtype": "f16", "pairs": "adjacent", "norm": False, "order": "head"},
        # Prompts of a batch, ragged, with norms of the heads, into pages that hold all heads of a token side by side.
        {"name": "append_bf16_6x_2000_32+8x128", "op": "append", "sequences": 6, "new": 700, "new_to": 2000, "context": 1, "context_to": 500, "page": 64,
         "q_heads": 32, "kv_heads": 8, "dim": 128, "rotary": 128, "dtype": "bf16", "pairs": "halves", "norm": True, "order": "token"},
        # Decode of one sequence: latency.
        {"name": "decode_f16_1x1000_32/8x128", "op": "attend", "sequences": 1, "new": 1, "new_to": 1, "context": 999, "context_to": 999, "shared": 0,
         "page": 16, "q_heads": 32, "kv_heads": 8, "dim": 128, "dtype": "f16", "order": "head"},
        # Decode of 16 sequences with 2048 tokens behind them, a key head to each query head.
        {"name": "decode_f16_16x2048_32x128", "op": "attend", "sequences": 16, "new": 1, "new_to": 1, "context": 2047, "context_to": 2047, "shared": 0,
         "page": 64, "q_heads": 32, "kv_heads": 32, "dim": 128, "dtype": "f16", "order": "head"},
        # Decode of 64 sequences of very different lengths, shared key heads.
        {"name": "decode_bf16_64x100..16384_32/8", "op": "attend", "sequences": 64, "new": 1, "new_to": 1, "context": 99, "context_to": 16383, "shared": 0,
         "page": 16, "q_heads": 32, "kv_heads": 8, "dim": 128, "dtype": "bf16", "order": "token"},
        # The next 509 tokens of one prompt behind 2046 earlier ones, beside 15 sequences that decode.
        {"name": "mixed_f16_16x1..509_32/8x128", "op": "attend", "sequences": 16, "new": 1, "new_to": 509, "context": 400, "context_to": 2046, "shared": 0,
         "page": 16, "q_heads": 32, "kv_heads": 8, "dim": 128, "dtype": "f16", "order": "head", "one_long": True},
        # Four whole prompts of about 4096 tokens.
        {"name": "prompt_bf16_4x4096_32/8x128", "op": "attend", "sequences": 4, "new": 4033, "new_to": 4096, "context": 0, "context_to": 0, "shared": 0,
         "page": 64, "q_heads": 32, "kv_heads": 8, "dim": 128, "dtype": "bf16", "order": "head"},
        # Decode of 32 sequences behind one system prompt of 8192 tokens.
        {"name": "shared_bf16_32x8192+_32/8x128", "op": "attend", "sequences": 32, "new": 1, "new_to": 1, "context": 60, "context_to": 700, "shared": 8192,
         "page": 64, "q_heads": 32, "kv_heads": 8, "dim": 128, "dtype": "bf16", "order": "head"},
        # Short questions of eight users behind one document of 4000 tokens.
        {"name": "shared_f16_8x4000+30..90_16/4x64", "op": "attend", "sequences": 8, "new": 30, "new_to": 90, "context": 1, "context_to": 1, "shared": 4000,
         "page": 16, "q_heads": 16, "kv_heads": 4, "dim": 64, "dtype": "f16", "order": "token"},
    ]


def _log(rng, lo, hi):
    """A whole number of [lo, hi], even over the logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    while True:
        case = _draw(rng)
        w = work(case)
        if case["op"] != "attend":
            if w["bytes"] <= 1.7e8:
                return case
            continue
        new, length = _tokens(case)
        scores = case["sequences"] * max(new) * case["q_heads"] * max(length)
        if w["flops"] <= 5.4e11 and w["bytes"] <= 8e8 and scores <= 2.2e9 and case["sequences"] * max(length) * case["kv_heads"] <= 8.4e6:
            return case


def _draw(rng):
    op = rng.choice(("heads", "append", "attend", "attend", "attend"))
    kv_heads, group = rng.choice((1, 2, 4, 8, 8, 12, 32)), rng.choice((1, 1, 2, 4, 4, 5, 8, 16))
    while kv_heads * group > 64:
        group = rng.choice((1, 1, 2, 4, 4, 5, 8, 16))
    case = {"op": op, "q_heads": kv_heads * group, "kv_heads": kv_heads, "dim": rng.choice((64, 128, 128, 128, 80, 96, 256))}
    rotation = {"rotary": case["dim"] // rng.choice((1, 1, 1, 2)), "pairs": rng.choice(("adjacent", "halves")), "norm": rng.random() < 0.5}
    if op == "heads":
        return {**case, **rotation, "tokens": _log(rng, 1, 16384), "dtype": rng.choice(("f16", "bf16", "f32")), "far": _log(rng, 512, 1 << 20)}
    case |= {"dtype": rng.choice(("f16", "bf16")), "page": rng.choice((8, 16, 16, 32, 64, 64, 128, 256)), "order": rng.choice(("head", "token"))}
    decode = rng.random() < 0.5
    case["sequences"] = _log(rng, 1, 128) if decode else _log(rng, 1, 32)
    hi = 1 if decode else _log(rng, 2, 4096)
    case["new"], case["new_to"] = 1 if decode else _log(rng, 1, hi), hi
    if op == "append":
        hi = _log(rng, 1, 2000)
        return {**case, **rotation, "context": _log(rng, 1, hi), "context_to": hi}
    case["shared"] = _log(rng, 64, 16384) // case["page"] * case["page"] if rng.random() < 0.35 else 0
    hi = _log(rng, 1, 1000 if case["shared"] else 16384)
    return {**case, "context": _log(rng, 1, hi), "context_to": hi}


def _spread(lo, hi, n):
    """n whole numbers from lo to hi, even over the logarithm, in no order; both ends are among them where n allows."""
    if lo == hi:
        return [lo] * n
    steps = [hi if n == 1 else round(math.exp(math.log(lo) + (math.log(hi) - math.log(lo)) * i / (n - 1))) for i in range(n)]
    step = next(s for s in range(n * 5 // 8 or 1, n * 2 + 2) if math.gcd(s, n) == 1)
    return [steps[i * step % n] for i in range(n)]


def _tokens(case):
    """New tokens and whole length of each sequence, the shared prefix included."""
    n = case["sequences"]
    new = [case["new_to"]] + [case["new"]] * (n - 1) if case.get("one_long") else _spread(case["new"], case["new_to"], n)
    return new, [case.get("shared", 0) + a + b for a, b in zip(_spread(case["context"], case["context_to"], n), new)]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = _DTYPES[case["dtype"]]
    D, Hq, Hkv = case["dim"], case["q_heads"], case["kv_heads"]

    def normal(*shape, dtype=dt, std=1.0, mean=0.0):
        return torch.randn(*shape, generator=g, device="cuda").mul_(std).add_(mean).to(dtype)

    def whole(values):
        return torch.tensor(values, device="cuda", dtype=torch.int32)

    s = {"op": case["op"]}
    if case["op"] != "attend":
        s["pairs"] = case["pairs"]
        s["inv_freq"] = _THETA ** (-torch.arange(0, case["rotary"], 2, device="cuda", dtype=torch.float64) / case["rotary"])
        s["q_weight"], s["k_weight"] = (normal(D, std=0.1, mean=1.0), normal(D, std=0.1, mean=1.0)) if case["norm"] else (None, None)
    if case["op"] == "heads":
        T = case["tokens"]
        qkv = normal(T, (Hq + 2 * Hkv) * D)
        s["positions"] = torch.randint(0, case["far"], (T,), generator=g, device="cuda", dtype=torch.int32)
    else:
        new, length = _tokens(case)
        T, B, size = sum(new), len(new), case["page"]
        s["longest"], s["most"] = max(length), max(new)
        s["lengths"] = whole(length)
        s["starts"] = None if s["most"] == 1 else whole([sum(new[:i]) for i in range(B + 1)])
        # every sequence's pages, those of the shared prefix the same for all; the others in random order over the pool
        first = case.get("shared", 0) // size
        rest = [-(-n // size) - first for n in length]
        pool = first + sum(rest)
        order = torch.randperm(pool, generator=g, device="cuda", dtype=torch.int32)
        behind = torch.tensor([first + sum(rest[:i]) for i in range(B)], device="cuda")
        column = torch.arange(first + max(rest), device="cuda")
        place = torch.where(column < first, column, behind[:, None] + column - first).clamp_(max=pool - 1)
        s["page_table"] = order[place].contiguous()
        s["shared_pages"] = order[:first].clone() if first else None
        shape = (pool, Hkv, size, D) if case["order"] == "head" else (pool, size, Hkv, D)
        s["k_pages"], s["v_pages"] = (t if case["order"] == "head" else t.transpose(1, 2) for t in (normal(*shape), normal(*shape)))
        qkv = normal(T, (Hq + 2 * Hkv) * D)
    # slices of one projection's result
    s["q"], s["k"], s["v"] = (t.unflatten(1, (-1, D)) for t in qkv.split((Hq * D, Hkv * D, Hkv * D), dim=1))
    if case["op"] == "attend":
        s["q"] = s["q"].contiguous()                # it comes rotated from the step before
        del s["k"], s["v"]
    return s


def run(s):
    if own:
        return _own(s)
    return {"heads": _heads, "append": _append, "attend": _attend}[s["op"]](s)


def _own(s):
    import hexmi
    if s["op"] == "heads":
        q, k = hexmi.qk_norm_rope(s["q"], s["k"], s["q_weight"], s["k_weight"], s["inv_freq"], s["positions"], eps=_EPS, pairs=s["pairs"])
        return {"q": q, "k": k}
    if s["op"] == "append":
        q = hexmi.paged_append(s["k"], s["v"], s["k_pages"], s["v_pages"], s["page_table"], s["lengths"], s["starts"], k_weight=s["k_weight"],
                               inv_freq=s["inv_freq"], eps=_EPS, pairs=s["pairs"], q=s["q"], q_weight=s["q_weight"])
        return {"q": q, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
    return hexmi.paged_attention(s["q"], s["k_pages"], s["v_pages"], s["page_table"], s["lengths"], s["starts"], shared_pages=s["shared_pages"])


def _turned(x, weight, inv_freq, positions, pairs):
    """The rows of [tokens, heads, D], normed and rotated, in 32 bits and angles in 64, rounded once."""
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
    return torch.cat((turned, rest), -1).to(x.dtype)


def _heads(s):
    return {n: _turned(s[n], s[n + "_weight"], s["inv_freq"], s["positions"], s["pairs"]) for n in ("q", "k")}


def _where(s):
    """Sequence and position of each new token."""
    B, T = s["lengths"].numel(), s["q"].shape[0]
    starts = s["starts"].long() if s["starts"] is not None else torch.arange(B + 1, device="cuda")
    row = torch.arange(T, device="cuda")
    seq = torch.searchsorted(starts[1:].contiguous(), row, right=True)
    return seq, s["lengths"].long()[seq] - starts[seq + 1] + row


def _append(s):
    seq, position = _where(s)
    size = s["k_pages"].shape[2]
    page, slot = s["page_table"].long()[seq, position // size], position % size
    s["k_pages"][page, :, slot] = _turned(s["k"], s["k_weight"], s["inv_freq"], position, s["pairs"])
    s["v_pages"][page, :, slot] = s["v"]
    return {"q": _turned(s["q"], s["q_weight"], s["inv_freq"], position, s["pairs"]), "k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _attend(s):
    """Every sequence's pages side by side, its queries padded to the most of any; masked scores, softmax, sums, in 32 bits."""
    q, B = s["q"], s["lengths"].numel()
    T, Hq, D = q.shape
    _, Hkv, size, _ = s["k_pages"].shape
    table = s["page_table"].long()[:, :-(-s["longest"] // size)]
    k, v = (p[table].transpose(1, 2).flatten(2, 3).float() for p in (s["k_pages"], s["v_pages"]))              # [B, Hkv, L, D]
    seq, position = _where(s)
    row = torch.arange(T, device="cuda")
    first = s["starts"].long()[seq] if s["starts"] is not None else row
    queries = torch.zeros(B, s["most"], Hq, D, device="cuda")
    queries[seq, row - first] = q.float() / math.sqrt(D)
    last = torch.zeros(B, s["most"], device="cuda", dtype=torch.long)
    last[seq, row - first] = position
    queries = queries.unflatten(2, (Hkv, Hq // Hkv)).permute(0, 2, 1, 3, 4).flatten(2, 3)                      # [B, Hkv, most * G, D]
    scores = torch.matmul(queries, k.transpose(2, 3)).unflatten(2, (s["most"], Hq // Hkv))
    after = torch.arange(k.shape[2], device="cuda") > last[:, None, :, None, None]
    scores = scores.masked_fill_(after, -math.inf)
    scores = scores.sub_(scores.amax(-1, keepdim=True)).exp_()
    total = scores.sum(-1, keepdim=True)
    out = torch.matmul(scores.flatten(2, 3), v).unflatten(2, (s["most"], Hq // Hkv)) / total                   # [B, Hkv, most, G, D]
    return out[seq, :, row - first].flatten(1, 2).to(q.dtype)


def exact(case, seed):
    """run()'s outputs in 64 bits, from the definitions."""
    s = prepare(case, seed)
    if case["op"] == "heads":
        return {n: _exact_rows(s[n], s[n + "_weight"], s["inv_freq"], s["positions"], case) for n in ("q", "k")}
    new, length = _tokens(case)
    at = torch.cat([torch.arange(L - n, L, device="cuda") for n, L in zip(new, length)])
    if case["op"] == "append":
        k = _exact_rows(s["k"], s["k_weight"], s["inv_freq"], at, case)
        k_pages, v_pages = s["k_pages"].double(), s["v_pages"].double()
        done = 0
        for b, n in enumerate(new):
            here = at[done:done + n]
            page = s["page_table"][b].long()[torch.div(here, case["page"], rounding_mode="floor")]
            k_pages[page, :, here % case["page"]] = k[done:done + n]
            v_pages[page, :, here % case["page"]] = s["v"][done:done + n].double()
            done += n
        return {"q": _exact_rows(s["q"], s["q_weight"], s["inv_freq"], at, case), "k_pages": k_pages, "v_pages": v_pages}
    G, D = case["q_heads"] // case["kv_heads"], case["dim"]
    out, done = torch.empty(*s["q"].shape, device="cuda", dtype=torch.float64), 0
    for b, (n, L) in enumerate(zip(new, length)):
        pages = s["page_table"][b, :-(-L // case["page"])].long()
        hidden = torch.arange(L, device="cuda")[None, :] > at[done:done + n, None]
        for h in range(case["kv_heads"]):
            k, v = (t[pages, h].reshape(-1, D)[:L].double() for t in (s["k_pages"], s["v_pages"]))
            for j in range(h * G, h * G + G):
                p = torch.softmax((s["q"][done:done + n, j].double() @ k.T / math.sqrt(D)).masked_fill(hidden, -math.inf), dim=1)
                out[done:done + n, j] = p @ v
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
    size = 4 if case["dtype"] == "f32" else 2
    D, Hq, Hkv = case["dim"], case["q_heads"], case["kv_heads"]
    if case["op"] == "heads":
        n = case["tokens"] * (Hq + Hkv) * D
        return {"bytes": 2 * n * size + 4 * case["tokens"] + 4 * case["rotary"] + (2 * D * size if case["norm"] else 0),
                "flops": n * (7 if case["norm"] else 3)}
    new, length = _tokens(case)
    T, B = sum(new), len(new)
    if case["op"] == "append":
        return {"bytes": 2 * T * (Hq + 2 * Hkv) * D * size + 8 * B + 4 * case["rotary"] + (2 * D * size if case["norm"] else 0),
                "flops": T * (Hq + Hkv) * D * (7 if case["norm"] else 3)}
    shared = case["shared"]
    keys = shared + sum(L - shared for L in length)
    pairs = sum(n * (L - n) + n * (n + 1) // 2 for n, L in zip(new, length))
    return {"bytes": 2 * keys * Hkv * D * size + 2 * T * Hq * D * size + 4 * (B + keys // case["page"]), "flops": 4 * pairs * Hq * D}

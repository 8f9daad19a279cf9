"""What a serving step of long contexts adds to the library: tables of a step made on the device from the sequences' lengths,
a cache held in 4 bits (its write, single tokens and prompts attending over it), and log probabilities of a step's tokens.

A case is one call of a public entry point on what a serving program holds there.  ``own`` False: the same results from
elementary torch operations.  Sequences of a batch have unequal lengths, pages lie in no order in the pool.

The 4-bit cache: a row (a token's key or value of one head) is cut into groups of 32 neighbouring values.  A group has a step
s with 4 significant bits and a zero point z of 0..15, each value a code c of 0..15, and stands for (c - z) s.  A page of 64
tokens and one head is 64 rows of key codes (two a byte, the lower one first), 64 rows of a 16-bit word a group (the upper 16
bits of s as a float, whose lowest four are zero, with z in them), and then the same of the values.
"""
from __future__ import annotations

import math
import random

import torch

own = False

PAGE, GROUP = 64, 32
BF, F32, F64, I32 = torch.bfloat16, torch.float32, torch.float64, torch.int32
DEV = "cuda"
EPS = 1e-6
VOCAB = 151936              # the vocabulary of the benchmark's configurations


def listed():
    return [
        # tables of a decode step of 64 running sequences, and of a step that brings 65,536 tokens of 256 prompts
        {"name": "tables-64-single", "kind": "tables", "seqs": 64, "tokens": 64, "before": 4096, "width": 512, "behind": 0},
        {"name": "tables-256-prompts", "kind": "tables", "seqs": 256, "tokens": 65536, "before": 20000, "width": 2048, "behind": 177},
        # a token's keys and values into the 4-bit cache (32 + 2 x 8 heads of 128), and a step of prompts' tokens
        {"name": "write-1", "kind": "write", "seqs": 1, "tokens": 1, "before": 100, "heads": 32, "kv_heads": 8, "dim": 128},
        {"name": "write-5-prompts", "kind": "write", "seqs": 5, "tokens": 4096, "before": 70, "heads": 32, "kv_heads": 8, "dim": 128},
        # single tokens over the 4-bit cache: one sequence at the small model's heads, a batch of 8, a large batch of long ones
        {"name": "decode-1x2048", "kind": "attend", "seqs": 1, "tokens": 1, "before": 2047, "heads": 16, "kv_heads": 8, "dim": 128, "window": 0},
        {"name": "decode-8x4096", "kind": "attend", "seqs": 8, "tokens": 8, "before": 4095, "heads": 32, "kv_heads": 8, "dim": 128, "window": 0},
        {"name": "decode-32x16384", "kind": "attend", "seqs": 32, "tokens": 32, "before": 16383, "heads": 32, "kv_heads": 8, "dim": 128, "window": 0},
        # a few tokens a sequence onto long contexts (a turn's short continuation)
        {"name": "few-4x6", "kind": "attend", "seqs": 4, "tokens": 24, "before": 8192, "heads": 32, "kv_heads": 8, "dim": 128, "window": 0},
        # a whole prompt, and chunks of three prompts behind what they hold already, through a window, heads of 64
        {"name": "prompt-4096", "kind": "attend", "seqs": 1, "tokens": 4096, "before": 0, "heads": 32, "kv_heads": 8, "dim": 128, "window": 0},
        {"name": "chunks-3x900", "kind": "attend", "seqs": 3, "tokens": 2700, "before": 5000, "heads": 16, "kv_heads": 2, "dim": 64, "window": 4096},
        # log probabilities of a decode step's tokens, and of a scored prompt's
        {"name": "logprobs-8", "kind": "logprobs", "rows": 8, "vocab": VOCAB, "top": 5},
        {"name": "logprobs-2048", "kind": "logprobs", "rows": 2048, "vocab": VOCAB, "top": 20},
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    what = rng.choice(["tables", "write", "single", "few", "prompt", "logprobs"])
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 8])
    dim = rng.choice([64, 128])
    if what == "tables":
        seqs = _log(rng, 1, 256)
        tokens = max(seqs, _log(rng, 1, 65536))
        before = _log(rng, 1, 20000)
        return {"kind": "tables", "seqs": seqs, "tokens": tokens, "before": before, "width": (2 * (before + tokens)) // PAGE + rng.randint(2, 300),
                "behind": rng.choice([0, rng.randint(1, 300)])}
    if what == "write":
        seqs = _log(rng, 1, 32)
        return {"kind": "write", "seqs": seqs, "tokens": max(seqs, _log(rng, 1, 4096)), "before": _log(rng, 1, 300), "heads": heads,
                "kv_heads": kv_heads, "dim": dim}
    if what == "single":
        seqs = _log(rng, 1, 64)
        return {"kind": "attend", "seqs": seqs, "tokens": seqs, "before": _log(rng, 1, min(32768, 500000 // seqs)), "heads": heads,
                "kv_heads": kv_heads, "dim": dim, "window": rng.choice([0, 0, rng.randint(1, 4096)])}
    if what == "few":
        seqs = _log(rng, 1, 8)
        return {"kind": "attend", "seqs": seqs, "tokens": seqs * rng.randint(2, 16) + rng.randint(0, seqs - 1), "before": _log(rng, 16, 16384),
                "heads": heads, "kv_heads": kv_heads, "dim": dim, "window": rng.choice([0, 0, rng.randint(1, 4096)])}
    if what == "prompt":
        seqs = rng.randint(1, 4)
        tokens = _log(rng, 64 * seqs, 4096)
        return {"kind": "attend", "seqs": seqs, "tokens": tokens, "before": rng.choice([0, _log(rng, 1, 4096)]), "heads": heads,
                "kv_heads": kv_heads, "dim": dim, "window": rng.choice([0, 0, rng.randint(64, 4096)])}
    return {"kind": "logprobs", "rows": _log(rng, 1, 2048), "vocab": _log(rng, 500, VOCAB), "top": rng.randint(0, 20)}


# ----------------------------------------------------------------------------- a step's lengths (plain numbers)
def _spread(total, parts, rng, least=1):
    """``total`` as ``parts`` unequal numbers of at least ``least``."""
    weight = [rng.uniform(0.5, 1.5) for _ in range(parts)]
    out = [least + int((total - least * parts) * w / sum(weight)) for w in weight]
    out[0] += total - sum(out)
    return out


def _lengths(case):
    """What each sequence holds before the step (about ``before``; a lone sequence exactly) and brings with it; the same for
    every seed, so that the outputs have the same shapes."""
    rng = random.Random(case["tokens"] * 1000003 + case["before"])
    B, before = case["seqs"], case["before"]
    new = _spread(case["tokens"], B, rng)
    held = [before if B == 1 else int(before * (1.0 - 0.5 * rng.random())) for _ in range(B)]
    return held, new


def _pages_of(case, held, new, gen):
    """Pages of the sequences, one after the other, in no order, and where each sequence's begin; a few more are in the pool."""
    count = [-(-(h + n) // PAGE) for h, n in zip(held, new)]
    start = [0]
    for c in count:
        start.append(start[-1] + c)
    pool = start[-1] + 3
    pages = torch.randperm(pool, generator=gen, device=DEV)[:start[-1]].to(I32)
    return pages, torch.tensor(start, dtype=I32, device=DEV), pool, max(count)


# ----------------------------------------------------------------------------- the 4-bit rows
def _quantise(x):
    """Codes [..., n], steps and zero points [..., n / 32] of float32 rows."""
    g = x.reshape(*x.shape[:-1], -1, GROUP)
    lo, hi = g.amin(-1).clamp(max=0.0), g.amax(-1).clamp(min=0.0)
    bits = ((hi - lo) / 15.0).view(I32)
    s = ((bits + 0x80000) & -0x100000).view(F32)
    safe = torch.where(s > 0, s, torch.ones_like(s))
    z = torch.round(-lo / safe).clamp(0, 15)
    c = (torch.round(g / safe[..., None]) + z[..., None]).clamp(0, 15)
    return torch.where(s[..., None] > 0, c, torch.zeros_like(c)).reshape(x.shape), s, torch.where(s > 0, z, torch.zeros_like(z))


def _stands_for(c, s, z):
    g = c.reshape(*c.shape[:-1], -1, GROUP)
    return ((g - z[..., None]) * s[..., None]).reshape(c.shape)


def _bytes_of(x):
    """Rows [pages, heads, 64, n] as a page's bytes: codes, then words."""
    c, s, z = _quantise(x)
    c = c.to(torch.uint8)
    codes = (c[..., 0::2] | (c[..., 1::2] << 4)).flatten(2)
    words = ((s.view(I32) >> 16) | z.to(I32)).to(torch.int16).flatten(2)
    return torch.cat([codes, words.view(torch.uint8)], dim=2)


def _values_of(pool, dim):
    """Keys and values [pages, heads, 64, dim] float32 that a pool's bytes stand for."""
    n, out = PAGE * dim // 2, []
    for part in pool.chunk(2, dim=2):
        b = part[..., :n].to(I32).unflatten(2, (PAGE, dim // 2))
        c = torch.stack([b & 15, b >> 4], dim=-1).flatten(3).to(F32)
        w = part[..., n:].contiguous().view(torch.int16).to(I32).unflatten(2, (PAGE, dim // GROUP))
        out.append(_stands_for(c, ((w & 0xFFF0) << 16).view(F32), (w & 15).to(F32)))
    return out


def _pool(pages, heads, dim, gen):
    """A pool that holds earlier tokens everywhere; values with a share of larger ones, as keys and values have."""
    parts = []
    for _ in range(2):
        x = torch.randn((pages, heads, PAGE, dim), generator=gen, device=DEV)
        x.mul_(torch.exp(0.5 * torch.randn((1, heads, 1, dim), generator=gen, device=DEV)))
        parts.append(_bytes_of(x))
        del x
    return torch.cat(parts, dim=2)


# ----------------------------------------------------------------------------- states
def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    rand = lambda *shape: torch.randn(shape, generator=gen, device=DEV)  # noqa: E731
    if case["kind"] == "logprobs":
        logits = rand(case["rows"], case["vocab"]).mul_(2.5)
        tokens = torch.randint(case["vocab"], (case["rows"],), generator=gen, device=DEV).to(I32)
        return {"kind": "logprobs", "logits": logits, "tokens": tokens, "top": case["top"]}
    held, new = _lengths(case)
    pages, start, n_pool, most = _pages_of(case, held, new, gen)
    ints = lambda v: torch.tensor(v, dtype=I32, device=DEV)  # noqa: E731
    st = {"kind": case["kind"], "pages": pages, "page_start": start, "pos0": ints(held), "n_new": ints(new), "max_new": max(new),
          "max_len": max(h + n for h, n in zip(held, new)), "tokens": case["tokens"]}
    if case["kind"] == "tables":
        return {**st, "tokens": case["tokens"] + case["behind"], "width": max(case["width"], most)}
    # what the step's tables say, for the calls that take them
    cu = torch.cumsum(torch.cat([ints([0]), st["n_new"]]), 0).to(I32)
    seq = torch.repeat_interleave(torch.arange(case["seqs"], device=DEV), st["n_new"].long(), output_size=case["tokens"])
    pos = torch.arange(case["tokens"], device=DEV) - cu.long()[seq] + st["pos0"].long()[seq]
    slot = pages.long()[start.long()[seq] + pos // PAGE] * PAGE + pos % PAGE
    table = torch.zeros((case["seqs"], most + 5), dtype=I32, device=DEV)
    column = torch.arange(most + 5, device=DEV)
    holds = column[None] < (start[1:] - start[:-1])[:, None]
    table[holds] = pages
    st |= {"cu": cu, "seq": seq.to(I32), "pos": pos.to(I32), "slot": slot.to(I32), "table": table, "seq_len": st["pos0"] + st["n_new"],
           "heads": case["heads"], "kv_heads": case["kv_heads"], "dim": case["dim"],
           "pool": _pool(n_pool, case["kv_heads"], case["dim"], gen)}
    if case["kind"] == "write":
        freq = 1e6 ** (-torch.arange(0, case["dim"], 2, dtype=F64, device=DEV) / case["dim"])
        angle = pos[:, None].to(F64) * freq
        return {**st, "qkv": rand(case["tokens"], (case["heads"] + 2 * case["kv_heads"]) * case["dim"]), "q_weight": 1 + 0.2 * rand(case["dim"]),
                "k_weight": 1 + 0.2 * rand(case["dim"]), "cos": angle.cos().to(F32), "sin": angle.sin().to(F32)}
    return {**st, "q": rand(case["tokens"], case["heads"], case["dim"]).to(BF), "scale": case["dim"] ** -0.5, "window": case["window"]}


# ----------------------------------------------------------------------------- one pass
def run(st):
    if own:
        return _own(st)
    return {"tables": _plain_tables, "write": _plain_write, "attend": _plain_attend, "logprobs": _plain_logprobs}[st["kind"]](st)


def _own(st):
    from questwend_b200.kernels import ops
    if st["kind"] == "tables":
        t = ops.step_tables(st["pages"], st["page_start"], st["pos0"], st["n_new"], st["tokens"], st["width"])
        return [t.cu_seqlens, t.seq_len, t.tok_seq, t.tok_pos, t.page_table, t.slot_map]
    if st["kind"] == "write":
        q = ops.kv4_store(st["qkv"], st["q_weight"], st["k_weight"], st["cos"], st["sin"], st["slot"], st["pool"], st["heads"],
                          st["kv_heads"], st["dim"], st["dim"], EPS, BF)
        k, v, _ = ops.kv4_read(st["pool"], st["pages"], st["page_start"], st["seq_len"], st["max_len"], st["dim"], BF)
        return [q, k, v]
    if st["kind"] == "attend":
        tables = ops.StepTables(st["cu"], st["seq_len"], st["seq"], st["pos"], st["table"], st["slot"], st["pos0"], st["pages"], st["page_start"])
        return [ops.kv4_attention(st["q"], st["pool"], tables, st["max_new"], st["max_len"], st["scale"], window=st["window"])]
    r = ops.token_logprobs(st["logits"], st["tokens"], top=st["top"])
    return [r.logprob, r.entropy, r.top_ids, r.top_logprobs]


def _plain_tables(st):
    B, T, W = st["pos0"].numel(), st["tokens"], st["width"]
    cu = torch.nn.functional.pad(torch.cumsum(st["n_new"], 0), (1, 0))
    t = torch.arange(T, device=DEV)
    seq = torch.searchsorted(cu, t, right=True) - 1
    live = seq < B
    row = seq.clamp(max=B - 1)
    pos = t - cu[row] + st["pos0"].long()[row]
    at = st["page_start"].long()[row] + pos // PAGE
    slot = st["pages"].long()[at.clamp(max=st["pages"].numel() - 1)] * PAGE + pos % PAGE
    none = torch.full_like(t, -1)
    column = torch.arange(W, device=DEV)
    count = (st["page_start"][1:] - st["page_start"][:-1]).long()
    entry = (st["page_start"].long()[:-1, None] + column).clamp(max=st["pages"].numel() - 1)
    table = torch.where(column < count[:, None], st["pages"][entry], torch.zeros_like(st["pages"][:1]))
    return [cu.to(I32), st["pos0"] + st["n_new"], torch.where(live, seq, none).to(I32), torch.where(live, pos, none).to(I32), table,
            torch.where(live, slot, none).to(I32)]


def _turned(x, weight, cos, sin):
    """Heads [T, H, dim]: RMS norm with a weight, then the rotation of the pairs (i, i + dim / 2)."""
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight
    a, b = x.chunk(2, dim=-1)
    c, s = cos[:, None], sin[:, None]
    return torch.cat([a * c - b * s, a * s + b * c], dim=-1)


def _plain_write(st):
    H, KV, D = st["heads"], st["kv_heads"], st["dim"]
    x = st["qkv"].view(-1, H + 2 * KV, D)
    q = _turned(x[:, :H], st["q_weight"], st["cos"], st["sin"])
    k = _turned(x[:, H:H + KV], st["k_weight"], st["cos"], st["sin"])
    # the pages as they are, the step's rows in them, nothing behind a sequence's last token
    B = st["pos0"].numel()
    held = (st["page_start"][1:] - st["page_start"][:-1]).long()
    of = torch.repeat_interleave(torch.arange(B, device=DEV), held, output_size=st["pages"].numel())
    first = (torch.arange(st["pages"].numel(), device=DEV) - st["page_start"].long()[of]) * PAGE
    place = first[:, None] + torch.arange(PAGE, device=DEV)
    live = (place < st["seq_len"].long()[of][:, None])[:, None, :, None]
    at = st["page_start"].long()[st["seq"].long()] + st["pos"].long() // PAGE
    out = [q.to(BF)]
    for old, new in zip(_values_of(st["pool"][st["pages"].long()], D), (k, x[:, H + KV:])):
        old[at, :, st["pos"].long() % PAGE] = _stands_for(*_quantise(new.contiguous()))
        out.append(torch.where(live, old, torch.zeros_like(old)).to(BF))
    return out


def _plain_attend(st):
    B, H, KV, D, N = st["pos0"].numel(), st["heads"], st["kv_heads"], st["dim"], st["max_new"]
    wide = -(-st["max_len"] // PAGE)
    k, v = (x.unflatten(0, (B, wide)).transpose(1, 2).flatten(2, 3) for x in _values_of(st["pool"][st["table"][:, :wide].long().flatten()], D))
    i = torch.arange(N, device=DEV)
    at = (st["cu"].long()[:-1, None] + i).clamp(max=st["q"].shape[0] - 1)
    q = st["q"][at].to(F32).unflatten(2, (KV, H // KV)).permute(0, 2, 3, 1, 4).flatten(2, 3)            # [B, KV, H / KV * N, D]
    pos = (st["pos0"].long()[:, None] + i)[:, :, None]
    j = torch.arange(wide * PAGE, device=DEV)
    sees = (j <= pos) & (j < st["seq_len"].long()[:, None, None])
    if st["window"]:
        sees = sees & (j > pos - st["window"])
    score = torch.matmul(q, k.transpose(2, 3)).unflatten(2, (H // KV, N)).mul_(st["scale"])
    score.masked_fill_(~sees[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = score.sub_(torch.where(top.isfinite(), top, torch.zeros_like(top))).exp_()
    total = p.sum(-1, keepdim=True)
    # what no sequence holds counts for nothing, whatever the page has there
    v = torch.where((j < st["seq_len"].long()[:, None])[:, None, :, None], v, torch.zeros_like(v))
    o = torch.matmul(p.flatten(2, 3), v).unflatten(2, (H // KV, N)) / total
    o = o.permute(0, 3, 1, 2, 4).reshape(B, N, H * D)
    return [o[st["seq"].long(), st["pos"].long() - st["pos0"].long()[st["seq"].long()]].to(BF)]


def _plain_logprobs(st):
    x = st["logits"]
    m = x.amax(-1, keepdim=True)
    e = (x - m).exp()
    total = e.sum(-1, dtype=F64)
    norm = total.log()
    spread = ((x - m) * e).sum(-1, dtype=F64) / total
    at = x.gather(1, st["tokens"].long()[:, None])[:, 0]
    # the largest first, of equal ones the lowest id: the number's bits in their order above the id
    bits = (x + 0.0).view(I32).long()
    order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits)
    key = (order << 32) | (0x7FFFFFFF - torch.arange(x.shape[1], device=DEV))
    ids = 0x7FFFFFFF - (key.topk(st["top"], dim=1).values & 0xFFFFFFFF)
    lps = (x.gather(1, ids).to(F64) - m - norm[:, None]).to(F32)
    return [(at.to(F64) - m[:, 0] - norm).to(F32), (norm - spread).to(F32), ids.to(I32), lps]


# ----------------------------------------------------------------------------- what a pass cannot do without
def _visible(case):
    held, new = _lengths(case)
    pairs = keys = 0
    for h, n in zip(held, new):
        w = case.get("window", 0) or (h + n)
        pairs += sum(min(p + 1, w) for p in range(h, h + n))
        keys += min(h + n, w + n - 1)
    return pairs, keys


def work(case):
    if case["kind"] == "logprobs":
        R, V, top = case["rows"], case["vocab"], case["top"]
        return {"bytes": R * V * 4 + R * (12 + 8 * top), "flops": 5 * R * V}
    if case["kind"] == "tables":
        T, B = case["tokens"] + case["behind"], case["seqs"]
        return {"bytes": 4 * (3 * T + B * case["width"] + 6 * B + B * (case["before"] * 3 // 4 // PAGE)), "flops": T}
    H, KV, D, T = case["heads"], case["kv_heads"], case["dim"], case["tokens"]
    row = KV * (D + D // 8)                                             # bytes of a token's keys and values
    if case["kind"] == "write":
        held, new = _lengths(case)
        pages = sum(-(-(h + n) // PAGE) for h, n in zip(held, new))
        read_back = sum(h + n for h, n in zip(held, new)) * row + pages * PAGE * KV * D * 2 * 2
        return {"bytes": T * ((H + 2 * KV) * D * 4 + D * 4 + H * D * 2 + row) + read_back, "flops": 10 * T * (H + 2 * KV) * D}
    pairs, keys = _visible(case)
    return {"bytes": keys * row + T * H * D * 2 * 2, "flops": 4 * pairs * H * D}


# ----------------------------------------------------------------------------- from the definitions, in 64 bits
def _exact_rows(x):
    """What rows [..., n] in 64 bits stand for, group by group."""
    g = x.unflatten(-1, (-1, GROUP))
    lo = torch.minimum(g.min(-1).values, torch.zeros((), dtype=F64, device=x.device))
    hi = torch.maximum(g.max(-1).values, torch.zeros((), dtype=F64, device=x.device))
    mantissa, exponent = torch.frexp((hi - lo) / 15)
    s = torch.ldexp(torch.floor(mantissa * 16 + 0.5) / 16, exponent)
    ok = s > 0
    d = torch.where(ok, s, torch.ones_like(s))
    z = torch.round(-lo / d)
    c = torch.clamp(torch.round(g / d[..., None]), min=-z[..., None], max=15 - z[..., None])
    return torch.where(ok[..., None], c * s[..., None], torch.zeros_like(c)).flatten(-2)


def _exact_page(pool, page, head, dim):
    """Keys and values [64, dim] in 64 bits of a page and head, from the bytes' definition."""
    out = []
    half = pool.shape[2] // 2
    for b in (pool[page, head, :half], pool[page, head, half:]):
        codes, words = b[:PAGE * dim // 2].long(), b[PAGE * dim // 2:].long().view(-1, 2)
        c = torch.empty(PAGE * dim, dtype=F64, device=b.device)
        c[0::2], c[1::2] = (codes % 16).to(F64), (codes // 16).to(F64)
        w = words[:, 0] + 256 * words[:, 1]
        exponent, fraction, z = w // 128, (w % 128) // 16, w % 16       # s = (1 + fraction / 8) 2^(exponent - 127)
        s = torch.where(exponent > 0, torch.ldexp(1 + fraction.to(F64) / 8, exponent - 127), torch.zeros_like(fraction, dtype=F64))
        out.append(((c.view(-1, GROUP) - z[:, None]) * s[:, None]).view(PAGE, dim))
    return out


def _exact_sequence(st, b, head):
    pages = st["pages"][int(st["page_start"][b]):int(st["page_start"][b + 1])].long()
    half = st["pool"].shape[2] // 2
    out = []
    for lo in (0, half):
        raw = st["pool"][pages, head, lo:lo + half].long()
        n = PAGE * st["dim"] // 2
        c = torch.stack([raw[:, :n] % 16, raw[:, :n] // 16], -1).to(F64).view(len(pages) * PAGE, -1, GROUP)
        w = (raw[:, n::2] + 256 * raw[:, n + 1::2]).view(len(pages) * PAGE, -1)
        s = torch.where(w >= 128, torch.ldexp(1 + ((w % 128) // 16).to(F64) / 8, w // 128 - 127), torch.zeros((), dtype=F64, device=w.device))
        out.append(((c - (w % 16)[..., None]) * s[..., None]).flatten(1)[:int(st["seq_len"][b])])
    return out


def exact(case, seed):
    if case["kind"] == "tables":
        return None                                                     # whole numbers
    st = prepare(case, seed)
    if case["kind"] == "logprobs":
        parts = []
        for x, t in zip(st["logits"].split(64), st["tokens"].long().split(64)):
            lp = torch.log_softmax(x.to(F64), dim=1)
            value, ids = lp.sort(dim=1, descending=True, stable=True)
            parts.append([lp.gather(1, t[:, None])[:, 0], -(lp.exp() * lp).sum(1), ids[:, :case["top"]].to(I32), value[:, :case["top"]]])
        return [torch.cat(p) for p in zip(*parts)]
    H, KV, D = case["heads"], case["kv_heads"], case["dim"]
    if case["kind"] == "attend":
        out = torch.empty((case["tokens"], H, D), dtype=F64, device=DEV)
        cu = st["cu"].tolist()
        for b in range(case["seqs"]):
            for h in range(KV):
                k, v = _exact_sequence(st, b, h)
                for lo in range(cu[b], cu[b + 1], 1024):
                    hi = min(lo + 1024, cu[b + 1])
                    q = st["q"][lo:hi, h * (H // KV):(h + 1) * (H // KV)].to(F64)
                    score = torch.einsum("thd,jd->htj", q, k) * st["scale"]
                    back = st["pos"][lo:hi, None].long() - torch.arange(k.shape[0], device=DEV)
                    hidden = (back < 0) | (back >= (case["window"] or 1 << 40))
                    p = torch.softmax(score.masked_fill(hidden, -math.inf), dim=-1)
                    out[lo:hi, h * (H // KV):(h + 1) * (H // KV)] = torch.einsum("htj,jd->thd", p, v)
        return [out.flatten(1)]
    x = st["qkv"].to(F64).view(-1, H + 2 * KV, D)

    def turned(x, weight):
        x = x / torch.sqrt((x ** 2).sum(-1, keepdim=True) / D + EPS) * weight.to(F64)
        turn = torch.complex(st["cos"].to(F64), st["sin"].to(F64))[:, None]
        y = torch.complex(x[..., :D // 2].contiguous(), x[..., D // 2:].contiguous()) * turn
        return torch.cat([y.real, y.imag], -1)

    rows = [_exact_rows(turned(x[:, H:H + KV], st["k_weight"])), _exact_rows(x[:, H + KV:])]
    out = [torch.zeros((st["pages"].numel(), KV, PAGE, D), dtype=F64, device=DEV) for _ in range(2)]
    start, length, page = st["page_start"].tolist(), st["seq_len"].tolist(), st["pages"].tolist()
    for b in range(case["seqs"]):
        before, first = int(st["pos0"][b]), int(st["cu"][b])
        for j in range(start[b], start[b + 1]):
            base = (j - start[b]) * PAGE
            end = min(PAGE, length[b] - base)
            kept = min(max(before - base, 0), end)
            for part in range(2):
                if kept:
                    for h in range(KV):
                        out[part][j, h, :kept] = _exact_page(st["pool"], page[j], h, D)[part][:kept]
                t = first + base + kept - before
                out[part][j, :, kept:end] = rows[part][t:t + end - kept].transpose(0, 1)
    return [turned(x[:, :H], st["q_weight"]).clone(), *out]

"""The 4-bit cache, attention over it, a step's tables and log probabilities, plainly, in 64 bits (NumPy)."""
from __future__ import annotations

import numpy as np

PAGE, GROUP = 64, 32


def quantise(x):
    """Rows [..., n] float64 -> (codes uint8 [..., n], words uint16 [..., n / 32])."""
    x = np.asarray(x, dtype=np.float64)
    g = x.reshape(*x.shape[:-1], -1, GROUP)
    finite = np.isfinite(g).all(-1)
    g = np.where(finite[..., None], g, 0.0)
    lo, hi = np.minimum(g.min(-1), 0.0), np.maximum(g.max(-1), 0.0)
    with np.errstate(over="ignore"):
        mantissa, exponent = np.frexp((hi - lo) / 15)
        s = np.ldexp(np.floor(mantissa * 16 + 0.5) / 16, exponent)
    finite &= s < 2.0 ** 120
    s = np.where(finite & (s >= 2.0 ** -126), s, 0.0)
    d = np.where(s > 0, s, 1.0)
    z = np.where(s > 0, np.minimum(np.rint(-lo / d), 15), 0)
    c = np.where(s[..., None] > 0, np.clip(np.rint(g / d[..., None]) + z[..., None], 0, 15), 0)
    words = (s.astype(np.float32).view(np.uint32) >> 16).astype(np.uint16) | z.astype(np.uint16)
    words = np.where(finite, words, 0x7FC0).astype(np.uint16)
    return c.reshape(x.shape).astype(np.uint8), words


def stands_for(codes, words):
    g = codes.astype(np.float64).reshape(*codes.shape[:-1], -1, GROUP)
    w = words.astype(np.uint32)
    s = ((w & 0xFFF0) << 16).view(np.float32).astype(np.float64)
    return ((g - (w & 15)[..., None]) * s[..., None]).reshape(codes.shape)


def pack(k, v):
    """Keys and values [pages, heads, 64, n] -> the pool's bytes [pages, heads, bytes]."""
    parts = []
    for x in (k, v):
        c, w = quantise(x)
        parts += [(c[..., 0::2] | (c[..., 1::2] << 4)).reshape(*c.shape[:2], -1), np.ascontiguousarray(w).view(np.uint8).reshape(*c.shape[:2], -1)]
    return np.concatenate(parts, axis=2)


def unpack(pool, dim):
    """The pool's bytes -> (key codes, key words, value codes, value words)."""
    out, at = [], 0
    for _ in range(2):
        n = PAGE * dim // 2
        b = pool[..., at:at + n].reshape(*pool.shape[:2], PAGE, dim // 2)
        out.append(np.stack([b & 15, b >> 4], -1).reshape(*pool.shape[:2], PAGE, dim))
        at += n
        n = PAGE * dim // GROUP * 2
        out.append(np.ascontiguousarray(pool[..., at:at + n]).view(np.uint16).reshape(*pool.shape[:2], PAGE, dim // GROUP))
        at += n
    return out


def values(pool, dim):
    kc, kw, vc, vw = unpack(pool, dim)
    return stands_for(kc, kw), stands_for(vc, vw)


def norm_rope(x, weight, cos, sin, eps):
    """Heads [T, H, n] float64: RMS norm (weight or None), rotation of the first 2 * cos.shape[1] numbers."""
    if weight is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * weight
    if cos is None:
        return x
    h = cos.shape[1]
    c, s = cos[:, None], sin[:, None]
    a, b = x[..., :h], x[..., h:2 * h]
    return np.concatenate([a * c - b * s, a * s + b * c, x[..., 2 * h:]], -1)


def attention(q, k, v, pos, scale, window=0):
    """q [n, Hq, d], k and v [len, Hkv, d] of one sequence, pos [n]; returns (out [n, Hq, d], the same of |v|, the largest sum of
    |q k| scale of a pair) - the last two bound what roundings can do."""
    n, Hq, d = q.shape
    G = Hq // k.shape[1]
    out, mass, big = np.zeros((n, Hq, d)), np.zeros((n, Hq, d)), np.zeros((n, Hq, 1))
    for h in range(Hq):
        kk, vv = k[:, h // G], v[:, h // G]
        for i in range(n):
            lo = max(0, pos[i] - window + 1) if window else 0
            ks, vs = kk[lo:pos[i] + 1], vv[lo:pos[i] + 1]
            if not len(ks):
                continue
            s = ks @ q[i, h] * scale
            p = np.exp(s - s.max())
            p /= p.sum()
            out[i, h], mass[i, h] = p @ vs, p @ np.abs(vs)
            big[i, h] = (np.abs(ks) @ np.abs(q[i, h])).max() * scale
    return out, mass, big


def step_tables(pages, page_start, pos0, n_new, n_tokens, width):
    """(cu, seq_len, tok_seq, tok_pos, page_table, slot_map) as lists of whole numbers."""
    B = len(pos0)
    cu = [0]
    seq, pos, slot = [], [], []
    for b in range(B):
        cu.append(cu[-1] + n_new[b])
        mine = pages[page_start[b]:page_start[b + 1]]
        for i in range(n_new[b]):
            p = pos0[b] + i
            seq.append(b)
            pos.append(p)
            slot.append(mine[p // PAGE] * PAGE + p % PAGE if p // PAGE < len(mine) else -1)
    behind = [-1] * (n_tokens - len(seq))
    table = [(list(pages[page_start[b]:page_start[b + 1]]) + [0] * width)[:width] for b in range(B)]
    return cu, [p + n for p, n in zip(pos0, n_new)], seq + behind, pos + behind, table, slot + behind


def logprobs(x, tokens, top):
    """(logprob [R], entropy [R], ids [R, top], lps [R, top], E|d|, E d^2 with d = x - max) of rows of logits."""
    x = np.asarray(x, dtype=np.float64)
    m = x.max(-1, keepdims=True)
    with np.errstate(divide="ignore", invalid="ignore"):
        d = x - m
        e = np.exp(d)
        S = e.sum(-1, keepdims=True)
        lp = d - np.log(S)
        p = e / S
        dd = np.where(p > 0, d, 0.0)
        H = -(np.where(p > 0, p * lp, 0.0)).sum(-1)
    ids = np.argsort(-x, axis=-1, kind="stable")[:, :top]
    return (np.take_along_axis(lp, np.asarray(tokens)[:, None], 1)[:, 0], H, ids, np.take_along_axis(lp, ids, 1), (p * np.abs(dd)).sum(-1),
            (p * dd * dd).sum(-1))

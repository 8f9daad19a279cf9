"""Writing the 4-bit cache, reading it back, attention over it, and a step's tables, against plain 64-bit implementations."""
import numpy as np
import pytest
import torch

import plain_kv4 as pk
from questwend_b200.kernels import ops
from questwend_b200.kernels.ops import KernelError, StepTables

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, BF = torch.float32, torch.bfloat16
EPS = 1e-6


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def f64(t):
    return t.detach().to(torch.float64).cpu().numpy()


# ----------------------------------------------------------------------------- tables
@pytest.mark.parametrize("pos0,n_new,behind", [([0], [1], 0), ([63, 64, 0], [1, 1, 1], 0), ([5, 0, 200, 64], [70, 0, 3, 1], 11), ([100], [3000], 0),
                                               ([7] * 300, [1, 0, 2] * 100, 5), ([70] * 14000, [1] * 14000, 3), ([0, 0], [0, 0], 4)])
@pytest.mark.parametrize("extra", [0, 2])
def test_step_tables(pos0, n_new, behind, extra):
    rng = np.random.default_rng(len(pos0) + behind)
    count = [-(-(p + n) // 64) + (extra if i % 2 else 0) for i, (p, n) in enumerate(zip(pos0, n_new))]
    start = np.concatenate([[0], np.cumsum(count)]).tolist()
    pages = rng.permutation(start[-1] + 5)[:start[-1]].tolist()
    T, width = sum(n_new) + behind, max(count) + 3 * extra + (1 if max(count) == 0 else 0)
    want = pk.step_tables(pages, start, pos0, n_new, T, width)
    t = ops.step_tables(ints(pages), ints(start), ints(pos0), ints(n_new), T, width)
    for got, ref in zip((t.cu_seqlens, t.seq_len, t.tok_seq, t.tok_pos, t.page_table, t.slot_map), want):
        assert got.dtype == torch.int32 and got.tolist() == ref
    only = ops.step_tables(ints(pages), ints(start), ints(pos0), ints(n_new), T, width, tokens=False)
    assert only.tok_seq is None and torch.equal(only.page_table, t.page_table)
    narrow = ops.step_tables(ints(pages), ints(start), ints(pos0), ints(n_new), T, 1)
    assert torch.equal(narrow.page_table, t.page_table[:, :1]) and torch.equal(narrow.slot_map, t.slot_map)


def test_step_tables_with_too_few_pages_and_starts_beyond_them():
    t = ops.step_tables(ints([4, 2]), ints([0, 1, 9]), ints([60, 0]), ints([8, 200]), 208, 4)
    assert t.slot_map[:8].tolist() == [4 * 64 + p for p in range(60, 64)] + [-1] * 4         # one page held, two needed
    assert t.slot_map[8:72].tolist() == [2 * 64 + p for p in range(64)] and (t.slot_map[72:] == -1).all()
    assert t.page_table.tolist() == [[4, 0, 0, 0], [2, 0, 0, 0]]


def test_step_tables_refusals():
    a = ints([0, 1])
    for args in [(a, a, a, a, 1, 1), (a, ints([0, 1, 2]), a, ints([1]), 1, 1), (a, ints([0, 1, 2]), a, a, -1, 1), (a, ints([0, 1, 2]), a, a, 1, -1),
                 (a, ints([0]), ints([]), ints([]), 1, 1), (a, ints([0] * 58002), ints([0] * 58001), ints([0] * 58001), 1, 1)]:
        with pytest.raises(KernelError, match="step_tables"):
            ops.step_tables(*args)
    with pytest.raises(KernelError, match="int32"):
        ops.step_tables(a.long(), ints([0, 1, 2]), a, a, 1, 1)


# ----------------------------------------------------------------------------- write and read
def _write_case(seed, T, Hq, Hkv, hd, rot, pages):
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((T, (Hq + 2 * Hkv) * hd)).astype(np.float32) * np.exp(rng.standard_normal((T, 1))).astype(np.float32)
    angle = rng.uniform(0, 1000, (T, rot // 2))
    slots = rng.permutation(pages * 64)[:T].astype(np.int32)
    pool = pk.pack(rng.standard_normal((pages, Hkv, 64, hd)), rng.standard_normal((pages, Hkv, 64, hd)))
    return x, np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32), slots, pool, rng


def _expected_pool(pool, k, v, slots, hd):
    parts = pk.unpack(pool, hd)
    for t, s in enumerate(slots):
        if not 0 <= s < pool.shape[0] * 64:
            continue
        for x, (c, w) in ((k, parts[:2]), (v, parts[2:])):
            codes, words = pk.quantise(x[t])
            c[s // 64, :, s % 64], w[s // 64, :, s % 64] = codes, words
    return parts


@pytest.mark.parametrize("Hq,Hkv,hd,rot,norm", [(4, 2, 128, 128, True), (3, 1, 64, 64, True), (8, 8, 128, 64, False), (2, 2, 32, 0, False),
                                                (5, 1, 96, 40, True), (6, 3, 256, 256, True), (16, 8, 128, 128, True), (9, 3, 64, 64, False)])
@pytest.mark.parametrize("T", [1, 7, 130])
@pytest.mark.parametrize("dtype", [F32, BF])
def test_store(T, Hq, Hkv, hd, rot, norm, dtype):
    x, cos, sin, slots, pool, rng = _write_case(T + hd, T, Hq, Hkv, hd, rot, 4)
    if T > 3:
        slots[1], slots[3] = -1, 4 * 64                  # no place: behind the last sequence, beyond the pool
    qw, kw = ((1 + 0.3 * rng.standard_normal((2, hd))).astype(np.float32) if norm else (None, None))
    dev = lambda a: None if a is None else torch.from_numpy(a).to(DEV)
    on_gpu = torch.from_numpy(pool).to(DEV)
    q = ops.kv4_store(dev(x), dev(qw), dev(kw), dev(cos) if rot else None, dev(sin) if rot else None, dev(slots), on_gpu, Hq, Hkv, hd, rot, EPS, dtype)
    heads = x.astype(np.float64).reshape(T, -1, hd)
    c64, s64 = (cos.astype(np.float64), sin.astype(np.float64)) if rot else (None, None)
    up = lambda w: None if w is None else w.astype(np.float64)
    # codes and words are choices: equal, all of them (the norm, the rotation and the choice are made in 64 bits)
    want = _expected_pool(pool, pk.norm_rope(heads[:, Hq:Hq + Hkv], up(kw), c64, s64, float(np.float32(EPS))), heads[:, Hq + Hkv:], slots, hd)
    for got, ref in zip(pk.unpack(on_gpu.cpu().numpy(), hd), want):
        assert (got == ref).all()
    ref = pk.norm_rope(heads[:, :Hq], up(qw), c64, s64, EPS)
    normed = pk.norm_rope(heads[:, :Hq], up(qw), None, None, EPS)
    # 32-bit: the norm's factor (a sum of hd squares: hd / 32 + 5 additions a term, a root, a division), two products, two products and a sum
    size = np.abs(normed).max(-1, keepdims=True) * 2
    assert (np.abs(f64(q) - ref) <= (hd / 32 + 12) * 2.0 ** -24 * size + (2.0 ** -8 if dtype == BF else 0) * np.abs(ref)).all()
    assert q.dtype == dtype and tuple(q.shape) == (T, Hq, hd)
    before = on_gpu.clone()
    q2 = ops.kv4_store(dev(x), dev(qw), dev(kw), dev(cos) if rot else None, dev(sin) if rot else None, dev(slots), on_gpu, Hq, Hkv, hd, rot, EPS, dtype,
                       store_kv=False)
    assert torch.equal(on_gpu, before) and torch.equal(q, q2)


@pytest.mark.parametrize("size", [1e25, 1e-25, 1e-40])
@pytest.mark.parametrize("eps,factor", [(1e-6, 1.0), (1e-38, 1.7), (0.0, 0.3)])
@pytest.mark.parametrize("hd", [64, 128])
def test_store_of_large_and_small_numbers(size, eps, factor, hd):
    """Squares that 32 bits do not hold, an eps that counts or does not, a rotation that scales."""
    T, Hkv = 20, 2
    x, cos, sin, slots, pool, rng = _write_case(3, T, 1, Hkv, hd, hd, 2)
    x = (x * size).astype(np.float32)
    cos, sin = (cos * factor).astype(np.float32), (sin * factor).astype(np.float32)
    kw = (1 + 0.3 * rng.standard_normal(hd)).astype(np.float32)
    dev = lambda a: torch.from_numpy(a).to(DEV)
    on_gpu = dev(pool)
    ops.kv4_store(dev(x), None, dev(kw), dev(cos), dev(sin), dev(slots), on_gpu, 1, Hkv, hd, hd, eps, BF)
    h = x.astype(np.float64).reshape(T, -1, hd)
    k = pk.norm_rope(h[:, 1:1 + Hkv], kw.astype(np.float64), cos.astype(np.float64), sin.astype(np.float64), float(np.float32(eps)))
    for got, ref in zip(pk.unpack(on_gpu.cpu().numpy(), hd), _expected_pool(pool, k, h[:, 1 + Hkv:], slots, hd)):
        assert (got == ref).all()


def test_store_of_groups_at_the_border():
    """Numbers halfway between two codes, zeros, equal numbers, tiny and huge ones, and some that are not finite."""
    hd = 128
    x = np.zeros((12, 3 * hd), dtype=np.float32)
    x[0, hd:] = np.tile(np.arange(32) / 2 - 3.5, 8)                                 # step 1: every second one is a tie
    x[1, hd:] = np.tile(np.arange(32) / 2, 8)
    x[2, hd:] = -np.tile(np.arange(32) / 2, 8)
    x[3, hd:], x[4, hd:], x[5, hd:], x[6, hd:] = 2.5, -1.0, 1e-42, 0.0
    x[7, hd:] = np.tile([9e36, -9e36] + [1.0] * 30 + [3e37] + [1.0] * 31, 4)
    x[8, hd], x[9, 2 * hd + 5], x[10, hd + 40] = np.nan, np.inf, -np.inf
    x[11, hd:] = np.tile(np.nextafter(np.float32(np.arange(32) / 2 - 3.5), np.float32(100)), 8)
    slots = np.arange(12, dtype=np.int32)
    pool = np.full((1, 1, ops.kv4_page_bytes(hd)), 255, dtype=np.uint8)
    on_gpu = torch.from_numpy(pool).to(DEV)
    ops.kv4_store(torch.from_numpy(x).to(DEV), None, None, None, None, ints(slots.tolist()), on_gpu, 1, 1, hd, 0, 0.0, F32)
    h = x.astype(np.float64).reshape(12, 3, hd)
    for got, ref in zip(pk.unpack(on_gpu.cpu().numpy(), hd), _expected_pool(pool, h[:, 1:2], h[:, 2:], slots, hd)):
        assert (got == ref).all()


def _cache(seed, lens, Hkv, hd, spread=1.0, spare=2, stale=255):
    """A pool for sequences of these lengths, pages in no order; places that hold no token are filled with ``stale`` bytes (NaN)."""
    rng = np.random.default_rng(seed)
    count = [-(-n // 64) for n in lens]
    start = np.concatenate([[0], np.cumsum(count)]).astype(int)
    n_pages = int(start[-1]) + spare
    order = rng.permutation(n_pages)[:start[-1]]
    k = rng.standard_normal((n_pages, Hkv, 64, hd)) * spread
    v = rng.standard_normal((n_pages, Hkv, 64, hd)) + 0.3
    pool = pk.pack(k, v)
    kv = pk.values(pool, hd)
    seqs = [[x[order[start[b]:start[b + 1]]].transpose(0, 2, 1, 3).reshape(-1, Hkv, hd)[:n] for x in kv] for b, n in enumerate(lens)]
    raw = pool.reshape(n_pages, Hkv, -1)
    live = np.zeros((n_pages, 64), dtype=bool)
    for b, n in enumerate(lens):
        for j in range(count[b]):
            live[order[start[b] + j], :max(0, min(64, n - 64 * j))] = True
    at = 0
    for size in (hd // 2, hd // 16) * 2:                   # rows of codes and of words, of keys and of values
        part = raw[:, :, at:at + 64 * size].reshape(n_pages, Hkv, 64, size)
        part[~np.broadcast_to(live[:, None], part.shape[:3])] = stale
        raw[:, :, at:at + 64 * size] = part.reshape(n_pages, Hkv, -1)
        at += 64 * size
    return torch.from_numpy(raw).to(DEV), order.tolist(), start.tolist(), seqs, rng


def _tables(order, start, pos0, n_new, behind=0, width=None):
    T = sum(n_new) + behind
    return ops.step_tables(ints(order), ints(start), ints(pos0), ints(n_new), T, width or max(1, max(b - a for a, b in zip(start, start[1:]))))


@pytest.mark.parametrize("lens", [[1], [64], [65, 3, 128], [200, 0, 130]])
@pytest.mark.parametrize("Hkv,hd", [(2, 128), (1, 64), (3, 32), (1, 96)])
@pytest.mark.parametrize("dtype", [F32, BF])
def test_read(lens, Hkv, hd, dtype):
    pool, order, start, seqs, _ = _cache(3, lens, Hkv, hd)
    k, v, table = ops.kv4_read(pool, ints(order), ints(start), ints(lens), max(lens), hd, dtype)
    assert k.dtype == dtype and tuple(k.shape) == (start[-1], Hkv, 64, hd) and tuple(table.shape) == (len(lens), -(-max(lens) // 64))
    for b, n in enumerate(lens):
        for got, ref in zip((k, v), seqs[b]):
            pages = got[table[b, :-(-n // 64)].long()].transpose(1, 2).reshape(-1, Hkv, hd)
            assert (f64(pages[:n]) == ref).all() and (pages[n:] == 0).all()             # exact in both types
        assert table[b].tolist() == [start[b] + j if 64 * j < n else 0 for j in range(table.shape[1])]


def test_read_marked():
    """A token with a value that is not finite: values of zero, keys of NaN, in that head only."""
    pool, order, start, seqs, _ = _cache(4, [70], 2, 64)
    raw = pool.view(torch.uint8)
    word = 64 * 32 + 64 * 4 + 64 * 32 + 5 * 4             # the values' words begin behind keys' codes and words and values' codes
    raw[order[0], 1, word:word + 2] = torch.tensor([0xC0, 0x7F], dtype=torch.uint8, device=DEV)
    args = (pool, ints(order), ints(start), ints([70]), 70, 64, F32)
    k, v, _ = ops.kv4_read(*args)
    assert v[0, 1, 5, :32].isnan().all() and not v[0, 1, 5, 32:].isnan().any() and not k.isnan().any()
    km, vm, _ = ops.kv4_read(*args, marked=True)
    assert km[0, 1, 5].isnan().all() and (vm[0, 1, 5] == 0).all() and not vm.isnan().any()
    km[0, 1, 5], vm[0, 1, 5] = k[0, 1, 5], v[0, 1, 5]
    assert torch.equal(km, k) and torch.equal(vm.nan_to_num(), v.nan_to_num())


# ----------------------------------------------------------------------------- attention
def tolerance(dtype, hd, mass, big, out, n_keys):
    """A score is off by at most (hd + 2) 2^-23 of the sum of |q k| scale (32-bit sums, whose additions may be cut and not rounded,
    and the products by scale and log2 e), which changes weights by twice that; the sums over the keys by 2^-23 a key, the
    weights' exponential by 2^-21.  bfloat16 forms round a weight (2^-8 of it) and the result (2^-8).  A weight under 2^-126 may be
    lost: 2^-122 a key, with values below 16."""
    u = 2.0 ** -8 if dtype == BF else 0.0
    return (u + 2.0 ** -21 + 2 * (hd + 2) * 2.0 ** -23 * big + n_keys * 2.0 ** -23) * mass + (u + 2.0 ** -23) * np.abs(out) + n_keys * 2.0 ** -122


def forms(q):
    return ["auto", "plain", "rows", "read"] if q.dtype == BF and q.shape[2] in (64, 128) else ["auto"]


def _check(pool, tables, seqs, q, pos0, n_new, max_len, scale, window):
    qd, t, want = f64(q), 0, []
    for b, n in enumerate(n_new):
        want.append((t, n, *pk.attention(qd[t:t + n], *seqs[b], [pos0[b] + i for i in range(n)], scale, window)))
        t += n
    for impl in forms(q):
        got = ops.kv4_attention(q, pool, tables, max(n_new), max_len, scale, window=window, impl=impl)
        assert got.dtype == q.dtype and tuple(got.shape) == (q.shape[0], q.shape[1] * q.shape[2])
        got = f64(got).reshape(q.shape)
        for b, (at, n, out, mass, big) in enumerate(want):
            lim = tolerance(q.dtype, q.shape[2], mass, big, out, min(pos0[b] + n, window or 1 << 30))
            bad = ~(np.abs(got[at:at + n] - out) <= lim)
            assert not bad.any(), (impl, b, np.abs(got[at:at + n] - out).max(), (np.abs(got[at:at + n] - out) / np.maximum(lim, 1e-30)).max(),
                                   np.argwhere(bad)[:5].tolist())
        assert (got[t:] == 0).all(), impl


SIZES = [(4, 1, 128), (8, 2, 64), (3, 3, 128), (2, 1, 64), (16, 2, 128), (10, 2, 128), (12, 1, 64), (32, 1, 128)]
ODD = [(2, 1, 32), (3, 1, 96), (4, 2, 256)]


@pytest.mark.parametrize("Hq,Hkv,hd", SIZES + ODD)
@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("window", [0, 1, 50, 64, 200])
def test_single_tokens(Hq, Hkv, hd, dtype, window):
    lens = [1, 64, 65, 130, 700, 17, 1030]
    pool, order, start, seqs, rng = _cache(Hq + hd, lens, Hkv, hd)
    pos0, n_new = [n - 1 for n in lens], [1] * len(lens)
    q = torch.from_numpy(rng.standard_normal((len(lens), Hq, hd))).to(dtype).to(DEV)
    _check(pool, _tables(order, start, pos0, n_new), seqs, q, pos0, n_new, max(lens), hd ** -0.5, window)


@pytest.mark.parametrize("Hq,Hkv,hd", SIZES[:5] + ODD[:2])
@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("window", [0, 3, 70])
@pytest.mark.parametrize("lens,n_new", [([5], [5]), ([64, 300], [2, 7]), ([70, 1, 200], [3, 1, 16]), ([130, 66], [70, 2])])
def test_few_tokens_and_prompts(Hq, Hkv, hd, dtype, window, lens, n_new):
    pool, order, start, seqs, rng = _cache(Hq + hd + len(lens), lens, Hkv, hd)
    pos0 = [a - b for a, b in zip(lens, n_new)]
    q = torch.from_numpy(rng.standard_normal((sum(n_new), Hq, hd))).to(dtype).to(DEV)
    _check(pool, _tables(order, start, pos0, n_new), seqs, q, pos0, n_new, max(lens), hd ** -0.5, window)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("hd", [64, 128])
def test_a_longer_prompt(dtype, hd):
    lens, n_new = [520, 333], [500, 333]
    pool, order, start, seqs, rng = _cache(9, lens, 1, hd)
    pos0 = [a - b for a, b in zip(lens, n_new)]
    q = torch.from_numpy(rng.standard_normal((sum(n_new), 2, hd))).to(dtype).to(DEV)
    for window in (0, 100):
        _check(pool, _tables(order, start, pos0, n_new), seqs, q, pos0, n_new, max(lens), hd ** -0.5, window)


@pytest.mark.parametrize("Hq,Hkv,hd", [(8, 2, 128), (6, 2, 64)])
@pytest.mark.parametrize("window", [0, 1500])
def test_few_tokens_behind_long_contexts(Hq, Hkv, hd, window):
    """The prompt kernel cuts the keys of such a step into pieces, joined by a kernel of its own."""
    lens, n_new = [5000, 700, 2950], [20, 33, 1]
    pool, order, start, seqs, rng = _cache(Hq, lens, Hkv, hd)
    pos0 = [a - b for a, b in zip(lens, n_new)]
    q = torch.from_numpy(rng.standard_normal((sum(n_new) + 3, Hq, hd))).to(BF).to(DEV)
    t = _tables(order, start, pos0, n_new, behind=3)
    _check(pool, t, seqs, q, pos0, n_new, max(lens), hd ** -0.5, window)
    before = ops.LAUNCHES[0]
    ops.kv4_attention(q, pool, t, max(n_new), max(lens), 0.1, window=window, impl="read")
    assert ops.LAUNCHES[0] - before == 3                   # pages, pieces, join


@pytest.mark.parametrize("dtype", [F32, BF])
def test_large_scores(dtype):
    """Scores of hundreds: one key carries all the weight; and a maximum that grows along the sequence."""
    pool, order, start, seqs, rng = _cache(5, [900], 1, 128, spread=30.0)
    q = torch.from_numpy(rng.standard_normal((1, 4, 128)) * 20).to(dtype).to(DEV)
    _check(pool, _tables(order, start, [899], [1]), seqs, q, [899], [1], 900, 128 ** -0.5, 0)
    lens = [600]
    k = np.zeros((10, 1, 64, 64))
    k[..., 0] = np.arange(640).reshape(10, 1, 64) / 10.0
    pool = pk.pack(k, rng.standard_normal((10, 1, 64, 64)))
    seqs = [[x.transpose(0, 2, 1, 3).reshape(-1, 1, 64)[:600] for x in pk.values(pool, 64)]]
    q = torch.ones(1, 2, 64).to(dtype).to(DEV)
    _check(torch.from_numpy(pool).to(DEV), _tables(list(range(10)), [0, 10], [599], [1]), seqs, q, [599], [1], 600, 1.0, 0)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("n_new", [1, 3, 100])
def test_padded_steps(dtype, n_new):
    """Tokens behind the last sequence's (and sequences that bring nothing): zeros there, nothing else changes."""
    lens, new = [150, 0, 120], [n_new, 0, min(n_new, 5)]
    pool, order, start, seqs, rng = _cache(6, lens, 2, 64)
    pos0 = [a - b for a, b in zip(lens, new)]
    q = torch.from_numpy(rng.standard_normal((sum(new) + 9, 4, 64))).to(dtype).to(DEV)
    _check(pool, _tables(order, start, pos0, new, behind=9), seqs, q, pos0, new, max(lens), 0.125, 0)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("n_new", [4, 90])
def test_a_token_that_is_not_finite_reaches_those_that_see_it_only(dtype, n_new):
    hd, L = 128, 200
    pool, order, start, seqs, rng = _cache(7, [L], 2, hd)
    t = _tables(order, start, [L - n_new], [n_new])
    q = torch.from_numpy(rng.standard_normal((n_new, 4, hd))).to(dtype).to(DEV)
    clean = {f: ops.kv4_attention(q, pool, t, n_new, L, 0.1, impl=f).view(n_new, 4, hd) for f in forms(q)}
    at = L - 2
    page, row = order[at // 64], at % 64
    for part in (0, 1):                                  # a key's word, a value's word, of head 1
        broken = pool.clone()
        word = part * 64 * (hd // 2 + hd // 16) + 64 * hd // 2 + row * (hd // 16)
        broken[page, 1, word:word + 2] = torch.tensor([0xC0, 0x7F], dtype=torch.uint8, device=DEV)
        for f in forms(q):
            got = ops.kv4_attention(q, broken, t, n_new, L, 0.1, impl=f).view(n_new, 4, hd)
            assert torch.equal(got[:, :2], clean[f][:, :2]), f                            # the other head's queries
            assert torch.equal(got[:-2, 2:], clean[f][:-2, 2:]), f                        # tokens before it
            assert got[-2:, 2:, :32].isnan().all(), f


@pytest.mark.parametrize("Hq,Hkv,hd,n_new,window", [(8, 2, 128, 1, 0), (8, 2, 64, 1, 0), (8, 2, 128, 3, 0), (4, 4, 128, 1, 500), (32, 2, 64, 1, 0)])
def test_attention_does_not_depend_on_the_batch(Hq, Hkv, hd, n_new, window):
    """Bit for bit: alone or with others, and whether the runs of a sequence are joined by a cluster's blocks or, where a longer sequence
    could be in the batch, by a second kernel."""
    lens = [300, 1000, 70, 2100]
    pool, order, start, seqs, rng = _cache(8, lens, Hkv, hd)
    new, B = [n_new] * len(lens), len(lens)
    q = torch.from_numpy(rng.standard_normal((B * n_new, Hq, hd))).to(BF).to(DEV)
    pos0 = [n - n_new for n in lens]
    run = lambda q, t, most: ops.kv4_attention(q, pool, t, n_new, most, 0.09, window=window, impl="rows")
    whole = run(q, _tables(order, start, pos0, new), max(lens))
    assert torch.equal(whole, run(q, _tables(order, start, pos0, new, width=150), 150 * 64))
    for b in range(B):
        alone = run(q[b * n_new:(b + 1) * n_new].contiguous(), _tables(order[start[b]:start[b + 1]], [0, start[b + 1] - start[b]], [pos0[b]], [n_new]), lens[b])
        assert torch.equal(whole[b * n_new:(b + 1) * n_new], alone)


@pytest.mark.parametrize("impl", ["plain", "rows"])
def test_lengths_beyond_what_was_said_are_cut_off(impl):
    """More tokens on the device than ``max_len``, or than the page table holds, pages that the pool does not have: what is not there is not
    seen, and nothing beyond the scratch is written."""
    pool, order, start, seqs, rng = _cache(11, [900], 1, 128)
    q = torch.from_numpy(rng.standard_normal((1, 4, 128))).to(BF).to(DEV)
    t = _tables(order, start, [899], [1])
    whole = ops.kv4_attention(q, pool, t, 1, 900, 0.1, impl=impl)
    assert ops.kv4_attention(q, pool, t, 1, 64, 0.1, impl=impl).isfinite().all()
    narrow = t._replace(page_table=t.page_table[:, :3].contiguous())
    first = ops.kv4_attention(q, pool, narrow, 1, 900, 0.1, impl=impl)
    ref = pk.attention(f64(q), *(x[:192] for x in seqs[0]), [191], 0.1)
    assert (np.abs(f64(first).reshape(1, 4, 128) - ref[0]) <= tolerance(BF, 128, ref[1], ref[2], ref[0], 192)).all()
    wrong = t.page_table.clone()
    wrong[0, 3:] = pool.shape[0]
    wrong[0, 4] = -5
    gone = ops.kv4_attention(q, pool, t._replace(page_table=wrong), 1, 900, 0.1, impl=impl)
    assert (f64(gone).reshape(1, 4, 128) - ref[0] <= tolerance(BF, 128, ref[1], ref[2], ref[0], 192)).all()
    assert torch.equal(whole, ops.kv4_attention(q, pool, t, 1, 900, 0.1, impl=impl))


def test_a_replayed_graph_and_another_stream():
    lens = [500, 130]
    pool, order, start, seqs, rng = _cache(12, lens, 2, 128)
    q = torch.from_numpy(rng.standard_normal((2, 8, 128))).to(BF).to(DEV)
    pos0, starts, pages = ints([300, 100]), ints(start), ints(order)
    want = [ops.kv4_attention(q, pool, ops.step_tables(pages, starts, p, ints([1, 1]), 2, 8), 1, 512, 0.1) for p in (pos0, pos0 + 29)]
    ones = ints([1, 1])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(ops.kv4_attention(q, pool, ops.step_tables(pages, starts, pos0, ones, 2, 8), 1, 512, 0.1), want[0])
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.kv4_attention(q, pool, ops.step_tables(pages, starts, pos0, ones, 2, 8)._replace(pages=None), 1, 512, 0.1)
    graph.replay()
    assert torch.equal(out, want[0])
    pos0 += 29
    graph.replay()
    assert torch.equal(out, want[1])


def test_attention_refusals():
    pool, order, start, _, _ = _cache(1, [70], 2, 64)
    t = _tables(order, start, [69], [1])
    q = torch.zeros(1, 4, 64, device=DEV)
    for args, kw in [((q, pool, t, 0, 70, 1.0), {}), ((q, pool, t, 1, 0, 1.0), {}), ((q, pool, t, 1, 70, 1.0), {"window": -1}),
                     ((q, pool, t, 1, 70, 1.0), {"impl": "none"}), ((q, pool, t, 1, 70, 1.0), {"impl": "rows"}), ((q, pool, t, 1, 70, 1.0), {"impl": "read"}),
                     ((q.bfloat16(), pool, t._replace(pages=None), 1, 70, 1.0), {"impl": "read"}), ((torch.zeros(1, 3, 64, device=DEV), pool, t, 1, 70, 1.0), {}),
                     ((torch.zeros(2, 4, 64, device=DEV), pool, t, 1, 70, 1.0), {}), ((torch.zeros(1, 4, 128, device=DEV), pool, t, 1, 70, 1.0), {}),
                     ((q, pool.clone().view(-1)[:9216].view(2, 1, 4608), t._replace(pos0=ints([1, 2])), 1, 70, 1.0), {})]:
        with pytest.raises(KernelError, match="kv4"):
            ops.kv4_attention(*args, **kw)
    with pytest.raises(KernelError, match="float32 or bfloat16"):
        ops.kv4_attention(q.half(), pool, t, 1, 70, 1.0)
    with pytest.raises(KernelError, match="16 bytes"):
        shifted = torch.zeros(pool.numel() + 8, dtype=torch.uint8, device=DEV)[8:].view(pool.shape)
        ops.kv4_attention(q, shifted, t, 1, 70, 1.0)


def test_store_and_read_refusals():
    pool = torch.zeros(2, 1, 4608, dtype=torch.uint8, device=DEV)
    x, s = torch.zeros(1, 3 * 64, device=DEV), ints([0])
    with pytest.raises(KernelError, match="kv4_store"):
        ops.kv4_store(x, None, None, None, None, ints([0, 1]), pool, 1, 1, 64, 0, 0.0, F32)
    with pytest.raises(KernelError, match="kv4_store"):
        ops.kv4_store(x, None, None, None, None, s, pool, 2, 1, 64, 0, 0.0, F32)
    with pytest.raises(KernelError, match="rotary"):
        ops.kv4_store(x, None, None, None, None, s, pool, 1, 1, 64, 66, 0.0, F32)
    with pytest.raises(KernelError, match="cos"):
        ops.kv4_store(x, None, None, torch.zeros(1, 31, device=DEV), torch.zeros(1, 31, device=DEV), s, pool, 1, 1, 64, 64, 0.0, F32)
    with pytest.raises(KernelError, match="entries"):
        ops.kv4_store(x, torch.zeros(63, device=DEV), None, None, None, s, pool, 1, 1, 64, 0, 0.0, F32)
    with pytest.raises(KernelError, match="kv4_read"):
        ops.kv4_read(pool, s, s, s, 64, 64, F32)
    with pytest.raises(KernelError, match="does not hold"):
        ops.kv4_read(pool, s, ints([0, 1]), s, 64, 128, F32)


def test_calls_through_ctypes_and_with_other_whole_numbers_give_the_same_bits(monkeypatch):
    rng = np.random.default_rng(3)
    B, Hq, Hkv, hd = 3, 8, 2, 64
    pos0, n_new, start = ints([100, 0, 63]), ints([2, 1, 3]), ints([0, 2, 3, 5])
    qkv = torch.from_numpy(rng.standard_normal((6, (Hq + 2 * Hkv) * hd)).astype(np.float32)).to(DEV)
    weight, angle = torch.rand(hd, device=DEV) + 0.5, torch.rand(6, hd // 2, device=DEV)
    logits = torch.from_numpy(rng.standard_normal((5, 3000)).astype(np.float32)).to(DEV)

    def step(whole):
        t = ops.step_tables(ints([4, 1, 0, 2, 3]), start, pos0, n_new, whole(6), whole(2))
        pool = torch.zeros(5, Hkv, ops.kv4_page_bytes(hd), dtype=torch.uint8, device=DEV)
        q = ops.kv4_store(qkv, weight, weight, angle.cos(), angle.sin(), t.slot_map, pool, whole(Hq), whole(Hkv), whole(hd), whole(hd), np.float32(1e-6), BF)
        k, v, table = ops.kv4_read(pool, t.pages, t.page_start, t.seq_len, whole(102), whole(hd), F32)
        outs = [ops.kv4_attention(x, pool, t, whole(3), whole(102), np.float32(0.1), whole(0), impl=impl)
                for x, impl in ((q, "rows"), (q, "read"), (q, "auto"), (q, "plain"), (q.float(), "auto"))]
        return [x for x in t if x is not None] + [q, pool, k, v, table] + outs + list(ops.token_logprobs(logits, ints([0, 1, 2, 3, 4]), top=5))

    first, host = step(int), ops._HOST
    monkeypatch.setattr(ops, "_host_wanted", False)
    ops._bind_host(None)
    try:
        plain = step(int)
    finally:
        ops._bind_host(host)
    for other in (plain, step(np.int64)):
        assert len(first) == len(other) and all(torch.equal(a, b) for a, b in zip(first, other))

"""The forms of the attention over the 4-bit cache against each other: page tables that change from call to call, that are too narrow, that name
pages which are not there; steps of unequal sequences."""
import numpy as np
import pytest
import torch

import plain_kv4 as pk
from questwend_b200.kernels import ops
from questwend_b200.kernels.ops import KernelError
from test_gpu_kv4 import BF, DEV, F32, _cache, _check, _tables, f64, forms, ints, tolerance

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hd,lens,n_new", [(128, [200, 500], [70, 30]), (64, [130, 700, 64], [60, 100, 64]), (128, [3000, 640], [20, 5])])
def test_calls_one_behind_the_other_read_their_own_pages(hd, lens, n_new):
    """Two steps whose page tables lie in the same memory, in turn and without a pause: nobody sees the other's table."""
    steps, want = [], []
    for turn in (1, -1):
        its, new = lens[::turn], n_new[::turn]
        pool, order, start, _, rng = _cache(21, its, 2, hd)
        pos0 = [a - b for a, b in zip(its, new)]
        q = torch.from_numpy(rng.standard_normal((sum(new), 4, hd))).to(BF).to(DEV)
        steps.append((q, pool, _tables(order, start, pos0, new), max(new), max(its), hd ** -0.5))
    for step in steps:
        torch.cuda.synchronize()
        want.append(ops.kv4_attention(*step, impl="read"))
        torch.cuda.synchronize()
        assert (want[-1].float() - ops.kv4_attention(*step, impl="rows").float()).abs().max() < 0.1
    got = [ops.kv4_attention(*steps[i % 2], impl="read") for i in range(40)]
    assert all(torch.equal(out, want[i % 2]) for i, out in enumerate(got))


@pytest.mark.parametrize("hd", [64, 128])
def test_a_step_that_brings_nothing(hd):
    """Padding alone, as pages read back as well: zeros, and what comes behind the call finds them and its own memory."""
    pool, order, start, _, _ = _cache(22, [300, 70], 2, hd)
    t = _tables(order, start, [300, 70], [0, 0], behind=40)
    q = torch.ones(40, 8, hd, dtype=BF, device=DEV)
    for impl in forms(q):
        for _ in range(20):
            out = ops.kv4_attention(q, pool, t, 40, 300, 0.1, impl=impl)
            behind = out + 1
            again = torch.full_like(out, 3.0)
            assert (out == 0).all() and (behind == 1).all() and (again == 3).all()


@pytest.mark.parametrize("hd,group", [(128, 4), (64, 3)])
@pytest.mark.parametrize("window", [0, 50, 700])
@pytest.mark.parametrize("n_new", [1, 90])
def test_a_sequence_longer_than_its_row_of_the_page_table(hd, group, window, n_new):
    """Keys that the table does not name are not seen; rows that then see nothing are zeros.  The same in every form."""
    lens, pos0, width = [900, 130], [900 - n_new, 129], 3
    pool, order, start, seqs, rng = _cache(23, lens, 2, hd)
    q = torch.from_numpy(rng.standard_normal((n_new + 1, 2 * group, hd))).to(BF).to(DEV)
    t = _tables(order, start, pos0, [n_new, 1], width=width)
    _check(pool, t, [[x[:64 * width] for x in s] for s in seqs], q, pos0, [n_new, 1], 900, hd ** -0.5, window)
    for most in (192, 130, 64, 1):                        # a bound that does not hold: as many pages as it says are read, and no more
        got = f64(ops.kv4_attention(q, pool, t, n_new, most, hd ** -0.5, window=window, impl="read")).reshape(n_new + 1, 2 * group, hd)
        pages = -(-most // 64)
        for b, (at, n) in enumerate(((0, n_new), (n_new, 1))):
            out, mass, big = pk.attention(f64(q[at:at + n]), *(x[:64 * pages] for x in seqs[b]), [pos0[b] + i for i in range(n)], hd ** -0.5, window)
            assert (np.abs(got[at:at + n] - out) <= tolerance(BF, hd, mass, big, out, 192)).all(), (most, b)


def test_a_sequence_longer_than_the_table_in_pieces():
    """Few tokens behind a long context, whose keys the prompt kernel cuts into pieces: the join knows of the table's end too."""
    hd, L, n_new = 128, 6000, 12
    pool, order, start, seqs, rng = _cache(24, [L], 1, hd)
    q = torch.from_numpy(rng.standard_normal((n_new, 4, hd))).to(BF).to(DEV)
    for width, window in ((40, 0), (40, 4000), (40, 100), (93, 0)):
        t = _tables(order, start, [L - n_new], [n_new], width=width)
        before = ops.LAUNCHES[0]
        ops.kv4_attention(q, pool, t, n_new, L, hd ** -0.5, window=window, impl="read")
        assert ops.LAUNCHES[0] - before == (2 if window == 100 else 3)
        _check(pool, t, [[x[:64 * width] for x in seqs[0]]], q, [L - n_new], [n_new], L, hd ** -0.5, window)


@pytest.mark.parametrize("impl", ["read", "auto"])
def test_lengths_of_fewer_sequences_are_refused(impl):
    """The table of the pages that are read back has a row for each length: with fewer than sequences the others' rows would lie behind it."""
    pool, order, start, _, _ = _cache(25, [200, 100], 2, 64)
    t = _tables(order, start, [0, 0], [200, 100])
    q = torch.zeros(300, 4, 64, dtype=BF, device=DEV)
    for more in ({"seq_len": ints([200]), "page_start": ints(start[:2])}, {"seq_len": ints([200])}, {"seq_len": None},
                 {"seq_len": ints([200, 100, 0]), "page_start": ints(start + start[-1:])}):
        with pytest.raises(KernelError, match="2 sequences"):
            ops.kv4_attention(q, pool, t._replace(**more), 200, 200, 0.1, impl=impl)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("lens", [[200, 120], [4000, 60]])
def test_counts_beyond_the_tokens_that_there_are(hd, lens):
    """A step that was made for fewer tokens than its sequences bring: the tokens that there are get what they would, nothing is written behind them."""
    T, new, pos0 = 70, [40, 60], [lens[0] - 40, lens[1] - 60]
    pool, order, start, seqs, rng = _cache(26, lens, 2, hd)
    q = torch.from_numpy(rng.standard_normal((100, 4, hd))).to(BF).to(DEV)
    whole = _tables(order, start, pos0, new)
    t = ops.step_tables(ints(order), ints(start), ints(pos0), ints(new), T, whole.page_table.shape[1])
    assert t.cu_seqlens.tolist() == [0, 40, 100]
    for impl in forms(q):
        got = ops.kv4_attention(q[:T].contiguous(), pool, t, 60, max(lens), hd ** -0.5, impl=impl)
        at = 0
        for b, n in enumerate((40, 30)):
            out, mass, big = pk.attention(f64(q[at:at + n]), *seqs[b], [pos0[b] + i for i in range(n)], hd ** -0.5)
            assert (np.abs(f64(got[at:at + n]).reshape(out.shape) - out) <= tolerance(BF, hd, mass, big, out, max(lens))).all(), (impl, b)
            at += n


@pytest.mark.parametrize("hd,group", [(128, 4), (64, 2), (32, 2)])
@pytest.mark.parametrize("lens,n_new,window", [([900, 200], [1, 1], 0), ([900, 200], [80, 40], 0), ([900, 200], [80, 40], 300), ([3000, 130], [20, 1], 0),
                                               ([300, 64], [300, 10], 0)])
def test_pages_that_the_pool_does_not_have_are_not_seen(hd, group, lens, n_new, window):
    """In every form, whatever stands around them; a row that sees no other page is zero."""
    pool, order, start, seqs, rng = _cache(27, lens, 2, hd)
    gone = [{2, 3, 7} if lens[0] > 500 else {0, 2}, {0}]
    for b in range(2):
        for n, j in enumerate(sorted(gone[b])):
            order[start[b] + j] = [pool.shape[0], -5, pool.shape[0] + 1000][n]
    pos0 = [a - b for a, b in zip(lens, n_new)]
    q = torch.from_numpy(rng.standard_normal((sum(n_new), 2 * group, hd))).to(BF).to(DEV)
    t, qd = _tables(order, start, pos0, n_new), f64(q)
    got = {f: f64(ops.kv4_attention(q, pool, t, max(n_new), max(lens), hd ** -0.5, window=window, impl=f)).reshape(qd.shape) for f in forms(q)}
    at = 0
    for b, n in enumerate(n_new):
        for i in range(n):
            pos = pos0[b] + i
            seen = [j for j in range(max(0, pos - window + 1) if window else 0, pos + 1) if j // 64 not in gone[b]]
            out, mass, big = pk.attention(qd[at:at + 1], *(x[seen] for x in seqs[b]), [len(seen) - 1], hd ** -0.5)
            for f, y in got.items():
                assert (np.abs(y[at] - out[0]) <= tolerance(BF, hd, mass, big, out, max(lens))[0]).all(), (f, b, i)
            at += 1
    k, v, table = ops.kv4_read(pool, t.pages, t.page_start, t.seq_len, max(lens), hd, F32, marked=True)
    assert [(r < 0).nonzero().flatten().tolist() for r in table] == [sorted(gone[b] | set(range(-(-lens[b] // 64), table.shape[1]))) for b in range(2)]
    assert all((x[start[b] + j] == 0).all() for x in (k, v) for b in range(2) for j in gone[b])


@pytest.mark.parametrize("scale", [0.0, -0.125, float("nan"), float("inf"), 1e-40, 1e35])
def test_a_scale_that_is_not_above_0_is_refused(scale):
    """By every form: a hidden key's score would not be the lowest one, and the forms would not agree on what comes of it."""
    pool, order, start, _, _ = _cache(28, [70], 1, 64)
    t = _tables(order, start, [60], [10])
    for dtype in (BF, F32):
        q = torch.ones(10, 2, 64, dtype=dtype, device=DEV)
        for impl in forms(q):
            with pytest.raises(KernelError, match="scale above 0"):
                ops.kv4_attention(q, pool, t, 10, 70, scale, impl=impl)


@pytest.mark.parametrize("scale", [2.0 ** -60, 3.0])
def test_small_and_large_scales(scale):
    """With a large scale one key has nearly all the weight, and where its number is 0 the result is what the others' tiny weights leave.  As rows a number
    c s - z s is formed from two sums over the keys, of p c s and of p z s (exact products): each is off by at most 2^-23 a key of
    itself, and both are at most 15 s times the weights' sum, 1 behind the division.  So 2 x 15 s 2^-23 a key comes on top of ``tolerance``,
    which counts errors of p (c s - z s) alone."""
    lens, n_new, hd = [300, 100], [100, 7], 64
    pool, order, start, seqs, rng = _cache(29, lens, 1, hd)
    words = pk.unpack(pool.cpu().numpy(), hd)[3].astype(np.uint32)
    step = float(((words[(words & 0x7F80) != 0x7F80] & 0xFFF0) << 16).view(np.float32).max())
    pos0 = [a - b for a, b in zip(lens, n_new)]
    q = torch.from_numpy(rng.standard_normal((sum(n_new), 2, hd))).to(BF).to(DEV)
    t = _tables(order, start, pos0, n_new)
    for window in (0, 50):
        for impl in forms(q):
            got, at = f64(ops.kv4_attention(q, pool, t, max(n_new), max(lens), scale, window=window, impl=impl)).reshape(-1, 2, hd), 0
            for b, n in enumerate(n_new):
                out, mass, big = pk.attention(f64(q[at:at + n]), *seqs[b], [pos0[b] + i for i in range(n)], scale, window)
                more = 0.0 if impl in ("plain", "read") else 2 * 15 * step * lens[b] * 2.0 ** -23
                assert (np.abs(got[at:at + n] - out) <= tolerance(BF, hd, mass, big, out, lens[b]) + more).all(), (impl, b, window)
                at += n


def _sampled(q, got, seqs, pos0, n_new, hd, scale, at_most=12):
    """Some of the tokens of every sequence, its first and last among them, against the 64-bit implementation."""
    rng, t = np.random.default_rng(0), 0
    for b, n in enumerate(n_new):
        for i in sorted({0, n - 1, *rng.integers(0, n, at_most).tolist()}):
            out, mass, big = pk.attention(f64(q[t + i:t + i + 1]), *seqs[b], [pos0[b] + i], scale)
            lim = tolerance(q.dtype, hd, mass, big, out, pos0[b] + n)
            assert (np.abs(f64(got[t + i]).reshape(out.shape) - out) <= lim).all(), (b, i)
        t += n


@pytest.mark.parametrize("Hq,Hkv,hd,lens,n_new,listed", [(128, 1, 64, [8192], [8192], True), (72, 1, 64, [70, 14600], [1, 14600], True),
                                                         (128, 1, 128, [8200], [8195], False), (8, 1, 64, [500, 131073, 64], [1, 131073, 1], True)])
def test_prompts_too_long_for_rows(Hq, Hkv, hd, lens, n_new, listed):
    """What the rows form refuses goes another way, by itself: groups beyond 64 heads, tables without a list of pages, single tokens beside a long prompt."""
    pool, order, start, seqs, rng = _cache(30, lens, Hkv, hd)
    pos0 = [a - b for a, b in zip(lens, n_new)]
    q = torch.randn(sum(n_new), Hq, hd, generator=torch.Generator().manual_seed(1)).to(BF).to(DEV)
    t = _tables(order, start, pos0, n_new)
    if not listed:
        t = t._replace(pages=None, page_start=None)
    with pytest.raises(KernelError, match="as rows"):
        ops.kv4_attention(q, pool, t, max(n_new), max(lens), hd ** -0.5, impl="rows")
    _sampled(q, ops.kv4_attention(q, pool, t, max(n_new), max(lens), hd ** -0.5), seqs, pos0, n_new, hd, hd ** -0.5)


def test_more_tokens_of_a_sequence_than_the_prompt_kernels_grid_takes():
    """As a bound that says so: read back it is refused, by itself it goes plainly."""
    pool, order, start, seqs, rng = _cache(31, [100], 1, 64)
    q = torch.from_numpy(rng.standard_normal((20, 64, 64))).to(BF).to(DEV)
    t, most = _tables(order, start, [80], [20]), 65535 * 2 + 1
    for impl, words in (("read", "too many tokens"), ("rows", "as rows")):
        with pytest.raises(KernelError, match=words):
            ops.kv4_attention(q, pool, t, most, 100, 0.125, impl=impl)
    assert torch.equal(ops.kv4_attention(q, pool, t, most, 100, 0.125), ops.kv4_attention(q, pool, t, 20, 100, 0.125, impl="plain"))
    _sampled(q, ops.kv4_attention(q, pool, t, most - 1, 100, 0.125, impl="read"), seqs, [80], [20], 64, 0.125)


def test_steps_without_sequences_or_heads_are_refused():
    pool, order, start, _, _ = _cache(32, [100], 2, 64)
    t = _tables(order, start, [50], [50])
    none = t._replace(pos0=ints([]), cu_seqlens=ints([0]), seq_len=ints([]), page_start=ints([0]))
    for q, tables, its in ((torch.zeros(50, 4, 64), none, pool), (torch.zeros(50, 0, 64), t, pool), (torch.zeros(50, 4, 64), t, pool[:, :0].contiguous())):
        for impl in ("auto", "plain", "rows", "read"):
            with pytest.raises(KernelError, match="kv4_attention"):
                ops.kv4_attention(q.to(BF).to(DEV), its, tables, 50, 100, 0.1, impl=impl)


def _peak(call):
    """The result and the bytes that the call asked for beside it at most.  (Asked for: a cached block that is given may be up to 1 MB larger.)"""
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    asked = lambda which: torch.cuda.memory_stats()[f"requested_bytes.all.{which}"]
    before = asked("current")
    out = call()
    torch.cuda.synchronize()
    return out, asked("peak") - before - out.numel() * out.element_size()


@pytest.mark.parametrize("Hq,Hkv,hd", [(16, 8, 128), (15, 5, 64), (6, 3, 128)])
@pytest.mark.parametrize("lens,n_new", [([2500, 300], [1, 1]), ([2500, 300, 1500], [5, 40, 1]), ([700, 500], [400, 60])])
def test_heads_a_few_at_a_time(Hq, Hkv, hd, lens, n_new, monkeypatch):
    """Where all heads at once would take more memory than a call may: the same results, as rows bit for bit, in that much less memory."""
    pool, order, start, seqs, rng = _cache(33, lens, Hkv, hd)
    pos0, behind = [a - b for a, b in zip(lens, n_new)], 3
    q = torch.from_numpy(rng.standard_normal((sum(n_new) + behind, Hq, hd))).to(BF).to(DEV)
    wide = _tables(order, start, pos0, n_new, behind=behind, width=200)           # a table of 200 pages: runs joined by scratch memory
    t = _tables(order, start, pos0, n_new, behind=behind)
    run = lambda impl, t, most: _peak(lambda: ops.kv4_attention(q, pool, t, max(n_new), most, hd ** -0.5, impl=impl))
    rows, rows_bytes = run("rows", wide, 200 * 64)
    read, read_bytes = run("read", t, max(lens))
    each_rows, each_read = q.shape[0] * (Hq // Hkv) * 25 * (hd + 2) * 4, start[-1] * 64 * hd * 4
    assert rows_bytes >= Hkv * each_rows and read_bytes >= Hkv * each_read
    for heads in {1, 2, 3} - {Hkv}:
        monkeypatch.setattr(ops, "KV4_WORK_BYTES", heads * each_rows)
        before = ops.LAUNCHES[0]
        got, took = run("rows", wide, 200 * 64)
        assert torch.equal(got, rows) and took <= heads * each_rows + 1024 and ops.LAUNCHES[0] - before == 2 * -(-Hkv // ops._heads_at_once(Hkv, each_rows))
        monkeypatch.setattr(ops, "KV4_WORK_BYTES", heads * each_read)
        got, took = run("read", t, max(lens))
        assert (got.float() - read.float()).abs().max() <= 2.0 ** -7 * read.float().abs().max() and took <= 2 * heads * each_read + 4096
        _check(pool, t, seqs, q, pos0, n_new, max(lens), hd ** -0.5, 0)
    monkeypatch.setattr(ops, "KV4_WORK_BYTES", 1)                                   # a head's runs are too much: not as rows by itself
    _check(pool, wide, seqs, q, pos0, n_new, 200 * 64, hd ** -0.5, 0)
    got, took = run("auto", wide._replace(pages=None, page_start=None), 200 * 64)
    assert torch.equal(got, ops.kv4_attention(q, pool, wide, max(n_new), 200 * 64, hd ** -0.5, impl="plain")) and took <= 1024


def test_pages_of_some_heads():
    pool, order, start, _, _ = _cache(34, [200, 70], 5, 64)
    args = (pool, ints(order), ints(start), ints([200, 70]), 200, 64, BF)
    k, v, table = ops.kv4_read(*args)
    for first, n in ((0, 5), (0, 2), (2, 3), (4, 1)):
        its = ops.kv4_read(*args, heads=(first, n))
        assert torch.equal(its[0], k[:, first:first + n]) and torch.equal(its[1], v[:, first:first + n]) and torch.equal(its[2], table)
    plain = ops.kv4_read(*args[:-1], F32, heads=(3, 2))
    assert torch.equal(plain[0], k[:, 3:].float()) and torch.equal(plain[1], v[:, 3:].float())
    for heads in ((-1, 2), (0, 0), (4, 2), (5, 1)):
        with pytest.raises(KernelError, match="heads from"):
            ops.kv4_read(*args, heads=heads)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("hd,L,n_new", [(128, 200, 4), (128, 200, 90), (64, 1100, 1), (64, 1100, 30), (96, 200, 5)])
@pytest.mark.parametrize("window", [0, 70])
def test_what_is_not_finite_makes_all_of_its_head_nan_wherever_it_lies(dtype, hd, L, n_new, window):
    """A key's or a value's group, in pages that are seen wholly, in the last one and at a window's edge: the same in every form."""
    pool, order, start, seqs, rng = _cache(35, [L], 2, hd)
    t = _tables(order, start, [L - n_new], [n_new])
    q = torch.from_numpy(rng.standard_normal((n_new, 4, hd))).to(dtype).to(DEV)
    clean = {f: ops.kv4_attention(q, pool, t, n_new, L, 0.1, window=window, impl=f).view(n_new, 4, hd) for f in forms(q)}
    for at in (3, 64, L - n_new - 60, L - n_new, L - 2):
        for part in (0, 1):
            group = at % (hd // 32)
            broken = pool.clone()
            word = part * 64 * (hd // 2 + hd // 16) + 64 * hd // 2 + (at % 64) * (hd // 16) + 2 * group
            broken[order[at // 64], 1, word:word + 2] = torch.tensor([0xC0, 0x7F], dtype=torch.uint8, device=DEV)
            sees = torch.tensor([at <= p and (not window or at > p - window) for p in range(L - n_new, L)], device=DEV)
            for f in forms(q):
                got = ops.kv4_attention(q, broken, t, n_new, L, 0.1, window=window, impl=f).view(n_new, 4, hd)
                assert torch.equal(got[:, :2], clean[f][:, :2]) and torch.equal(got[~sees], clean[f][~sees]), (f, at, part)
                assert got[sees][:, 2:].isnan().all(), (f, at, part)

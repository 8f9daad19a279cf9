"""Log probabilities of tokens, entropies and the most probable tokens, against a plain 64-bit implementation."""
import math

import numpy as np
import pytest
import torch

import plain_kv4 as pk
from questwend_b200.kernels import ops
from questwend_b200.kernels.ops import KernelError, TokenLogprobs

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -23


def check(x, tokens, top):
    r = ops.token_logprobs(torch.from_numpy(x).to(DEV), torch.tensor(tokens, dtype=torch.int32, device=DEV), top=top)
    lp, H, ids, lps, mean, square = pk.logprobs(x, tokens, top)
    # ln S: an exponential is off by (2 + 1.173 |d|) units of 2^-23 (its stated bound), a sum of at most 16 + 5 + 8 terms one after the
    # other, five changes of the reference (an exponential, a product) and then 1 / 32 of the segments + 5 by half a unit each; then the differences x - m and (x - m) - ln S, and ln's own unit
    lnS = (2 + 1.2 * mean + (70 + x.shape[1] / 8192 / 32) / 2) * U

    def near(got, ref, lim):
        got = got.cpu().numpy().astype(np.float64)
        with np.errstate(invalid="ignore"):
            return bool(((got == ref) | (np.abs(got - ref) <= lim)).all())              # equal: infinities

    d = lambda v: np.abs(v) * U * 2 + U * 32                                            # |v| + |ln S| below 2 |v| + 32
    assert near(r.logprob, lp, lnS + d(lp))
    # U / S: the same errors on terms of |d|, and d's own rounding
    assert near(r.entropy, H, lnS + (2 * mean + 1.2 * square + mean * (72 + x.shape[1] / 8192 / 32)) * U + U * 32)
    assert r.top_ids.dtype == torch.int32 and r.top_ids.cpu().numpy().tolist() == ids.tolist()
    if top:
        assert near(r.top_logprobs, lps, lnS[:, None] + d(lps))
    return r


@pytest.mark.parametrize("V", [1, 5, 100, 1021, 8192, 8193, 30001, 151936])
@pytest.mark.parametrize("R", [1, 3, 17])
@pytest.mark.parametrize("top", [0, 1, 5, 20, 64])
def test_rows(R, V, top):
    rng = np.random.default_rng(R * V + top)
    x = (rng.standard_normal((R, V)) * rng.uniform(0.1, 8)).astype(np.float32)
    check(x, rng.integers(0, V, R).tolist(), min(top, V))


@pytest.mark.parametrize("R,V", [(300, 5000), (700, 20000), (3, 270000), (2, 262144)])
def test_many_rows(R, V):
    rng = np.random.default_rng(R)
    check((rng.standard_normal((R, V)) * 3).astype(np.float32), rng.integers(0, V, R).tolist(), 7)


@pytest.mark.parametrize("V", [64, 9000, 20000])
@pytest.mark.parametrize("order", ["equal", "zeros of both signs", "rising", "falling", "few values", "one holds all", "strided"])
def test_ties_and_orders(V, order):
    """Equal logits (the lower id first), sorted ones (the largest lie together), values that fall on the same threads."""
    rng = np.random.default_rng(V)
    i = np.arange(V)
    x = {"equal": np.full(V, 1.25), "zeros of both signs": np.where(i % 2, 0.0, -0.0), "rising": i / 100.0, "falling": -i / 100.0,
         "few values": rng.integers(0, 3, V), "one holds all": np.where(i == V // 2, 60.0, 0.0),
         "strided": np.where(i % 256 == 3, 5.0 + i / V, 0.0)}[order]
    x = np.stack([x, x[::-1]]).astype(np.float32)
    for top in (1, 20, 64):
        check(x, [0, V - 1], top)


def test_large_and_masked_logits():
    rng = np.random.default_rng(3)
    x = (rng.standard_normal((8, 20000)) * 2).astype(np.float32)
    x[0] += 3e4
    x[1] *= 100
    x[2, 100:] = -np.inf                                    # most tokens cannot be
    x[3, :17000] = -np.inf                                  # a whole segment
    x[4, 1:] = -np.inf                                      # one token left
    x[5] = np.where(rng.random(20000) < 0.5, np.finfo(np.float32).min, x[5])          # masked by the type's lowest value
    x[6] = np.finfo(np.float32).min                         # all of them: as good as each other
    x[7] = np.where(rng.random(20000) < 0.5, 3e38, -3e38)
    r = check(x, [5, 7, 3, 17500, 0, int(np.argmax(x[5])), 3, int(np.argmax(x[7]))], 30)
    assert float(r.logprob[4]) == 0.0 and float(r.entropy[4]) == 0.0
    got = ops.token_logprobs(torch.from_numpy(x).to(DEV), torch.tensor([0, 0, 500, 5, 9, 0, 0, 0], dtype=torch.int32, device=DEV))
    assert got.logprob[2:5].tolist() == [-math.inf] * 3


def test_rows_without_a_distribution():
    x = torch.zeros(4, 9000, device=DEV)
    x[0, 8500] = math.nan
    x[1] = -math.inf
    x[2, 7] = math.inf
    x[3, 5:] = math.nan
    tokens = torch.tensor([1, 1, 7, 2], dtype=torch.int32, device=DEV)
    r = ops.token_logprobs(x, tokens, top=6)
    assert r.logprob.isnan().all() and r.entropy.isnan().all() and r.top_logprobs.isnan().all()
    assert r.top_ids[0].tolist() == [0, 1, 2, 3, 4, 5] and r.top_ids[1].tolist() == [0, 1, 2, 3, 4, 5]
    assert r.top_ids[2].tolist() == [7, 0, 1, 2, 3, 4] and r.top_ids[3].tolist() == [0, 1, 2, 3, 4, -1]


def test_tokens_outside_the_vocabulary():
    x = torch.zeros(3, 10, device=DEV)
    r = ops.token_logprobs(x, torch.tensor([-1, 10, 3], dtype=torch.int32, device=DEV))
    assert r.logprob.isnan().tolist() == [True, True, False] and not r.entropy.isnan().any()


def test_a_row_does_not_depend_on_the_others():
    g = torch.Generator().manual_seed(1)
    x = (torch.randn(40, 30000, generator=g) * 3).to(DEV)
    t = torch.arange(40, dtype=torch.int32, device=DEV)
    whole = ops.token_logprobs(x, t, top=9)
    two = ops.token_logprobs(x.repeat(8, 1), t.repeat(8), top=9)            # many rows: no clusters
    assert all(torch.equal(a, b[:40]) for a, b in zip(whole, two))
    for i in (0, 17, 39):
        one = ops.token_logprobs(x[i:i + 1].contiguous(), t[i:i + 1].contiguous(), top=9)
        assert all(torch.equal(a[i:i + 1], b) for a, b in zip(whole, one))


@pytest.mark.parametrize("R", [2, 300])
def test_logits_that_do_not_begin_at_16_bytes(R):
    x = (torch.randn(R * 9000 + 1, generator=torch.Generator().manual_seed(4)) * 3).to(DEV)
    t = torch.zeros(R, dtype=torch.int32, device=DEV)
    odd = x[1:].view(R, 9000)
    got, want = ops.token_logprobs(odd, t, top=5), ops.token_logprobs(odd.clone(), t, top=5)
    assert torch.equal(got.top_ids, want.top_ids)
    for a, b in ((got.logprob, want.logprob), (got.entropy, want.entropy), (got.top_logprobs, want.top_logprobs)):
        assert (a - b).abs().max() <= 1e-5                  # another order of the sums


def test_out_and_a_replayed_graph():
    g = torch.Generator().manual_seed(2)
    x = (torch.randn(5, 20000, generator=g) * 3).to(DEV)
    t = torch.zeros(5, dtype=torch.int32, device=DEV)
    out = ops.token_logprobs(x, t, top=4)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.token_logprobs(x, t, top=4, out=out)
    y = (torch.randn(5, 20000, generator=g) * 3).to(DEV)
    x.copy_(y)
    t.fill_(77)
    graph.replay()
    want = ops.token_logprobs(y, torch.full_like(t, 77), top=4)
    assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_refusals():
    x, t = torch.zeros(2, 10, device=DEV), torch.zeros(2, dtype=torch.int32, device=DEV)
    for args, kw in [((x, t[:1]), {}), ((x, t), {"top": 11}), ((x, t), {"top": -1}), ((torch.zeros(2, 100, device=DEV), t), {"top": 65}),
                     ((x, t), {"top": 1, "out": ops.token_logprobs(x, t, top=2)})]:
        with pytest.raises(KernelError, match="token_logprobs"):
            ops.token_logprobs(*args, **kw)
    with pytest.raises(KernelError, match="float32"):
        ops.token_logprobs(x.bfloat16(), t)
    with pytest.raises(KernelError, match="contiguous"):
        ops.token_logprobs(torch.zeros(10, 2, device=DEV).t(), t)
    empty = ops.token_logprobs(torch.zeros(0, 10, device=DEV), t[:0], top=2)
    assert tuple(empty.top_ids.shape) == (0, 2)

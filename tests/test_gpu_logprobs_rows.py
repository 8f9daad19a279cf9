"""Rows whose list of alternatives is found one by one (more threads hold a candidate than the list's memory does), few and many rows."""
import math

import numpy as np
import pytest
import torch

from questwend_b200.kernels import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("V,R", [(40000, 1), (40000, 3), (40000, 300), (151936, 2), (151936, 70), (300001, 2)])
@pytest.mark.parametrize("numbers", [0, 1, 2, 7])
@pytest.mark.parametrize("top", [1, 5, 20, 64])
def test_rows_with_fewer_numbers_than_alternatives(V, R, numbers, top):
    """All logits NaN but a few: these in their order, then nothing (id -1), to the end of the list."""
    rng = np.random.default_rng(V + numbers)
    at = rng.choice(V, numbers, replace=False)
    x = np.full((R, V), math.nan, dtype=np.float32)
    x[:, at] = rng.integers(-3, 3, numbers)
    order = sorted(range(numbers), key=lambda i: (-x[0, at[i]], at[i]))
    want = ([int(at[i]) for i in order] + [-1] * top)[:top]
    r = ops.token_logprobs(torch.from_numpy(x).to(DEV), torch.zeros(R, dtype=torch.int32, device=DEV), top=top)
    assert r.logprob.isnan().all() and r.entropy.isnan().all() and r.top_logprobs.isnan().all()
    assert r.top_ids.tolist() == [want] * R


@pytest.mark.parametrize("V,R", [(40000, 2), (151936, 2), (151936, 70)])
@pytest.mark.parametrize("left", [1, 3, 40])
def test_rows_most_of_whose_tokens_cannot_be(V, R, left):
    """Minus infinity but for a few: these first, then the lowest ids among the rest, with probability 0."""
    rng = np.random.default_rng(V + left)
    at = rng.choice(V, left, replace=False)
    x = np.full((R, V), -math.inf, dtype=np.float32)
    x[:, at] = rng.standard_normal(left)
    top = 20
    want = ([int(at[i]) for i in np.argsort(-x[0, at], kind="stable")] + [i for i in range(left + top) if i not in set(at.tolist())])[:top]
    r = ops.token_logprobs(torch.from_numpy(x).to(DEV), torch.full((R,), int(at[0]), dtype=torch.int32, device=DEV), top=top)
    assert r.top_ids.tolist() == [want] * R and r.logprob.isfinite().all() and r.entropy.isfinite().all()
    n = min(left, top)
    assert r.top_logprobs[:, :n].isfinite().all() and (r.top_logprobs[:, n:] == -math.inf).all()

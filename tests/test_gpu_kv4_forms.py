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

"""The 4-bit cache's format and the plain implementations that the GPU tests compare with (CPU)."""
import ctypes

import numpy as np
import pytest
import torch

import plain_kv4 as pk
from questwend_b200.kernels import build, ops
from questwend_b200.kernels.limits import kv4_refusal
from questwend_b200.kernels.ops import KernelError


@pytest.mark.parametrize("dim,size", [(32, 2304), (64, 4608), (128, 9216), (256, 18432)])
def test_page_bytes(dim, size):
    assert ops.kv4_page_bytes(dim) == size
    x = np.random.default_rng(0).standard_normal((2, 3, 64, dim))
    assert pk.pack(x, x).shape == (2, 3, size)


@pytest.mark.parametrize("dim", [0, -32, 16, 48, 100, 288])
def test_head_sizes_that_are_refused(dim):
    assert "multiple of 32" in kv4_refusal(dim)
    with pytest.raises(KernelError, match="multiple of 32"):
        ops.kv4_page_bytes(dim)


def test_a_number_is_within_half_a_step_and_exact_in_bfloat16():
    """Inside the 16 numbers a group stands for, half a step; the lowest and highest may lie outside: 15 steps are the range but for
    the step's rounding (1/16 at most, so 15/16 of a step in all) and the zero point's (half a step)."""
    rng = np.random.default_rng(1)
    x = rng.standard_normal((50, 96)) * np.exp(3 * rng.standard_normal((50, 1)))
    x[0], x[1, :32], x[2] = 0.0, 1.5, np.abs(x[2])
    c, w = pk.quantise(x)
    y = pk.stands_for(c, w)
    s = np.repeat(((w.astype(np.uint32) & 0xFFF0) << 16).view(np.float32).astype(np.float64), 32, -1)
    z = np.repeat(w & 15, 32, -1).astype(np.float64)
    inside = (x >= -z * s) & (x <= (15 - z) * s)
    assert (np.abs(x - y)[inside] <= 0.5 * s[inside] * (1 + 1e-12)).all()
    assert (np.abs(x - y) <= (0.5 + 15 / 16) * s * (1 + 1e-12)).all()
    assert (y == torch.from_numpy(y).to(torch.bfloat16).to(torch.float64).numpy()).all()
    assert (y[0] == 0).all() and (np.sign(y) * np.sign(x) >= 0).all()


def test_what_is_not_finite_and_what_is_tiny():
    x = np.ones((5, 64))
    x[0, 3], x[1, 40], x[2] = np.nan, np.inf, 1e-45
    x[3, 0], x[3, 1], x[4, 0] = 9e36, -9e36, 3e37             # a step of 1.2e36; of 2e36, 2^120 is 1.33e36
    y = pk.stands_for(*pk.quantise(x))
    one = 15 * 0.065625                                         # a fifteenth to 4 significant bits is 0.0625 1.05
    assert np.isnan(y[0, :32]).all() and np.isclose(y[0, 32:], one, rtol=1e-12).all()
    assert np.isnan(y[1, 32:]).all() and np.isclose(y[1, :32], one, rtol=1e-12).all()
    assert (y[2] == 0).all()
    assert np.isfinite(y[3]).all() and abs(y[3, 0] / 9e36 - 1) < 0.1 and np.isnan(y[4, :32]).all()


@pytest.mark.parametrize("call", [
    lambda t: ops.step_tables(t, t, t, t, 1, 1), lambda t: ops.token_logprobs(torch.zeros(1, 4), t),
    lambda t: ops.kv4_read(torch.zeros(1, 1, 2304, dtype=torch.uint8), t, t, t, 1, 32, torch.float32),
    lambda t: ops.kv4_store(torch.zeros(1, 96), None, None, None, None, t, torch.zeros(1, 1, 2304, dtype=torch.uint8), 1, 1, 32, 0, 0.0, torch.float32),
    lambda t: ops.kv4_attention(torch.zeros(1, 1, 32), torch.zeros(1, 1, 2304, dtype=torch.uint8), ops.StepTables(t, t, t, t, t, t, t), 1, 1, 1.0)])
def test_tensors_off_the_gpu_are_refused(call):
    with pytest.raises(KernelError, match="CUDA tensor"):
        call(torch.zeros(1, dtype=torch.int32))


def test_plain_tables():
    cu, length, seq, pos, table, slot = pk.step_tables([7, 3, 9], [0, 2, 2, 3], [60, 0, 5], [6, 0, 2], 9, 2)
    assert cu == [0, 6, 6, 8] and length == [66, 0, 7] and seq == [0] * 6 + [2, 2, -1]
    assert pos == [60, 61, 62, 63, 64, 65, 5, 6, -1] and table == [[7, 3], [0, 0], [9, 0]]
    assert slot == [7 * 64 + 60, 7 * 64 + 61, 7 * 64 + 62, 7 * 64 + 63, 3 * 64, 3 * 64 + 1, 9 * 64 + 5, 9 * 64 + 6, -1]


@pytest.mark.parametrize("way", ["native", "plain"])
def test_pieces(way):
    make = ops._plain_pieces
    if way == "native":
        module = build.host_calls()
        if module is None:
            pytest.skip("no native module")
        make = module.pieces
    like = torch.zeros(3)
    a, b, c, d = make(like, torch.int32, (2, 5), torch.float32, (7,), torch.bfloat16, (0, 3), torch.uint8, (1, 2, 3, 4))
    assert [tuple(t.shape) for t in (a, b, c, d)] == [(2, 5), (7,), (0, 3), (1, 2, 3, 4)]
    assert [t.dtype for t in (a, b, c, d)] == [torch.int32, torch.float32, torch.bfloat16, torch.uint8]
    assert all(t.is_contiguous() and t.device == like.device and not t.requires_grad for t in (a, b, c, d))
    for i, t in enumerate((a, b, d)):
        t.fill_(i + 1)
    assert (a == 1).all() and (b == 2).all() and (d == 3).all() and all(t.data_ptr() % 64 == a.data_ptr() % 64 for t in (b, d) if way == "native")
    keep = b.clone()
    del a, d
    assert torch.equal(b, keep) and torch.equal(b.view(torch.int32).view(torch.float32), keep)
    if way == "native":
        for args in [(like,), (like, torch.int32), (1, torch.int32, (2,)), (like, 3, (2,)), (like, torch.int32, [2]), (like, torch.int32, (-1,))]:
            with pytest.raises((TypeError, ValueError)):
                make(*args)


def test_here():
    module = build.host_calls()
    if module is None:
        pytest.skip("no native module")
    t = torch.zeros(2)
    assert module.here(0) and module.here(0, None, None) and not module.here(0, t) and not module.here(0, None, 3)
    with pytest.raises(TypeError):
        module.here()
    with pytest.raises(TypeError):
        module.here("0", t)


def test_ready():
    module = build.host_calls()
    if module is None:
        pytest.skip("no native module")
    t = torch.zeros(2)
    assert module.ready() == -1 and module.ready(None, None, None) == -1 and module.ready(t, torch.float32, 1) == -1 and module.ready(3, None, None) == -1
    for args in [(t,), (t, torch.float32), (0, t, torch.float32, 1)]:
        with pytest.raises(TypeError):
            module.ready(*args)


def test_arguments_as_they_are(monkeypatch):
    """What goes natively as it is goes through ctypes as objects: the types that the launchers take."""
    t = torch.zeros(3)
    monkeypatch.setattr(ops, "_HOST", None)
    seen = []
    monkeypatch.setattr(ops, "_call", lambda module, fn, *args, kernels=1: seen.append((module, fn, kernels, args)))
    ops._run("m", "f", t, None, 7, np.int64(-3), True, 0.5, "the stream", kernels=2)
    (module, fn, kernels, args), = seen
    assert (module, fn, kernels) == ("m", "f", 2) and args[-1] == "the stream"
    assert [type(a) for a in args[:-1]] == [ctypes.c_void_p] * 2 + [ctypes.c_int] * 3 + [ctypes.c_float]
    assert [a.value for a in args[:-1]] == [t.data_ptr(), None, 7, -3, 1, 0.5]
    with pytest.raises(TypeError):
        ops._run("m", "f", "no number", None)


def test_a_tensor_of_another_device_is_refused(monkeypatch):
    """Not the device that is current: refused, with what to do, whichever way the check goes."""
    class Elsewhere:
        device = "cuda:1"

        def get_device(self):
            return 1
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    for host in (None, ops._HOST):
        monkeypatch.setattr(ops, "_HOST", host)
        with pytest.raises(KernelError, match="use torch.cuda.device"):
            ops._here("kv4_store", None, Elsewhere())
